"""The workloads that the quantized paged cache and shared prefixes are measured on.

One case is what a decoder block that serves requests asks of its paged K/V
cache: the rotary embedding with the write of keys and values in 8 or 4 bits and
their reading back (``write``), the reading of whole sequences (``read``),
attention over the quantized pages (``attn``), and attention of sequences that
share a long prefix (``shared``, over plain or quantized pages). Sizes are those
of the repository's own workloads: 32 / 8 heads of 128, 14 / 2 heads of 64 and 8 /
8 of 128, prompts of up to a few thousand tokens, decode batches of 1 to 256.

With ``own`` false, ``run`` computes a case in plain torch operations, in 32
bits, rounded once at the end; with ``own`` true it makes the library's calls.
``exact`` computes a case in 64 bits, sequence by sequence. What a cache holds in
8 or 4 bits stands for T(code * scale + bias), T the type of q, k and v.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"
THETA = 5e5


# ---- the cases -------------------------------------------------------------------

def _case(kind, name, **values):
    c = {"kind": kind, **values}
    return {"name": name, **c} if name else c


def _write(name, B, T, heads, page, bits, group, dtype, part=1):
    """T new tokens of B empty requests (fewer of some); the rotated dims are D / part."""
    Hq, Hkv, D = heads
    return _case("write", name, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, bits=bits, group=group, dtype=dtype, part=part)


def _read(name, B, heads, L, page, bits, group, dtype):
    """Sequences of up to L keys."""
    Hq, Hkv, D = heads
    return _case("read", name, B=B, Hkv=Hkv, D=D, L=L, page=page, bits=bits, group=group, dtype=dtype)


def _attn(name, B, heads, T, L, page, bits, group, dtype):
    """T query tokens at the end of up to L keys."""
    Hq, Hkv, D = heads
    return _case("attn", name, B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, L=L, page=page, bits=bits, group=group, dtype=dtype)


def _shared(name, B, groups, heads, T, P, L, page, bits, group, dtype):
    """B sequences in ``groups`` groups, each with a prefix of P keys of its own and up to L
    more in each sequence, the T query tokens among them; bits 0: plain pages."""
    Hq, Hkv, D = heads
    return _case("shared", name, B=B, groups=groups, Hq=Hq, Hkv=Hkv, D=D, T=T, P=P, L=L, page=page, bits=bits, group=group,
                 dtype=dtype)


_LLAMA, _QWEN, _MHA = (32, 8, 128), (14, 2, 64), (8, 8, 128)


def listed():
    return [
        # The first token of each request of a serving batch. Latency alone.
        _write("write_decode", 64, 1, _LLAMA, 16, 8, 64, "bf16"),
        # Prompts enter the cache and are read back for their own attention.
        _write("write_prompts", 4, 2048, _LLAMA, 16, 8, 64, "bf16"),
        # Odd prompts of a small model that rotates half of each head, 4 bits.
        _write("write_odd", 3, 517, _QWEN, 64, 4, 32, "fp16", part=2),
        # Long ragged sequences leave the cache whole, as for another machine.
        _read("read_long", 16, _LLAMA, 8192, 16, 8, 64, "bf16"),
        # A few short ones, 4 bits.
        _read("read_short", 3, _QWEN, 1500, 64, 4, 64, "fp16"),
        # A decode step over long ragged caches, 8 and 4 bits.
        _attn("decode_8bit", 64, _LLAMA, 1, 8192, 16, 8, 64, "bf16"),
        _attn("decode_4bit", 64, _LLAMA, 1, 8192, 64, 4, 64, "fp16"),
        # One user's decode step. Latency.
        _attn("decode_one", 1, _QWEN, 1, 1000, 16, 8, 32, "bf16"),
        # A chunk of each of three prompts against longer caches.
        _attn("chunk", 3, _QWEN, 500, 4000, 16, 4, 64, "fp16"),
        # A decode step of a batch behind one long instruction.
        _shared("shared_decode", 64, 1, _LLAMA, 1, 8192, 512, 16, 0, 0, "bf16"),
        # Four such groups over a quantized cache, three draft tokens checked at once.
        _shared("shared_groups", 32, 4, _LLAMA, 4, 2048, 600, 64, 8, 64, "bf16"),
        # A small batch in 32 bits, the prefix no whole number of splits.
        _shared("shared_fp32", 7, 1, _MHA, 3, 1008, 90, 16, 0, 0, "fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("write", "write", "read", "attn", "attn", "attn", "shared", "shared", "shared"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32"))
    heads = rng.choice((_LLAMA, _QWEN, _MHA))
    page, bits, group = rng.choice((8, 16, 16, 64)), rng.choice((8, 4)), rng.choice((32, 64))
    if kind == "write":
        T = _log(rng, 1, 2048)
        return _write(None, _log(rng, 1, min(64, max(2, 8192 // T))), T, heads, page, bits, group, dtype, rng.choice((1, 1, 2)))
    if kind == "read":
        L = _log(rng, 1, 8192)
        return _read(None, _log(rng, 1, min(64, max(2, 65536 // L))), heads, L, page, bits, group, dtype)
    if kind == "attn":
        T = rng.choice((1, 1, _log(rng, 2, 8), _log(rng, 2, 1024)))
        L = T + _log(rng, 1, 4000)
        return _attn(None, _log(rng, 1, 64 if T == 1 else 16 if T <= 8 else 2), heads, T, L, page, bits, group, dtype)
    B, T = _log(rng, 2, 64), rng.choice((1, 1, _log(rng, 2, 6)))
    bits = rng.choice((0, 0, bits))
    return _shared(None, B, rng.randint(1, max(1, B // 4)), heads, T, page * max(1, _log(rng, 100, 4000) // page),
                   T + _log(rng, 1, 500), page, bits, group if bits else 0, dtype)


# ---- inputs (made from the seed alone) ----------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _randint(g, lo, hi, shape):
    """Whole numbers lo .. hi, hi included, as int32."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV, dtype=torch.int32)


def _pool(case, g, pages):
    """One pool of pages: values of type T, or the codes and the (scale, bias) of every group."""
    Hkv, D, page, bits, dt = (case[k] for k in ("Hkv", "D", "page", "bits", "dtype"))
    dt = DTYPES[dt]
    if not bits:
        return _randn(g, pages, Hkv, page, D, dtype=dt)
    codes = torch.randint(0, 256, (pages, Hkv, page, D * bits // 8), generator=g, device=DEV, dtype=torch.uint8)
    low = -2.5 + 0.5 * torch.randn((pages, Hkv, page, D // case["group"]), generator=g, device=DEV)
    span = (5.0 + torch.rand(low.shape, generator=g, device=DEV)) / (2 ** bits - 1)
    return codes, torch.stack([span, low], -1).to(dt)


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    dt, page, Hkv, D = DTYPES[case["dtype"]], case["page"], case["Hkv"], case["D"]
    st = {"case": case}
    if kind == "write":
        B, T, Hq = case["B"], case["T"], case["Hq"]
        new = _randint(g, (T + 1) // 2, T, (B,))
        per = -(-T // page)
        st["table"] = torch.randperm(B * per, generator=g, device=DEV).to(torch.int32).reshape(B, per)
        # Tokens of request b sit at the end of its T rows, behind padding rows.
        row = torch.arange(T, device=DEV)[None, :] - (T - new)[:, None]
        pos = row.clamp(min=0)
        slots = st["table"].long().gather(1, pos // page) * page + pos % page
        st["slots"] = torch.where(row >= 0, slots, torch.full_like(slots, -1))
        st["pos"], st["lens"] = pos.to(torch.int32), new
        half = D // case["part"] // 2
        inv = THETA ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        ang = torch.arange(max(T, 64), dtype=torch.float64, device=DEV)[:, None] * inv
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        st["q"], st["k"], st["v"] = (_randn(g, B, T, h, D, dtype=dt) for h in (Hq, Hkv, Hkv))
        st["kp"], st["vp"] = ((torch.zeros(B * per, Hkv, page, D * case["bits"] // 8, dtype=torch.uint8, device=DEV),
                               torch.zeros(B * per, Hkv, page, D // case["group"], 2, dtype=dt, device=DEV)) for _ in range(2))
        return st
    B, L = case["B"], case["L"]
    if kind == "shared":
        T, P, groups = case["T"], case["P"], case["groups"]
        own_pages, first = -(-L // page), P // page
        pages = torch.randperm(groups * first + B * own_pages, generator=g, device=DEV).to(torch.int32)
        # Group n holds the sequences from n B / groups on.
        starts = torch.arange(groups + 1, device=DEV) * B // groups
        member = torch.searchsorted(starts, torch.arange(B, device=DEV), right=True) - 1
        st["table"] = torch.cat([pages[:groups * first].reshape(groups, first)[member],
                                 pages[groups * first:].reshape(B, own_pages)], 1).contiguous()
        st["starts"], st["plens"] = starts.to(torch.int32), torch.full((groups,), P, dtype=torch.int32, device=DEV)
        st["lens"] = P + _randint(g, T, L, (B,))
        count = pages.numel()
    else:
        T = case.get("T", 1)
        per = -(-L // page)
        count = B * per
        st["table"] = torch.randperm(count, generator=g, device=DEV).to(torch.int32).reshape(B, per)
        # prompts shorter than the T rows of a padded batch leave their first rows empty
        st["lens"] = _randint(g, (T + 1) // 2, L, (B,))
    if kind != "read":
        st["q"] = _randn(g, B, case["Hq"], T, D, dtype=dt, scale=2.0)
    st["kp"], st["vp"] = _pool(case, g, count), _pool(case, g, count)
    return st


# ---- one pass: the library's calls -----------------------------------------------------

def _library():
    """The package, imported by the first pass: a pass is the library's call alone."""
    bi = sys.modules.get("mlx_batch_invariant_amd")
    if bi is None:
        pkg = os.path.join(os.getcwd(), "mlx-batch-invariant_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import mlx_batch_invariant_amd as bi
    return bi


def _own(st):
    bi, case = _library(), st["case"]
    kind = case["kind"]
    kp, vp = st["kp"], st["vp"]
    if case["bits"]:
        kp, vp = (bi.QuantizedPages(*p, case["bits"], case["group"]) for p in (kp, vp))
    if kind == "write":
        q = bi.rope_quantized_cache(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pos"], st["slots"], kp, vp)
        return [q, *bi.read_quantized_cache(kp, vp, st["table"], st["lens"])]
    if kind == "read":
        return list(bi.read_quantized_cache(kp, vp, st["table"], st["lens"]))
    more = dict(scale=case["D"] ** -0.5, mask="causal")
    if kind == "shared":
        more.update(shared_starts=st["starts"], shared_lens=st["plens"])
        if not case["bits"]:
            return bi.batch_invariant_shared_prefix_attention(st["q"], kp, vp, st["table"], st["lens"], **more)
    return bi.batch_invariant_quantized_paged_attention(st["q"], kp, vp, st["table"], st["lens"], **more)


# ---- one pass: the plain form ------------------------------------------------------------

def _values(codes, groups, bits):
    """What codes [..., D bits / 8] and groups [..., D / g, 2] stand for, of the groups' type. (The
    product of a code and a 16-bit scale is exact in 32 bits; the others take 64.)"""
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    wide = torch.float64 if groups.dtype == torch.float32 else torch.float32
    c = codes.reshape(*groups.shape[:-1], -1).to(wide)
    x = c * groups[..., :1].to(wide) + groups[..., 1:].to(wide)
    return x.float().to(groups.dtype).reshape(codes.shape)


def _gather(pool, case, table):
    """The rows of every sequence, [B, Hkv, L, D], of type T."""
    bits = case["bits"]

    def rows(t):
        t = t[table.long()].transpose(1, 2)             # [B, Hkv, pages, page, ...]
        return t.reshape(*t.shape[:2], -1, *t.shape[4:])

    return _values(rows(pool[0]), rows(pool[1]), bits) if bits else rows(pool)


def _quantize(x, bits, group):
    """Codes [..., D bits / 8] and groups [..., D / group, 2] of x, of x's type."""
    top = 2 ** bits - 1
    y = x.reshape(*x.shape[:-1], -1, group).float()
    low, high = y.amin(-1), y.amax(-1)
    # quotients next to a border between two codes: in 64 bits, rounded to 32
    scale = ((high - low).double() / top).float().to(x.dtype).float()
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = ((y - low[..., None]).double() / scale[..., None].double()).float()
    codes = q.round().clamp(0, top).to(torch.uint8).reshape(x.shape)
    if bits == 4:
        codes = codes[..., 0::2] | codes[..., 1::2] << 4
    return codes, torch.stack([scale, low], -1).to(x.dtype)


def _plain_write(st):
    case, dt = st["case"], st["q"].dtype
    page, half = case["page"], case["D"] // case["part"] // 2
    at = st["pos"].long()
    cos, sin = (t[at][:, :, None, :] for t in (st["cos"], st["sin"]))

    def turned(x):
        # a sum of a product and a rounded product, rounded once: in 64 bits, as
        # a key's value may be next to a border between two codes
        x = x.float()
        a, b = x[..., :half], x[..., half:2 * half]
        y1 = a.double() * cos - (b * sin).double()
        y2 = b.double() * cos + (a * sin).double()
        return torch.cat([y1.float(), y2.float(), x[..., 2 * half:]], -1).to(dt)

    keep = st["slots"] >= 0
    slot = st["slots"][keep]
    for pool, x in ((st["kp"], turned(st["k"])), (st["vp"], st["v"])):
        for held, new in zip(pool, _quantize(x[keep], case["bits"], case["group"])):
            held[slot // page, :, slot % page] = new
    return [turned(st["q"]).transpose(1, 2).contiguous(), *_plain_read(st)]


def _plain_read(st):
    L = st["table"].shape[1] * st["case"]["page"]
    held = (torch.arange(L, device=DEV) < st["lens"][:, None])[:, None, :, None]
    both = (_gather(st[p], st["case"], st["table"]) for p in ("kp", "vp"))
    return [torch.where(held, x, torch.zeros((), dtype=x.dtype, device=DEV)) for x in both]


def _plain_attn(st):
    case, q = st["case"], st["q"].float()
    B, Hq, Hkv, D, T = (case[k] for k in ("B", "Hq", "Hkv", "D", "T"))
    k, v = (_gather(st[p], case, st["table"]).float() for p in ("kp", "vp"))
    L = k.shape[2]
    s = torch.matmul(q.reshape(B, Hkv, -1, D), k.transpose(2, 3).contiguous()).reshape(B, Hq, T, L) * D ** -0.5
    seen = st["lens"][:, None] - T + 1 + torch.arange(T, device=DEV)           # [B, T]
    visible = (torch.arange(L, device=DEV) < seen[:, :, None])[:, None]
    s = torch.where(visible, s, torch.full((), -math.inf, device=DEV))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(B, Hkv, -1, L), v).reshape(B, Hq, T, D)
    return torch.where(total > 0, out / total, torch.zeros_like(out)).to(st["q"].dtype)


def run(st):
    if own:
        return _own(st)
    return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn, "shared": _plain_attn}[st["case"]["kind"]](st)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    kind, es = case["kind"], 4 if case["dtype"] == "fp32" else 2
    B, Hkv, D, bits = case["B"], case["Hkv"], case["D"], case["bits"]
    row = D * bits / 8 + D // case["group"] * 2 * es if bits else D * es        # bytes of one key's row
    if kind == "write":
        T, Hq, page = case["T"], case["Hq"], case["page"]
        tokens, rot = B * (T + (T + 1) // 2) / 2, D // case["part"]
        dense = -(-T // page) * page * B
        return {"bytes": es * D * (2 * B * T * Hq + 2 * tokens * Hkv) + 2 * Hkv * row * tokens + B * T * 12
                + max(T, 64) * rot * 4 + 2 * Hkv * D * es * dense + 4 * B * (1 + T / page),
                "flops": 3 * rot * (B * T * Hq + tokens * Hkv) + 10 * tokens * Hkv * D}
    L = case["L"]
    if kind == "read":
        keys = B * (L + 1) / 2
        dense = -(-L // case["page"]) * case["page"] * B
        return {"bytes": 2 * Hkv * (row * keys + D * es * dense), "flops": 4 * Hkv * D * keys}
    T, Hq = case["T"], case["Hq"]
    if kind == "shared":
        mine = (L + T) / 2
        pairs = T * (case["P"] + mine - (T - 1) / 2)
        held = case["groups"] * case["P"] + B * mine
    else:
        keys = (L + (T + 1) // 2) / 2
        pairs = T * (keys - (T - 1) / 2) if keys >= T else keys * (keys + 1) / 2
        held = B * keys
    return {"bytes": 2 * Hkv * row * held + es * B * 2 * T * Hq * D, "flops": 4 * B * pairs * Hq * D}


# ---- the same in 64 bits ------------------------------------------------------------------

def _exact_rows(case, pool, table, n):
    """Rows 0 .. n - 1 of one sequence, [Hkv, n, D], in 64 bits: each the value of type T that it stands for."""
    at = torch.arange(n, device=DEV)
    page, row = table.long()[at // case["page"]], at % case["page"]
    if not case["bits"]:
        return pool[page, :, row].transpose(0, 1).double()
    codes, groups = (t[page, :, row].transpose(0, 1) for t in pool)
    if case["bits"] == 4:
        wide = torch.empty(*codes.shape[:2], 2 * codes.shape[2], dtype=torch.int64, device=DEV)
        wide[..., 0::2], wide[..., 1::2] = codes % 16, codes // 16
        codes = wide
    scale, bias = (x.double().repeat_interleave(case["group"], -1) for x in groups.unbind(-1))
    return torch.addcmul(bias, codes.double(), scale).to(DTYPES[case["dtype"]]).double()


def _exact_attn(case, st):
    B, Hq, Hkv, D, T = (case[k] for k in ("B", "Hq", "Hkv", "D", "T"))
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["lens"].tolist()):
        k, v = (_exact_rows(case, st[p], st["table"][b], n) for p in ("kp", "vp"))
        first = max(0, T - n)                             # rows in front of the sequence see nothing
        at = torch.arange(n - T + first, n, device=DEV).unsqueeze(1)
        hide = torch.arange(n, device=DEV).unsqueeze(0) > at
        for h in range(Hq):
            s = st["q"][b, h, first:].double() @ k[h // (Hq // Hkv)].t().contiguous() / math.sqrt(D)
            out[b, h, first:] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v[h // (Hq // Hkv)]
    return out


def _exact_read(case, st):
    L = st["table"].shape[1] * case["page"]
    both = torch.zeros(2, case["B"], case["Hkv"], L, case["D"], dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["lens"].tolist()):
        for i, p in enumerate(("kp", "vp")):
            both[i, b, :, :n] = _exact_rows(case, st[p], st["table"][b], n)
    return list(both)


def _exact_write(case, st):
    dt, D, group, top = DTYPES[case["dtype"]], case["D"], case["group"], 2 ** case["bits"] - 1
    half = D // case["part"] // 2
    at = st["pos"].long()
    turn = torch.complex(st["cos"].double()[at], st["sin"].double()[at])[:, :, None, :]

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:2 * half].double()) * turn
        return torch.cat([z.real, z.imag, x[..., 2 * half:].double()], -1)

    def held(x):
        """Rows of type T after a stay in the cache."""
        y = x.to(dt).double().unflatten(-1, (D // group, group))
        low = y.min(-1, keepdim=True).values
        scale = ((y.max(-1, keepdim=True).values - low) / top).to(dt).double()
        scale[scale == 0] = 1
        code = torch.round((y - low) / scale).clamp(max=top)
        return (low + code * scale).to(dt).double().flatten(-2)

    T, L = case["T"], st["table"].shape[1] * case["page"]
    both = torch.zeros(2, case["B"], case["Hkv"], L, D, dtype=torch.float64, device=DEV)
    keys = turned(st["k"])
    for b, n in enumerate(st["lens"].tolist()):
        for i, x in enumerate((keys, st["v"])):
            both[i, b, :, :n] = held(x[b, T - n:]).transpose(0, 1)
    return [turned(st["q"]).transpose(1, 2).contiguous(), *both]


def exact(case, seed):
    st = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attn": _exact_attn, "shared": _exact_attn}[case["kind"]](case, st)
