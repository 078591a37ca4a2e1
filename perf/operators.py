"""The workloads that the paged-serving operators are measured on.

One case is one call of a decoder block that serves requests from a paged K/V
cache: the block table and the slots of the new tokens (``slots``), the rotary
embedding with the write into the pages (``rope``), the attention over the cache
with capped scores, a distance bias, a document mask or a prefix mask
(``attn``), and the norms around the block with gate and residual (``norm``).
Sizes are those of the repository's own workloads: 32 / 8 heads of 128 and 14 /
2 heads of 64, hidden sizes 4096 and 896, prompts of up to a few thousand
tokens, decode batches of 1 to 256.

With ``own`` false, ``run`` computes a case in plain torch operations, in 32
bits, rounded once at the end; with ``own`` true it makes the library's calls.
``exact`` computes a case in 64 bits, sequence by sequence.
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
EPS = 1e-5


# ---- the cases -------------------------------------------------------------------

def _case(kind, name, **values):
    c = {"kind": kind, **values}
    return {"name": name, **c} if name else c


def _slots(name, B, T, L, page):
    """B requests with up to T new tokens each, at most L tokens held and new."""
    return _case("slots", name, B=B, T=T, L=L, page=page)


def _rope(name, B, T, heads, L, page, axes, part, tables, dtype):
    """The rotated head dims are D / part; tables in 32 bits or in the inputs' type."""
    Hq, Hkv, D = heads
    return _case("rope", name, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, L=L, page=page, axes=axes, part=part, tables=tables,
                 dtype=dtype)


def _attn(name, B, heads, T, L, page, dtype, causal=True, ragged=True, cap=0.0, slopes=False, docs=0, prefix=False):
    """T query tokens at the end of up to L keys; page 0: contiguous caches;
    docs: the mean length of a document, 0 for no document mask."""
    Hq, Hkv, D = heads
    return _case("attn", name, B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, L=L, page=page, dtype=dtype, causal=causal,
                 ragged=ragged, cap=cap, slopes=slopes, docs=docs, prefix=prefix)


def _norm(name, rows, D, dtype, post, pre, gate, scale):
    return _case("norm", name, rows=rows, D=D, dtype=dtype, post=post, pre=pre, gate=gate, scale=scale)


_LLAMA, _QWEN, _MHA = (32, 8, 128), (14, 2, 64), (8, 8, 128)


def listed():
    return [
        # One decode step of a serving batch: a slot for each sequence's next
        # token, a new page for a sixteenth of them. Latency alone.
        _slots("slots_decode", 64, 1, 8192, 16),
        # A batch of prompt chunks enters the cache.
        _slots("slots_prompts", 256, 2048, 8192, 16),
        # A decode step's queries, keys and values of one block.
        _rope("rope_decode", 64, 1, _LLAMA, 1024, 16, 1, 1, "fp32", "bf16"),
        # Prompts with images: a time, a height and a width position per token.
        _rope("rope_three_axes", 4, 2048, _LLAMA, 2048, 16, 3, 1, "fp32", "bf16"),
        # Odd chunks of a small model that rotates half of each head, two axes.
        _rope("rope_partial", 3, 517, _QWEN, 1500, 64, 2, 2, "same", "fp16"),
        # A decode step over long ragged paged caches with capped scores.
        _attn("attn_cap_decode", 64, _LLAMA, 1, 8192, 16, "bf16", causal=False, cap=50.0),
        # Whole prompts with capped scores.
        _attn("attn_cap_prefill", 4, _LLAMA, 2048, 2048, 0, "bf16", ragged=False, cap=50.0),
        # A chunk of each of three prompts against longer caches, with a bias
        # that grows with the distance.
        _attn("attn_bias_chunk", 3, _QWEN, 500, 4000, 16, "fp16", slopes=True),
        # Documents packed into one long row.
        _attn("attn_documents", 1, _LLAMA, 8192, 8192, 0, "bf16", ragged=False, docs=700),
        # Prompts whose first part is seen from everywhere, in 32 bits.
        _attn("attn_prefix_fp32", 2, _MHA, 601, 601, 0, "fp32", ragged=False, cap=30.0, prefix=True),
        # The norms around one block for a decode step, and for a prompt batch
        # with a gate.
        _norm("norm_decode", 16, 4096, "bf16", True, True, "none", 1.0),
        _norm("norm_prompts", 16384, 4096, "bf16", True, True, "channel", 0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("slots", "rope", "rope", "attn", "attn", "attn", "attn", "norm", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32"))
    if kind == "slots":
        L = _log(rng, 64, 8192)
        return _slots(None, _log(rng, 1, 256), _log(rng, 1, min(L, 2048)), L, rng.choice((1, 8, 16, 16, 64, 256)))
    if kind == "rope":
        T = _log(rng, 1, 2048)
        B = _log(rng, 1, min(64, max(2, 8192 // T)))
        return _rope(None, B, T, rng.choice((_LLAMA, _QWEN, _MHA)), T + _log(rng, 1, 1000), rng.choice((8, 16, 64)),
                     rng.choice((1, 2, 3)), rng.choice((1, 1, 2)), rng.choice(("fp32", "same")), dtype)
    if kind == "attn":
        heads = rng.choice((_LLAMA, _QWEN, _MHA))
        mods = rng.choice(("cap", "cap", "slopes", "docs", "prefix", "all"))
        T = rng.choice((1, _log(rng, 2, 1024)))
        L = T + _log(rng, 1, 2000)
        B = _log(rng, 1, 64 if T == 1 else 2)
        every = mods == "all"
        return _attn(None, B, heads, T, L, rng.choice((0, 0, 8, 16, 64)), dtype, causal=mods != "cap" or T > 1,
                     ragged=rng.random() < 0.7, cap=rng.choice((20.0, 50.0)) if every or mods == "cap" else 0.0,
                     slopes=every or mods == "slopes", docs=_log(rng, 20, 800) if every or mods == "docs" else 0,
                     prefix=every or mods == "prefix")
    return _norm(None, _log(rng, 1, 16384), rng.choice((896, 4096, 4097, 1000)), dtype, *rng.choice(
        ((True, True), (True, True), (False, True), (True, False))), rng.choice(("none", "channel", "row")),
        rng.choice((1.0, 0.5)))


# ---- inputs (made from the seed alone) ----------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _randint(g, lo, hi, shape):
    """Whole numbers lo .. hi, hi included, as int32."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV, dtype=torch.int32)


def _requests(case, g):
    """Token counts held and new of each request, a block table with the held
    pages in it, and the free pages, in a random order of the pool's pages."""
    B, T, L, page = (case[k] for k in ("B", "T", "L", "page"))
    new = _randint(g, (T + 1) // 2, T, (B,))
    held = (torch.rand(B, generator=g, device=DEV) * (L - new + 1)).to(torch.int32)
    per = -(-L // page)
    pages = torch.randperm(B * per + 8, generator=g, device=DEV).to(torch.int32)
    table = pages[:B * per].reshape(B, per)
    kept = torch.arange(per, device=DEV)[None, :] < ((held + page - 1) // page)[:, None]
    free = torch.cat([table[~kept], pages[B * per:]])
    return held, new, torch.where(kept, table, torch.zeros_like(table)), free


def _tables(case, n):
    """cos and sin of positions [0, n): rotated pairs of dims along the columns."""
    half = case["D"] // case["part"] // 2
    inv = THETA ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    ang = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    dt = torch.float32 if case["tables"] == "fp32" else DTYPES[case["dtype"]]
    return ang.cos().to(dt), ang.sin().to(dt)


def _sections(case):
    """Pairs of dims that turn with each axis: all; 3/8 and 5/8; 2/8, 3/8 and 3/8."""
    half = case["D"] // case["part"] // 2
    return {1: (half,), 2: (half // 8 * 3, half // 8 * 5), 3: (half // 4, half // 8 * 3, half // 8 * 3)}[case["axes"]]


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    st = {"case": case}
    if kind == "slots":
        st["held"], st["new"], st["table"], st["free"] = _requests(case, g)
        return st
    dt = DTYPES[case["dtype"]]
    if kind == "rope":
        B, T, Hq, Hkv, D, L, page = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "L", "page"))
        held, new, table, free = _requests(case, g)
        # Tokens of request b sit at the end of its T rows, behind padding rows.
        row = torch.arange(T, device=DEV)[None, :] - (T - new)[:, None]
        pos = (held[:, None] + row).clamp(min=0)
        per = table.shape[1]
        full = torch.randperm(B * per, generator=g, device=DEV).reshape(B, per)
        slots = full.gather(1, pos.long() // page) * page + pos % page
        st["slots"] = torch.where(row >= 0, slots, torch.full_like(slots, -1))
        extra = _randint(g, 0, 40, (case["axes"] - 1, B, T)) if case["axes"] > 1 else pos[:0].reshape(0, B, T)
        st["pos"] = torch.cat([pos[None].to(torch.int32), extra]) if case["axes"] > 1 else pos[None].to(torch.int32)
        st["cos"], st["sin"] = _tables(case, max(L, 64))
        st["q"], st["k"], st["v"] = (_randn(g, B, T, h, D, dtype=dt) for h in (Hq, Hkv, Hkv))
        st["kp"], st["vp"] = (torch.zeros(B * per, Hkv, page, D, dtype=dt, device=DEV) for _ in range(2))
        return st
    if kind == "attn":
        B, Hq, Hkv, D, T, L, page = (case[k] for k in ("B", "Hq", "Hkv", "D", "T", "L", "page"))
        st["q"] = _randn(g, B, Hq, T, D, dtype=dt, scale=3.0)
        per = -(-L // page) if page else 0
        shape = (B * per, Hkv, page, D) if page else (B, Hkv, L, D)
        st["k"], st["v"] = _randn(g, *shape, dtype=dt), _randn(g, *shape, dtype=dt)
        st["table"] = torch.randperm(B * per, generator=g, device=DEV).to(torch.int32).reshape(B, per) if page else None
        # prompts shorter than the T rows of a padded batch leave their first rows empty
        st["lens"] = _randint(g, (T + 1) // 2, L, (B,)) if case["ragged"] else torch.full((B,), L, dtype=torch.int32, device=DEV)
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device=DEV) / Hq) if case["slopes"] else None
        st["docs"] = None
        if case["docs"]:
            first = torch.rand((B, per * page if page else L), generator=g, device=DEV) < 1.0 / case["docs"]
            st["docs"] = first.cumsum(1).to(torch.int32)
        st["prefix"] = (torch.rand(B, generator=g, device=DEV) * L / 2).to(torch.int32) if case["prefix"] else None
        return st
    rows, D = case["rows"], case["D"]
    st["x"], st["res"] = _randn(g, rows, D, dtype=dt, scale=1.5), _randn(g, rows, D, dtype=dt, scale=4.0)
    st["post"], st["pre"] = ((1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dt) for _ in range(2))
    gate = {"none": None, "channel": (D,), "row": (rows, D)}[case["gate"]]
    st["gate"] = None if gate is None else _randn(g, *gate, dtype=dt)
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
    if kind == "slots":
        got = bi.paged_slots(st["held"], st["new"], st["table"], st["free"], page_size=case["page"], max_new=case["T"])
        return [got.slots, got.positions, got.kv_lens, got.cursor, st["table"]]
    if kind == "rope":
        q = bi.rope_paged_cache(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["pos"], st["slots"], st["kp"],
                                st["vp"], sections=_sections(case))
        return [q, st["kp"], st["vp"]]
    if kind == "attn":
        more = dict(scale=case["D"] ** -0.5, mask="causal" if case["causal"] else None, softcap=case["cap"] or None,
                    slopes=st["slopes"], doc_ids=st["docs"], prefix_lens=st["prefix"])
        if st["table"] is not None:
            return bi.batch_invariant_paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], **more)
        return bi.batch_invariant_attention(st["q"], st["k"], st["v"], kv_lens=st["lens"], **more)
    y, h = bi.batch_invariant_residual_rms_norm(st["x"], st["res"], st["post"] if case["post"] else None,
                                                st["pre"] if case["pre"] else None, EPS, gate=st["gate"],
                                                scale=case["scale"], post_norm=case["post"], pre_norm=case["pre"])
    return [y, h] if case["pre"] else [y]


# ---- one pass: the plain form ------------------------------------------------------------

def _plain_slots(st):
    case = st["case"]
    T, page = case["T"], case["page"]
    held, new, table, free = st["held"], st["new"], st["table"], st["free"]
    have, want = (held + page - 1) // page, (held + new + page - 1) // page
    need = want - have
    incl = need.cumsum(0)
    fits = (want <= table.shape[1]) & ((need == 0) | (incl <= free.shape[0]))
    col = torch.arange(table.shape[1], device=DEV)[None, :]
    fresh = fits[:, None] & (col >= have[:, None]) & (col < want[:, None])
    pick = ((incl - need)[:, None] + col - have[:, None]).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(fresh, free[pick], table))
    row = torch.arange(T, device=DEV)[None, :] - (T - new)[:, None]
    live = fits[:, None] & (row >= 0)
    pos = torch.where(live, held[:, None] + row, torch.zeros_like(row)).to(torch.int32)
    slots = table.gather(1, pos.long() // page).long() * page + pos % page
    lens = torch.where(fits, held + new, held)
    cursor = torch.where(fits, need, torch.zeros_like(need)).sum().to(torch.int32).reshape(1)
    return [torch.where(live, slots, torch.full_like(slots, -1)), pos, lens, cursor, table]


def _plain_rope(st):
    case = st["case"]
    page, half = case["page"], case["D"] // case["part"] // 2
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=DEV),
                                   torch.tensor(_sections(case), device=DEV), output_size=half)
    at = st["pos"].long()[axis].permute(1, 2, 0)                      # [B, T, half]
    col = torch.arange(half, device=DEV)
    cos, sin = (t.float()[at, col][:, :, None, :] for t in (st["cos"], st["sin"]))

    def turned(x):
        x = x.float()
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)

    dt = st["q"].dtype
    keep = st["slots"] >= 0
    slot = st["slots"][keep]
    st["kp"][slot // page, :, slot % page] = turned(st["k"])[keep].to(dt)
    st["vp"][slot // page, :, slot % page] = st["v"][keep]
    return [turned(st["q"]).to(dt).transpose(1, 2).contiguous(), st["kp"], st["vp"]]


def _plain_attn(st):
    case, q = st["case"], st["q"].float()
    B, Hq, Hkv, D, T = (case[k] for k in ("B", "Hq", "Hkv", "D", "T"))
    k, v = st["k"], st["v"]
    if st["table"] is not None:
        pages = st["table"].long()
        k, v = (t[pages].transpose(1, 2).reshape(B, Hkv, -1, D) for t in (k, v))
    L = k.shape[2]
    s = torch.matmul(q.reshape(B, Hkv, -1, D), k.float().transpose(2, 3).contiguous()).reshape(B, Hq, T, L)
    s *= D ** -0.5
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    pos = st["lens"][:, None] - T + torch.arange(T, device=DEV)        # [B, T]
    key = torch.arange(L, device=DEV)
    if st["slopes"] is not None:
        far = (pos[:, :, None] - key).abs().float()
        s = s - st["slopes"][None, :, None, None] * far[:, None]
    end = st["lens"][:, None].expand(B, T)
    if case["causal"]:
        seen = pos + 1
        if st["prefix"] is not None:
            seen = torch.maximum(seen, torch.minimum(st["prefix"], st["lens"])[:, None])
        end = torch.where(pos >= 0, seen, torch.zeros_like(seen))
    visible = key < end[:, :, None]
    if st["docs"] is not None:
        mine = torch.where(pos >= 0, st["docs"].gather(1, pos.clamp(min=0).long()), torch.full_like(pos, -1))
        visible = visible & (st["docs"][:, None, :L] == mine[:, :, None])
    visible = visible[:, None]
    s = torch.where(visible, s, torch.full((), -math.inf, device=DEV))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(B, Hkv, -1, L), v.float()).reshape(B, Hq, T, D)
    return torch.where(total > 0, out / total, torch.zeros_like(out)).to(st["q"].dtype)


def _plain_norm(st):
    case, dt = st["case"], st["x"].dtype

    def norm(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()

    u = st["x"].float()
    if case["post"]:
        u = norm(u, st["post"])
    if st["gate"] is not None:
        u = u * st["gate"].float()
    y = st["res"].float() + u * case["scale"]
    return [y.to(dt), norm(y, st["pre"]).to(dt)] if case["pre"] else [y.to(dt)]


def run(st):
    if own:
        return _own(st)
    return {"slots": _plain_slots, "rope": _plain_rope, "attn": _plain_attn, "norm": _plain_norm}[st["case"]["kind"]](st)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    kind, es = case["kind"], 4 if case.get("dtype") == "fp32" else 2
    if kind == "slots":
        B, T, page = case["B"], case["T"], case["page"]
        tokens = B * (T + (T + 1) // 2) / 2
        # lengths in and out, slots and positions out, one table entry read or
        # taken from the free list and written for every page that is touched
        return {"bytes": 12 * B + 12 * B * T + 12 * (B + tokens / page), "flops": 0}
    if kind == "rope":
        B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
        tokens = B * (T + (T + 1) // 2) / 2
        rot = D // case["part"]
        tab = 4 if case["tables"] == "fp32" else es
        return {"bytes": es * D * (2 * B * T * Hq + 4 * tokens * Hkv) + B * T * (8 + 4 * case["axes"])
                + min(B * T, max(case["L"], 64)) * rot * tab,
                "flops": 3 * rot * (B * T * Hq + tokens * Hkv)}
    if kind == "attn":
        B, Hq, Hkv, D, T, L = (case[k] for k in ("B", "Hq", "Hkv", "D", "T", "L"))
        keys = (L + (T + 1) // 2) / 2 if case["ragged"] else L
        pairs = T * keys
        if case["causal"]:
            pairs = T * (keys - (T - 1) / 2) if keys >= T else keys * (keys + 1) / 2
        if case["prefix"]:                                            # a prefix of L / 4 keys on average
            first = max(0.0, L / 4 - max(0.0, keys - T))
            pairs += first * first / 2
        if case["docs"]:
            pairs = min(pairs, T * case["docs"])
        return {"bytes": es * B * (2 * min(keys, pairs) * Hkv * D + 2 * T * Hq * D), "flops": 4 * B * pairs * Hq * D}
    n = case["rows"] * case["D"]
    per = 3 + case["pre"] + (case["gate"] == "row")
    return {"bytes": es * (per * n + case["D"] * (case["post"] + case["pre"] + (case["gate"] == "channel"))),
            "flops": n * (4 * case["post"] + 4 * case["pre"] + 3)}


# ---- the same in 64 bits ------------------------------------------------------------------

def _exact_attn(case, st):
    B, Hq, Hkv, D, T = (case[k] for k in ("B", "Hq", "Hkv", "D", "T"))
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=DEV)
    lens = st["lens"].tolist()
    for b in range(B):
        n = lens[b]
        if st["table"] is None:
            k, v = st["k"][b, :, :n].double(), st["v"][b, :, :n].double()
        else:
            rows = torch.arange(n, device=DEV)
            page = st["table"][b].long()[rows // case["page"]]
            k, v = (st[x][page, :, rows % case["page"]].transpose(0, 1).double() for x in ("k", "v"))
        at = torch.arange(n - T, n, device=DEV).unsqueeze(1)
        j = torch.arange(n, device=DEV).unsqueeze(0)
        hide = torch.zeros(T, n, dtype=torch.bool, device=DEV)
        if case["causal"]:
            hide = j > at
            if st["prefix"] is not None:
                hide = hide & (j >= st["prefix"][b])
            hide = hide | (at < 0)
        if st["docs"] is not None:
            ids = st["docs"][b, :n]
            hide = hide | (ids[None, :] != ids[at.clamp(min=0)]) | (at < 0)
        for h in range(Hq):
            s = st["q"][b, h].double() @ k[h // (Hq // Hkv)].t().contiguous() / math.sqrt(D)
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][h].double() * (at - j).abs().double()
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1).nan_to_num(0.0)
            out[b, h] = p @ v[h // (Hq // Hkv)]
    return out


def _exact_rope(case, st):
    B, T, page = case["B"], case["T"], case["page"]
    half = case["D"] // case["part"] // 2
    c, s = (torch.empty(B, T, 1, half, dtype=torch.float64, device=DEV) for _ in range(2))
    d = 0
    for a, n in enumerate(_sections(case)):
        rows = st["pos"][a].long()
        c[:, :, 0, d:d + n] = st["cos"].double()[rows, d:d + n]
        s[:, :, 0, d:d + n] = st["sin"].double()[rows, d:d + n]
        d += n

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:2 * half].double()) * torch.complex(c, s)
        return torch.cat([z.real, z.imag, x[..., 2 * half:].double()], -1)

    k, kp, vp = turned(st["k"]), st["kp"].double(), st["vp"].double()
    for b in range(B):
        rows = torch.nonzero(st["slots"][b] >= 0)[:, 0]
        at = st["slots"][b, rows]
        kp[at // page, :, at % page] = k[b, rows]
        vp[at // page, :, at % page] = st["v"][b, rows].double()
    return [turned(st["q"]).transpose(1, 2).contiguous(), kp, vp]


def _exact_norm(case, st):
    u, y = st["x"].double(), st["res"].double()
    if case["post"]:
        u = u * torch.rsqrt(u.square().mean(1, keepdim=True) + EPS) * st["post"].double()
    y = y + case["scale"] * (u if st["gate"] is None else u * st["gate"].double())
    if not case["pre"]:
        return [y]
    return [y, y * torch.rsqrt(y.square().mean(1, keepdim=True) + EPS) * st["pre"].double()]


def exact(case, seed):
    if case["kind"] == "slots":
        return None                                   # whole numbers only
    st = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "norm": _exact_norm}[case["kind"]](case, st)
