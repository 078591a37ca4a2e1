"""Plain 64-bit (or whole-number) forms of the paged-serving operators, for the tests."""

from __future__ import annotations

import torch


def slots(lens, news, table, free, page, T, cursor=0):
    """paged_slots request by request on Python lists: (slots, positions, lens,
    cursor, table)."""
    B, cap = len(lens), (len(table[0]) if table else 0) * page
    table = [list(r) for r in table]
    at = min(max(cursor, 0), len(free))
    end, out_slots, out_pos, out_lens = at, [], [], []
    for b in range(B):
        n, new = min(max(lens[b], 0), cap), max(news[b], 0)
        have, want = -(-n // page), -(-(n + new) // page)
        fits = want <= len(table[b]) and new <= T
        need = want - have if fits else 0
        end += need
        ok = fits and (need == 0 or end <= len(free))
        if ok:
            for j in range(need):
                table[b][have + j] = free[end - need + j]
            if need:
                at = end
        row_s, row_p = [-1] * T, [0] * T
        if ok:
            for i in range(new):
                p = n + i
                page_no = table[b][p // page]
                row_s[T - new + i] = page_no * page + p % page if page_no >= 0 else -1
                row_p[T - new + i] = p
        out_slots.append(row_s)
        out_pos.append(row_p)
        out_lens.append(n + new if ok else n)
    return out_slots, out_pos, out_lens, at, table


def rope(x, cos, sin, pos, sections):
    """x [B, T, H, D] in 64 bits, positions [A, B, T] (clamped into the tables)."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    half = cos.shape[1]
    c, s = (torch.empty(*x.shape[:2], 1, half, dtype=torch.float64) for _ in range(2))
    d = 0
    for a, n in enumerate(sections):
        row = pos[a].long().clamp(0, cos.shape[0] - 1)
        c[:, :, 0, d:d + n], s[:, :, 0, d:d + n] = cos[row, d:d + n], sin[row, d:d + n]
        d += n
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def residual_norm(x, res, w1, w2, eps, gate=None, scale=1.0, post=True, pre=True):
    x, y = x.double(), res.double()
    ones = torch.ones(x.shape[-1], dtype=torch.float64)
    if post:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (ones if w1 is None else w1.double())
    y = y + (x if gate is None else x * gate.double()) * scale
    h = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * (ones if w2 is None else w2.double())
    return y, h if pre else None


def attention(q, k, v, scale, lens, causal, softcap=None, slopes=None, docs=None, prefix=None):
    """q [B, Hq, T, D], k / v [B, Hkv, L, D] in 64 bits: the outputs, and per
    output the softmax of |v| and the row's largest score terms (for the bounds:
    sum |q k| scale, slope x distance). Masked keys take no part, whatever K and
    V hold there; a row that sees none is 0."""
    q, k, v = q.double(), k.double(), v.double()
    B, Hq, T, D = q.shape
    L, G = k.shape[2], Hq // k.shape[1]
    out, absv = (torch.zeros(B, Hq, T, D, dtype=torch.float64) for _ in range(2))
    dot, bias = (torch.zeros(B, Hq, T, 1, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        n = L if lens is None else min(max(int(lens[b]), 0), L)
        for t in range(T):
            p = n - T + t
            end = n if not causal else 0 if p < 0 else max(p + 1, min(int(prefix[b]), n) if prefix is not None else 0)
            keys = torch.arange(end)
            if docs is not None:
                keys = keys[docs[b, :end] == docs[b, p]] if p >= 0 else keys[:0]
            if not len(keys):
                continue
            kk, vv = (x[b, :, keys].repeat_interleave(G, 0) for x in (k, v))
            qq = q[b, :, t, :, None]
            s = (kk @ qq)[..., 0] * scale
            dot[b, :, t, 0] = (kk.abs() @ qq.abs()).amax((1, 2)) * scale
            if softcap is not None:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                far = slopes[:, None].double() * (p - keys).abs()
                bias[b, :, t, 0] = far.abs().amax(1)
                s = s - far
            w = torch.softmax(s, 1)[:, None]
            out[b, :, t], absv[b, :, t] = (w @ vv)[:, 0], (w @ vv.abs())[:, 0]
    return out, absv, dot, bias


def attention_allowance(want, absv, dot, bias, dtype, D, nsplit, softcap=None):
    """How far an output may be from the 64-bit one. Half a step of the result, and
    2 A (e_p + e_acc + 2 e_s) with A the softmax of |v|:
      e_p   = 2^-17 (bf16) / 2^-21 (f16) / 0: a weight is carried as hi + lo;
      e_acc = (2 x 256 + 2 nsplit) 2^-24: one rounding per MFMA block and merge;
      e_s     a score's error: (D + 2) 2^-24 of sum |q k| scale; 12 2^-24 softcap
              for the cap (of 1 - 2 / (x + 1): 2 from x = exp2, 6 from the
              reciprocal and its argument, 1 from the difference, 2 from the
              factor and its rounding); 4 2^-24 of the largest slope x distance
              (slope, its factor, the sum)."""
    e = 2.0 ** -24
    e_p = {torch.bfloat16: 2.0 ** -17, torch.float16: 2.0 ** -21, torch.float32: 0.0}[dtype]
    e_s = (D + 2) * e * dot + 12 * e * (softcap or 0.0) + 4 * e * bias
    fi = torch.finfo(dtype)
    return fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps + 2 * absv * (e_p + (512 + 2 * nsplit) * e + 2 * e_s)
