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
    """q [B, Hq, T, D], k / v [B, Hkv, L, D] in 64 bits. Masked keys take no
    part, whatever K and V hold there; a row that sees none is 0."""
    q, k, v = q.double(), k.double(), v.double()
    B, Hq, T, D = q.shape
    L, G = k.shape[2], Hq // k.shape[1]
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64)
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
            for h in range(Hq):
                s = k[b, h // G, keys] @ q[b, h, t] * scale
                if softcap is not None:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s - slopes[h].double() * (p - keys).abs()
                out[b, h, t] = torch.softmax(s, 0) @ v[b, h // G, keys]
    return out
