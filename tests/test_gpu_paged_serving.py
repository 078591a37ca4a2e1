"""Requests served from a paged cache through one decoder block: slots, rotary
embedding with the write, attention with capped scores and a distance bias, the
norms around the block, over a padded batch of prompts, a second chunk of some,
and decode steps. Each attention is checked against the 64-bit formula over the
keys and values kept beside; a request's results are its bits when served alone
from other pages."""

import pytest
import torch

import paged_ref as ref
from helpers import DT, bits, gen, randn

pytestmark = pytest.mark.gpu
I32 = torch.int32
HQ, HKV, D, H, PAGE, COLS = 6, 2, 64, 256, 16, 12


class _Server:
    def __init__(self, dt, B, seed):
        g = gen(seed)
        self.dt, self.B = DT[dt], B
        self.wqkv = randn(((HQ + 2 * HKV) * D, H), self.dt, gen(1), H ** -0.5)
        self.wo = randn((H, HQ * D), self.dt, gen(2), (HQ * D) ** -0.5)
        self.norms = [(1 + randn((H,), torch.float32, gen(3 + i), 0.1)).to(self.dt) for i in range(2)]
        ang = torch.outer(torch.arange(PAGE * COLS).double(), 1e4 ** (-torch.arange(24).double() / 24))
        self.cos, self.sin = ang.cos().float().cuda(), ang.sin().float().cuda()   # 48 of 64 dims turn
        n = B * COLS + 5
        self.free = torch.randperm(n, generator=g).to(I32).cuda()
        self.kp, self.vp = (torch.full((n, PAGE, HKV, D), float("nan"), dtype=self.dt, device="cuda").transpose(1, 2)
                            for _ in range(2))
        self.table = torch.full((B, COLS), -1, dtype=I32, device="cuda")
        self.lens = torch.zeros(B, dtype=I32, device="cuda")
        self.cursor = torch.zeros(1, dtype=I32, device="cuda")
        self.slopes = (2.0 ** -torch.arange(1, HQ + 1)).cuda()

    def step(self, x, residual, new):
        """x, residual [B, T, H]; new tokens of each request, in its last rows."""
        import mlx_batch_invariant_amd as bi
        B, T, _ = x.shape
        plan = bi.paged_slots(self.lens, new, self.table, self.free, page_size=PAGE, max_new=T, cursor=self.cursor)
        qkv = bi.batch_invariant_matmul(x, self.wqkv.t())
        q, k, v = (t.reshape(B, T, -1, D) if not t.is_contiguous() else t.view(B, T, -1, D)
                   for t in qkv.split([HQ * D, HKV * D, HKV * D], -1))
        q = bi.rope_paged_cache(q, k, v, self.cos, self.sin, plan.positions, plan.slots, self.kp, self.vp)
        a = bi.batch_invariant_paged_attention(q, self.kp, self.vp, self.table, plan.kv_lens, mask="causal", softcap=20.0,
                                               slopes=self.slopes)
        o = bi.batch_invariant_matmul(a.transpose(1, 2).reshape(B, T, HQ * D), self.wo.t())
        y, h = bi.batch_invariant_residual_rms_norm(o, residual, *self.norms, 1e-5, scale=0.5)
        self.lens, self.cursor = plan.kv_lens, plan.cursor
        return plan, q, a, y, h

    def keys(self, b):
        """Keys and values of request b, out of its pages in order."""
        n = int(self.lens[b])
        at = self.table[b].long().repeat_interleave(PAGE)[:n]
        row = torch.arange(n, device="cuda") % PAGE
        return self.kp[at, :, row].transpose(0, 1), self.vp[at, :, row].transpose(0, 1)


def _schedule(B):
    """New tokens of every request at each step: prompts, later chunks, decode."""
    return [[37, 1, 90][:B], [0, 50, 20][:B]] + [[1] * B] * 6


def _inputs(dt, step, b, n):
    g = gen(1000 * step + b)
    return randn((n, H), DT[dt], g), randn((n, H), DT[dt], g, 2.0)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_served_requests(dt):
    B = 3
    together = _Server(dt, B, 50)
    alone = [_Server(dt, 1, 60 + b) for b in range(B)]
    for s, counts in enumerate(_schedule(B)):
        T = max(counts)
        x, res = torch.zeros(B, T, H, dtype=DT[dt], device="cuda"), torch.zeros(B, T, H, dtype=DT[dt], device="cuda")
        for b, n in enumerate(counts):
            x[b, T - n:], res[b, T - n:] = _inputs(dt, s, b, n)
        new = torch.tensor(counts, dtype=I32, device="cuda")
        plan, q, a, y, h = together.step(x, res, new)
        assert plan.kv_lens.tolist() == [sum(c[b] for c in _schedule(B)[:s + 1]) for b in range(B)]
        held = together.table[together.table >= 0]
        assert held.unique().numel() == held.numel() == int(together.cursor)
        for b, n in enumerate(counts):
            if n == 0:
                continue
            # 64-bit attention over the request's own keys and values
            k, v = together.keys(b)
            mine = q[b:b + 1, :, T - n:].cpu()
            want, absv, dot, bias = ref.attention(mine, k[None].cpu(), v[None].cpu(), D ** -0.5, None, True, 20.0,
                                                  together.slopes.cpu())
            allow = ref.attention_allowance(want, absv, dot, bias, DT[dt], D, 1, 20.0)
            assert ((a[b:b + 1, :, T - n:].double().cpu() - want).abs() <= allow).all()
            # the request alone, from pages of its own
            one = alone[b]
            _, _, a1, y1, h1 = one.step(x[b:b + 1, T - n:].contiguous(), res[b:b + 1, T - n:].contiguous(),
                                        new[b:b + 1])
            k1, v1 = one.keys(0)
            assert bits(k1) == bits(k) and bits(v1) == bits(v)
            assert bits(a1[0]) == bits(a[b, :, T - n:])
            assert bits(y1[0]) == bits(y[b, T - n:]) and bits(h1[0]) == bits(h[b, T - n:])


def test_decode_step_in_a_graph():
    """A decode step captured once and replayed with the lengths and cursor handed
    on, against the same steps run eagerly."""
    B = 3
    eager, graphed = _Server("bf16", B, 70), _Server("bf16", B, 70)
    x0, r0 = (torch.stack([t[i] for t in (_inputs("bf16", 0, b, 40) for b in range(B))]) for i in range(2))
    new = torch.full((B,), 40, dtype=I32, device="cuda")
    for srv in (eager, graphed):
        srv.step(x0, r0, new)
    x, r = torch.zeros(B, 1, H, dtype=torch.bfloat16, device="cuda"), torch.zeros(B, 1, H, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(B, dtype=I32, device="cuda")
    lens, cursor = graphed.lens.clone(), graphed.cursor.clone()

    def step():
        graphed.lens, graphed.cursor = lens, cursor
        return graphed.step(x, r, one)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                          # the pages and rows it writes are written again below
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, _, a, y, h = step()
    for s in range(10):                                 # crosses a page
        xs, rs = (torch.stack([t[i] for t in (_inputs("bf16", 1 + s, b, 1) for b in range(B))]) for i in range(2))
        x.copy_(xs)
        r.copy_(rs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = eager.step(xs, rs, one)
        assert torch.equal(plan.kv_lens, want[0].kv_lens) and torch.equal(plan.slots, want[0].slots)
        for got, w in zip((a, y, h), want[2:]):
            assert bits(got) == bits(w)
        lens.copy_(plan.kv_lens)
        cursor.copy_(plan.cursor)
    del graph
