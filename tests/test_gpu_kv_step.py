"""The operators together, as a program uses them: tables, rotation, append and attention of one step after another, eager
and captured, against the same steps in 64 bits on the cache that the kernels wrote."""
import math

import pytest
import torch

from oracle import kv_oracle as K
from pasa_amd.kv_cache import KVCache8, append_kv, cached_attention, extend_block_tables
from pasa_amd.rotary import RotaryAxes, grid_positions, rope_axes

pytestmark = pytest.mark.gpu


class Program:
    """Requests that grow by some tokens a step: rows of a fixed batch size, the rest of it padding."""

    def __init__(self, device, R, Hq, Hk, D, page, pages, width, tokens):
        self.device, self.tokens, self.D = device, tokens, D
        i32 = dict(dtype=torch.int32, device=device)
        self.cache = KVCache8.empty(pages, Hk, D, page, device=device)
        self.tables = torch.full((R, width), -1, **i32)
        self.lens, self.new = torch.zeros(R, **i32), torch.zeros(R, **i32)
        self.free, self.left = torch.arange(pages, **i32), torch.tensor([pages], **i32)
        self.axes = RotaryAxes.sections((D // 2, D // 4, D // 4), pairing="halves", shared=True, device=device)
        self.q = torch.zeros(tokens, Hq, D, dtype=torch.bfloat16, device=device)
        self.k, self.v = (torch.zeros(tokens, Hk, D, dtype=torch.bfloat16, device=device) for _ in range(2))

    def step(self):
        s = extend_block_tables(self.tables, self.lens, self.new, self.free, self.left, self.cache.page_size, self.tokens)
        pos = s.positions.expand(3, -1)                     # text: the same position on every axis
        q, k = rope_axes(self.q, self.k, pos, self.axes)
        append_kv(self.cache, k, self.v, s.slots)
        o = cached_attention(q, self.cache, self.tables, s.lens, s.cu_q, causal=True)
        self.lens.copy_(s.lens)
        self.left.copy_(s.num_free)
        return o, q, k, s

    def fill(self, new, seed):
        g = torch.Generator().manual_seed(seed)
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        for t in (self.q, self.k, self.v):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))

    def check(self, o, q, k, s, what):
        c, tables = self.cache, self.tables.tolist()
        lens, cu = s.lens.tolist(), s.cu_q.tolist()
        ref, _, bound, _ = K.attention(q.cpu(), c.k.cpu(), c.v.cpu(), c.k_exp.cpu(), c.v_exp.cpu(), tables, lens, cu,
                                       self.D ** -0.5, True)
        tol = bound * (1 + 2.0 ** -8) + 2.0 ** -8 * ref.abs() + 2.0 ** -133
        worst = float(((o.cpu().double() - ref).abs() / tol)[:cu[-1]].max()) if cu[-1] else 0.0
        rot = K.rope(self.q.cpu()[None], s.positions.cpu().expand(3, 1, -1), self.axes.inv_freq.cpu(), self.axes.axis.cpu(), "halves")[0]
        assert float((q.cpu().double() - rot).abs().max()) <= 2.0 ** -8 * float(rot.abs().max()) + 2.0 ** -18
        # What the cache holds of the step's keys: half a code's step, 2^-4, of the value, or of the smallest normal code.
        page = c.page_size
        kv, vv = (t.cpu() for t in c.values())
        for i, slot in enumerate(s.slots.tolist()):
            if slot < 0:
                continue
            for held, x, e in ((kv, k, c.k_exp), (vv, self.v, c.v_exp)):
                got, want = held[slot // page, :, slot % page], x[i].cpu().float()
                step = 2.0 ** -4 * want.abs() + 2.0 ** -10 * 2.0 ** e[slot // page].cpu().float()[:, None]
                assert bool(((got - want).abs() <= step).all()), (what, i)
        assert bool((o[cu[-1]:] == 0).all())
        print(f"[step] {what}: worst {worst:.3f} of the tolerance", flush=True)
        assert worst <= 1, what


def test_steps_of_ragged_requests(device):
    p = Program(device, 5, 6, 3, 64, 16, 60, 16, 90)
    for i, new in enumerate(([30, 1, 0, 20, 7], [1, 1, 1, 1, 1], [1, 1, 1, 1, 1], [5, 0, 60, 1, 3], [40, 1, 1, 0, 17], [1, 1, 1, 1, 1])):
        p.fill(new, i)
        p.check(*p.step(), f"step {i}")
    assert p.lens.tolist() == [78, 5, 64, 24, 30]


def test_pages_run_out(device):
    """Tokens that no page is left for are neither written nor seen; the requests go on with what they have."""
    p = Program(device, 3, 2, 2, 64, 16, 6, 8, 70)
    p.fill([40, 20, 10], 1)
    o, q, k, s = p.step()
    assert s.lens.tolist() == [40, 20, 10][:1] + [20, 10] and s.num_free.tolist() == [0]
    p.fill([20, 1, 20], 2)
    o, q, k, s = p.step()
    assert s.lens.tolist() == [48, 21, 16] and s.num_free.tolist() == [0]
    assert (s.slots >= 0).sum().item() == 8 + 1 + 6


def test_captured_step(device):
    """One captured step, replayed on other tokens and lengths, between eager steps of a second program."""
    a, b = (Program(device, 4, 4, 2, 128, 32, 40, 8, 24) for _ in range(2))
    for p in (a, b):
        p.fill([9, 3, 5, 7], 0)
        p.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        o, q, k, s = a.step()
    torch.cuda.synchronize()
    for i, new in enumerate(([1, 1, 1, 1], [6, 6, 6, 6], [1, 0, 20, 2], [0, 0, 0, 0], [1, 1, 1, 1])):
        a.fill(new, 10 + i)
        b.fill(new, 10 + i)
        want = b.step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(s.slots, want[3].slots) and torch.equal(a.lens, b.lens), i
        for x, y in ((a.cache.k, b.cache.k), (a.cache.v, b.cache.v), (a.cache.k_exp, b.cache.k_exp), (a.cache.v_exp, b.cache.v_exp)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), i
        b.check(*want, f"replay {i}")


def test_two_graphs(device):
    """Two captured attentions with workspaces of their own, replayed in turn and at once on two streams."""
    g0 = torch.Generator().manual_seed(3)
    c = KVCache8.empty(64, 2, 128, 64, device=device)
    for i in range(0, 64 * 64, 512):
        k, v = torch.randn(2, 512, 2, 128, generator=g0).to(torch.bfloat16).to(device)
        append_kv(c, k, v, torch.arange(i, i + 512, device=device))
    i32 = dict(dtype=torch.int32, device=device)
    tables = torch.arange(64, **i32).view(2, 32)
    lens = torch.tensor([2000, 1500], **i32)
    qs = [torch.randn(2, 4, 128, generator=g0).to(torch.bfloat16).to(device) for _ in range(2)]
    want = [cached_attention(q, c, tables, lens, causal=True).clone() for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cached_attention(q, c, tables, lens, causal=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams if i % 2 else [torch.cuda.current_stream()] * 2):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), i


def test_video_chunks_against_dense(device):
    """Three chunks of a small video, each attending to all so far: near the dense attention on the unquantised keys and
    values.  A code is off by at most 2^-4 of its value: outputs stay within 2^-3 of the largest value's size."""
    H, D, page = 2, 128, 64
    frames, h, w = 2, 6, 10
    n = frames * h * w
    axes = RotaryAxes.video(D, device=device)
    cache = KVCache8.empty(16, H, D, page, device=device)
    table = torch.randperm(16, device=device).to(torch.int32)[None]
    g = torch.Generator().manual_seed(4)
    ks, vs = [], []
    for chunk in range(3):
        q, k, v = torch.randn(3, 1, n, H, D, generator=g).to(torch.bfloat16).to(device)
        pos = grid_positions(frames, h, w, first_frame=chunk * frames, device=device)
        q, k = rope_axes(q, k, pos, axes)
        ks.append(k)
        vs.append(v)
        at = torch.arange(chunk * n, chunk * n + n, device=device)
        append_kv(cache, k[0], v[0], table[0, at // page].long() * page + at % page)
        lens = torch.tensor([chunk * n + n], dtype=torch.int32, device=device)
        o = cached_attention(q[0], cache, table, lens)
        kk, vv = torch.cat(ks, 1)[0].double(), torch.cat(vs, 1)[0].double()
        ref = torch.stack([torch.softmax(q[0, :, i].double() @ kk[:, i].t() / math.sqrt(D), -1) @ vv[:, i] for i in range(H)], 1)
        assert float((o.double() - ref).abs().max()) <= 2.0 ** -3 * float(vv.abs().max())
        cos = float((o.double() * ref).sum() / (o.double().norm() * ref.norm()))
        print(f"[step] chunk {chunk}: cosine to the unquantised attention {cos:.6f}", flush=True)
        assert cos > 0.99
