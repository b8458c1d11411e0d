"""Calls at the edges of what the cache's attention and the rotary embedding are documented to take: rows in front of
the first request, requests of one length, appends of many runs, captured backward passes beside living graphs, pieces
that do not line up."""
import random

import pytest
import torch

from oracle import kv_oracle as K
from pasa_amd.kv_cache import cached_attention
from pasa_amd.rotary import RotaryAxes, rope_axes
from test_gpu_kv_append import check as append_check, make_cache, tokens
from test_gpu_kv_attention import check, compare, make
from test_gpu_rotary import close as against, make as values

pytestmark = pytest.mark.gpu


# (heads of q, of k, head dim, new, cached): rows of one tile, split rows, tiles of 128 and of 256 rows, those split.
@pytest.mark.parametrize("Hq,Hk,D,new,kv", [
    (2, 2, 128, [1, 1], [40, 70]), (4, 1, 64, [3, 9], [90, 700]), (2, 1, 128, [2, 1], [9000, 8000]),
    (8, 1, 64, [40, 60], [300, 200]), (8, 1, 128, [90, 80], [500, 130]), (8, 1, 128, [70, 60], [6000, 5000])])
@pytest.mark.parametrize("front", [1, 37])
def test_rows_in_front_of_the_first_request(device, Hq, Hk, D, new, kv, front):
    c, q, tables, kv, cu = make(device, kv, new, Hq, Hk, D, 64, torch.bfloat16, seed=front)
    pad = torch.full((front, Hq, D), float("nan"), dtype=q.dtype, device=device)
    q = torch.cat([pad, q, pad])
    cu = [n + front for n in cu]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    torch.full((64, *q.shape), 7.0, dtype=q.dtype, device=device)  # what a new tensor finds in its memory
    o, lse = cached_attention(q, c, i32(tables), i32(kv), i32(cu), causal=True, return_lse=True)
    out = torch.full_like(q, 3.0)
    cached_attention(q, c, i32(tables), i32(kv), i32(cu), causal=True, out=out)
    torch.cuda.synchronize()
    for rows in (slice(0, front), slice(cu[-1], None)):
        assert bool((o[rows] == 0).all()) and bool((lse[rows] == -float("inf")).all())
        assert bool((out[rows] == 3).all())
    mine = slice(cu[0], cu[-1])
    assert torch.equal(out[mine], o[mine])
    want, _ = check((c, q[mine].contiguous(), tables, kv, [n - front for n in cu]), f"front {front}", causal=True)
    # Another place of the rows in their tiles: another running maximum, and p rounded at another point.
    assert torch.allclose(o[mine].float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -6 * float(want.float().abs().max()))


def test_captured_gradient_beside_a_living_graph(device):
    axes = RotaryAxes.video(64, device=device)
    pos = torch.randint(0, 5000, (3, 33), dtype=torch.int32).to(device)
    q, k = values((2, 33, 4, 64), torch.float16).requires_grad_(), values((2, 33, 2, 64), torch.float16, 1).requires_grad_()
    gq, gk = values(q.shape, q.dtype, 2), values(k.shape, k.dtype, 3)
    alive = rope_axes(q, k, pos, axes)
    with pytest.raises(ValueError, match="graph of this leaf"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            rope_axes(q, k, pos, axes)
    torch.cuda.synchronize()
    q1, k1 = q.detach().requires_grad_(), k.detach().requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rope_axes(q1, k1, pos, axes)
        grads = torch.autograd.grad(out, (q1, k1), (gq, gk))
    for i in range(3):
        pos.copy_(torch.randint(0, 5000, (3, 33), dtype=torch.int32).to(device))
        with torch.no_grad():
            q.mul_(1.01)
            gk.mul_(0.99)
        eager = rope_axes(q, k, pos, axes)
        want = torch.autograd.grad(eager, (q, k), (gq, gk))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((*out, *grads), (*eager, *want)):
            assert torch.equal(a, b), i
    assert alive[0].requires_grad


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("T,H,D,dims", [(1, 1, 8, (8,)), (1, 70, 128, (44, 42, 42)), (5, 3, 96, (32, 32)), (9000, 3, 64, (16, 8, 8)),
                                        (8193, 1, 32, (16, 16)), (3, 2, 256, (256,)), (7, 9, 48, (20, 28)), (7, 9, 48, (20, 22))])
def test_whole_pieces_and_others(device, dtype, pairing, T, H, D, dims):
    """16-byte pieces, and the same values an element off them."""
    axes = RotaryAxes.sections(dims, pairing=pairing, device=device)
    pos = torch.randint(0, 3000, (len(dims), T), dtype=torch.int32).to(device)
    x = values((T, H, D), dtype, T)
    whole, k = rope_axes(x, x[:, :1], pos, axes)
    close = lambda y, x, *a, **kw: against(y[None], x[None], *a, **kw)
    close(whole, x, pos, axes, inverse=False, what="whole pieces")
    close(k, x[:, :1], pos, axes, inverse=False, what="whole pieces, k")
    room = torch.empty(T * H * D + 1, dtype=dtype, device=device)
    off = room[1:].view(T, H, D)
    off.copy_(x)
    close(rope_axes(off, None, pos, axes)[0], x, pos, axes, inverse=False, what="an element off")
    rope_axes(off, None, pos, axes, inplace=True)
    close(off, x, pos, axes, inverse=False, what="an element off, in place")


@pytest.mark.parametrize("T,H,D,page,lengths", [(2500, 8, 128, 64, [1, 1, 2, 5, 13, 16, 40, 64]), (2500, 8, 64, 16, [1, 3, 15, 16]),
                                                (5000, 16, 128, 16, [1, 1, 1, 2]), (5000, 16, 64, 128, [1, 60, 128]), (1100, 2, 96, 32, [1, 7])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_runs_in_one_append(device, dtype, T, H, D, page, lengths):
    """Workgroups that take several tokens: short runs side by side, long ones together, a page to each."""
    rng = random.Random(T + page)
    slots = []
    while len(slots) < T:
        n = min(rng.choice(lengths), T - len(slots), page)
        slots.append((n, rng.randrange(page - n + 1)))
        slots += [None] * (n - 1)
    runs = [s for s in slots if s is not None]
    ids = rng.sample(range(len(runs) + 2), len(runs))
    slots = [i * page + at + j for i, (n, at) in zip(ids, runs) for j in range(n)]
    for i in rng.sample(range(T), 5):
        slots[i] = rng.choice([-1, 10 ** 13])  # ends a run: what is left of it is skipped too
        rest = i + 1
        while rest < T and slots[rest] % page != 0 and slots[rest] // page == (slots[i - 1] // page if i else -1):
            slots[rest] = -1
            rest += 1
    c = make_cache(device, len(runs) + 2, H, D, page, seed=T)
    k, v = tokens(T, H, D, dtype, T, spread=2.0)
    append_check(c, k, v, slots, f"{len(runs)} runs of {T} tokens, page {page}")


# (heads of q, of k, head dim, new, cached): a part of a tile, several, a part of the last; of 16, 32, 128, 256 rows; split.
@pytest.mark.parametrize("Hq,Hk,D,new,kv", [
    (2, 2, 128, 3, 70), (8, 2, 64, 5, 700), (8, 1, 128, 7, 5000), (8, 1, 64, 20, 300), (8, 1, 128, 20, 900),
    (8, 1, 128, 70, 6000), (4, 1, 64, 100, 5000), (1, 1, 128, 300, 310)])
@pytest.mark.parametrize("window", [None, 100])
def test_requests_of_one_length(device, Hq, Hk, D, new, kv, window):
    """Without row starts: every request has its own tiles, and the result is that with row starts, within the bounds."""
    c, q, tables, kv, cu = make(device, [kv, kv - 7, kv - new], [new] * 3, Hq, Hk, D, 32, torch.float16, seed=new)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    o, lse = cached_attention(q, c, i32(tables), i32(kv), causal=True, window=window, return_lse=True)
    torch.cuda.synchronize()
    want = K.attention(q.cpu(), c.k.cpu(), c.v.cpu(), c.k_exp.cpu(), c.v_exp.cpu(), tables, kv, cu, D ** -0.5, True, window)
    compare(o, lse, *want, f"{new} tokens each")
