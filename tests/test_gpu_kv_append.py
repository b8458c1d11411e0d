"""New keys and values into the cache in 8 bits: codes and exponents equal to the oracle's, bit for bit."""
import random

import pytest
import torch

from oracle import kv_oracle as K
from pasa_amd.kv_cache import KVCache8, append_kv

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def make_cache(device, pages, heads, head_dim, page, seed=0):
    """A cache that holds values: normal codes of every size, exponents from -12 to 3."""
    c = KVCache8.empty(pages, heads, head_dim, page, device=device)
    g = torch.Generator().manual_seed(seed)
    for t in (c.k, c.v):
        x = torch.randn(t.shape, generator=g) * torch.exp(2 * torch.randn(t.shape, generator=g))
        t.copy_(x.clamp(-448, 448).to(E4M3).to(device))
    c.k[..., head_dim:] = 0
    c.v[:, :, head_dim:] = 0
    for t in (c.k_exp, c.v_exp):
        t.copy_(torch.randint(-12, 4, t.shape, generator=g).to(torch.int8))
    return c


def same(c, ref, what):
    for name in ("k", "v", "k_exp", "v_exp"):
        a, b = getattr(c, name).cpu(), ref[name]
        if a.dtype == E4M3:
            a, b = a.view(torch.uint8), b.view(torch.uint8)
            a, b = (torch.where((t & 0x7f) == 0x7f, torch.full_like(t, 0x7f), t) for t in (a, b))  # either NaN
        n = int((a != b).sum())
        print(f"[append] {what}: {name}: {n} of {a.numel()} differ", flush=True)
        assert n == 0, f"{what}: {name} at {(a != b).nonzero()[:4].tolist()}"


def check(c, k, v, slots, what):
    ref = {n: getattr(c, n).cpu().clone() for n in ("k", "v", "k_exp", "v_exp")}
    slots = torch.as_tensor(slots, dtype=torch.int64)
    K.append(ref["k"], ref["v"], ref["k_exp"], ref["v_exp"], k.cpu(), v.cpu(), slots, c.head_dim)
    append_kv(c, k, v, slots.to(c.k.device))
    torch.cuda.synchronize()
    same(c, ref, what)


def tokens(T, H, D, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, T, H, D, generator=g) * torch.exp(spread * torch.randn(2, T, H, 1, generator=g))
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("H,D", [(1, 128), (3, 64), (2, 80), (2, 5), (1, 1)])
def test_single_tokens(device, dtype, page, H, D):
    c = make_cache(device, 40, H, D, page)
    k, v = tokens(33, H, D, dtype, spread=3.0)
    rng = random.Random(page)
    slots = [p * page + rng.choice([0, 1, page - 1, rng.randrange(page)]) for p in rng.sample(range(40), 33)]
    check(c, k, v, slots, f"{dtype} page {page} D {D}")


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dtype,H,D", [(torch.bfloat16, 2, 128), (torch.float16, 1, 64), (torch.float32, 2, 96)])
@pytest.mark.parametrize("runs", [[1], [16], [63, 1, 64], [65, 130, 7, 300], [128, 128], [1500]])
def test_runs(device, dtype, H, D, page, runs):
    """Runs that begin and end anywhere in a page, over pages in any order, with slots to skip between and behind."""
    rng = random.Random(page + len(runs))
    slots, need = [], sum(-(-n // page) + 1 for n in runs)
    ids = rng.sample(range(need + 3), need + 3)
    for n in runs:
        at = rng.choice([0, 0, page - 1, rng.randrange(page)])
        mine = [ids.pop() for _ in range(-(-(at + n) // page))]
        slots += [mine[(at + i) // page] * page + (at + i) % page for i in range(n)] + rng.choice([[], [-1], [-1, 10 ** 12]])
    slots += [-1] * 3
    c = make_cache(device, need + 3, H, D, page)
    k, v = tokens(len(slots), H, D, dtype, len(slots))
    check(c, k, v, slots, f"runs {runs} page {page}")


def test_token_by_token_grows_the_scale(device):
    """A page filled one token at a time, each larger than the last: every append scales what is there."""
    c = make_cache(device, 3, 2, 64, 16)
    for i in range(20):
        k, v = tokens(1, 2, 64, torch.bfloat16, i) * 1.7 ** i
        check(c, k, v, [16 + i] if i < 16 else [32 + i - 16], f"token {i}")


def test_values_at_the_edges(device):
    """Zeros, subnormals, 448 * 2^e and its neighbours, halves between two codes, infinities, NaN, the largest floats."""
    top = torch.finfo(torch.float32).max
    rows = [[0.0] * 8, [448.0, -448.0, 447.9, 1.0, 2 ** -9, 2 ** -10, 3 * 2 ** -11, -2 ** -10],
            [448.0001, 17.0, 18.0, 19.0, 1.0625, 1.1875, -1.0625, 2 ** -9 * 1.5], [float("inf"), 1.0, -3.0, 0.5, 0, 0, 0, 0],
            [float("nan"), float("-inf"), 2.0, 0, 0, 0, 0, 1.0], [top, -top, 1.0, 2.0 ** 60, 2.0 ** 50, 0, 0, 0],
            [1e-45, 1e-40, 0, 0, 0, 0, 0, -1e-44], [2.0 ** -50, 2.0 ** -42, 2.0 ** -60, 0, 0, 0, 0, 0], [float("nan")] * 8]
    x = torch.tensor(rows)[:, None, :].cuda()
    for page in (16, 64):
        c = make_cache(device, len(rows) + 1, 1, 8, page)
        check(c, x, -x.flip(2), [i * page for i in range(len(rows))], f"begins a page of {page}")
        c = make_cache(device, len(rows) + 1, 1, 8, page)
        check(c, x, x.flip(0), [i * page + 3 for i in range(len(rows))], f"goes on in a page of {page}")
    assert not torch.isnan(c.values()[0][8, 0, :3].float()).any()


def test_strides_and_alignment(device):
    page = 16
    big = tokens(40, 6, 128, torch.bfloat16)
    k, v = big[0][::2, 1:4], big[1][:20, 3:]                        # token and head strides
    check(make_cache(device, 4, 3, 128, page), k, v, list(range(5, 25)), "strides")
    flat = tokens(1, 1, 20 * 3 * 64 + 1, torch.float16)[0, 0, 0]
    off = flat[1:].view(20, 3, 64)                                  # not on 16 bytes
    check(make_cache(device, 4, 3, 64, page), off, off.flip(0).contiguous(), list(range(20)), "off 16 bytes")
    hm = tokens(3, 20, 64, torch.bfloat16)[0].transpose(0, 1)       # head-major
    check(make_cache(device, 4, 3, 64, page), hm, hm, list(range(20, 40)), "head-major")
    one = tokens(20, 1, 64, torch.bfloat16)[0].expand(20, 3, 64)    # the same for every head
    check(make_cache(device, 4, 3, 64, page), one, one, list(range(20)), "expanded")


def test_the_same_slots_again_and_two_calls(device):
    """The same tokens twice give the same page; what other pages hold stays."""
    c = make_cache(device, 6, 2, 128, 64)
    k, v = tokens(50, 2, 128, torch.bfloat16)
    slots = torch.arange(70, 120, device=device)
    append_kv(c, k, v, slots)
    once = [t.clone() for t in (c.k, c.v, c.k_exp, c.v_exp)]
    append_kv(c, k, v, slots)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(once, (c.k, c.v, c.k_exp, c.v_exp)))
    append_kv(c, k[:0], v[:0], slots[:0])
    append_kv(c, k, v, torch.full_like(slots, -1))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(once, (c.k, c.v, c.k_exp, c.v_exp)))


def test_graph(device):
    c = make_cache(device, 12, 2, 64, 16)
    k, v = tokens(30, 2, 64, torch.bfloat16)
    slots = torch.arange(30, device=device)
    append_kv(c, k, v, slots)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        append_kv(c, k, v, slots)
    for i in range(3):
        slots.copy_(torch.arange(30, device=device) + 37 * i)
        k.mul_(1.3)
        ref = {n: getattr(c, n).cpu().clone() for n in ("k", "v", "k_exp", "v_exp")}
        K.append(ref["k"], ref["v"], ref["k_exp"], ref["v_exp"], k.cpu(), v.cpu(), slots.cpu(), 64)
        g.replay()
        torch.cuda.synchronize()
        same(c, ref, f"replay {i}")
