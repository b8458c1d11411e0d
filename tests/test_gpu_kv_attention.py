"""Attention to the cache in 8 bits, against the oracle in 64 bits on the codes themselves.

Tolerance of an output: the oracle's bound of the kernel's arithmetic (p in fp16, fp32 scores and sums), then half a
step of the output's type; fp16 also half of its smallest subnormal."""
import math
import random

import pytest
import torch

from oracle import kv_oracle as K
from pasa_amd.kv_cache import KVCache8, cached_attention

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(device, kv, new, Hq, Hk, D, page, dtype, seed=0, spare=2, exps=(-9, -5), extra_width=1):
    """Requests of kv cached tokens, new of them queries, in pages in any order; what no request holds is NaN codes."""
    rng = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in kv]
    P = sum(pages) + spare
    c = KVCache8.empty(P, Hk, D, page, device=device)
    k = torch.full((P, Hk, page, c.k.shape[3]), 0x7f, dtype=torch.uint8)
    v = torch.full((P, Hk, c.k.shape[3], page), 0xff, dtype=torch.uint8)
    ids = list(range(P))
    rng.shuffle(ids)
    width = max([1] + pages) + extra_width
    tables = []
    for n, p in zip(kv, pages):
        mine = [ids.pop() for _ in range(p)]
        tables.append(mine + [rng.choice([-1, 0, 10 ** 9])] * (width - p))
        for j, i in enumerate(mine):
            m = min(page, n - j * page)
            code = lambda *s: (torch.randn(s, generator=g) * 90).clamp(-448, 448).to(E4M3).view(torch.uint8)
            k[i, :, :m] = 0
            v[i, :, :, :m] = 0
            k[i, :, :m, :D] = code(Hk, m, D)
            v[i, :, :D, :m] = code(Hk, D, m)
    c.k.view(torch.uint8).copy_(k)
    c.v.view(torch.uint8).copy_(v)
    for t in (c.k_exp, c.v_exp):
        t.copy_(torch.randint(exps[0], exps[1] + 1, t.shape, generator=g).to(torch.int8))
    q = (torch.randn(sum(new), Hq, D, generator=g) * 1.5).to(dtype).to(device)
    cu = [0] + torch.tensor(new).cumsum(0).tolist()
    return c, q, tables, kv, cu


def check(case, what, **kw):
    c, q, tables, kv, cu = case
    dev = q.device
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    scale = kw.pop("scale", None)
    o, lse = cached_attention(q, c, i32(tables), i32(kv), i32(cu), return_lse=True, scale=scale, **kw)
    torch.cuda.synchronize()
    s = q.shape[2] ** -0.5 if scale is None else scale
    ref, ref_lse, bound, lse_bound = K.attention(q.cpu(), c.k.cpu(), c.v.cpu(), c.k_exp.cpu(), c.v_exp.cpu(), tables, kv, cu,
                                                 s, kw.get("causal", False), kw.get("window"))
    compare(o, lse, ref, ref_lse, bound, lse_bound, what)
    return o, lse


def compare(o, lse, ref, ref_lse, bound, lse_bound, what):
    o, lse = o.cpu(), lse.cpu()
    tol = bound * (1 + 2.0 ** -8) + HALF_STEP[o.dtype] * ref.abs() + (2.0 ** -25 if o.dtype == torch.float16 else 2.0 ** -133)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(o), nan), f"{what}: NaN in other places"
    err = torch.where(nan, 0.0, (o.double() - ref).abs())
    worst = float((err / torch.where(nan, 1.0, tol)).max()) if o.numel() else 0.0
    print(f"[attention] {what}: worst {worst:.3f} of the tolerance", flush=True)
    assert worst <= 1, what
    empty = ref_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty), what
    assert bool((o[empty] == 0).all()), what
    ok = ~empty & ~torch.isnan(ref_lse)
    assert torch.equal(torch.isnan(lse), torch.isnan(ref_lse)), what
    assert bool(((lse.double() - ref_lse).abs()[ok] <= lse_bound[ok]).all()), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hk,D", [(1, 1, 128), (4, 4, 64), (10, 2, 128), (7, 1, 96), (40, 1, 64), (3, 3, 7)])
def test_single_tokens(device, dtype, page, Hq, Hk, D):
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 130, 0, 300, 511]
    check(make(device, kv, [1] * len(kv), Hq, Hk, D, page, dtype), f"{dtype} page {page} {Hq}/{Hk} x {D}", causal=True)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [None, 1, 50, 200])
@pytest.mark.parametrize("new,kv", [([2, 3, 4], [2, 70, 300]), ([40, 1, 0, 17], [90, 1, 33, 17]), ([130], [257]), ([70, 5], [20, 5])])
def test_masks(device, causal, window, new, kv):
    """Few and many new tokens, more of them than cached ones (rows before the first key), with and without a window."""
    for D, Hq, Hk, dtype, page in ((128, 4, 2, torch.bfloat16, 32), (64, 3, 3, torch.float16, 64)):
        check(make(device, kv, new, Hq, Hk, D, page, dtype, seed=sum(kv)), f"causal {causal} window {window} new {new} D {D}",
              causal=causal, window=window)


@pytest.mark.parametrize("new", [1, 16, 150])
def test_long_and_split(device, new):
    """Thousands of keys: parts of the keys joined, and pages that were given back in between."""
    case = make(device, [5000, 3001], [new, max(1, new - 3)], 2, 1, 128, 64, torch.bfloat16)
    check(case, f"long, {new} new", causal=True)
    c, q, tables, kv, cu = case
    for j in (0, 1, 2, 17, 40):
        tables[0][j] = -1
    tables[1][46] = 10 ** 8
    check(case, f"long, {new} new, dropped pages", causal=True, window=4000)
    tables[1][:] = [-1] * len(tables[1])
    check(case, f"long, {new} new, a request without pages")


def test_scales_far_apart(device):
    """Pages whose exponents lie 40 apart, in both directions, and zero pages with the lowest one."""
    for lo, hi in ((-30, 10), (-50, -50), (8, 9)):
        c, q, tables, kv, cu = make(device, [400, 70], [1, 33], 2, 2, 64, 16, torch.bfloat16, exps=(lo, hi))
        c.k_exp.fill_(-8)
        c.v[3:5] = 0
        c.v_exp[3:5] = -50
        check((c, q, tables, kv, cu), f"value exponents {lo} .. {hi}", causal=True)


def test_large_scores(device):
    """Scores of some hundreds: one key takes all the weight.  fp32 scores are off by (D + 8) 2^-24 of their terms."""
    c, q, tables, kv, cu = make(device, [200, 65], [3, 65], 2, 1, 64, 32, torch.float16, exps=(-3, -3))
    c.k_exp.fill_(0)
    check((c, q, tables, kv, cu), "large scores", causal=True)


def test_nan_reaches_only_who_sees_it(device):
    """NaN codes in keys and values: rows that see the key are NaN (all channels for a key, the channel for a value),
    rows that the causal mask or the window keeps from it are what they were."""
    for new in (1, 40, 150):
        kv = [200, 150]
        new = [new, min(new, 100)]
        case = make(device, kv, new, 2, 2, 64, 16, torch.bfloat16, seed=5)
        c, q, tables, _, cu = case
        # Request 0: a value channel of key 180; request 1: a value of key 149, the last, and of key 60.
        for r, j, d in ((0, 180, 3), (1, 149, 40), (1, 60, 63)):
            c.v.view(torch.uint8)[tables[r][j // 16], :, d, j % 16] = 0x7f
        check(case, f"NaN value, {new} new", causal=True)
        check(case, f"NaN value, {new} new, window", causal=True, window=15)
        for r, j, d in ((0, 190, 1),):
            c.k.view(torch.uint8)[tables[r][j // 16], 1, j % 16, d] = 0xff
        check(case, f"NaN key, {new} new", causal=True)
        check(case, f"NaN key, {new} new, all seen")
        check(case, f"NaN key, {new} new, one key", causal=True, window=1)


def test_uniform_rows_strides_out_and_padding(device):
    c, q, tables, kv, cu = make(device, [90, 33, 64], [4, 4, 4], 6, 3, 64, 32, torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    t, n = i32(tables), i32(kv)
    want = cached_attention(q, c, t, n, i32(cu), causal=True)
    assert torch.equal(cached_attention(q, c, t, n, causal=True), want), "cu_q None: the same number for each request"
    # q as a slice of a projection, out head-major.
    wide = torch.randn(12, 10, 64, device=device).to(torch.bfloat16)
    wide[:, 2:8] = q
    out = torch.full((6, 12, 64), 7.0, device=device, dtype=torch.bfloat16)
    got = cached_attention(wide[:, 2:8], c, t, n, i32(cu), causal=True, out=out.transpose(0, 1))
    assert got.data_ptr() == out.data_ptr() and torch.equal(out.transpose(0, 1), want)
    flat = torch.empty(q.numel() + 1, device=device, dtype=torch.bfloat16)[1:].view(q.shape).copy_(q)
    assert torch.equal(cached_attention(flat, c, t, n, i32(cu), causal=True), want), "off 16 bytes"
    # Rows behind the last request: left as they were in a given tensor, 0 in a new one.
    more = torch.cat([q, torch.full_like(q[:5], float("nan"))])
    buf = torch.full_like(more, 9.0)
    cached_attention(more, c, t, n, i32(cu), causal=True, out=buf)
    assert torch.equal(buf[:12], want) and bool((buf[12:] == 9).all())
    new, lse = cached_attention(more, c, t, n, i32(cu), causal=True, return_lse=True)
    assert torch.equal(new[:12], want) and bool((new[12:] == 0).all()) and bool((lse[12:] == -math.inf).all())
    # Keys from max_kv_len on are not looked at.
    few = cached_attention(q, c, t, n, i32(cu), max_kv_len=33)
    ref, _, _, _ = K.attention(q.cpu(), c.k.cpu(), c.v.cpu(), c.k_exp.cpu(), c.v_exp.cpu(), tables, [33, 33, 33], cu, 0.125)
    assert float((few.cpu().double() - ref).abs().max()) <= 2.0 ** -7 * float(ref.abs().max())
    assert bool((cached_attention(q, c, t, n, i32(cu), max_kv_len=0) == 0).all())
    assert cached_attention(q[:0], c, t, n, i32([0, 0, 0, 0])).shape == (0, 6, 64)
    # The table as columns of a wider one.
    tw = torch.full((3, t.shape[1] + 5), 2, dtype=torch.int32, device=device)
    tw[:, :t.shape[1]] = t
    assert torch.equal(cached_attention(q, c, tw[:, :t.shape[1]], n, i32(cu), causal=True), want)


def test_row_starts_out_of_range_stay_in_bounds(device):
    """Row starts and lengths that no caller means: rows outside q are neither read nor written."""
    c, q, tables, kv, cu = make(device, [90, 33], [4, 4], 2, 1, 64, 16, torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    for starts in ([0, 5, 100], [-7, 4, 8], [0, 2 ** 31 - 1, 2 ** 31 - 1], [8, 4, 0], [5, 3, 8]):
        cached_attention(q, c, i32(tables), i32(kv), i32(starts), causal=True)
    cached_attention(q, c, i32(tables), i32([2 ** 31 - 1, -4]), i32(cu), causal=True)
    torch.cuda.synchronize()
    assert torch.isfinite(cached_attention(q, c, i32(tables), i32(kv), i32(cu), causal=True)).all()


def test_same_bits_on_every_call_and_stream(device):
    case = make(device, [3000, 700, 64], [1, 3, 2], 8, 2, 128, 64, torch.bfloat16)
    c, q, tables, kv, cu = case
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    args = i32(tables), i32(kv), i32(cu)
    want = cached_attention(q, c, *args, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = cached_attention(q, c, *args, causal=True)
    b = cached_attention(q, c, *args, causal=True)                 # both at once, each with its own workspace
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, want) and torch.equal(b, want)


def test_offsets_past_32_bits(device):
    """A cache of more than 2^32 bytes of codes: pages at its far end."""
    page, H, D = 128, 8, 128
    P = 2 ** 32 // (page * H * D) + 3
    c = KVCache8.empty(P, H, D, page, device=device)
    g = torch.Generator().manual_seed(1)
    small, q, tables, kv, cu = make(device, [300], [2], 8, 8, 128, page, torch.bfloat16)
    at = [P - 1, 0, P - 2]
    for j, i in enumerate(tables[0][:3]):
        c.k.view(torch.uint8)[at[j]] = small.k.view(torch.uint8)[i]
        c.v.view(torch.uint8)[at[j]] = small.v.view(torch.uint8)[i]
        c.k_exp[at[j]], c.v_exp[at[j]] = small.k_exp[i], small.v_exp[i]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    want = cached_attention(q, small, i32(tables), i32(kv), i32(cu), causal=True)
    got = cached_attention(q, c, i32([at]), i32(kv), i32(cu), causal=True)
    # A part of the keys for each workgroup goes by the table's width; both tables hold at most four pages.
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -6 * float(want.float().abs().max())
    from pasa_amd.kv_cache import append_kv
    k, v = torch.randn(2, 1, H, D, device=device, generator=torch.Generator(device=device).manual_seed(3)).to(torch.bfloat16)
    append_kv(c, k, v, torch.tensor([(P - 1) * page], device=device))
    append_kv(small, k, v, torch.tensor([tables[0][0] * page], device=device))
    assert torch.equal(c.k.view(torch.uint8)[P - 1, :, 0], small.k.view(torch.uint8)[tables[0][0], :, 0])
    assert torch.equal(c.v.view(torch.uint8)[P - 1, :, :, 0], small.v.view(torch.uint8)[tables[0][0], :, :, 0])
