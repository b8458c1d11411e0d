"""Rotary embedding from positions on several axes, against the oracle in 64 bits.

Tolerance of a channel, before any run: the angle's share of a turn is rounded once to fp32 (at most half a turn, so
2^-25 of one, 2 pi 2^-25 < 2^-22 rad), the sine and cosine add 2^-22, the rotation three fp32 roundings of terms of at
most |x0| + |x1|: together under 2^-20 (|x0| + |x1|).  Then half a step of the output's type."""
import pytest
import torch

from oracle import kv_oracle as K
from pasa_amd import rotary
from pasa_amd.rotary import RotaryAxes, grid_positions, rope_axes

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def say(msg):
    print(f"[rotary] {msg}", flush=True)


def close(got, x, positions, axes, inverse=False, what=""):
    got, x = got.detach().cpu(), x.detach().cpu()
    if positions.dim() == 2:
        positions = positions[:, None]
    pos = positions.expand(-1, x.shape[0], -1).cpu()
    ref = K.rope(x, pos, axes.inv_freq.cpu(), axes.axis.cpu(), axes.pairing, inverse)
    n = axes.inv_freq.numel()
    size = x.double().abs()
    pair = size.clone()
    if axes.pairing == "halves":
        pair[..., :n] += size[..., n:2 * n]
        pair[..., n:2 * n] += size[..., :n]
    else:
        pair[..., 0:2 * n:2] += size[..., 1:2 * n:2]
        pair[..., 1:2 * n:2] += size[..., 0:2 * n:2]
    tiny = torch.finfo(x.dtype).smallest_normal * HALF_STEP[x.dtype] * 2
    tol = HALF_STEP[x.dtype] * ref.abs() + 2.0 ** -20 * pair * (1 + HALF_STEP[x.dtype]) + tiny
    err = (got.double() - ref).abs()
    worst = float((err / tol).max())
    say(f"{what} {tuple(x.shape)} {x.dtype} {axes.pairing}: worst {worst:.3f} of the tolerance")
    assert got.dtype == x.dtype and worst <= 1
    if 2 * n < x.shape[-1]:
        assert torch.equal(got[..., 2 * n:], x[..., 2 * n:]), "channels behind the pairs are copied"


def make(shape, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * 3).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("B,S,Hq,Hk,D,dims", [
    (1, 1, 1, 1, 2, (2, 0, 0)), (1, 7, 12, 12, 128, (44, 42, 42)), (2, 65, 5, 1, 64, (16, 16, 16)),
    (1, 130, 3, 2, 80, (26, 28, 26)), (1, 33, 2, 2, 7, (2, 2, 2)), (1, 40, 40, 8, 256, (64, 96, 96)), (3, 9, 1, 1, 34, (2, 4, 2))])
def test_shapes(device, dtype, pairing, B, S, Hq, Hk, D, dims):
    axes = RotaryAxes.sections(dims, pairing=pairing, shared=pairing == "halves", device=device)
    q, k = make((B, S, Hq, D), dtype), make((B, S, Hk, D), dtype, 1)
    g = torch.Generator().manual_seed(2)
    pos = torch.randint(0, 5000, (3, B, S), generator=g, dtype=torch.int32).to(device)
    keep = q.clone(), k.clone()
    oq, ok = rope_axes(q, k, pos, axes)
    assert torch.equal(q, keep[0]) and torch.equal(k, keep[1])
    close(oq, q, pos, axes, what="q")
    close(ok, k, pos, axes, what="k")
    bq, _ = rope_axes(q, None, pos, axes, inverse=True)
    close(bq, q, pos, axes, inverse=True, what="inverse")


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32])
def test_far_and_fractional_positions(device, dtype):
    axes = RotaryAxes.video(128, device=device)
    far = torch.tensor([[0, 1, 2 ** 24 - 1, 2 ** 24, 1000003], [3, -7, 2 ** 24, 12345678, 5], [0, 2, 4, -(2 ** 23), 9]])
    if dtype == torch.int64:
        far[0, 3] = 2 ** 31 + 12345
    pos = far.to(dtype)
    if dtype == torch.float32:
        pos[0, 0] = 0.375
    q = make((1, 5, 3, 128), torch.float32)
    oq, none = rope_axes(q, None, pos.to(device), axes)
    assert none is None
    close(oq, q, pos.to(device), axes, what="far")


def test_strides_and_in_place(device):
    axes = RotaryAxes.video(64, device=device)
    pos = grid_positions(2, 3, 5, first_frame=9, device=device)
    # Head-major tensors, a slice of a projection, an offset that leaves rows off 16 bytes, and an expanded input.
    bhsd = make((2, 4, 30, 64), torch.bfloat16)
    close(rope_axes(bhsd.transpose(1, 2), None, pos, axes)[0], bhsd.transpose(1, 2), pos, axes, what="head-major")
    proj = make((2, 30, 3 * 4 * 64), torch.bfloat16)
    q, k, _ = proj.unflatten(2, (12, 64)).split(4, 2)
    before = proj.clone()
    want_q, want_k = rope_axes(q, k, pos, axes)
    got_q, got_k = rope_axes(q, k, pos, axes, inplace=True)
    assert got_q.data_ptr() == q.data_ptr() and torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    assert torch.equal(proj[..., 8 * 64:], before[..., 8 * 64:])
    close(want_q, before.unflatten(2, (12, 64))[:, :, :4], pos, axes, what="slice")
    odd = make((2 * 30 * 4 * 64 + 3,), torch.bfloat16)[3:].view(2, 30, 4, 64)
    close(rope_axes(odd, None, pos, axes)[0], odd, pos, axes, what="off 16 bytes")
    wide = make((2, 30, 1, 64), torch.float16).expand(2, 30, 4, 64)
    out, _ = rope_axes(wide, None, pos, axes)
    close(out, wide, pos, axes, what="expanded")
    with pytest.raises(ValueError, match="share memory"):
        rope_axes(wide, None, pos, axes, inplace=True)
    with pytest.raises(ValueError, match="share memory"):
        rope_axes(bhsd.transpose(1, 2), bhsd.transpose(1, 2), pos, axes, inplace=True)


def test_agrees_with_the_prologue_tables(device):
    """The complex fp64 table form of the prologue kernel on the same angles: both round one fp64/fp32 rotation to bf16."""
    from pasa_amd.prologue import apply_qk_rope_inplace_cossin_complex
    axes = RotaryAxes.video(128, device=device)
    pos = grid_positions(3, 4, 5, device=device)
    q = make((1, 60, 2, 128), torch.bfloat16)
    angle = (pos[axes.axis.long()].double() * axes.inv_freq[:, None]).t()
    t = q.transpose(1, 2).contiguous()
    ref, _ = apply_qk_rope_inplace_cossin_complex(t.clone(), t.clone(), angle.cos(), angle.sin())
    got, _ = rope_axes(q, None, pos, axes)
    d = (got.transpose(1, 2).float() - ref.float()).abs()
    step = 2.0 ** -7 * ref.float().abs() + 2.0 ** -18
    assert bool((d <= step).all()), "at most one bf16 step apart, where a value lies next to a border"
    assert float((d > 0).float().mean()) < 1e-3


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_gradient(device, pairing):
    axes = RotaryAxes.sections((8, 6, 6), pairing=pairing, device=device)
    pos = torch.randint(0, 999, (3, 17), dtype=torch.int32).to(device)
    q, k = make((2, 17, 4, 24), torch.float32).requires_grad_(), make((2, 17, 2, 24), torch.float32, 1).requires_grad_()
    oq, ok = rope_axes(q, k, pos, axes)
    gq, gk = torch.randn_like(oq), torch.randn_like(ok)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk), retain_graph=True)
    close(dq, gq, pos, axes, inverse=True, what="dq")
    close(dk, gk, pos, axes, inverse=True, what="dk")
    # Differences: the rotation is linear, so a step of any size gives the slope; fp32 rounds it by 2^-20.
    step = torch.randn_like(q)
    with torch.no_grad():
        diff = (rope_axes(q + step, None, pos, axes)[0].double() - rope_axes(q - step, None, pos, axes)[0].double()) / 2
    along = float((diff * gq.double()).sum())
    assert abs(along - float((dq.double() * step.double()).sum())) <= 2.0 ** -18 * float((diff.abs() * gq.double().abs()).sum() + (dq.double() * step.double()).abs().sum())
    # One gradient alone, a broadcast one, and only one leaf.
    (only_k,) = torch.autograd.grad(ok, k, gk, retain_graph=True)
    assert torch.equal(only_k, dk)
    (ones,) = torch.autograd.grad(oq.sum(), q)
    close(ones, torch.ones_like(q), pos, axes, inverse=True, what="sum")
    k2 = k.detach()
    oq, ok = rope_axes(q, k2, pos, axes)
    (again,) = torch.autograd.grad(oq, q, gq)
    assert torch.equal(again, dq)
    # An input that is expanded takes the sum over what it was expanded to.
    one = make((1, 17, 1, 24), torch.float32, 3).requires_grad_()
    out, _ = rope_axes(one.expand(2, 17, 4, 24), None, pos, axes)
    (d1,) = torch.autograd.grad(out, one, gq)
    assert torch.allclose(d1, dq.sum((0, 2), keepdim=True), rtol=0, atol=8 * 2.0 ** -24 * float(dq.abs().sum((0, 2)).max()))


def test_nothing_to_do_and_refusals_on_the_gpu(device):
    axes = RotaryAxes.video(64, device=device)
    q = torch.empty(0, 3, 64, device=device, dtype=torch.bfloat16)
    assert rope_axes(q, None, torch.empty(3, 0, device=device, dtype=torch.int32), axes)[0].shape == (0, 3, 64)
    q = make((4, 3, 64), torch.bfloat16)
    pos = torch.zeros(3, 4, device=device, dtype=torch.int32)
    with pytest.raises(ValueError, match="positions is on"):
        rope_axes(q, None, pos.cpu(), axes)
    with pytest.raises(ValueError, match="no gradient"):
        rope_axes(q.float().requires_grad_(), None, pos, axes, inplace=True)
    # An axis outside the positions reads the nearest one.
    wild = RotaryAxes(axes.inv_freq, torch.full_like(axes.axis, 99), "interleaved")
    last = RotaryAxes(axes.inv_freq, torch.full_like(axes.axis, 2), "interleaved")
    pos[2] = 5
    assert torch.equal(rope_axes(q, None, pos, wild)[0], rope_axes(q, None, pos, last)[0])


def test_streams_and_graph(device):
    axes = RotaryAxes.video(128, device=device)
    q, k = make((77, 6, 128), torch.bfloat16), make((77, 2, 128), torch.bfloat16, 1)
    pos = torch.randint(0, 5000, (3, 77), dtype=torch.int32).to(device)
    want = [t.clone() for t in rope_axes(q, k, pos, axes)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = rope_axes(q, k, pos, axes)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = rope_axes(q, k, pos, axes)
    for i in range(3):
        pos.copy_(torch.randint(0, 5000, (3, 77), dtype=torch.int32).to(device))
        q.mul_(1.01)
        eager = rope_axes(q, k, pos, axes)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(b[0], eager[0]) and torch.equal(b[1], eager[1]), i
