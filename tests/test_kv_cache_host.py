"""Refusals of the rotary embedding, the block tables and the cache in 8 bits, in Python and at the C entries: all of
them before any HIP call, so none needs a GPU."""
import ctypes

import pytest
import torch

from pasa_amd import _lib, kv_cache, rotary
from pasa_amd.kv_cache import KVCache8, append_kv, cached_attention, extend_block_tables
from pasa_amd.rotary import RotaryAxes, grid_positions, rope_axes

bf, f16, f32, i32, i64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64


# ---------------------------------------------------------------- Python --

def test_no_cpu_path():
    axes = RotaryAxes.video(64)
    with pytest.raises(ValueError, match="ROCm device"):
        rope_axes(torch.zeros(2, 1, 64, dtype=bf), None, torch.zeros(3, 2, dtype=i32), axes)
    c = KVCache8.empty(2, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="ROCm device"):
        append_kv(c, torch.zeros(2, 1, 64, dtype=bf), torch.zeros(2, 1, 64, dtype=bf), torch.zeros(2, dtype=i64))
    z = torch.zeros(1, dtype=i32)
    with pytest.raises(ValueError, match="ROCm device"):
        cached_attention(torch.zeros(1, 1, 64, dtype=bf), c, z[None], z)
    with pytest.raises(ValueError, match="ROCm device"):
        extend_block_tables(z[None].clone(), z, z, z, z, 64, 1)


def test_rotary_axes():
    a = RotaryAxes.video(128)
    assert a.inv_freq.shape == (64,) and a.axis.tolist() == [0] * 22 + [1] * 21 + [2] * 21
    assert float(a.inv_freq[0]) == 1 and abs(float(a.inv_freq[22 + 20]) - 10000 ** (-40 / 42)) < 1e-18
    s = RotaryAxes.sections((4, 0, 4), theta=100.0, pairing="halves", shared=True)
    assert s.axis.tolist() == [0, 0, 2, 2]
    assert torch.allclose(s.inv_freq, torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64), rtol=1e-15)
    for dims in ((3, 2), (), (0, 0), (-2, 4)):
        with pytest.raises(ValueError, match="dims"):
            RotaryAxes.sections(dims)
    g = grid_positions(2, 2, 3, first_frame=5)
    assert g[:, 0].tolist() == [5, 0, 0] and g[:, 7].tolist() == [6, 0, 1] and g[:, 11].tolist() == [6, 1, 2]


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(4, 64, dtype=bf)), "q must be"), (dict(q=torch.zeros(4, 2, 64, dtype=torch.float64)), "dtype"),
    (dict(q=torch.zeros(4, 2, 128, dtype=bf)[..., ::2]), "contiguous"), (dict(k=torch.zeros(5, 2, 64, dtype=bf)), "k must"),
    (dict(k=torch.zeros(4, 2, 32, dtype=bf)), "k must"), (dict(k=torch.zeros(4, 2, 64, dtype=f16)), "k must"),
    (dict(positions=torch.zeros(3, 5, dtype=i32)), "positions must"), (dict(positions=torch.zeros(4, dtype=i32)), "positions must"),
    (dict(positions=torch.zeros(3, 2, 4, dtype=i32)), "positions must"), (dict(positions=torch.zeros(3, 4, dtype=torch.int16)), "dtype"),
    (dict(axes=RotaryAxes(torch.zeros(4), torch.zeros(4, dtype=i32))), "RotaryAxes"),
    (dict(axes=RotaryAxes(torch.zeros(4, dtype=torch.float64), torch.zeros(3, dtype=i32))), "RotaryAxes"),
    (dict(axes=RotaryAxes(torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=i32), "thirds")), "pairing"),
    (dict(positions=torch.zeros(3, 4, requires_grad=True)), "positions")])
def test_rope_refusals(change, match):
    a = dict(q=torch.zeros(4, 2, 64, dtype=bf), k=torch.zeros(4, 1, 64, dtype=bf), positions=torch.zeros(3, 4, dtype=i32),
             axes=RotaryAxes.video(64))
    a.update(change)
    with pytest.raises(ValueError, match=match):
        rope_axes(a["q"], a["k"], a["positions"], a["axes"])


def test_shares_memory():
    t = torch.zeros(4, 6, 8)
    for ok in (t, t.transpose(0, 1), t[::2, 1:3], t[:, :1].squeeze(1), t.permute(2, 0, 1), t[:0]):
        assert not _lib.shares_memory(ok)
    for bad in (t[:, :1].expand(4, 6, 8), torch.zeros(20).as_strided((4, 8), (3, 1))):
        assert _lib.shares_memory(bad)


@pytest.mark.parametrize("change,match", [
    (dict(lens=torch.zeros(3, dtype=i32)), "lens and new_tokens"), (dict(new=torch.zeros(2, dtype=i64)), "int32"),
    (dict(num_free=torch.zeros(2, dtype=i32)), "num_free"), (dict(free=torch.zeros(2, 2, dtype=i32)), "free_pages"),
    (dict(page=48), "page_size"), (dict(page=256), "page_size"), (dict(tokens=-1), "negative"),
    (dict(tables=torch.zeros(2, 4, dtype=i64)), "block_tables"), (dict(tables=torch.zeros(2, 0, dtype=i32)), "block_tables"),
    (dict(tables=torch.zeros(4, 2, dtype=i32).t()), "block_tables"), (dict(tables=torch.zeros(1, 4, dtype=i32).expand(2, 4)), "block_tables"),
    (dict(tables=torch.zeros(4097, 1, dtype=i32), lens=torch.zeros(4097, dtype=i32), new=torch.zeros(4097, dtype=i32)), "4097 requests"),
    (dict(tables=torch.zeros(0, 1, dtype=i32), lens=torch.zeros(0, dtype=i32), new=torch.zeros(0, dtype=i32)), "0 requests")])
def test_table_refusals(change, match):
    a = dict(tables=torch.zeros(2, 4, dtype=i32), lens=torch.zeros(2, dtype=i32), new=torch.zeros(2, dtype=i32),
             free=torch.zeros(4, dtype=i32), num_free=torch.zeros(1, dtype=i32), page=64, tokens=3)
    a.update(change)
    with pytest.raises(ValueError, match=match):
        extend_block_tables(*a.values())


def test_cache_refusals():
    with pytest.raises(ValueError, match="page_size"):
        KVCache8.empty(2, 1, 64, 8, device="cpu")
    for d in (0, 129):
        with pytest.raises(ValueError, match="head_dim"):
            KVCache8.empty(2, 1, d, device="cpu")
    good = KVCache8.empty(3, 2, 80, 32, device="cpu")
    assert good.k.shape == (3, 2, 32, 128) and good.v.shape == (3, 2, 128, 32) and (good.num_pages, good.heads, good.page_size) == (3, 2, 32)
    k, v = good.values()
    assert k.shape == v.shape == (3, 2, 32, 80) and not k.any() and not v.any()
    x, s = torch.zeros(1, 2, 80, dtype=bf), torch.zeros(1, dtype=i64)
    for bad, match in ((KVCache8(good.k.float(), good.v, good.k_exp, good.v_exp, 80), "float8"),
                       (KVCache8(good.k, good.k, good.k_exp, good.v_exp, 80), "v must be"),
                       (KVCache8(good.k, good.v, good.k_exp.int(), good.v_exp, 80), "int8"),
                       (KVCache8(good.k, good.v, good.k_exp, good.v_exp[:2], 80), "int8"),
                       (KVCache8(good.k.transpose(2, 3).contiguous().transpose(2, 3), good.v, good.k_exp, good.v_exp, 80), "contiguous")):
        with pytest.raises(ValueError, match=match):
            append_kv(bad, x, x, s)


@pytest.mark.parametrize("change,match", [
    (dict(k=torch.zeros(2, 3, 64, dtype=bf)), "k must be"), (dict(v=torch.zeros(2, 2, 32, dtype=bf)), "v must be"),
    (dict(k=torch.zeros(2, 64, dtype=bf)), "k must be"), (dict(k=torch.zeros(2, 2, 64, dtype=torch.int32)), "dtype"),
    (dict(v=torch.zeros(2, 2, 64, dtype=f16)), "one dtype"), (dict(v=torch.zeros(3, 2, 64, dtype=bf)), "one dtype"),
    (dict(k=torch.zeros(2, 2, 128, dtype=bf)[..., ::2]), "contiguous"),
    (dict(v=torch.zeros(2, 2, 64, dtype=bf, requires_grad=True)), "no gradient"), (dict(slots=torch.zeros(2, dtype=i32)), "slots"),
    (dict(slots=torch.zeros(3, dtype=i64)), "slots must")])
def test_append_refusals(change, match):
    a = dict(k=torch.zeros(2, 2, 64, dtype=bf), v=torch.zeros(2, 2, 64, dtype=bf), slots=torch.zeros(2, dtype=i64))
    a.update(change)
    with pytest.raises(ValueError, match=match):
        append_kv(KVCache8.empty(3, 2, 64, device="cpu"), **a)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(4, 3, 64, dtype=bf)), "q must be"), (dict(q=torch.zeros(4, 2, 32, dtype=bf)), "q must be"),
    (dict(q=torch.zeros(4, 64, dtype=bf)), "q must be"), (dict(q=torch.zeros(4, 2, 64)), "dtype"),
    (dict(q=torch.zeros(4, 0, 64, dtype=bf)), "q must be"), (dict(q=torch.zeros(4, 2, 128, dtype=bf)[..., ::2]), "contiguous"),
    (dict(q=torch.zeros(4, 2, 64, dtype=bf, requires_grad=True)), "no gradient"),
    (dict(block_tables=torch.zeros(2, 4, dtype=i64)), "block_tables"), (dict(lens=torch.zeros(3, dtype=i32)), "lens must"),
    (dict(lens=torch.zeros(2, dtype=i64)), "lens must"), (dict(cu_q=torch.zeros(2, dtype=i32)), "cu_q must"),
    (dict(cu_q=torch.zeros(3, dtype=i64)), "cu_q must"), (dict(q=torch.zeros(5, 2, 64, dtype=bf), cu_q=None), "give cu_q"),
    (dict(window=0), "window"), (dict(max_kv_len=-1), "max_kv_len"), (dict(out=torch.zeros(4, 2, 64, dtype=f16)), "out must"),
    (dict(out=torch.zeros(4, 1, 64, dtype=bf).expand(4, 2, 64)), "share memory"),
    (dict(out=torch.zeros(4, 2, 128, dtype=bf)[..., ::2]), "out must")])
def test_attention_refusals(change, match):
    a = dict(q=torch.zeros(4, 2, 64, dtype=bf), block_tables=torch.zeros(2, 4, dtype=i32), lens=torch.zeros(2, dtype=i32),
             cu_q=torch.zeros(3, dtype=i32))
    a.update(change)
    q = a.pop("q")
    with pytest.raises(ValueError, match=match):
        cached_attention(q, KVCache8.empty(3, 2, 64, device="cpu"), a.pop("block_tables"), a.pop("lens"), a.pop("cu_q"), **a)


def test_out_may_not_be_q():
    c, z = KVCache8.empty(3, 2, 64, device="cpu"), torch.zeros(2, dtype=i32)
    big = torch.zeros(6, 2, 64, dtype=bf)
    with pytest.raises(ValueError, match="share memory"):
        cached_attention(big[:4], c, torch.zeros(2, 4, dtype=i32), z, out=big[1:5])


# ---------------------------------------------------------------- the C entries --

FAKE = 0x1000  # never dereferenced: every call below fails validation first


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def status(lib, rc, code, text):
    assert rc == code, (rc, lib.pasa_last_error())
    assert text.encode() in lib.pasa_last_error(), lib.pasa_last_error()


def rope_tensor(**kw):
    t = _lib.RopeTensor(kw.get("in_", FAKE), kw.get("out", FAKE))
    t.heads = kw.get("heads", 2)
    return ctypes.byref(t)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), -1, "q is NULL"), (dict(q=rope_tensor(in_=None)), -1, "q has a NULL"), (dict(k=rope_tensor(out=None)), -1, "k has a NULL"),
    (dict(q=rope_tensor(heads=0)), -2, "heads"), (dict(k=rope_tensor(heads=70000)), -6, "heads"), (dict(pos=None), -1, "NULL"),
    (dict(freq=None), -1, "NULL"), (dict(dtype=7), -7, "dtype"), (dict(pos_type=3), -7, "positions"), (dict(D=1), -3, "head_dim"),
    (dict(D=257), -3, "head_dim"), (dict(pairs=0), -2, "pairs"), (dict(pairs=33), -2, "pairs"), (dict(axes=0), -2, "axes"),
    (dict(pairing=2), -9, "pairing"), (dict(inverse=2), -9, "inverse"), (dict(B=-1), -2, "batch"), (dict(B=1 << 20, S=1 << 20), -6, "overflow")])
def test_c_rope(lib, change, code, text):
    a = dict(q=rope_tensor(), k=None, pos=FAKE, pos_type=0, pa=8, pb=0, ps=1, axes=3, freq=FAKE, axis=FAKE, pairs=32, B=1, S=8, D=64,
             pairing=0, inverse=0, dtype=0, stream=None)
    a.update(change)
    status(lib, lib.pasa_rope_axes(*a.values()), code, text)


def test_c_rope_nothing(lib):
    assert lib.pasa_rope_axes(rope_tensor(), None, None, 0, 0, 0, 0, 3, None, None, 32, 1, 0, 64, 0, 0, 0, None) == 0


@pytest.mark.parametrize("change,code,text", [
    (dict(tables=None), -1, "NULL"), (dict(slots=None), -1, "NULL"), (dict(free=None), -1, "NULL"), (dict(requests=0), -2, "requests"),
    (dict(requests=4097), -6, "4097 requests"), (dict(width=0), -2, "width"), (dict(stride=3), -2, "table_stride"), (dict(tokens=-1), -2, "tokens"),
    (dict(tokens=1 << 31), -6, "2^31"), (dict(page=24), -4, "page_size"), (dict(page=8), -4, "page_size"), (dict(lens_out=FAKE * 2), -9, "lens_out"),
    (dict(num_out=FAKE * 4), -9, "num_free_out")])
def test_c_tables(lib, change, code, text):
    a = dict(tables=FAKE, stride=4, width=4, lens=FAKE * 2, new=FAKE * 3, requests=2, free=FAKE, cap=5, num=FAKE * 4, page=64, tokens=3,
             cu=FAKE, slots=FAKE, pos=FAKE, lens_out=FAKE * 5, num_out=FAKE * 6, stream=None)
    a.update(change)
    status(lib, lib.pasa_block_tables(*a.values()), code, text)


def kv8(**kw):
    a = dict(k=FAKE, v=FAKE, k_exp=FAKE, v_exp=FAKE, num_pages=4, heads=2, page_size=64, dim=128, head_dim=128)
    a.update(kw)
    return ctypes.byref(_lib.Kv8(*a.values()))


CACHES = [(dict(k=None), -1, "NULL"), (dict(v_exp=None), -1, "NULL"), (dict(dim=96), -3, "dim 96"), (dict(head_dim=129), -3, "head_dim"),
          (dict(head_dim=0), -3, "head_dim"), (dict(page_size=256), -4, "page_size"), (dict(num_pages=0), -2, "pages"),
          (dict(heads=1 << 17), -6, "heads"), (dict(num_pages=1 << 31), -6, "pages"), (dict(v=FAKE + 8), -9, "16-byte")]


@pytest.mark.parametrize("cache,code,text", CACHES)
def test_c_cache(lib, cache, code, text):
    status(lib, lib.pasa_kv8_append(kv8(**cache), FAKE, FAKE, FAKE, 3, 256, 128, 256, 128, 0, None), code, text)
    status(lib, lib.pasa_kv8_attn(kv8(**cache), attn(), FAKE, 1 << 30, None), code, text)


@pytest.mark.parametrize("change,code,text", [(dict(k=None), -1, "NULL"), (dict(slots=None), -1, "NULL"), (dict(tokens=-1), -2, "tokens"),
                                              (dict(tokens=1 << 31), -6, "tokens"), (dict(dtype=3), -7, "dtype")])
def test_c_append(lib, change, code, text):
    a = dict(cache=kv8(), k=FAKE, v=FAKE, slots=FAKE, tokens=3, kt=256, kh=128, vt=256, vh=128, dtype=0, stream=None)
    a.update(change)
    status(lib, lib.pasa_kv8_append(*a.values()), code, text)


def attn(**kw):
    a = dict(q=FAKE, o=FAKE, lse=None, qt=256, qh=128, ot=256, oh=128, tables=FAKE, stride=4, width=4, lens=FAKE, cu=FAKE, tokens=8, requests=2,
             heads=2, max_kv=256, window=0, causal=1, zero=0, dtype=0, scale=0.1)
    a.update(kw)
    return ctypes.byref(_lib.Kv8Attn(*a.values()))


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), -1, "NULL"), (dict(lens=None), -1, "NULL"), (dict(tokens=-1), -2, "tokens"), (dict(requests=0), -2, "requests"),
    (dict(heads=3), -2, "q_heads"), (dict(max_kv=-1), -2, "max_kv"), (dict(tokens=1 << 31), -6, "tokens"), (dict(dtype=2), -7, "dtype"),
    (dict(scale=0.0), -9, "scale"), (dict(scale=float("nan")), -9, "scale"), (dict(scale=-1.0), -9, "scale"), (dict(scale=1e30), -9, "scale"),
    (dict(window=-1), -9, "window"), (dict(width=0), -2, "width"), (dict(stride=2), -2, "table_stride"), (dict(cu=None, tokens=7), -2, "same number")])
def test_c_attn(lib, change, code, text):
    status(lib, lib.pasa_kv8_attn(kv8(), attn(**change), FAKE, 1 << 30, None), code, text)


def test_c_attn_workspace(lib):
    need = lib.pasa_kv8_attn_workspace_bytes(2, 2, 2, 2, 128, 1 << 16)
    assert need > 0 and lib.pasa_kv8_attn_workspace_bytes(0, 2, 2, 2, 128, 1 << 16) == 0
    assert lib.pasa_kv8_attn_workspace_bytes(2, 2, 3, 2, 128, 1 << 16) == 0
    big = dict(tokens=2, max_kv=1 << 16, width=1 << 10, stride=1 << 10)
    status(lib, lib.pasa_kv8_attn(kv8(), attn(**big), None, 0, None), -8, "workspace")
    status(lib, lib.pasa_kv8_attn(kv8(), attn(**big), FAKE, need - 1, None), -8, "workspace")
    status(lib, lib.pasa_kv8_attn(kv8(), attn(**big), FAKE + 4, need, None), -9, "aligned")
    status(lib, lib.pasa_kv8_attn(kv8(), None, FAKE, 0, None), -1, "NULL")
