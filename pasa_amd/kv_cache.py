"""A paged key/value cache in 8 bits, and the attention that reads it, on MI355X.

One step of chunk-wise video generation, or of text tokens served one at a time:

    step = extend_block_tables(tables, lens, new_tokens, free_pages, num_free, cache.page_size, tokens)
    q, k = rope_axes(q, k, positions, axes)              # pasa_amd.rotary
    append_kv(cache, k, v, step.slots)
    o = cached_attention(q, cache, tables, step.lens, step.cu_q, causal=True)

Everything stays on the GPU: nothing here synchronises or reads a length back, so a step can be captured in a graph.
Keys and values are e4m3 codes with one power-of-two scale for each page of tokens and head (``KVCache8``), half the
bytes of bf16 and half the time of an attention that is bound by them.  There is no CPU path, and no gradient.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
PAGE_SIZES = (16, 32, 64, 128)
EXP_MIN, EXP_MAX = -50, 50
MAX_TABLE_REQUESTS = 4096
MAX_KEYS = 0x7fffff00  # of a request


@dataclass
class KVCache8:
    """k: float8_e4m3fn [pages, heads, page_size, dim]; v: float8_e4m3fn [pages, heads, dim, page_size]; k_exp, v_exp:
    int8 [pages, heads].  A value is its code times 2 ** exponent.  dim is 64 or 128; channels from head_dim on are 0."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor
    head_dim: int

    @classmethod
    def empty(cls, num_pages: int, heads: int, head_dim: int, page_size: int = 64, device="cuda") -> "KVCache8":
        """A cache of zeros.  head_dim 1 .. 128 (kept as 64 or 128 channels); page_size 16, 32, 64 or 128."""
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size} not in {PAGE_SIZES}")
        if not 1 <= head_dim <= 128:
            raise ValueError(f"head_dim {head_dim} not in [1, 128]")
        dim = 64 if head_dim <= 64 else 128
        codes = lambda *s: torch.zeros(s, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        exps = lambda: torch.full((num_pages, heads), EXP_MIN, dtype=torch.int8, device=device)
        return cls(codes(num_pages, heads, page_size, dim), codes(num_pages, heads, dim, page_size), exps(), exps(), head_dim)

    @property
    def num_pages(self) -> int:
        return self.k.shape[0]

    @property
    def heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def values(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """fp32 keys and values [pages, heads, page_size, head_dim] that the codes stand for."""
        k = torch.ldexp(self.k.float(), self.k_exp.int()[..., None, None])
        v = torch.ldexp(self.v.float(), self.v_exp.int()[..., None, None]).transpose(2, 3)
        return k[..., :self.head_dim], v[..., :self.head_dim]

    def _struct(self) -> "_lib.Kv8":
        k, v = self.k, self.v
        if k.dim() != 4 or k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
            raise ValueError("a cache's k and v are 4-d float8_e4m3fn tensors")
        pages, heads, page, dim = k.shape
        if v.shape != (pages, heads, dim, page):
            raise ValueError(f"v must be {[pages, heads, dim, page]} for k {list(k.shape)}, got {list(v.shape)}")
        for t in (self.k_exp, self.v_exp):
            if t.dtype != torch.int8 or t.shape != (pages, heads):
                raise ValueError(f"k_exp and v_exp must be int8 {[pages, heads]}, got {t.dtype} {list(t.shape)}")
        for t in (k, v, self.k_exp, self.v_exp):
            if not t.is_contiguous() or t.device != k.device:
                raise ValueError("a cache's tensors must be contiguous and on one device")
        return _lib.Kv8(k.data_ptr(), v.data_ptr(), self.k_exp.data_ptr(), self.v_exp.data_ptr(), pages, heads, page, dim,
                        int(self.head_dim))


def _call(device: torch.device, fn: str, *args) -> None:
    """The library's call with ``device`` current, on its current stream."""
    if device.type != "cuda":
        raise ValueError("the cache kernels need ROCm device tensors (there is no CPU path)")
    _lib.on_stream(device, fn, *args)


def _check_ints(device, dtype=torch.int32, **ts) -> None:
    for name, t in ts.items():
        if t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} tensor, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


def _meets(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory that ``a`` spans meets ``b``'s."""
    ends = lambda t: (t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))))
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = ends(a), ends(b)
    return a0 < b1 and b0 < a1


def _check_tables(tables: torch.Tensor) -> None:
    if tables.dim() != 2 or tables.dtype != torch.int32 or tables.shape[1] < 1 or tables.stride(1) != 1 or \
            (tables.shape[0] > 1 and tables.stride(0) < tables.shape[1]):
        raise ValueError(f"block_tables must be int32 [requests, width] with rows apart, got {tables.dtype} {tuple(tables.shape)}")


# ---------------------------------------------------------------- block tables --

@dataclass
class BlockTableStep:
    """What a step needs of the requests' lengths: cu_q int32 [requests + 1], slots int64 [tokens], positions int32
    [tokens], lens int32 [requests] and num_free int32 [1] after the step."""
    cu_q: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    lens: torch.Tensor
    num_free: torch.Tensor


def extend_block_tables(block_tables: torch.Tensor, lens: torch.Tensor, new_tokens: torch.Tensor,
                        free_pages: torch.Tensor, num_free: torch.Tensor, page_size: int, tokens: int) -> BlockTableStep:
    """Pages, slots and positions for ``new_tokens`` [requests] more tokens behind ``lens`` [requests] cached ones.

    Requests take pages in order from the end of free_pages[:num_free] and ``block_tables`` [requests, width] gets
    them in place, behind the ceil(lens / page_size) that it holds.  ``tokens``: the step's size on the host; new
    tokens beyond it are not taken, and slots and positions behind the last one are -1.  A token that no page is left
    for, or that the table is too narrow for, has slot -1 and ``lens`` of the result leaves it out.  All int32; at
    most 4,096 requests.  The inputs but for the tables stay as they are."""
    _check_tables(block_tables)
    R = block_tables.shape[0]
    dev = block_tables.device
    _check_ints(dev, lens=lens, new_tokens=new_tokens, free_pages=free_pages, num_free=num_free)
    if lens.shape != (R,) or new_tokens.shape != (R,) or num_free.numel() != 1 or free_pages.dim() != 1:
        raise ValueError(f"lens and new_tokens must be [{R}], num_free one number, free_pages a list, got "
                         f"{tuple(lens.shape)}, {tuple(new_tokens.shape)}, {tuple(num_free.shape)}, {tuple(free_pages.shape)}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} not in {PAGE_SIZES}")
    if not 1 <= R <= MAX_TABLE_REQUESTS:
        raise ValueError(f"{R} requests: 1 to {MAX_TABLE_REQUESTS} are taken")
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens {tokens} is negative")
    cu_q, after, left, positions = lens.new_empty(2 * R + 2 + tokens).split((R + 1, R, 1, tokens))
    slots = lens.new_empty(tokens, dtype=torch.int64)
    _call(dev, "pasa_block_tables", block_tables.data_ptr(), max(block_tables.stride(0), block_tables.shape[1]),
          block_tables.shape[1], lens.data_ptr(), new_tokens.data_ptr(), R, free_pages.data_ptr(), free_pages.numel(),
          num_free.data_ptr(), page_size, tokens, cu_q.data_ptr(), slots.data_ptr(), positions.data_ptr(),
          after.data_ptr(), left.data_ptr())
    return BlockTableStep(cu_q, slots, positions, after, left)


# ---------------------------------------------------------------- append --

def append_kv(cache: KVCache8, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Write k and v [tokens, heads, head_dim] (bf16, fp16 or fp32) into the cache at ``slots`` (int64 [tokens]:
    page * page_size + offset; negative ones are skipped), in place.

    Tokens in a row with consecutive slots of one page share the page's scale: the smallest power of two that holds
    their largest magnitude and, unless they begin the page (offset 0), what the page holds already, whose codes are
    scaled along.  Values are rounded to the nearest code; what is not finite is kept as NaN.  A page is written by
    one such run in a call: its contents are unspecified if there are two."""
    st = cache._struct()
    dev = cache.k.device
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape[1] != cache.heads or t.shape[2] != cache.head_dim:
            raise ValueError(f"{name} must be [tokens, {cache.heads}, {cache.head_dim}], got {tuple(t.shape)}")
        if t.dtype not in _DTYPES:
            raise ValueError(f"{name}: dtype {t.dtype} is not bfloat16, float16 or float32")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the cache on {dev}")
        if t.shape[2] > 1 and t.numel() and t.stride(2) != 1:
            raise ValueError(f"{name}: the channels must be contiguous, got stride {t.stride(2)}")
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
        raise ValueError("append_kv has no gradient: call it under torch.no_grad()")
    if v.dtype != k.dtype or v.shape != k.shape:
        raise ValueError(f"k and v must have one dtype and shape, got {k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)}")
    _check_ints(dev, torch.int64, slots=slots)
    if slots.shape != (k.shape[0],):
        raise ValueError(f"slots must be [{k.shape[0]}], got {tuple(slots.shape)}")
    _call(dev, "pasa_kv8_append", ctypes.byref(st), k.data_ptr(), v.data_ptr(), slots.data_ptr(), k.shape[0], k.stride(0),
          k.stride(1), v.stride(0), v.stride(1), _DTYPES[k.dtype])


# ---------------------------------------------------------------- attention --

def cached_attention(q: torch.Tensor, cache: KVCache8, block_tables: torch.Tensor, lens: torch.Tensor,
                     cu_q: Optional[torch.Tensor] = None, *, scale: Optional[float] = None, causal: bool = False,
                     window: Optional[int] = None, max_kv_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Softmax attention of q [tokens, q_heads, head_dim] (bf16 or fp16) to the cache.

    block_tables: int32 [requests, width]; lens: int32 [requests], cached tokens with the new ones; cu_q: int32
    [requests + 1], ascending, first row of each request's new tokens, or None if each has tokens / requests of them.  New token i
    of n is at position lens - n + i.  It sees every cached key, or with ``causal`` those up to its own, or with
    ``window`` the last ``window`` up to its own (and, without ``causal``, those behind it).  A table entry of -1 hides
    its page, as where early frames were given back.  Rows that see no key are 0.  q_heads is a multiple of the
    cache's heads, query heads h * group .. share key head h.

    ``scale``: of the scores, default head_dim ** -0.5.  ``max_kv_len``: a bound of lens known on the host (default:
    the table's width); the work is split by it, and keys from there on are not read.  ``out``: where the result
    goes; rows of no request (in front of the first, behind the last) stay as they were there, and are 0 in a new tensor.  ``return_lse``: also the
    natural logarithm of each row's sum of exponentials, fp32 [tokens, q_heads] (-inf where a row sees nothing)."""
    st = cache._struct()
    dev = cache.k.device
    if q.dim() != 3 or q.shape[2] != cache.head_dim or q.shape[1] < 1 or q.shape[1] % cache.heads:
        raise ValueError(f"q must be [tokens, a multiple of {cache.heads}, {cache.head_dim}], got {tuple(q.shape)}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"q: dtype {q.dtype} is not bfloat16 or float16")
    if q.device != dev:
        raise ValueError(f"q is on {q.device}, the cache on {dev}")
    if q.requires_grad and torch.is_grad_enabled():
        raise ValueError("cached_attention has no gradient: call it under torch.no_grad()")
    T, H, D = q.shape
    if D > 1 and q.numel() and q.stride(2) != 1:
        raise ValueError(f"q: the channels must be contiguous, got stride {q.stride(2)}")
    _check_tables(block_tables)
    if block_tables.device != dev:
        raise ValueError(f"block_tables is on {block_tables.device}, not on {dev}")
    R, width = block_tables.shape
    _check_ints(dev, lens=lens)
    if R < 1 or lens.shape != (R,):
        raise ValueError(f"lens must be [{R}] for block_tables {tuple(block_tables.shape)}, got {tuple(lens.shape)}")
    if cu_q is not None:
        _check_ints(dev, cu_q=cu_q)
        if cu_q.shape != (R + 1,):
            raise ValueError(f"cu_q must be [{R + 1}], got {tuple(cu_q.shape)}")
    elif T % R:
        raise ValueError(f"{T} tokens are not the same number for each of {R} requests: give cu_q")
    if window is not None and window < 1:
        raise ValueError(f"window {window} must be at least 1")
    if max_kv_len is not None and max_kv_len < 0:
        raise ValueError(f"max_kv_len {max_kv_len} is negative")
    max_kv = width * cache.page_size if max_kv_len is None else min(width * cache.page_size, int(max_kv_len))
    if max_kv > MAX_KEYS:
        raise ValueError(f"a request of {max_kv} keys: at most {MAX_KEYS} are taken (max_kv_len bounds them)")
    if out is None:
        o = q.new_empty((T, H, D))
    else:
        o = out
        if o.shape != q.shape or o.dtype != q.dtype or o.device != dev or (o.numel() and D > 1 and o.stride(2) != 1):
            raise ValueError(f"out must be {q.dtype} {tuple(q.shape)} on {dev} with contiguous channels, got {o.dtype} {tuple(o.shape)} on {o.device}")
        if o.requires_grad and torch.is_grad_enabled():
            raise ValueError("cached_attention has no gradient: out must not require one")
        if _lib.shares_memory(o) or _meets(o, q):
            raise ValueError("out: its rows and heads must not share memory with each other or with q")
    lse = q.new_empty((T, H), dtype=torch.float32) if return_lse else None
    need = _lib.load().pasa_kv8_attn_workspace_bytes(T, R, H, cache.heads, cache.k.shape[3], max_kv)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    args = _lib.Kv8Attn(q.data_ptr(), o.data_ptr(), None if lse is None else lse.data_ptr(), q.stride(0), q.stride(1),
                        o.stride(0), o.stride(1), block_tables.data_ptr(), max(block_tables.stride(0), width), width,
                        lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), T, R, H, max_kv,
                        0 if window is None else int(window), int(bool(causal)), int(out is None), _DTYPES[q.dtype],
                        D ** -0.5 if scale is None else float(scale))
    _call(dev, "pasa_kv8_attn", ctypes.byref(st), ctypes.byref(args), None if ws is None else ws.data_ptr(), need)
    return o if lse is None else (o, lse)
