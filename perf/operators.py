"""The operators of a step with a key/value cache, as they are measured: their cases, their inputs, one pass through
each, and the same in elementary torch operations.

A step of chunk-wise video generation (or of text tokens served one at a time) extends the requests' block tables,
rotates the new tokens' q and k by their positions, appends k and v to the cache in 8 bits, and attends to the cache:

* ``tables``    block tables, slots and positions from the requests' lengths
* ``rotate``    rotary embedding from positions on several axes, forward or forward and gradient
* ``append``    k and v in 8 bits with a power-of-two scale for each page of tokens and head
* ``attention`` softmax attention to the cache

The cache: k codes [pages, heads, page, D], v codes [pages, heads, D, page], both e4m3, and int8 exponents
[pages, heads] for each: a value is its code times 2 ** exponent.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3 = torch.float8_e4m3fn
E_MIN, E_MAX, CODE_MAX = -50, 50, 448.0


# ---------------------------------------------------------------- cases --

def listed():
    return [
        # One step of 256 text requests: every one takes one slot, a few of them a new page.  The smallest launch.
        dict(name="tables, 256 single tokens", kind="tables", requests=256, kv=8192, new=1, page=64, ragged=True),
        # A batch of prompts and video chunks, ragged: many slots and pages at once.
        dict(name="tables, ragged prompts", kind="tables", requests=48, kv=32760, new=3600, page=64, ragged=True),
        # One new token of each of 64 requests, shared key heads, positions on three axes, pairs from the two halves.
        dict(name="rotate, 64 single tokens", kind="rotate", batch=1, seq=64, q_heads=40, kv_heads=8, head_dim=128,
             rotated=128, pairing="halves", dtype="bf16", grad=False),
        # Self-attention of a whole 720p video: 21 x 45 x 80 tokens of 40 heads.  Bound by memory.
        dict(name="rotate, 720p video", kind="rotate", batch=1, seq=75600, q_heads=40, kv_heads=40, head_dim=128,
             rotated=128, pairing="interleaved", dtype="bf16", grad=False),
        # A training step's forward and gradient at 480p, two clips, head dim 64 with 48 rotated channels.
        dict(name="rotate, 480p with gradient", kind="rotate", batch=2, seq=32760, q_heads=12, kv_heads=12, head_dim=64,
             rotated=48, pairing="interleaved", dtype="fp16", grad=True),
        # One new token of each of 64 requests, somewhere in its page.
        dict(name="append, 64 single tokens", kind="append", requests=64, new=1, kv_heads=8, head_dim=128, page=64,
             dtype="bf16", ragged=False, padding=0),
        # Three 720p frames (10,800 tokens) of 40 heads, pages of 128 tokens.
        dict(name="append, 3 frames at 720p", kind="append", requests=1, new=10800, kv_heads=40, head_dim=128, page=128,
             dtype="bf16", ragged=False, padding=0),
        # One query to one 480p frame: the smallest attention, all latency.
        dict(name="attention, 1 token to 1,560", kind="attention", requests=1, kv=1560, new=1, q_heads=12, kv_heads=12,
             head_dim=128, page=64, causal=True, window=0, dtype="bf16", ragged=False),
        # Text serving: 64 requests of up to 8,192 tokens, five query heads to a key head.
        dict(name="attention, 64 ragged tokens", kind="attention", requests=64, kv=8192, new=1, q_heads=40, kv_heads=8,
             head_dim=128, page=64, causal=True, window=0, dtype="bf16", ragged=True),
        # Single tokens behind a whole 720p video, 40 key heads: as many bytes as the cache has.
        dict(name="attention, 2 tokens to 75,600", kind="attention", requests=2, kv=75600, new=1, q_heads=40, kv_heads=40,
             head_dim=128, page=128, causal=True, window=0, dtype="bf16", ragged=False),
        # Ragged prompts with a causal window, head dim 64, small pages, fp16.
        dict(name="attention, ragged window", kind="attention", requests=12, kv=6000, new=1500, q_heads=32, kv_heads=8,
             head_dim=64, page=16, causal=True, window=2048, dtype="fp16", ragged=True),
        # One 720p frame's 3,600 queries to the 75,600 tokens of the video so far, 40 heads: the largest, bound by MFMA.
        dict(name="attention, frame to 720p video", kind="attention", requests=1, kv=75600, new=3600, q_heads=40,
             kv_heads=40, head_dim=128, page=64, causal=False, window=0, dtype="bf16", ragged=False),
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tables", "rotate", "append", "attention", "attention"])
    if kind == "tables":
        requests = _log(rng, 1, 1024)
        new = rng.choice([1, 1, _log(rng, 1, max(1, min(4096, 80000 // requests)))])
        return dict(kind=kind, requests=requests, kv=_log(rng, 1, 75600), new=new, page=rng.choice([16, 32, 64, 128]),
                    ragged=rng.random() < 0.7)
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 40])
    group = rng.choice([1, 1, 1, 2, 4, 5, 7, 8])
    q_heads = kv_heads * group if kv_heads * group <= 64 else kv_heads
    head_dim = rng.choice([64, 128, 128])
    if kind == "rotate":
        grad = rng.random() < 0.3
        seq = _log(rng, 1, max(1, min(75600, (75600 * 40 * 128 // (2 if grad else 1)) // (q_heads * head_dim))))
        return dict(kind=kind, batch=rng.choice([1, 2]) if seq <= 37800 else 1, seq=seq, q_heads=q_heads, kv_heads=kv_heads,
                    head_dim=head_dim, rotated=rng.choice([head_dim, head_dim, 48]),
                    pairing=rng.choice(["interleaved", "halves"]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), grad=grad)
    page = rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "append":
        requests = _log(rng, 1, 128)
        new = _log(rng, 1, max(1, 10800 // requests))
        return dict(kind=kind, requests=requests, new=new, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype,
                    ragged=rng.random() < 0.7, padding=rng.choice([0, 0, rng.randint(1, 9)]))
    if rng.random() < 0.5:  # single tokens (or the few of a speculated step)
        new = rng.choice([1, 1, 1, 2, 4])
        requests = _log(rng, 1, 128)
        kv = _log(rng, 16, max(16, min(75600, 2 * 75600 * 40 // (requests * kv_heads))))
    else:
        requests = _log(rng, 1, 16)
        new = _log(rng, 16, 4096)
        kv = _log(rng, new, max(new, min(75600, 3600 * 75600 * 40 // (4 * requests * new * q_heads))))
    return dict(kind=kind, requests=requests, kv=max(kv, new), new=new, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, causal=rng.random() < 0.7, window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]), dtype=dtype,
                ragged=rng.random() < 0.6)


def _lens(c):
    """The requests' cached and new tokens.  Attention: the new ones are in the cache already (kv >= new, but for
    a ragged batch of 8 and more, whose last request has nothing cached).  They go with the case, not the seed."""
    r = random.Random("%s %s %s" % (c["kind"], c["requests"], c.get("kv", 0)))
    n, new = c["requests"], [c["new"]] * c["requests"]
    if c["ragged"] and c["new"] > 1:
        new = [c["new"]] + [r.randint(1, c["new"]) for _ in range(n - 1)]
    if c["kind"] == "append":
        return [0] * n, new
    kv = [c["kv"]] * n
    if c["ragged"]:
        kv = [c["kv"]] + [max(m, r.randint(max(1, c["kv"] // 16), c["kv"])) for m in new[1:]]
        if n >= 8:
            kv[-1] = 0
    return kv, new


# ---------------------------------------------------------------- inputs --

def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _exponent(amax):
    """The smallest e with amax <= 448 * 2 ** e, in [E_MIN, E_MAX]."""
    f, e = torch.frexp(amax)  # amax = f * 2 ** e, f in [0.5, 1); 448 = 0.875 * 2 ** 9
    e = e - torch.where(f <= CODE_MAX / 512, 9, 8)
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX)


def _codes(x, e):
    """e4m3 of x * 2 ** -e; what is not finite becomes e4m3's NaN."""
    y = torch.ldexp(x, -e).clamp(-CODE_MAX, CODE_MAX)
    return torch.where(torch.isfinite(x), y, float("nan")).to(E4M3)


def _values(codes, e):
    return torch.ldexp(codes.float(), e)


def _tokens(g, shape, spread):
    """Normal values whose channels differ in size, a few of them by far, as keys and values do."""
    x = torch.randn(shape, device=DEV, generator=g)
    c = torch.exp(spread * torch.randn(shape[-1], device=DEV, generator=g))
    return x.mul_(c).add_(0.3 * torch.randn(shape[-1], device=DEV, generator=g))


def _cache(g, pages, heads, page, dim):
    out = {}
    for name, spread in (("k", 0.5), ("v", 0.2)):
        x = _tokens(g, (pages, heads, page, dim), spread)
        e = _exponent(x.abs().amax((2, 3)))
        codes = _codes(x, e[..., None, None])
        out[name] = codes if name == "k" else codes.view(torch.uint8).transpose(2, 3).contiguous().view(E4M3)
        out[name + "_exp"] = e.to(torch.int8)
    return out


def _frequencies(c):
    """Three axes (time, height, width).  Interleaved: each axis has frequencies of its own, as video transformers have
    them; halves: one sequence of frequencies, whose runs go to the axes, as language models have them."""
    n = c["rotated"] // 2
    h = n // 3
    dims = [n - 2 * h, h, h]
    axis = [a for a, d in enumerate(dims) for _ in range(d)]
    if c["pairing"] == "halves":
        freq = [10000.0 ** (-i / n) for i in range(n)]
    else:
        freq = [10000.0 ** (-i / d) for d in dims for i in range(d)]
    return torch.tensor(freq, dtype=torch.float64, device=DEV), _i32(axis)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "rotate":
        dt = DTYPES[c["dtype"]]
        for name, heads in (("q", c["q_heads"]), ("k", c["kv_heads"])):
            s[name] = torch.randn(c["batch"], c["seq"], heads, c["head_dim"], device=DEV, generator=g).to(dt)
            if c["grad"]:
                s["d" + name] = torch.randn(s[name].shape, device=DEV, generator=g).to(dt)
                s[name].requires_grad_(True)
        t = torch.arange(c["seq"], device=DEV)
        first = torch.randint(0, 4096, (1,), device=DEV, generator=g)  # text before the video, or earlier chunks of it
        s["positions"] = torch.stack([first + t // 3600, t // 80 % 45, t % 80]).to(torch.int32)
        if c["pairing"] == "halves":
            s["positions"] += torch.randint(0, 100000, (1, c["seq"]), device=DEV, generator=g, dtype=torch.int32)
        s["inv_freq"], s["axis"] = _frequencies(c)
        return s

    kv, new = _lens(c)
    page = c["page"]
    s["cu_q"] = _i32([0] + torch.tensor(new).cumsum(0).tolist())
    if c["kind"] == "tables":
        width = -(-(max(kv) + max(new)) // page) + 2
        old = [-(-n // page) for n in kv]
        need = sum(-(-(n + m) // page) for n, m in zip(kv, new)) - sum(old)
        ids = torch.randperm(sum(old) + need + 8, device=DEV, generator=g).to(torch.int32)
        lp = torch.arange(width, device=DEV)[None]
        lens, had = _i32(kv), _i32(old)
        start = (had.cumsum(0) - had)[:, None]
        s["tables"] = torch.where(lp < had[:, None], ids[(start + lp).clamp(max=ids.numel() - 1)], -1).to(torch.int32)
        s.update(lens=lens, new=_i32(new), tokens=sum(new) + 5, page=page, free=ids[sum(old):].contiguous(),
                 num_free=_i32([need + 8]))
        return s

    dt = DTYPES[c["dtype"]]
    if c["kind"] == "append":
        r = random.Random("at %s" % c["requests"])
        at = [r.randrange(page) for _ in new]  # where in its page a request goes on
        pages = [-(-(a + n) // page) for a, n in zip(at, new)]
        ids = torch.randperm(sum(pages) + 4, device=DEV, generator=g)
        slots, done = [], 0
        for a, n, p in zip(at, new, pages):
            i = a + torch.arange(n, device=DEV)
            slots.append(ids[done + i // page] * page + i % page)
            done += p
        s["slots"] = torch.cat(slots + [torch.full((c["padding"],), -1, device=DEV)])
        s["runs"] = sum(pages)
        total = sum(new) + c["padding"]
        s["k"] = _tokens(g, (total, c["kv_heads"], c["head_dim"]), 0.5).to(dt)
        s["v"] = _tokens(g, (total, c["kv_heads"], c["head_dim"]), 0.2).to(dt)
        s["cache"] = _cache(g, sum(pages) + 4, c["kv_heads"], page, c["head_dim"])
        return s

    pages = [-(-n // page) for n in kv]
    width = max(1, max(pages))
    ids = torch.randperm(sum(pages) + 4, device=DEV, generator=g).to(torch.int32)
    had = _i32(pages)
    lp = torch.arange(width, device=DEV)[None]
    s["tables"] = torch.where(lp < had[:, None], ids[((had.cumsum(0) - had)[:, None] + lp).clamp(max=ids.numel() - 1)], -1).to(torch.int32)
    s["lens"], s["most_new"] = _i32(kv), max(new)
    s["q"] = (1.5 * torch.randn(sum(new), c["q_heads"], c["head_dim"], device=DEV, generator=g)).to(dt)
    s["cache"] = _cache(g, sum(pages) + 4, c["kv_heads"], page, c["head_dim"])
    return s


# ---------------------------------------------------------------- one pass --

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


def _own_tables(s):
    from pasa_amd import kv_cache
    step = kv_cache.extend_block_tables(s["tables"], s["lens"], s["new"], s["free"], s["num_free"], s["page"], s["tokens"])
    return {"tables": s["tables"], "cu_q": step.cu_q, "slots": step.slots, "positions": step.positions, "lens": step.lens,
            "num_free": step.num_free}


def _own_rotate(s):
    from pasa_amd import rotary
    axes = rotary.RotaryAxes(s["inv_freq"], s["axis"], s["case"]["pairing"])
    q, k = rotary.rope_axes(s["q"], s["k"], s["positions"], axes)
    if not s["case"]["grad"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _own_append(s):
    from pasa_amd import kv_cache
    c = s["cache"]
    kv_cache.append_kv(kv_cache.KVCache8(c["k"], c["v"], c["k_exp"], c["v_exp"], s["case"]["head_dim"]), s["k"], s["v"], s["slots"])
    return c


def _own_attention(s):
    from pasa_amd import kv_cache
    c, d = s["cache"], s["case"]
    return kv_cache.cached_attention(s["q"], kv_cache.KVCache8(c["k"], c["v"], c["k_exp"], c["v_exp"], d["head_dim"]),
                                     s["tables"], s["lens"], s["cu_q"], causal=d["causal"], window=d["window"] or None)


_OWN = {"tables": _own_tables, "rotate": _own_rotate, "append": _own_append, "attention": _own_attention}


def _plain_tables(s):
    table, page = s["tables"], s["page"]
    width = table.shape[1]
    lens, total = s["lens"].long(), s["tokens"]
    ends = s["new"].long().cumsum(0).clamp(max=total)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends])
    new = cu[1:] - cu[:-1]
    had = (lens + page - 1) // page
    need = ((lens + new + page - 1) // page).clamp(max=width) - had
    before = need.cumsum(0) - need
    got = torch.minimum((s["num_free"] - before).clamp(min=0), need)
    after = torch.minimum(lens + new, (had + got) * page)
    lp = torch.arange(width, device=DEV)[None]
    taken = (lp >= had[:, None]) & (lp < (had + got)[:, None])
    at = (s["num_free"] - 1 - (before[:, None] + lp - had[:, None])).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(taken, s["free"][at], table))
    t = torch.arange(total, device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True)
    real = r < lens.numel()
    r = r.clamp(max=lens.numel() - 1)
    pos = lens[r] + t - cu[r]
    page_id = table[r, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(real & (pos < after[r]) & (page_id >= 0), page_id * page + pos % page, -1)
    return {"tables": table, "cu_q": cu.int(), "slots": slots, "positions": torch.where(real, pos, -1).int(), "lens": after.int(),
            "num_free": (s["num_free"] - got.sum()).int()}


def _rotated(x, cos, sin, pairing):
    """x [B, S, H, D] in 32 bits; cos and sin [S, 1, pairs].  Channels behind the pairs stay."""
    n = cos.shape[-1]
    y, rest = x.float()[..., :2 * n], x.float()[..., 2 * n:]
    a, b = (y[..., :n], y[..., n:]) if pairing == "halves" else (y[..., 0::2], y[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    y = torch.cat([u, v], -1) if pairing == "halves" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([y, rest], -1).to(x.dtype)


def _plain_rotate(s):
    with torch.no_grad():
        angle = (s["positions"][s["axis"].long()].double() * s["inv_freq"][:, None]).t()[:, None]
        cos, sin = angle.cos().float(), angle.sin().float()
        pairing = s["case"]["pairing"]
        out = {"q": _rotated(s["q"], cos, sin, pairing), "k": _rotated(s["k"], cos, sin, pairing)}
        if s["case"]["grad"]:
            out.update(dq=_rotated(s["dq"], cos, -sin, pairing), dk=_rotated(s["dk"], cos, -sin, pairing))
    return out


def _plain_append(s):
    c, page, runs = s["cache"], s["case"]["page"], s["runs"]
    total = s["slots"].numel() - s["case"]["padding"]
    at, off = s["slots"][:total] // page, s["slots"][:total] % page
    # The tokens of one page follow each other: its number among the pages written.
    new = torch.cat([torch.ones_like(at[:1]), (at[1:] != at[:-1]).long()])
    n = new.cumsum(0) - 1
    ids = torch.zeros(runs, dtype=torch.long, device=DEV).scatter_(0, n, at)
    fresh = torch.zeros(runs, dtype=torch.bool, device=DEV).index_put_((n,), off == 0, accumulate=True)[:, None]
    for_k = _append_one(c["k"], c["k_exp"], s["k"][:total].float(), ids, n, off, fresh)
    for_v = _append_one(c["v"].view(torch.uint8).transpose(2, 3).view(E4M3), c["v_exp"], s["v"][:total].float(), ids, n, off, fresh)
    c["k"].view(torch.uint8).index_copy_(0, ids, for_k[0].view(torch.uint8))
    c["v"].view(torch.uint8).index_copy_(0, ids, for_v[0].view(torch.uint8).transpose(2, 3).contiguous())
    c["k_exp"].index_copy_(0, ids, for_k[1])
    c["v_exp"].index_copy_(0, ids, for_v[1])
    return c


def _append_one(codes, exps, x, ids, n, off, fresh):
    most = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    most = torch.zeros(ids.numel(), x.shape[1], device=DEV).index_reduce_(0, n, most, "amax")
    had = torch.where(fresh, E_MIN, exps[ids].int())
    e = torch.maximum(_exponent(most).int(), had)
    old = codes.view(torch.uint8)[ids].view(E4M3)
    moved = torch.ldexp(old.float(), torch.where(fresh, 0, had - e)[..., None, None]).to(E4M3)
    moved = moved.view(torch.uint8)
    moved[n, :, off] = _codes(x, e[n][..., None]).view(torch.uint8)
    return moved.view(E4M3), e.to(torch.int8)


def _plain_attention(s):
    c, d = s["cache"], s["case"]
    page, heads, dim, most = d["page"], d["kv_heads"], d["head_dim"], s["most_new"]
    group, table = d["q_heads"] // heads, s["tables"].clamp(min=0).long()
    n, width = table.shape
    k = _values(c["k"].view(torch.uint8)[table].view(E4M3), c["k_exp"][table].int()[..., None, None])
    k = k.transpose(1, 2).reshape(n, heads, width * page, dim)
    v = _values(c["v"].view(torch.uint8)[table].view(E4M3), c["v_exp"][table].int()[..., None, None])
    v = v.permute(0, 2, 1, 4, 3).reshape(n, heads, width * page, dim)
    cu = s["cu_q"].long()
    lens, new = s["lens"].long(), cu[1:] - cu[:-1]
    i = torch.arange(most, device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float() * dim ** -0.5
    q = q.reshape(n, most, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, group * most, dim)
    score = q @ k.transpose(2, 3)
    j, pos = torch.arange(width * page, device=DEV), (lens - new)[:, None] + i
    seen = (j < lens[:, None])[:, None].expand(n, most, -1)
    if d["causal"]:
        seen = seen & (j <= pos[..., None])
    if d["window"]:
        seen = seen & (j > pos[..., None] - d["window"])
    score.view(n, heads, group, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total > 0, total, 1.0)
    o = o.view(n, heads, group, most, dim).permute(0, 3, 1, 2, 4)
    t = torch.arange(s["q"].shape[0], device=DEV)
    r = torch.searchsorted(cu[1:], t, right=True)
    return o[r, t - cu[r]].reshape(t.numel(), heads * group, dim).to(s["q"].dtype)


_PLAIN = {"tables": _plain_tables, "rotate": _plain_rotate, "append": _plain_append, "attention": _plain_attention}


# ---------------------------------------------------------------- what a pass cannot do without --

def work(case):
    c = case
    if c["kind"] == "rotate":
        tokens = c["batch"] * c["seq"]
        n = tokens * (c["q_heads"] + c["kv_heads"]) * c["head_dim"] * (2 if c["grad"] else 1)
        return {"bytes": 2 * n * BYTES[c["dtype"]] + 12 * c["seq"], "flops": 3 * n}
    kv, new = _lens(c)
    total = sum(new)
    if c["kind"] == "tables":
        # Lengths in and out, one table entry for each request, slots and positions.
        return {"bytes": 20 * c["requests"] + 12 * (total + 5) + 8 * (total // c["page"]), "flops": 0}
    if c["kind"] == "append":
        n = 2 * total * c["kv_heads"] * c["head_dim"]
        return {"bytes": n * (BYTES[c["dtype"]] + 1) + 8 * total, "flops": 3 * n}
    pairs, keys = 0, 0
    for length, m in zip(kv, new):
        lo = length
        for i in range(m):
            p = length - m + i
            hi = min(length, p + 1) if c["causal"] else length
            first = max(0, p + 1 - c["window"]) if c["window"] else 0
            pairs += max(0, hi - first)
            lo = min(lo, first)
        keys += max(0, length - lo)
    return {"bytes": 2 * keys * c["kv_heads"] * c["head_dim"] + 2 * total * c["q_heads"] * c["head_dim"] * BYTES[c["dtype"]],
            "flops": 4 * pairs * c["q_heads"] * c["head_dim"]}


# ---------------------------------------------------------------- the definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "rotate":
            return _exact_rotate(s)
        if kind == "append":
            return _exact_append(s)
        if kind == "attention":
            return _exact_attention(s)
    return None  # tables: whole numbers


def _exact_rotate(s):
    n = s["inv_freq"].numel()
    where = s["positions"].double()[s["axis"].long()].t() * s["inv_freq"]
    turn = torch.polar(torch.ones_like(where), where)[None, :, None]
    halves = s["case"]["pairing"] == "halves"

    def one(x, w):
        y = x.double().clone()
        first, second = (slice(0, n), slice(n, 2 * n)) if halves else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * w
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"q": one(s["q"], turn), "k": one(s["k"], turn)}
    if s["case"]["grad"]:
        out.update(dq=one(s["dq"], turn.conj()), dk=one(s["dk"], turn.conj()))
    return out


def _exact_append(s):
    """The codes' values before they are rounded; the exponents have no such value."""
    c, page = s["cache"], s["case"]["page"]
    slots = s["slots"][s["slots"] >= 0]
    out = {"k_exp": None, "v_exp": None}
    for name in ("k", "v"):
        x = s[name][:slots.numel()].double()
        old = c[name].to(torch.float32).double()
        old = old if name == "k" else old.transpose(2, 3)
        held = old.clone()
        ids, n = torch.unique_consecutive(slots // page, return_inverse=True)
        had = c[name + "_exp"][ids].double()
        fresh = torch.zeros(ids.numel(), device=DEV).index_add_(0, n, (slots % page == 0).double().float()) > 0
        most = torch.zeros(ids.numel(), x.shape[1], device=DEV, dtype=torch.float64)
        for i in range(ids.numel()):
            mine = n == i
            most[i] = x[mine].abs().amax((0, 2))
        e = torch.ceil(torch.log2(most / CODE_MAX)).clamp(E_MIN, E_MAX)
        e = torch.where(fresh[:, None], e, torch.maximum(e, had))
        held[ids] = held[ids] * torch.where(fresh[:, None], 1.0, torch.exp2(had - e))[..., None, None]
        held[slots // page, :, slots % page] = x * torch.exp2(-e[n])[..., None]
        out[name] = held if name == "k" else held.transpose(2, 3).contiguous()
    return out


def _exact_attention(s):
    c, d = s["cache"], s["case"]
    heads, dim, page = d["kv_heads"], d["head_dim"], d["page"]
    group = d["q_heads"] // heads
    cu, lens = s["cu_q"].tolist(), s["lens"].tolist()
    out = torch.zeros(cu[-1], d["q_heads"], dim, dtype=torch.float64, device=DEV)
    for r, length in enumerate(lens):
        first, m = cu[r], cu[r + 1] - cu[r]
        if not length:
            continue
        ids = s["tables"][r, :-(-length // page)].long()
        j = torch.arange(length, device=DEV)
        pos = torch.arange(length - m, length, device=DEV)[:, None]
        hidden = (j > pos) if d["causal"] else torch.zeros(m, length, dtype=torch.bool, device=DEV)
        if d["window"]:
            hidden = hidden | (j <= pos - d["window"])
        for h in range(heads):
            k = c["k"][:, h].view(torch.uint8)[ids].view(E4M3).to(torch.float64) * 2.0 ** c["k_exp"][ids, h].double()[:, None, None]
            v = c["v"][:, h].view(torch.uint8)[ids].view(E4M3).to(torch.float64) * 2.0 ** c["v_exp"][ids, h].double()[:, None, None]
            k, v = k.reshape(-1, dim)[:length], v.transpose(1, 2).reshape(-1, dim)[:length]
            for i in range(h * group, (h + 1) * group):
                a = (s["q"][first:first + m, i].double() @ k.t()) / math.sqrt(dim)
                p = torch.softmax(a.masked_fill_(hidden, -math.inf), -1)
                out[first:first + m, i] = torch.nan_to_num(p @ v)
    return out
