"""CPU restatements in 64 bits of the key/value cache in 8 bits, its attention, its block tables and the rotary
embedding from positions: loops over requests, heads and tokens, from the formulas of include/pasa.h."""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
EXP_MIN, EXP_MAX = -50, 50


# ---------------------------------------------------------------- rotary --

def rope(x, positions, inv_freq, axis, pairing, inverse=False):
    """x [B, S, H, D]; positions [A, B, S].  fp64 [B, S, H, D]."""
    n = inv_freq.numel()
    y = x.double().clone()
    for i in range(n):
        a = positions[int(axis[i])].double() * float(inv_freq[i])
        a = (-a if inverse else a)[..., None]
        c0, c1 = (i, i + n) if pairing == "halves" else (2 * i, 2 * i + 1)
        x0, x1 = x[..., c0].double(), x[..., c1].double()
        y[..., c0] = x0 * a.cos() - x1 * a.sin()
        y[..., c1] = x1 * a.cos() + x0 * a.sin()
    return y


# ---------------------------------------------------------------- block tables --

def block_tables(tables, lens, new, free, num_free, page, tokens):
    """Python lists in, (tables, cu_q, slots, positions, lens, num_free) out."""
    tables = [list(r) for r in tables]
    left, cu, slots, pos, after = num_free, [0], [], [], []
    for r, (n, m) in enumerate(zip(lens, new)):
        m = min(max(m, 0), tokens - cu[-1])
        cu.append(cu[-1] + m)
        width = len(tables[r])
        have = -(-n // page)
        want = min(-(-(n + m) // page), width)
        while have < want and left > 0:
            left -= 1
            tables[r][have] = free[left]
            have += 1
        if have < want or n + m > width * page:
            end = min(n + m, have * page)
        else:
            end = n + m
        after.append(end)
        for i in range(m):
            p = n + i
            pos.append(p)
            id_ = tables[r][p // page] if p < end else -1
            slots.append(id_ * page + p % page if id_ >= 0 else -1)
    pad = tokens - cu[-1]
    return tables, cu, slots + [-1] * pad, pos + [-1] * pad, after, left


# ---------------------------------------------------------------- append --

def exponent(amax: float) -> int:
    """The smallest e in [-50, 50] with amax <= 448 * 2 ** e (the largest if there is none)."""
    e = EXP_MIN
    while e < EXP_MAX and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def to_code(x: torch.Tensor, e: int) -> torch.Tensor:
    y = torch.ldexp(x.double(), torch.tensor(-e)).clamp(-448, 448).float()
    return torch.where(torch.isfinite(x.double()), y, torch.tensor(float("nan"))).to(E4M3)


def append(k_codes, v_codes, k_exp, v_exp, k, v, slots, head_dim):
    """In place, on CPU tensors laid out as the cache's."""
    pages, heads, page, _ = k_codes.shape
    slots = [s if 0 <= s < pages * page else -2 for s in slots.tolist()]
    t = 0
    while t < len(slots):
        s, n = slots[t], 1
        if s < 0:
            t += 1
            continue
        while t + n < len(slots) and slots[t + n] == s + n and (s + n) % page:
            n += 1
        id_, off = s // page, s % page
        for h in range(heads):
            for codes, exps, x in ((k_codes[id_, h], k_exp, k), (v_codes[id_, h].view(torch.uint8).t().view(E4M3), v_exp, v)):
                new = x[t:t + n, h]
                fin = new.double()[torch.isfinite(new.double())]
                had = EXP_MIN if off == 0 else int(exps[id_, h])
                e = max(had, exponent(float(fin.abs().max()) if fin.numel() else 0.0))
                raw = codes.view(torch.uint8)
                if off and e != had:
                    others = [j for j in range(page) if not off <= j < off + n]
                    moved = torch.ldexp(codes.float()[others].double(), torch.tensor(had - e)).float().to(E4M3)
                    for j, row in zip(others, moved):
                        raw[j] = row.view(torch.uint8)
                raw[off:off + n] = 0
                raw[off:off + n, :head_dim] = to_code(new, e).view(torch.uint8)
                exps[id_, h] = e
        t += n


# ---------------------------------------------------------------- attention --

def attention(q, k_codes, v_codes, k_exp, v_exp, tables, lens, cu_q, scale, causal=False, window=None):
    """fp64 (o, lse, bound, lse_bound) of q [T, Hq, D]; the cache's tensors and tables on the CPU.  bound: what the kernel's
    arithmetic may add to o before its last rounding, from
      * p in fp16: half a step, 2^-11 of each term, once in the products (the sums are of unrounded p);
      * fp32 scores: (D + 8) 2^-24 of sum_d |q_d k_jd| each, as a relative error of p, in products and sums;
      * fp32 sums over n keys and exp2: (n + 8) 2^-24 in products and sums.
    lse_bound: the latter two once, and fp32's rounding of the result and its logarithm (2^-22 of it, and 2^-22)."""
    pages, heads, page, _ = k_codes.shape
    T, Hq, D = q.shape
    group = Hq // heads
    o = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    bound = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse_bound = torch.zeros(T, Hq, dtype=torch.float64)
    for r in range(len(lens)):
        a, b, n = cu_q[r], cu_q[r + 1], lens[r]
        ids = [tables[r][j] if j < len(tables[r]) else -1 for j in range(-(-n // page))]
        there = torch.tensor([0 <= ids[j // page] < pages for j in range(n)], dtype=torch.bool)
        safe = torch.tensor([i if 0 <= i < pages else 0 for i in ids], dtype=torch.long)
        for h in range(heads if n else 0):
            k = (k_codes[:, h].float().double()[safe] * 2.0 ** k_exp[safe, h].double()[:, None, None]).reshape(-1, k_codes.shape[3])[:n, :D]
            v = (v_codes[:, h].float().double()[safe] * 2.0 ** v_exp[safe, h].double()[:, None, None]).transpose(1, 2)
            v = v.reshape(-1, v_codes.shape[2])[:n, :D]
            j = torch.arange(n)
            for t in range(a, b):
                p_t = n - (b - a) + (t - a)
                see = there.clone()
                if causal:
                    see &= j <= p_t
                if window:
                    see &= j > p_t - window
                if not see.any():
                    continue
                kk, vv = k[see], v[see]
                for i in range(h * group, (h + 1) * group):
                    x = q[t, i].double()
                    s = (kk @ x) * scale
                    lse[t, i] = torch.logsumexp(s, 0)
                    p = torch.softmax(s, 0)
                    o[t, i] = p @ vv
                    mass = p @ vv.abs()
                    size = float(((kk.abs() @ x.abs()) * scale).max())
                    sums = ((D + 8) * size + len(s) + 8) * 2.0 ** -24
                    bound[t, i] = (2.0 ** -11 + 2 * sums) * mass
                    lse_bound[t, i] = sums + 2.0 ** -22 * (1 + abs(float(lse[t, i])))
    return o, lse, bound, lse_bound
