"""Caches of 8-bit codes in 64 bits, from the formulas.  TEST INFRASTRUCTURE ONLY: nothing in the shipped package may import this module.

A cache is a pair (codes, scales): codes int8 or float8_e4m3fn [pages, Hk, page_size, D] ("HND") or [pages, page_size, Hk, D] ("NHD"), scales
fp32 [pages, Hk, blocks].
"""
from __future__ import annotations

import math

import torch

from . import serving_oracle as SO

LARGEST = {torch.int8: 127, torch.float8_e4m3fn: 448}
SMALLEST = 2.0 ** -100


def numbers(codes):
    """What codes are as numbers, in 64 bits."""
    return codes.float().double()


def values(codes, scales, layout="HND"):
    """[pages, page_size, Hk, D] in 64 bits."""
    x = numbers(codes)
    x = x.transpose(1, 2) if layout == "HND" else x
    page = x.shape[1]
    s = scales.double().repeat_interleave(page // scales.shape[-1], dim=-1)  # [pages, Hk, page]
    return x * s.transpose(1, 2)[..., None]


def e4m3_numbers():
    """The finite e4m3 numbers that are not negative, in order: number i has the bits i."""
    return torch.tensor([(i & 7) * 2.0 ** -9 if i < 8 else (8 + (i & 7)) * 2.0 ** ((i >> 3) - 10) for i in range(127)], dtype=torch.float64)


def nearest(x, dtype):
    """The nearest codes to numbers in 64 bits, ties to the even one, as numbers."""
    if dtype == torch.int8:
        return torch.round(x).clamp(max=127)  # (half to even)
    grid = e4m3_numbers()
    size = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(grid, size.contiguous()).clamp(min=1, max=126)
    lo = hi - 1
    below, above = size - grid[lo], grid[hi] - size
    pick = torch.where((above < below) | ((above == below) & (hi % 2 == 0)), grid[hi], grid[lo])
    return torch.copysign(pick, x)


def append(k, v, k_cache, v_cache, slots, k_scale, v_scale, layout="HND"):
    """Returns new (k_cache, v_cache, k_scale, v_scale); all on the CPU."""
    res_codes, res_scales = [], []
    page = k_cache.shape[2] if layout == "HND" else k_cache.shape[1]
    pages, blocks = k_cache.shape[0], k_scale.shape[-1]
    size = page // blocks
    tokens = {}
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * page:
            tokens.setdefault(slot // size, {})[slot % size] = t
    for x, codes, scales in ((k, k_cache, k_scale), (v, v_cache, v_scale)):
        codes, scales = codes.clone(), scales.clone()
        by_place = codes if layout == "NHD" else codes.transpose(1, 2)  # [pages, page, Hk, D]
        for b, places in tokens.items():
            p, at = b // blocks, b % blocks
            rows = x[list(places.values())].float()  # [n, Hk, D]
            for h in range(x.shape[1]):
                row = rows[:, h].double()
                old = 0.0 if 0 in places else float(scales[p, h, at])
                if torch.isfinite(row).all():
                    # (in fp32, correctly rounded: the quotient of a 24-bit number and 127 or 7 lies on no middle, and next to none)
                    asked = float((row.abs().max().clamp(min=SMALLEST) / LARGEST[codes.dtype]).float())
                else:
                    asked = math.nan
                # (sizes: a block that the program gave a negative scale keeps its values; one of an infinite scale keeps that)
                now = math.nan if math.isnan(old) or math.isnan(asked) else old if math.isinf(old) else max(abs(old), asked)
                scales[p, h, at] = now
                held = by_place[p, at * size:(at + 1) * size, h]
                new = numbers(held)
                if 0 in places:
                    new = torch.zeros_like(new)
                elif now != old and now == now:
                    new = nearest(new * old / now, codes.dtype)  # (code * old has 31 bits; the quotient next to a middle but not on it differs by 2^-32 of itself)
                for i, q in enumerate(places):
                    new[q] = 0.0 if math.isnan(now) else nearest(row[i] / now, codes.dtype)
                held.copy_(new.float().to(codes.dtype))
        res_codes.append(codes)
        res_scales.append(scales)
    return (*res_codes, *res_scales)


def read(codes, scales, table, cu, total, dtype, layout="HND"):
    """[total, Hk, D]; rows of no sequence are NaN.  The product in fp32, as documented, and one rounding from there."""
    x = codes.float()
    x = x.transpose(1, 2) if layout == "HND" else x
    pages, page, hk, d = x.shape
    out = torch.full((total, hk, d), math.nan, dtype=dtype)
    cu = cu.tolist()
    for s in range(len(cu) - 1):
        for t in range(cu[s], min(cu[s + 1], total)):
            pos = t - cu[s]
            p = int(table[s, pos // page]) if pos // page < table.shape[1] else -1
            if not 0 <= p < pages:
                out[t] = 0
            elif scales is None:
                out[t] = codes[p, :, pos % page] if layout == "HND" else codes[p, pos % page]
            else:
                out[t] = (x[p, pos % page] * scales[p, :, pos % page // (page // scales.shape[-1])][:, None]).to(dtype)
    return out


def paged(q, k_cache, v_cache, k_scale, v_scale, table, lens, sm_scale=None, layout="HND"):
    """As serving_oracle.paged, with the bounds of the kernel over codes: q [S, H, D] or [S, M, H, D]."""
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    q4 = q if q.dim() == 4 else q[:, None]
    kv, vv = values(k_cache, k_scale, layout), values(v_cache, v_scale, layout)
    pages, page, hk, d = kv.shape
    v_size = numbers(v_cache).abs()
    v_size = v_size.transpose(1, 2) if layout == "HND" else v_size  # [pages, page, Hk, D], of the codes
    s_size = v_scale.double().abs().repeat_interleave(page // v_scale.shape[-1], dim=-1).transpose(1, 2)  # [pages, page, Hk]
    S, M, H, _ = q4.shape
    half_step = torch.finfo(q.dtype).eps / 2
    least = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134  # half a step of the output below its normal range
    o = torch.zeros(q4.shape, dtype=torch.float64)
    o_tol = torch.zeros_like(o)
    norm = torch.full((S, H, M), -math.inf, dtype=torch.float64)
    norm_tol = torch.zeros_like(norm)
    for s in range(S):
        n = min(max(int(lens[s]), 0), table.shape[1] * page)
        rows = table[s, :-(-n // page)].long()
        bad = (rows < 0) | (rows >= pages)
        hidden = bad.repeat_interleave(page)[:n]
        k, v, vc = (c[rows.masked_fill(bad, 0)].reshape(-1, hk, d)[:n] for c in (kv, vv, v_size))
        vs = s_size[rows.masked_fill(bad, 0)].reshape(-1, hk)[:n]
        for h in range(H):
            ki, vi, ci, si = (x[:, h * hk // H] for x in (k, v, vc, vs))
            for m in range(M):
                sees = (torch.arange(n) <= n - M + m) & ~hidden
                if not sees.any():
                    continue
                kk, vw, qi = ki[sees], vi[sees], q4[s, m, h].double()
                x = (kk @ qi) * sm_scale
                norm[s, h, m] = torch.logsumexp(x, 0)
                p = torch.exp(x - x.max())
                inv = 1 / p.sum()
                o[s, m, h] = (p @ vw) * inv
                # A score: D products summed in fp32, three factors, the exponent's argument and the exponential, each a few 2^-24 of
                # the sum of the terms' sizes or of 1; queries in bf16 enter as fp16, off by up to 2^-39 of the row's largest
                # (which is at least 2^14 there, and half of the least step is 2^-25).
                size = float(((kk.abs() @ qi.abs()) * abs(sm_scale)).max())
                score = (d + 16) * 2.0 ** -24 * size + 2.0 ** -21
                if q.dtype == torch.bfloat16:
                    score += 2.0 ** -39 * float(qi.abs().max()) * float(kk.abs().sum(1).max()) * abs(sm_scale)
                cnt = int(sees.sum())
                norm_tol[s, h, m] = score + cnt * 2.0 ** -24 + 2.0 ** -22 * abs(float(norm[s, h, m]))
                # A weight w = p vs is rounded to fp16, whose numbers in [1, 2) lie 2^-10 apart: off by half of that, 2^-11 of itself
                # (a bound of 2^-12, as if the step were 2^-11, is below what the rounding itself does); those below 2^-14 lie 2^-24 apart,
                # and the row's largest weight so far is at least 2^10 in their unit: off by 2^-25 / 2^10 = 2^-35 of it, and by no
                # more than themselves (the nearest number is no further than zero).  In fp32 before that: p below 2^-126 may be zero, products below
                # it lie 2^-149 apart.  Each reaches the output through its own code; the output is rounded once more.
                spread = (p @ vw.abs()) * inv
                w = p * si[sees]
                small = torch.minimum(w, 2.0 ** -35 * w.max()) + p.clamp(max=2.0 ** -126) * si[sees] + 2.0 ** -150
                o_tol[s, m, h] = half_step * (o[s, m, h].abs() + 2.0 ** -11 * spread) + 2.0 ** -11 * spread \
                    + (2 * score + 2 * cnt * 2.0 ** -24 + 2.0 ** -22) * spread + (small @ ci[sees]) * inv + least
    if q.dim() == 3:
        o, o_tol, norm, norm_tol = o[:, 0], o_tol[:, 0], norm[:, :, 0], norm_tol[:, :, 0]
    return o, norm, o_tol, norm_tol


assert_close = SO.assert_close
