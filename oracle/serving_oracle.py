"""Attention of packed sequences and of paged caches in 64 bits, from the formulas.  TEST INFRASTRUCTURE ONLY: nothing in the
shipped package may import this module.

``attend`` evaluates one sequence; ``varlen`` and ``paged`` take the operators' arguments apart into sequences and call it.  Each
returns the output, the natural log normalizer and the bounds that the tests compare with: how far a kernel may be off
that multiplies in fp32, rounds P and the output to 16 bits and keeps statistics in fp32.
"""
from __future__ import annotations

import math

import torch


def attend(q, k, v, causal, sm_scale, hidden=None):
    """q [M, H, D], k, v [N, Hk, D] -> o [M, H, D], log normalizer [H, M], bounds of both.  hidden [N]: keys that take no part.
    Keys that a query does not see are left out of its sums (an infinity there changes nothing)."""
    m, h, d = q.shape
    n, hk = k.shape[0], k.shape[1]
    half_step = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0  # fp16: P below the normal range is off by up to half of 2^-24
    dev = q.device
    o = torch.zeros(m, h, d, dtype=torch.float64, device=dev)
    o_tol = torch.zeros_like(o)
    norm = torch.full((h, m), -math.inf, dtype=torch.float64, device=dev)
    norm_tol = torch.zeros_like(norm)
    if n == 0 or m == 0:
        return o, norm, o_tol, norm_tol
    sees = torch.ones(m, n, dtype=torch.bool, device=dev)
    if causal:
        sees = torch.arange(n, device=dev)[None, :] <= torch.arange(m, device=dev)[:, None] + (n - m)
    if hidden is not None:
        sees = sees & ~hidden[None, :]
    some = sees.any(dim=1)
    for i in range(h):
        qi, ki, vi = q[:, i].double(), k[:, i // (h // hk)].double(), v[:, i // (h // hk)].double()
        clean = torch.isfinite(vi).all()
        s = torch.where(sees, (qi @ ki.t()) * sm_scale, -math.inf)
        top = torch.where(some, s.amax(dim=1), 0.0)
        p = torch.where(sees, torch.exp(s - top[:, None]), 0.0)
        total = p.sum(dim=1)
        inv = torch.where(some, 1.0 / total, 0.0)
        if clean:
            oi = p @ vi
        else:
            oi = torch.where(sees[:, :, None], p[:, :, None] * vi[None], 0.0).sum(dim=1)
        oi = torch.where(some[:, None], oi * inv[:, None], 0.0)
        o[:, i] = oi
        norm[i] = torch.where(some, top + total.log(), -math.inf)
        # fp32 products of D terms: each score is off by up to (D + 4) 2^-24 of the sum of its terms' sizes (and of the scale, the
        # exponent's argument and the exponential itself, each a few 2^-24 of the score or of 1)
        size = torch.where(sees, (qi.abs() @ ki.abs().t()) * sm_scale, 0.0).amax(dim=1)
        score = (d + 12) * 2.0 ** -24 * size + 2.0 ** -21
        norm_tol[i] = score + n * 2.0 ** -24 + 2.0 ** -22 * norm[i].abs().nan_to_num(posinf=0.0)
        spread = (p @ vi.abs().nan_to_num(posinf=0.0)) * inv[:, None]  # mean of |v| under P
        vmax = vi.abs().nan_to_num(posinf=0.0).amax()
        o_tol[:, i] = half_step * (spread + oi.abs().nan_to_num(posinf=0.0)) \
            + (2 * score + 2 * n * 2.0 ** -24)[:, None] * spread + n * tiny * vmax * inv[:, None] + torch.finfo(q.dtype).tiny
    return o, norm, o_tol, norm_tol


def varlen(q, k, v, cu_q, cu_k, causal, sm_scale=None):
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    norm = torch.zeros(q.shape[1], q.shape[0], dtype=torch.float64, device=q.device)
    o_tol, norm_tol = torch.zeros_like(o), torch.zeros_like(norm)
    cu_q, cu_k = cu_q.tolist(), cu_k.tolist()
    for s in range(len(cu_q) - 1):
        a, b, c, e = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        o[a:b], norm[:, a:b], o_tol[a:b], norm_tol[:, a:b] = attend(q[a:b], k[c:e], v[c:e], causal, sm_scale)
    return o, norm, o_tol, norm_tol


def paged(q, k_cache, v_cache, table, lens, sm_scale=None, layout="HND"):
    """q [S, H, D] or [S, M, H, D]; log normalizer [S, H] or [S, H, M]."""
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    q4 = q if q.dim() == 4 else q[:, None]
    if layout == "HND":
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    pages, page, hk, d = k_cache.shape
    res = []
    for s in range(q4.shape[0]):
        n = min(max(int(lens[s]), 0), table.shape[1] * page)
        rows = table[s, :-(-n // page)].long()
        bad = (rows < 0) | (rows >= pages)
        k, v = (c[rows.masked_fill(bad, 0)].reshape(-1, hk, d)[:n] for c in (k_cache, v_cache))
        hidden = bad.repeat_interleave(page)[:n]
        res.append(attend(q4[s], k, v.masked_fill(hidden[:, None, None], 0), True, sm_scale, hidden))
    o, norm, o_tol, norm_tol = (torch.stack(x) for x in zip(*res))
    if q.dim() == 3:
        o, o_tol, norm, norm_tol = o[:, 0], o_tol[:, 0], norm[:, :, 0], norm_tol[:, :, 0]
    return o, norm, o_tol, norm_tol


def assert_close(got, want, tol, what=""):
    """Infinities and NaN in the same places, everything else within its bound."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (what, "NaN in other places")
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), (what, "infinities in other places")
    fine = torch.isfinite(want)
    over = (got - want).abs()[fine] - tol[fine]
    if over.numel():
        worst = over.argmax()
        assert over[worst] <= 0, (what, "off by", float((got - want).abs()[fine][worst]), "allowed", float(tol[fine][worst]))
