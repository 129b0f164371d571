"""The paged cache of 8-bit codes where scales are far apart, of either sign or not finite, and where calls are large: against the formulas in 64 bits
(oracle/cache8_oracle.py)."""
import math

import pytest
import torch

from oracle import cache8_oracle as CO

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16
CODES = {"int8": INT8, "e4m3": E4M3}


def random_codes(shape, dtype, g):
    x = torch.randint(-127, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)
    if dtype == E4M3:
        x = torch.where((x & 127) == 127, torch.zeros_like(x), x).view(E4M3)
    return x


def make_cache(pages, hk, page, blocks, d, dtype, g, spread=1.0):
    codes = [random_codes((pages, hk, page, d), dtype, g) for _ in range(2)]
    scales = [torch.exp2(spread * torch.randn(pages, hk, blocks, generator=g)) / (70 if dtype == INT8 else 30) for _ in range(2)]
    return (*codes, *scales)


def attend(q, cache, table, lens, dev):
    import flag_attn

    kc, vc, ks, vs = (x.to(dev) for x in cache)
    o, norm = flag_attn.paged_attention(q.to(dev), kc, vc, table.to(dev), torch.as_tensor(lens, dtype=torch.int32).to(dev), return_log_normalizer=True,
                                        k_scale=ks, v_scale=vs)
    return o.cpu(), norm.cpu()


def check(q, cache, table, lens, dev, what=""):
    """Returns (output, its oracle)."""
    o, norm = attend(q, cache, table, lens, dev)
    want, want_norm, tol, norm_tol = CO.paged(q, *cache, table, lens)
    CO.assert_close(norm, want_norm, norm_tol, (what, "log normalizer"))
    CO.assert_close(o, want, tol, (what, "output"))
    seen = want_norm > -math.inf if q.dim() == 3 else (want_norm > -math.inf).transpose(1, 2)
    # what the bounds are worth: an output of zeros is outside of nearly all of them
    assert (want.abs() > tol)[seen].double().mean() > 0.9, what
    return o, want


# ---- value scales far apart: what a value weighs is p times its scale

@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("far", [30, 38, 44, 80, -38, -80])
def test_a_far_scale_under_keys_of_no_weight(gpu_device, codes, dtype, page, d, far):
    """The others keep their part, whether the keys whose values are 2^far as large come first, between them or last, and whether the tiles
    before and after them are full of such keys.  (Their own weight is about 2^-200.)"""
    g = torch.Generator().manual_seed(50)
    n = 320
    for begin, end in ((0, 1), (0, 64), (100, 101), (96, 160), (319, 320), (280, 320)):
        pages = -(-n // page)
        kc, vc, ks, vs = make_cache(pages, 1, page, page, d, CODES[codes], g)
        at = torch.arange(begin, end)
        kc.view(torch.int8)[at // page, 0, at % page] = -127 if codes == "int8" else -2  # e4m3: -448
        ks[at // page, 0, at % page] = 0.3 if codes == "int8" else 0.1
        vs[at // page, 0, at % page] *= 2.0 ** far
        q = torch.full((1, 4, d), 3.0) + 0.1 * torch.randn(1, 4, d, generator=g)
        check(q.to(dtype), (kc, vc, ks, vs), torch.arange(pages, dtype=torch.int32)[None], [n], gpu_device, (begin, end))


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 24])
def test_a_large_scale_that_other_rows_do_not_see(gpu_device, codes, page):
    """Of several new tokens, those that do not see the last keys are as exact as without them."""
    g = torch.Generator().manual_seed(51)
    lens, m, hk = [100, 64, 33], 4, 2
    pages = sum(-(-n // page) for n in lens)
    cache = make_cache(pages, hk, page, page, 64, CODES[codes], g)
    table, at = torch.zeros(3, 8, dtype=torch.int32), 0
    for s, n in enumerate(lens):
        table[s, :-(-n // page)] = torch.arange(at, at - (-n // page))
        at -= -n // page
        cache[3][int(table[s, (n - 1) // page]), :, (n - 1) % page] *= 2.0 ** 50
    q = torch.randn(3, m, 8, 64, generator=g).to(BF16)
    o, want = check(q, cache, table, lens, gpu_device)
    assert want[:, 3].abs().max() > 2.0 ** 30 and want[:, :3].abs().max() < 2.0 ** 10  # (of the oracle)


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_rows_that_weigh_the_same_values_differently(gpu_device, dtype):
    """Two kinds of keys, 2^40 apart in the scales of their values; one half of the rows gives the large ones weight 2^-40, the other half next to none."""
    g = torch.Generator().manual_seed(52)
    page, n, d = 16, 400, 64
    pages = n // page
    kc, vc, ks, vs = make_cache(pages, 1, page, page, d, INT8, g, spread=0.3)
    far = torch.rand(n, generator=g) < 0.5
    at = torch.arange(n)[far]
    vs[at // page, 0, at % page] *= 2.0 ** 40
    kc[..., 0] = 127
    kc[at // page, 0, at % page, 0] = -127
    ks.fill_(1.0 / 127)
    q = 0.2 * torch.randn(1, 8, d, generator=g)
    q[0, :4, 0] = 20 * math.log(2) * 8  # scores of +20 ln 2 and -20 ln 2: weights 2^-40 apart
    q[0, 4:, 0] = 40 * math.log(2) * 8
    check(q.to(dtype), (kc, vc, ks, vs), torch.arange(pages, dtype=torch.int32)[None], [n], gpu_device)


def test_far_scales_in_cut_launches(gpu_device):
    """Shares whose keys have values of very different sizes are joined."""
    g = torch.Generator().manual_seed(53)
    page, n, d = 16, 3000, 128
    pages = -(-n // page)
    kc, vc, ks, vs = make_cache(pages, 2, page, 4, d, INT8, g)
    vs *= torch.exp2(torch.randint(-60, 1, (pages, 1, 1), generator=g).float())
    vs[5] *= 2.0 ** 70
    kc[5] = -127
    ks[5] = 0.3
    wide = torch.zeros(1, 1300, dtype=torch.int32)
    wide[0, :pages] = torch.arange(pages)
    check((3 + 0.1 * torch.randn(1, 8, d, generator=g)).to(BF16), (kc, vc, ks, vs), wide, [n], gpu_device)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_entries_of_a_query_far_below_its_largest(gpu_device, codes):
    """Queries in bf16 enter in steps of 2^-38 of a largest entry of 1: one of 1.5 steps beside it is off by half a step, 2^-39."""
    g = torch.Generator().manual_seed(54)
    kc, vc, ks, vs = make_cache(2, 1, 16, 1, 64, CODES[codes], g)
    kc.view(torch.int8).zero_()
    kc[:, :, :, 1] = torch.arange(32).view(2, 1, 16).to(kc.dtype)
    ks.fill_(2.0 ** 37)
    q = torch.zeros(1, 2, 64)
    q[:, :, 0], q[0, 0, 1], q[0, 1, 1] = 1.0, 1.5 * 2.0 ** -38, 3 * 2.0 ** -38
    _, norm = attend(q.to(BF16), (kc, vc, ks, vs), torch.arange(2, dtype=torch.int32)[None], [32], gpu_device)
    _, want, _, tol = CO.paged(q.to(BF16), kc, vc, ks, vs, torch.arange(2, dtype=torch.int32)[None], [32])
    CO.assert_close(norm, want, tol)
    assert (norm - want).abs()[0, 0] > 0.6 * tol[0, 0] and (norm - want).abs()[0, 1] < 1e-5


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("m", [1, 3])
@pytest.mark.parametrize("least,most", [(112, 112), (-105, -105), (-105, 110), (-60, 60), (0, 0)])
def test_value_scales_near_the_ends_of_fp32(gpu_device, codes, page, m, least, most):
    """All values very large, or very small (as blocks of the smallest scale are), or of sizes drawn from a wide range, key by key; negative ones among them."""
    g = torch.Generator().manual_seed(55)
    lens, hk = [300, 150, m, 64], 2
    pages = sum(-(-n // page) for n in lens)
    kc, vc, ks, vs = make_cache(pages, hk, page, page, 64, CODES[codes], g)
    vs *= torch.exp2(torch.randint(least, most + 1, vs.shape, generator=g).float()) * torch.where(torch.rand(vs.shape, generator=g) < 0.5, -1.0, 1.0)
    table, at = torch.zeros(len(lens), 300 // page + 1, dtype=torch.int32), 0
    for s, n in enumerate(lens):
        table[s, :-(-n // page)] = torch.arange(at, at - (-n // page))
        at -= -n // page
    q = torch.randn(len(lens), m, 8, 64, generator=g).to(BF16)
    check(q if m > 1 else q[:, 0], (kc, vc, ks, vs), table, lens, gpu_device)


def test_scales_that_grow_along_a_sequence(gpu_device):
    """Every tile's values are larger than all before, or every tile's keys count more than all before: units and references move at each step."""
    g = torch.Generator().manual_seed(56)
    page, n = 16, 1536
    pages = n // page
    for grows in (2, 3):
        cache = list(make_cache(pages, 1, page, 1, 64, INT8, g, spread=0.2))
        cache[0].copy_(cache[0].abs())
        cache[grows] *= torch.exp2(torch.arange(pages).float() * (0.6 if grows == 3 else 0.05))[:, None, None]
        q = 0.3 + 0.1 * torch.randn(1, 8, 64, generator=g)
        for dtype in (BF16, FP16) if grows == 2 else (BF16,):
            check(q.to(dtype), cache, torch.arange(pages, dtype=torch.int32)[None], [n], gpu_device, grows)
