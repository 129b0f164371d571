"""Quantized writes into blocks that go on, over scales and codes that a program wrote itself: negative scales, zeros, infinities, NaN, and what
attention makes of infinite scales; bit by bit against the formulas in 64 bits (oracle/cache8_oracle.py)."""
import math

import pytest
import torch

from oracle import cache8_oracle as CO

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16 = torch.bfloat16
CODES = {"int8": INT8, "e4m3": E4M3}


def random_codes(shape, dtype, g):
    x = torch.randint(-127, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)
    if dtype == E4M3:
        x = torch.where((x & 127) == 127, torch.zeros_like(x), x).view(E4M3)
    return x


def same_numbers(a, b):
    """Equal, where the two zeros are one number and NaN equals NaN."""
    return torch.equal(torch.nan_to_num(a.cpu().float(), nan=1e30), torch.nan_to_num(b.cpu().float(), nan=1e30))


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("page,blocks,tokens", [(16, 1, 200), (16, 4, 200), (16, 1, 700), (16, 4, 700), (64, 1, 200), (128, 2, 700), (24, 3, 300)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "fp32"])
def test_scales_of_either_sign_that_are_held(gpu_device, codes, page, blocks, tokens, dtype):
    """A block that goes on compares with the size of its scale: the new one is the larger size, and what the block holds keeps its values."""
    import flag_attn

    g = torch.Generator().manual_seed(60)
    dev, hk, d, size = gpu_device, 2, 64, page // blocks
    pages = 2 * tokens // page + 2
    slots = torch.randperm(pages * page, generator=g)
    slots = slots[slots % size != 0][:tokens]  # (no block begins anew)
    x = [(torch.randn(tokens, hk, d, generator=g) * torch.exp2(3 * torch.randn(tokens, hk, 1, generator=g))).to(dtype) for _ in range(2)]
    held = [random_codes((pages, hk, page, d), CODES[codes], g) for _ in range(2)]
    top = CO.LARGEST[CODES[codes]]
    scales = [torch.exp2(4 * torch.randn(pages, hk, blocks, generator=g)) / top for _ in range(2)]
    for s in scales:
        s.mul_(torch.where(torch.rand(s.shape, generator=g) < 0.6, -1.0, 1.0))
        for i, bad in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan)):
            s[i % pages, 0, 0] = bad
    now = [t.to(dev) for t in (*held, *scales)]
    flag_attn.append_to_cache(x[0].to(dev), x[1].to(dev), now[0], now[1], slots.to(dev), k_scale=now[2], v_scale=now[3])
    want = CO.append(x[0], x[1], held[0], held[1], slots, scales[0], scales[1])
    assert same_numbers(now[2], want[2]) and same_numbers(now[3], want[3])
    assert same_numbers(now[0], want[0]) and same_numbers(now[1], want[1])


def test_a_negative_scale_is_no_reason_to_wrap(gpu_device):
    """By hand: codes of -5 under a row that asks for 1 become codes of 5 with the other sign; the lowest of int8, -128, the highest there is."""
    import flag_attn

    dev = gpu_device
    for kinds, top in ((INT8, 127.0), (E4M3, 448.0)):
        held = torch.zeros(1, 1, 16, 64)
        held[0, 0, 0, :4] = torch.tensor([top, -top, 1.0, -128.0])
        kc, vc = held.to(kinds).to(dev), held.to(kinds).to(dev)
        ks, vs = torch.full((1, 1, 1), -5.0, device=dev), torch.full((1, 1, 1), 5.0, device=dev)
        row = torch.full((1, 1, 64), top, dtype=torch.float32, device=dev)  # asks for a scale of 1
        flag_attn.append_to_cache(row, row, kc, vc, torch.tensor([3], device=dev), k_scale=ks, v_scale=vs)
        assert float(ks) == 5.0 and float(vs) == 5.0
        assert kc.float()[0, 0, 0, :4].tolist() == [-top, top, -1.0, 127.0 if kinds == INT8 else 128.0]
        assert vc.float()[0, 0, 0, :4].tolist() == [top, -top, 1.0, -128.0]
        assert (kc.float()[0, 0, 3] == vc.float()[0, 0, 3]).all() and not kc.float()[0, 0, 1].any()


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("m", [1, 4])
def test_infinite_scales_of_keys(gpu_device, codes, page, m):
    """A score of minus infinity leaves the key out, one of plus infinity makes the row NaN; rows that do not see the key are as before.  A row
    whose keys are all left out is a row of zeros."""
    import flag_attn

    g = torch.Generator().manual_seed(61)
    dev, n, hk, h, d = gpu_device, 100, 2, 8, 64
    pages = -(-n // page)
    kc, vc = (random_codes((pages, hk, page, d), CODES[codes], g) for _ in range(2))
    ks, vs = (torch.rand(pages, hk, page, generator=g) / 30 + 0.01 for _ in range(2))
    kc.view(torch.int8)[:, :, :, 0] = 64                               # (channel 0 of every key: 64, or 2 in e4m3)
    table, lens = torch.arange(pages, dtype=torch.int32)[None].to(dev), torch.tensor([n], dtype=torch.int32, device=dev)

    def attend(q, ks):
        q, ks = q.to(dev), ks.to(dev)
        q = q if m > 1 else q[:, 0]
        o, norm = flag_attn.paged_attention(q, kc.to(dev), vc.to(dev), table, lens, return_log_normalizer=True, k_scale=ks, v_scale=vs.to(dev))
        return (o.cpu(), norm.transpose(1, 2).cpu()) if m > 1 else (o.cpu()[:, None], norm.cpu()[:, None])

    q = torch.randn(1, m, h, d, generator=g).to(BF16)
    q[:, :, ::2, 1:] = 0                                               # these rows score by channel 0 alone, and positively before the scale
    q[:, :, ::2, 0] = 1.5
    at = n - 3                                                         # new token i of four sees keys up to 96 + i: the last three see it
    sees = torch.zeros(1, m, h // 2, dtype=torch.bool)
    sees[:, -3:] = True
    for kv in range(hk):
        far, low, high = ks.clone(), ks.clone(), ks.clone()
        far[at // page, kv, at % page], low[at // page, kv, at % page], high[at // page, kv, at % page] = -2.0 ** 40, -math.inf, math.inf
        mine = sees & ((torch.arange(0, h, 2) // (h // hk)) == kv)
        clean, clean_norm = attend(q, ks)
        (a, an), (b, bn), (c, cn) = (attend(q, x) for x in (far, low, high))
        assert torch.equal(a[:, :, ::2], b[:, :, ::2]) and torch.equal(an[:, :, ::2], bn[:, :, ::2])
        assert torch.isnan(c[:, :, ::2][mine]).all() and torch.isnan(cn[:, :, ::2][mine]).all()
        assert torch.equal(c[:, :, ::2][~mine], clean[:, :, ::2][~mine]) and torch.equal(cn[:, :, ::2][~mine], clean_norm[:, :, ::2][~mine])
    o, norm = attend(q, torch.full_like(ks, -math.inf))
    assert not o[:, :, ::2].any() and (norm[:, :, ::2] == -math.inf).all()
