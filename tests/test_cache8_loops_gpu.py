"""Quantized writes that go through several heads in one wave or workgroup, sizes on both sides of the choice between looking tokens up and mapping them,
and the longest blocks; bit by bit against the formulas in 64 bits (oracle/cache8_oracle.py)."""
import pytest
import torch

from oracle import cache8_oracle as CO

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16
CODES = {"int8": INT8, "e4m3": E4M3}


def same_numbers(a, b):
    """Equal, where the two zeros are one number and NaN equals NaN."""
    return torch.equal(torch.nan_to_num(a.cpu().float(), nan=1e30), torch.nan_to_num(b.cpu().float(), nan=1e30))


def check_write(slots, pages, hk, page, blocks, d, codes, dtype, g, dev, layout="HND"):
    """Rows of sizes far apart into a cache of random codes and scales, so that many blocks that go on have their codes converted.
    Returns how many did."""
    import flag_attn

    shape = (pages, hk, page, d) if layout == "HND" else (pages, page, hk, d)
    cache = []
    for _ in range(2):
        c = torch.randint(-127, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)
        cache.append(torch.where((c & 127) == 127, torch.zeros_like(c), c).view(codes))
    top = CO.LARGEST[codes]
    cache += [torch.exp2(2 * torch.randn(pages, hk, blocks, generator=g)) / top for _ in range(2)]
    x = [(torch.randn(len(slots), hk, d, generator=g) * torch.exp2(2 * torch.randn(len(slots), hk, 1, generator=g))).to(dtype) for _ in range(2)]
    slots = torch.as_tensor(slots)
    now = [t.to(dev) for t in cache]
    flag_attn.append_to_cache(x[0].to(dev), x[1].to(dev), now[0], now[1], slots.to(dev), tensor_layout=layout, k_scale=now[2], v_scale=now[3])
    want = CO.append(x[0], x[1], cache[0], cache[1], slots, cache[2], cache[3], layout)
    for got, w, name in zip(now, want, ("k_cache", "v_cache", "k_scale", "v_scale")):
        assert same_numbers(got, w), (name, int((got.cpu().float() != w.float()).sum()))
    # blocks that go on (their first place is not among the slots) and whose scale has grown
    size = page // blocks
    inside = slots[(slots >= 0) & (slots < pages * page)]
    begun = torch.zeros(pages * blocks, dtype=torch.bool)
    begun[inside[inside % size == 0] // size] = True
    grew = (want[2] > cache[2]).transpose(1, 2).reshape(pages * blocks, hk)
    return int(grew[~begun].sum())


def in_order(tokens, at, page, g, spare=1):
    """Tokens that fill pages in order, from place `at` on; pages in random order."""
    need = -(-(at + tokens) // page)
    where = torch.randperm(need + spare, generator=g)[:need]
    t = at + torch.arange(tokens)
    return where[t // page] * page + t % page, need + spare


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("tokens,hk,page,blocks,d", [
    (600, 64, 16, 1, 64),     # short blocks through the map: 10 workgroups, 102 < 128 units of a head of K or V
    (1030, 40, 8, 1, 64),     # two of them in a wave: 17 groups, 60 < 80
    (700, 80, 32, 1, 64),     # blocks of two steps of rows
    (200, 16, 16, 1, 64),     # short blocks by looking: 50 groups, 20 < 32
    (200, 8, 64, 1, 64),      # long blocks by looking: 200 groups, 5 < 16
    (200, 8, 64, 1, 128),
    (1500, 32, 128, 1, 128),  # long blocks through the map: 24 groups, 42 < 64
    (1500, 24, 48, 1, 64),    # of a number of rows that is no power of two: 32 groups, 32 < 48
    (256, 6, 96, 3, 80),
])
def test_heads_that_follow_each_other(gpu_device, codes, tokens, hk, page, blocks, d):
    """More heads of K and V than workgroups for them: each goes through several, the first block of the call goes on."""
    g = torch.Generator().manual_seed(70)
    size = page // blocks
    slots, pages = in_order(tokens, size // 2 + 1, page, g)
    slots = torch.cat([slots, torch.full((2,), -1)])
    assert check_write(slots[:tokens], pages, hk, page, blocks, d, CODES[codes], BF16, g, gpu_device) > 0
    # and in random order, half of the places
    some = torch.randperm(pages * page, generator=g)[: min(tokens, pages * page // 2)]
    assert check_write(some, pages, hk, page, blocks, d, CODES[codes], BF16, g, gpu_device) > 0


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("tokens", [252, 253, 255, 256, 257, 320])
@pytest.mark.parametrize("page,blocks,at", [(16, 1, 0), (16, 4, 5), (32, 32, 3), (256, 1, 100), (24, 2, 1), (64, 1, 7)])
def test_tokens_around_the_choice(gpu_device, codes, tokens, page, blocks, at):
    """Calls of up to 256 rows, padding among them, look their tokens up, larger ones map them."""
    g = torch.Generator().manual_seed(71)
    slots, pages = in_order(tokens, at, page, g, 2)
    for n in (0, 3):
        check_write(torch.cat([slots, torch.full((n,), -1)]).to(torch.int32), pages, 2, page, blocks, 64, CODES[codes], FP16, g, gpu_device)
    check_write(torch.randperm(pages * page, generator=g)[:tokens], pages, 2, page, blocks, 64, CODES[codes], FP16, g, gpu_device)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page,blocks", [(512, 1), (1024, 1), (2048, 2), (768, 1), (520, 1)])
def test_the_longest_blocks(gpu_device, codes, dtype, d, page, blocks):
    """Blocks of 512 to 1024 tokens, more than a workgroup keeps in registers: begun and gone on, few tokens and many, in order and not."""
    g = torch.Generator().manual_seed(72)
    dev, hk, size = gpu_device, 2, page // blocks
    for tokens, at in ((200, 0), (200, size - 100), (size + 130, 0), (size + 130, 300)):
        slots, pages = in_order(tokens, at, page, g)
        check_write(slots, pages, hk, page, blocks, d, CODES[codes], dtype, g, dev)
    for tokens in (250, 700):
        slots = torch.randperm(2 * page, generator=g)[:tokens]
        slots = slots[slots % size != 0]
        assert check_write(slots, 2, hk, page, blocks, d, CODES[codes], dtype, g, dev) > 0

