"""The paged cache of 8-bit codes on the GPU against its formulas in 64 bits: writes bit by bit, reads bit by bit, attention within bounds
that follow from its roundings (oracle/cache8_oracle.py), and the run of them together."""
import math

import pytest
import torch

from oracle import cache8_oracle as CO

pytestmark = pytest.mark.gpu

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
BF16, FP16 = torch.bfloat16, torch.float16
CODES = {"int8": INT8, "e4m3": E4M3}


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    assert a.dtype == b.dtype and a.shape == b.shape
    kind = {1: torch.int8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.contiguous().view(kind), b.contiguous().view(kind))


def same_numbers(a, b):
    """Equal, where the two zeros are one number and NaN equals NaN."""
    return torch.equal(torch.nan_to_num(a.cpu().float(), nan=1e30), torch.nan_to_num(b.cpu().float(), nan=1e30))


def random_codes(shape, dtype, g):
    x = torch.randint(-127, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)
    if dtype == E4M3:
        x = torch.where((x & 127) == 127, torch.zeros_like(x), x).view(E4M3)
    return x


def make_cache(pages, hk, page, blocks, d, dtype, g, layout="HND", spread=1.0):
    """(k_cache, v_cache, k_scale, v_scale) on the CPU, of random codes and scales that make numbers about 1."""
    shape = (pages, hk, page, d) if layout == "HND" else (pages, page, hk, d)
    codes = [random_codes(shape, dtype, g) for _ in range(2)]
    scales = [torch.exp2(spread * torch.randn(pages, hk, blocks, generator=g)) / (70 if dtype == INT8 else 30) for _ in range(2)]
    return (*codes, *scales)


def make_table(lens, page, pages, g):
    used = [-(-n // page) for n in lens]
    order = torch.randperm(pages, generator=g).to(torch.int32)
    assert sum(used) <= pages
    table = torch.zeros(len(lens), max(max(used), 1) + 1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    return table, order[at:]


def attend(q, cache, table, lens, dev, **kw):
    import flag_attn

    kc, vc, ks, vs = (x.to(dev) for x in cache)
    return flag_attn.paged_attention(q.to(dev), kc, vc, table.to(dev), torch.as_tensor(lens, dtype=torch.int32).to(dev),
                                     return_log_normalizer=True, k_scale=ks, v_scale=vs, **kw)


def check(q, cache, table, lens, dev, layout="HND", what="", **kw):
    o, norm = attend(q, cache, table, lens, dev, tensor_layout=layout, **kw)
    want, want_norm, tol, norm_tol = CO.paged(q, *cache, table, lens, layout=layout, **kw)
    CO.assert_close(norm.cpu(), want_norm, norm_tol, (what, "log normalizer"))
    CO.assert_close(o.cpu(), want, tol, (what, "output"))


# ---- attention

@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("h,hk,d", [(8, 2, 128), (4, 4, 64), (16, 1, 128), (20, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("page,blocks,layout", [(16, 1, "HND"), (16, 16, "NHD"), (32, 4, "HND"), (24, 3, "NHD"), (1, 1, "HND"), (48, 3, "HND"), (128, 1, "NHD")])
def test_attention(gpu_device, codes, dtype, h, hk, d, page, blocks, layout):
    g = torch.Generator().manual_seed(1)
    lens = [0, 1, 17, 33, 150, page, page + 1, 128, 129]
    pages = sum(-(-n // page) for n in lens) + 3
    cache = make_cache(pages, hk, page, blocks, d, CODES[codes], g, layout)
    table, free = make_table(lens, page, pages, g)
    for x in cache[2:]:  # what no sequence sees
        x[free.long()] = math.nan
    q = (2 * torch.randn(len(lens), h, d, generator=g)).to(dtype)
    check(q, cache, table, lens, gpu_device, layout)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("m,h,hk,d", [(2, 8, 2, 128), (4, 8, 2, 64), (7, 4, 4, 128), (9, 8, 2, 64), (5, 16, 1, 128), (33, 4, 2, 64)])
@pytest.mark.parametrize("page,blocks", [(16, 1), (32, 8), (24, 24)])
def test_several_new_tokens(gpu_device, codes, dtype, m, h, hk, d, page, blocks):
    """Rows that see different keys, sequences shorter than the new tokens."""
    g = torch.Generator().manual_seed(2)
    lens = [0, 1, m, m - 1, m + 1, 64, 100, 160]
    pages = sum(-(-n // page) for n in lens) + 2
    cache = make_cache(pages, hk, page, blocks, d, CODES[codes], g)
    table, _ = make_table(lens, page, pages, g)
    q = torch.randn(len(lens), m, h, d, generator=g).to(dtype)
    check(q, cache, table, lens, gpu_device)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("h,hk,d,m", [(8, 2, 128, 1), (2, 2, 64, 1), (8, 1, 64, 3)])
@pytest.mark.parametrize("lens,page", [([2500, 0, 3], 16), ([1, 5000], 64), ([900, 1000, 1100, 777, 40], 24), ([3500], 8)])
def test_cut_launches(gpu_device, codes, h, hk, d, m, lens, page):
    """Tables wide enough that the keys are shared out over the workgroups."""
    g = torch.Generator().manual_seed(3)
    pages = sum(-(-n // page) for n in lens) + 2
    cache = make_cache(pages, hk, page, 1, d, CODES[codes], g)
    table, _ = make_table(lens, page, pages, g)
    wide = torch.full((len(lens), max(table.shape[1], 20000 // page)), pages + 7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    q = torch.randn(len(lens), m, h, d, generator=g).to(BF16)
    check(q if m > 1 else q[:, 0], cache, wide, lens, gpu_device)


@pytest.mark.parametrize("seqs,hk,m,some", [(70, 8, 1, (0, 1, 5, 100, 300, 1500)), (32, 8, 1, (0, 0, 0, 3, 200, 1900)), (40, 4, 3, (0, 0, 129, 2000)), (65, 8, 1, (0,)), (40, 8, 2, (128, 256)),
                                            (16, 8, 1, (2000,)), (3, 8, 1, (1700, 1))])
def test_cut_launches_of_many_short_items(gpu_device, seqs, hk, m, some):
    """Shares that begin several items, empty ones among them, shares that end before an item's first chunk, more items than shares."""
    g = torch.Generator().manual_seed(12)
    lens = [some[i] for i in torch.randint(0, len(some), (seqs,), generator=g).tolist()]
    pages = sum(-(-n // 16) for n in lens) + 2
    cache = make_cache(pages, hk, 16, 16, 64, E4M3, g)
    table, _ = make_table(lens, 16, pages, g)
    wide = torch.zeros(seqs, 250, dtype=torch.int32)
    wide[:, :table.shape[1]] = table[:, :250]
    q = torch.randn(seqs, m, hk, 64, generator=g).to(BF16)
    check(q if m > 1 else q[:, 0], cache, wide, lens, gpu_device)


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("m", [1, 4])
def test_entries_that_are_no_page(gpu_device, page, m):
    g = torch.Generator().manual_seed(4)
    lens = [100, 200, 3 * page, 90]
    pages = sum(-(-n // page) for n in lens) + 2
    cache = make_cache(pages, 2, page, 2, 64, INT8, g)
    table, free = make_table(lens, page, pages, g)
    table[0, 1], table[1, 0], table[1, 3], table[3, -(-90 // page) - 1] = -1, pages, 1 << 30, -5
    table[2, :3] = -1  # a sequence without a page
    cache[2][0] = cache[2][0]
    q = torch.randn(4, m, 8, 64, generator=g).to(BF16)
    check(q if m > 1 else q[:, 0], cache, table, lens, gpu_device)
    check(q if m > 1 else q[:, 0], cache, table, [1 << 30, 77, 5, -3], gpu_device, what="lengths beyond the table")


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("qsize,kscale,vscale", [(1.0, 1.0, 2.0 ** -90), (2.0 ** -10, 2.0 ** 10, 2.0 ** 20), (100.0, 1.0, 1.0), (2.0 ** -12, 1.0, 2.0 ** 8), (1.0, 2.0 ** -60, 1.0)])
def test_sizes(gpu_device, dtype, qsize, kscale, vscale):
    """Queries and scales far from 1, heads of very different sizes in one group, scales of V that differ by 2^20."""
    if dtype == FP16 and vscale > 2.0 ** 10:
        vscale = 2.0 ** 6
    g = torch.Generator().manual_seed(5)
    lens, page = [70, 129, 40], 16
    kc, vc, ks, vs = make_cache(20, 2, page, 2, 64, INT8, g, spread=2.0)
    vs = vs * torch.exp2(torch.randint(-20, 1, vs.shape, generator=g).float())
    table, _ = make_table(lens, page, 20, g)
    q = qsize * torch.randn(3, 8, 64, generator=g)
    if dtype == BF16:
        q[:, ::2] *= 2.0 ** -30
        q[:, 3] *= 2.0 ** -120
    check(q.to(dtype), (kc, vc, ks * kscale, vs * vscale), table, lens, gpu_device)


def test_weights_far_below_the_largest_scale(gpu_device):
    """A value block 2^30 larger than the others, whose keys weigh nothing: the others keep their part."""
    g = torch.Generator().manual_seed(6)
    kc, vc, ks, vs = make_cache(8, 1, 16, 1, 64, INT8, g)
    vs[3] *= 2.0 ** 30
    kc[3] = -127
    q = torch.full((1, 4, 64), 3.0, dtype=BF16)
    table = torch.arange(8, dtype=torch.int32)[None]
    check(q, (kc, vc, ks, vs), table, [128], gpu_device)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_scales_that_are_not_finite(gpu_device, codes, page, bad):
    """They reach the rows that see a token of their block, and no other."""
    g = torch.Generator().manual_seed(7)
    lens, m = [64, 100, 50], 4
    pages = sum(-(-n // page) for n in lens) + 2
    for which in (2, 3):
        cache = make_cache(pages, 2, page, page, 64, CODES[codes], g)
        table, _ = make_table(lens, page, pages, g)
        q = torch.randn(3, m, 4, 64, generator=g).to(BF16)
        clean, clean_norm = attend(q, cache, table, lens, gpu_device)
        cache[which][int(table[0, 62 // page]), 1, 62 % page] = bad    # seen by the new tokens 2 and 3 of sequence 0
        cache[which][int(table[1, 10 // page]), 0, 10 % page] = bad    # seen by all of sequence 1
        cache[which][int(table[2, 49 // page]), 1, 49 % page] = bad    # seen by the last new token of sequence 2
        o, _ = attend(q, cache, table, lens, gpu_device)
        hit = torch.zeros(3, m, 4, dtype=torch.bool)
        hit[0, 2:, 2:] = hit[1, :, :2] = hit[2, 3:, 2:] = True
        o, clean = o.cpu(), clean.cpu()
        assert torch.equal(o[~hit], clean[~hit])
        if bad != bad:
            assert torch.isnan(o[hit]).all()
        elif which == 3:  # (codes are not zero: an infinity of either sign, or NaN of a zero code)
            assert not torch.isfinite(o[hit]).any()


def test_nan_codes_of_e4m3(gpu_device):
    """In K: rows that see the key are NaN.  In V: the channel is, in rows that see the key.  Elsewhere they change nothing."""
    g = torch.Generator().manual_seed(8)
    page, m, lens = 16, 3, [40, 61]
    cache = make_cache(9, 2, page, 1, 64, E4M3, g)
    table, free = make_table(lens, page, 9, g)
    for c in cache[:2]:
        c.view(torch.int8)[free.long()] = 127
        c.view(torch.int8)[int(table[0, 2]), :, 8:] = -1  # behind the last token
    q = torch.randn(2, m, 4, 64, generator=g).to(BF16)
    check(q, cache, table, lens, gpu_device)
    clean, _ = attend(q, cache, table, lens, gpu_device)
    cache[1].view(torch.int8)[int(table[0, 2]), 0, 7, 5] = 127   # token 39, the last: new token 2 sees it
    cache[1].view(torch.int8)[int(table[1, 0]), 1, 3, 60] = -1   # seen by all
    o, norm = attend(q, cache, table, lens, gpu_device)
    hit = torch.zeros(2, m, 4, 64, dtype=torch.bool)
    hit[0, 2, :2, 5] = hit[1, :, 2:, 60] = True
    assert torch.isnan(o.cpu()[hit]).all() and torch.equal(o.cpu()[~hit], clean.cpu()[~hit]) and torch.isfinite(norm).all()
    cache[0].view(torch.int8)[int(table[0, 2]), 0, 6, 0] = 127   # K of token 38: new tokens 1 and 2
    o, _ = attend(q, cache, table, lens, gpu_device)
    assert torch.isnan(o.cpu()[0, 1:, :2]).all() and torch.equal(o.cpu()[0, 0], clean.cpu()[0, 0])


def test_q_that_is_not_finite(gpu_device):
    """An infinity or NaN in a row of q stays in its row."""
    g = torch.Generator().manual_seed(9)
    cache = make_cache(9, 1, 16, 1, 64, INT8, g)
    table, _ = make_table([100], 16, 9, g)
    for dtype in (BF16, FP16):
        q = torch.randn(1, 6, 64, generator=g).to(dtype)
        clean, _ = attend(q, cache, table, [100], gpu_device)
        q[0, 1, 3], q[0, 4, 60] = math.inf, math.nan
        o, _ = attend(q, cache, table, [100], gpu_device)
        assert torch.equal(o[0, [0, 2, 3, 5]], clean[0, [0, 2, 3, 5]]) and torch.isnan(o[0, [1, 4]]).all()


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_strides(gpu_device, codes):
    """K and V interleaved in one tensor, scales too and in another order of dimensions, q and out as slices, a table with a stride."""
    import flag_attn

    g = torch.Generator().manual_seed(10)
    lens, page, pages, hk, d = [50, 129, 7], 16, 20, 2, 128
    cache = make_cache(pages, hk, page, 4, d, CODES[codes], g)
    table, _ = make_table(lens, page, pages, g)
    q = torch.randn(3, 8, d, generator=g).to(BF16)
    want, want_norm, tol, norm_tol = CO.paged(q, *cache, table, lens)
    dev = gpu_device
    both = torch.zeros(pages, 2, hk, page, d, dtype=torch.int8, device=dev)
    both[:, 0], both[:, 1] = cache[0].view(torch.int8).to(dev), cache[1].view(torch.int8).to(dev)
    both = both.view(CODES[codes])
    scales = torch.zeros(4, 3, pages, hk, device=dev)
    scales[:, 0], scales[:, 2] = cache[2].permute(2, 0, 1).to(dev), cache[3].permute(2, 0, 1).to(dev)
    wide_q = torch.zeros(3, 12, d, dtype=BF16, device=dev)
    wide_q[:, 2:10] = q.to(dev)
    wide_table = torch.zeros(table.shape[1], 3, dtype=torch.int32, device=dev)
    wide_table[:] = table.t()
    wide_out = torch.full((3, 12, d), 5.0, dtype=BF16, device=dev)
    o, norm = flag_attn.paged_attention(wide_q[:, 2:10], both[:, 0], both[:, 1], wide_table.t(), torch.tensor(lens, dtype=torch.int32, device=dev),
                                        return_log_normalizer=True, out=wide_out[:, 1:9], k_scale=scales[:, 0].permute(1, 2, 0), v_scale=scales[:, 2].permute(1, 2, 0))
    CO.assert_close(o.cpu(), want, tol, "output")
    CO.assert_close(norm.cpu(), want_norm, norm_tol, "log normalizer")
    assert (wide_out[:, 0] == 5).all() and (wide_out[:, 9:] == 5).all()


def test_expanded_scales(gpu_device):
    """One scale for all pages and heads (strides of zero) is read like any other."""
    g = torch.Generator().manual_seed(11)
    kc, vc, ks, vs = make_cache(12, 2, 16, 4, 64, E4M3, g)
    ks, vs = torch.full((1, 1, 1), 0.03).expand(12, 2, 4), torch.full((1, 1, 1), 0.02).expand(12, 2, 4)
    table, _ = make_table([100, 60], 16, 12, g)
    check(torch.randn(2, 4, 64, generator=g).to(FP16), (kc, vc, ks, vs), table, [100, 60], gpu_device)


# ---- writes

def write_case(pages, hk, page, blocks, d, codes, dtype, slots, g, layout="HND", x=None, spread=1.0):
    cache = make_cache(pages, hk, page, blocks, d, codes, g, layout)
    if x is None:
        x = [torch.randn(len(slots), hk, d, generator=g) * torch.exp2(spread * torch.randn(len(slots), hk, 1, generator=g)) for _ in range(2)]
    return [t.to(dtype) for t in x], cache, torch.as_tensor(slots)


def check_write(x, cache, slots, dev, layout="HND", what=""):
    import flag_attn

    kc, vc, ks, vs = (t.to(dev) for t in cache)
    versions = [t._version for t in (kc, vc, ks, vs)]
    flag_attn.append_to_cache(x[0].to(dev), x[1].to(dev), kc, vc, slots.to(dev), tensor_layout=layout, k_scale=ks, v_scale=vs)
    assert all(t._version > n for t, n in zip((kc, vc, ks, vs), versions))
    want = CO.append(x[0], x[1], cache[0], cache[1], slots, cache[2], cache[3], layout)
    for got, w, name in zip((ks, vs), want[2:], ("k_scale", "v_scale")):
        assert same_numbers(got, w), (what, name)
    for got, w, name in zip((kc, vc), want[:2], ("k_cache", "v_cache")):
        assert same_numbers(got, w), (what, name, int((got.cpu().float() != w.float()).sum()))
    return kc, vc, ks, vs


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hk,d", [(2, 128), (3, 64), (1, 16), (2, 48), (1, 80), (1, 256), (1, 512)])
@pytest.mark.parametrize("page,blocks,layout", [(16, 16, "HND"), (16, 1, "NHD"), (24, 3, "HND"), (1, 1, "NHD"), (64, 1, "HND")])
def test_write_in_any_order(gpu_device, codes, dtype, hk, d, page, blocks, layout):
    """Half of the slots of a cache in random order, some that it does not have."""
    g = torch.Generator().manual_seed(20)
    pages = max(3, 96 // page)
    slots = torch.randperm(pages * page, generator=g)[: pages * page // 2]
    slots[::7] = -1 - slots[::7]
    slots[3] = pages * page
    check_write(*write_case(pages, hk, page, blocks, d, CODES[codes], dtype, slots, g, layout), gpu_device, layout)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("tokens", [1, 1023, 1025, 1500])
@pytest.mark.parametrize("page,blocks,at", [(16, 1, 0), (16, 4, 5), (32, 32, 3), (256, 1, 100), (24, 2, 0)])
def test_write_prompts(gpu_device, codes, tokens, page, blocks, at):
    """Tokens that fill pages in order, from the first place or further in: few that look each other up, many through the map."""
    g = torch.Generator().manual_seed(21)
    need = -(-(at + tokens) // page)
    where = torch.randperm(need + 2, generator=g)[:need]
    t = at + torch.arange(tokens)
    slots = torch.cat([where[t // page] * page + t % page, torch.full((3,), -1)]).to(torch.int32)
    check_write(*write_case(need + 2, 1, page, blocks, 64, CODES[codes], BF16, slots, g), gpu_device)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_write_many_in_any_order(gpu_device, codes):
    """More tokens than look each other up, in random order and reversed."""
    g = torch.Generator().manual_seed(22)
    for slots in (torch.randperm(3000, generator=g)[:1800], torch.arange(2999, 1199, -1)):
        check_write(*write_case(125, 1, 24, 3, 32, CODES[codes], FP16, slots, g), gpu_device)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_token_by_token(gpu_device, codes):
    """A page filled by single tokens, larger and larger ones among them: the scale grows, what it holds is converted."""
    import flag_attn

    g = torch.Generator().manual_seed(23)
    cache = make_cache(3, 2, 16, 2, 64, CODES[codes], g)
    dev = gpu_device
    now = [t.to(dev) for t in cache]
    want = cache
    for i in range(16):
        x = [torch.randn(2, 2, 64, generator=g) * 2.0 ** (i % 5) for _ in range(2)]
        slots = torch.tensor([16 + i, i])
        flag_attn.append_to_cache(x[0].to(dev), x[1].to(dev), now[0], now[1], slots.to(dev), k_scale=now[2], v_scale=now[3])
        want = CO.append(x[0], x[1], want[0], want[1], slots, want[2], want[3])
        for a, b in zip(now, want):
            assert same_numbers(a, b), i


@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32], ids=["bf16", "fp16", "fp32"])
def test_ties(gpu_device, dtype):
    """Quotients on the middle between two codes, and as close to it as the type allows, go to the even one and to their side."""
    for codes, top, pages in ((INT8, 127.0, 4), (E4M3, 448.0, 4)):
        grid = torch.arange(0, 128).double() if codes == INT8 else CO.e4m3_numbers()
        middles = (grid[:-1] + grid[1:]) / 2
        x = torch.cat([middles, -middles, grid, torch.tensor([top] * 3, dtype=torch.float64)])
        x = torch.cat([x, torch.zeros(-len(x) % 64, dtype=torch.float64)]).view(-1, 1, 64)
        for shift in (0, -20 if dtype != FP16 else -4, 3 if dtype != FP16 else 2):
            rows = (x * 2.0 ** shift).to(dtype)
            kind = torch.int32 if dtype == torch.float32 else torch.int16
            ups = [(rows.view(kind) + e).view(dtype) for e in (0, 1, -1)]  # the next numbers of the type
            for i, r in enumerate(ups):
                r = torch.where(torch.isfinite(r) & (r.float().abs() <= top * 2.0 ** shift), r, torch.zeros((), dtype=dtype))
                r[:, 0, 0] = top * 2.0 ** shift  # the scale is a power of two
                n = r.shape[0]
                cache = (torch.zeros(pages, 1, 8, 64, dtype=torch.int8).view(codes), torch.zeros(pages, 1, 8, 64, dtype=torch.int8).view(codes),
                         torch.zeros(pages, 1, 1), torch.zeros(pages, 1, 1))
                assert n <= 8 * pages
                check_write([r, -r], cache, torch.arange(n), gpu_device, what=(codes, shift, i))


def test_near_ties_with_uneven_scales(gpu_device):
    """fp32 rows of the numbers next to (n + 1/2) s for scales of all mantissas."""
    g = torch.Generator().manual_seed(24)
    for codes, top in ((INT8, 127.0), (E4M3, 448.0)):
        grid = torch.arange(0, 127).double() if codes == INT8 else CO.e4m3_numbers()
        middles = (grid[:-1] + grid[1:]) / 2
        amax = torch.rand(96, generator=g) + 1
        s = (amax.double() / top).float().double()
        x = (middles[torch.randint(0, len(middles), (96, 64), generator=g)] * s[:, None]).float()
        x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=g, dtype=torch.int32)).view(torch.float32)
        x = torch.where(x.abs() < amax[:, None], x, torch.zeros(()))
        x[:, 0] = amax
        for blocks in (16, 1):
            rows = x[:, None] if blocks == 16 else torch.where(torch.arange(96)[:, None] % 16 == 0, x, x.clamp(max=amax.view(6, 16)[:, :1].repeat(1, 16).view(96, 1)))[:, None]
            cache = (torch.zeros(6, 1, 16, 64, dtype=torch.int8).view(codes), torch.zeros(6, 1, 16, 64, dtype=torch.int8).view(codes), torch.zeros(6, 1, blocks), torch.zeros(6, 1, blocks))
            check_write([rows, -rows], cache, torch.arange(96), gpu_device)


def test_rows_of_zeros_infinities_and_nan(gpu_device):
    """Zeros get the smallest scale; an infinity or NaN makes the block's scale NaN until it begins anew; tiny numbers keep their codes."""
    import flag_attn

    dev = gpu_device
    for codes, top in ((INT8, 127.0), (E4M3, 448.0)):
        for blocks in (16, 1):
            x = torch.randn(16, 1, 64, generator=torch.Generator().manual_seed(25))
            x[1] = 0
            x[2, 0, 3], x[3, 0, 4], x[4, 0, 0] = math.inf, math.nan, -math.inf
            x[5] = 2.0 ** -120
            x[6] = 3e38
            cache = (torch.zeros(3, 1, 16, 64, dtype=torch.int8).view(codes), torch.zeros(3, 1, 16, 64, dtype=torch.int8).view(codes), torch.zeros(3, 1, blocks), torch.zeros(3, 1, blocks))
            for keep in ([0, 1, 2, 3, 4, 5, 6], [1, 5], [0, 6], [5]):
                rows = x[keep].bfloat16()
                kc, vc, ks, vs = check_write([rows, -rows], cache, 16 + torch.tensor(keep), dev)
            assert float(ks[1, 0, 5 if blocks == 16 else 0]) == float(torch.tensor(2.0 ** -100 / top, dtype=torch.float64).float())
    # NaN stays where the block goes on, and goes where it begins anew
    cache = [t.to(dev) for t in (torch.zeros(1, 1, 16, 64, dtype=INT8), torch.zeros(1, 1, 16, 64, dtype=INT8), torch.full((1, 1, 1), math.nan), torch.full((1, 1, 1), 0.5))]
    row = torch.ones(1, 1, 64, dtype=BF16, device=dev)
    for slot, nan in ((3, True), (0, False), (4, False)):
        flag_attn.append_to_cache(row, row, cache[0], cache[1], torch.tensor([slot], device=dev), k_scale=cache[2], v_scale=cache[3])
        assert bool(torch.isnan(cache[2]).all()) == nan and float(cache[3]) == (0.5 if slot == 3 else float(torch.tensor(1 / 127)))


def test_write_strides(gpu_device):
    """k and v as slices of a projection, unaligned ones, caches and scales interleaved; nothing else is touched."""
    import flag_attn

    g = torch.Generator().manual_seed(26)
    dev, pages, hk, page, d = gpu_device, 5, 2, 16, 64
    slots = torch.randperm(pages * page, generator=g)[:40]
    for blocks in (16, 4):
        x, cache, _ = write_case(pages, hk, page, blocks, d, INT8, BF16, slots, g)
        want = CO.append(x[0], x[1], cache[0], cache[1], slots, cache[2], cache[3])
        both = torch.full((pages, 3, hk, page, d), 99, dtype=INT8, device=dev)
        both[:, 0], both[:, 1] = cache[0].to(dev), cache[1].to(dev)
        scales = torch.full((pages, 2, blocks, hk), 7.0, device=dev)
        scales[:, 0], scales[:, 1] = cache[2].transpose(1, 2).to(dev), cache[3].transpose(1, 2).to(dev)
        qkv = torch.zeros(40, 3 * hk, d, dtype=BF16, device=dev)
        qkv[:, :hk], qkv[:, 2 * hk:] = x[0].to(dev), x[1].to(dev)
        odd = torch.zeros(40, hk, d + 1, dtype=BF16, device=dev)
        odd[..., 1:] = x[1].to(dev)
        for k, v in ((qkv[:, :hk], qkv[:, 2 * hk:]), (qkv[:, :hk], odd[..., 1:])):
            flag_attn.append_to_cache(k, v, both[:, 0], both[:, 1], slots.to(dev), k_scale=scales[:, 0].transpose(1, 2), v_scale=scales[:, 1].transpose(1, 2))
            got = (both[:, 0], both[:, 1], scales[:, 0].transpose(1, 2), scales[:, 1].transpose(1, 2))
            for a, b in zip(got, want):
                assert same_numbers(a, b)
            assert (both[:, 2] == 99).all()


# ---- reads and copies

@pytest.mark.parametrize("codes", ["int8", "e4m3", None])
@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("page,blocks,layout,d", [(16, 1, "HND", 64), (24, 8, "NHD", 128), (1, 1, "HND", 64), (64, 64, "NHD", 16), (5, 1, "HND", 48)])
def test_read(gpu_device, codes, dtype, page, blocks, layout, d):
    import flag_attn

    g = torch.Generator().manual_seed(30)
    lens = [0, 37, 1, 0, 0, 64, 5, 100, 0]
    pages = sum(-(-n // page) for n in lens) + 2
    if codes is None:
        shape = (pages, 2, page, d) if layout == "HND" else (pages, page, 2, d)
        cache = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)] + [None, None]
    else:
        cache = make_cache(pages, 2, page, blocks, d, CODES[codes], g, layout)
    table, _ = make_table(lens, page, pages, g)
    table[1, 36 // page] = -1
    table[7, 0] = pages
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    total = int(cu[-1]) + 5
    dev = gpu_device
    kc, vc, ks, vs = (t.to(dev) if t is not None else None for t in cache)
    out = [torch.full((total, 2, d), 7.0, dtype=dtype, device=dev) for _ in range(2)]
    for res in (flag_attn.read_cache(kc, vc, table.to(dev), cu.to(dev), total, tensor_layout=layout, dtype=dtype, out=out, k_scale=ks, v_scale=vs),
                flag_attn.read_cache(kc, vc, table.to(dev), cu.to(dev), total, tensor_layout=layout, dtype=dtype, k_scale=ks, v_scale=vs),
                flag_attn.read_cache(kc, vc, table.to(dev), cu.to(dev), total, tensor_layout=layout, dtype=dtype, k_scale=ks, v_scale=vs)):
        for got, c, s in zip(res, cache[:2], cache[2:]):
            want = CO.read(c, s, table, cu, total, dtype, layout)
            assert same_numbers(got[: total - 5], want[: total - 5])
    assert all((t[total - 5:] == 7).all() for t in out)
    # lengths beyond the table are rows of zeros, also of a table without entries
    for wide in (table[:, :1], table[:, :0]):
        res = flag_attn.read_cache(kc, vc, wide.to(dev), cu.to(dev), total, tensor_layout=layout, dtype=dtype, k_scale=ks, v_scale=vs)
        for got, c, s in zip(res, cache[:2], cache[2:]):
            assert same_numbers(got[: total - 5], CO.read(c, s, wide, cu, total, dtype, layout)[: total - 5])


@pytest.mark.parametrize("layers", [0, 3])
@pytest.mark.parametrize("hk,page,blocks,d", [(2, 16, 16, 64), (1, 16, 1, 128), (3, 24, 3, 48), (8, 128, 128, 128)])
def test_copies(gpu_device, layers, hk, page, blocks, d):
    import flag_attn

    g = torch.Generator().manual_seed(31)
    pages, dev = 11, gpu_device
    kc, vc, ks, vs = (t.to(dev) for t in make_cache(pages * max(layers, 1), hk, page, blocks, d, INT8, g))
    if layers:
        kc, vc, ks, vs = (t.view(layers, pages, *t.shape[1:]) for t in (kc, vc, ks, vs))
    src, dst = torch.tensor([0, 3, 0, -1, 5, 99]), torch.tensor([7, 8, 9, 10, pages, 1])
    want = [t.clone() for t in (kc, vc, ks, vs)]
    for a, b in ((0, 7), (3, 8), (0, 9)):
        for t in want:
            if layers:
                t[:, b] = t[:, a]
            else:
                t[b] = t[a]
    versions = [t._version for t in (kc, vc, ks, vs)]
    flag_attn.copy_pages(kc, vc, src.to(dev), dst.to(dev), k_scale=ks, v_scale=vs)
    assert all(torch.equal(a, b) for a, b in zip((kc, vc, ks, vs), want))
    assert all(t._version > n for t, n in zip((kc, vc, ks, vs), versions))


# ---- as a program uses them

@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_prompt_chunks_steps_and_a_fork(gpu_device, codes):
    """A prompt in two chunks (write, read back, packed attention), steps of decoding, a fork that goes its own way: every
    result against the formulas over a cache that the oracle wrote."""
    import flag_attn
    from oracle import serving_oracle as SO

    g = torch.Generator().manual_seed(40)
    dev, h, hk, d, page, blocks, pages = gpu_device, 4, 2, 64, 16, 2, 12
    kinds = CODES[codes]
    cache = (torch.zeros(pages, hk, page, d, dtype=torch.int8).view(kinds), torch.zeros(pages, hk, page, d, dtype=torch.int8).view(kinds),
             torch.zeros(pages, hk, blocks), torch.zeros(pages, hk, blocks))
    own = [t.to(dev) for t in cache]
    scales = dict(k_scale=own[2], v_scale=own[3])
    table = torch.tensor([[4, 2, 9, 0], [7, 1, 3, 0]], dtype=torch.int32)
    lens = [0, 0]

    def rows(*n):
        return [torch.randn(*n, hk, d, generator=g).to(BF16) for _ in range(2)]

    def slots_of(counts):
        return torch.tensor([int(table[s, p // page]) * page + p % page for s, n in enumerate(counts) for p in range(lens[s], lens[s] + n)])

    for counts in ((21, 9), (5, 13)):  # chunks
        k, v = rows(sum(counts))
        slots = slots_of(counts)
        cache = CO.append(k, v, cache[0], cache[1], slots, cache[2], cache[3])
        flag_attn.append_to_cache(k.to(dev), v.to(dev), own[0], own[1], slots.to(dev), **scales)
        lens = [a + b for a, b in zip(lens, counts)]
        cu_q, cu_k = (torch.tensor([0, x[0], x[0] + x[1]], dtype=torch.int32) for x in (counts, lens))
        kk, vv = flag_attn.read_cache(own[0], own[1], table.to(dev), cu_k.to(dev), sum(lens), **scales)
        want_k, want_v = (CO.read(c, s, table, cu_k, sum(lens), BF16) for c, s in zip(cache[:2], cache[2:]))
        assert same_numbers(kk, want_k) and same_numbers(vv, want_v)
        q = torch.randn(sum(counts), h, d, generator=g).to(BF16)
        o = flag_attn.flash_attention_varlen(q.to(dev), kk, vv, cu_q.to(dev), cu_k.to(dev), causal=True)
        want, _, tol, _ = SO.varlen(q, want_k, want_v, cu_q, cu_k, True)
        SO.assert_close(o.cpu(), want, tol, "chunk")
    # sequence 1 becomes a copy of sequence 0: full pages are shared, the last one is copied
    src, dst = table[0, lens[0] // page].view(1), torch.tensor([6], dtype=torch.int32)
    flag_attn.copy_pages(own[0], own[1], src.to(dev), dst.to(dev), **scales)
    cache = tuple(t.clone() for t in cache)
    for t in cache:
        t.view(torch.int8 if t.element_size() == 1 else torch.int32)[6] = t.view(torch.int8 if t.element_size() == 1 else torch.int32)[int(src)]
    table[1] = table[0]
    table[1, lens[0] // page] = 6
    table[1, 2] = 5
    lens[1] = lens[0]
    for step in range(9):
        k, v = rows(2)
        slots = slots_of((1, 1))
        cache = CO.append(k, v, cache[0], cache[1], slots, cache[2], cache[3])
        flag_attn.append_to_cache(k.to(dev), v.to(dev), own[0], own[1], slots.to(dev), **scales)
        lens = [n + 1 for n in lens]
        q = torch.randn(2, h, d, generator=g).to(BF16)
        o, norm = flag_attn.paged_attention(q.to(dev), own[0], own[1], table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), return_log_normalizer=True, **scales)
        want, want_norm, tol, norm_tol = CO.paged(q, *cache, table, lens)
        CO.assert_close(o.cpu(), want, tol, step)
        CO.assert_close(norm.cpu(), want_norm, norm_tol, step)
    for a, b in zip(own, cache):
        assert same_numbers(a, b)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_a_captured_step(gpu_device, codes):
    """A step (write, attention) in a graph: replays follow the slots, lengths and rows that lie in its buffers, with eager work between; a
    second graph of the same caches and other buffers in turn with it."""
    import flag_attn

    g = torch.Generator().manual_seed(41)
    dev, page, pages = gpu_device, 16, 40
    cache = make_cache(pages, 2, page, 1, 64, CODES[codes], g)
    lens = [100, 37, 1, 250]
    table, _ = make_table([n + 20 for n in lens], page, pages, g)
    now = [t.to(dev) for t in cache]
    wide = torch.zeros(4, 1250, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    wide_dev = wide.to(dev)
    scales = dict(k_scale=now[2], v_scale=now[3])
    graphs = []
    for _ in range(2):
        b = dict(q=torch.zeros(4, 4, 64, dtype=BF16, device=dev), k=torch.zeros(4, 2, 64, dtype=BF16, device=dev), v=torch.zeros(4, 2, 64, dtype=BF16, device=dev),
                 slots=torch.full((4,), -1, device=dev), lens=torch.zeros(4, dtype=torch.int32, device=dev))

        def step(b=b):
            flag_attn.append_to_cache(b["k"], b["v"], now[0], now[1], b["slots"], **scales)
            return flag_attn.paged_attention(b["q"], now[0], now[1], wide_dev, b["lens"], **scales)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = step()
        graphs.append((graph, b, o))
    for i in range(6):
        graph, b, o = graphs[i % 2]
        lens = [n + 1 for n in lens]
        k, v = (torch.randn(4, 2, 64, generator=g).to(BF16) for _ in range(2))
        q = torch.randn(4, 4, 64, generator=g).to(BF16)
        slots = torch.tensor([int(table[s, (n - 1) // page]) * page + (n - 1) % page for s, n in enumerate(lens)])
        cache = CO.append(k, v, cache[0], cache[1], slots, cache[2], cache[3])
        for name, x in (("q", q), ("k", k), ("v", v), ("slots", slots), ("lens", torch.tensor(lens, dtype=torch.int32))):
            b[name].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want, _, tol, _ = CO.paged(q, *cache, table, lens)
        CO.assert_close(o.cpu(), want, tol, i)
        for a, c in zip(now, cache):
            assert same_numbers(a, c), i
        torch.randn(1000, 1000, device=dev).sum().item()


def test_another_stream_and_repeated_calls(gpu_device):
    """The same calls from the Python side, from the native host side and on another stream give the same bits."""
    import flag_attn

    g = torch.Generator().manual_seed(42)
    dev = gpu_device
    lens, page, pages = [700, 33], 16, 60
    cache = [t.to(dev) for t in make_cache(pages, 2, page, 4, 128, INT8, g)]
    table, _ = make_table(lens, page, pages, g)
    wide = torch.zeros(2, 1300, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table.to(dev)
    q = torch.randn(2, 8, 128, generator=g).to(BF16).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    scales = dict(k_scale=cache[2], v_scale=cache[3])
    cu = torch.tensor([0, 700, 733], dtype=torch.int32, device=dev)
    first = flag_attn.paged_attention(q, cache[0], cache[1], wide, n, **scales)
    first_read = flag_attn.read_cache(cache[0], cache[1], wide, cu, 733, **scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        assert same_bits(first, flag_attn.paged_attention(q, cache[0], cache[1], wide, n, **scales))
        assert all(same_bits(a, b) for a, b in zip(first_read, flag_attn.read_cache(cache[0], cache[1], wide, cu, 733, **scales)))
        with torch.cuda.stream(side):
            again = flag_attn.paged_attention(q, cache[0], cache[1], wide, n, **scales)
        side.synchronize()
        assert same_bits(first, again)


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
def test_offsets_beyond_32_bits(gpu_device, codes):
    """Caches of more than 2^32 bytes: the last pages and the first ones, in every operator."""
    import flag_attn

    g = torch.Generator().manual_seed(43)
    dev, hk, page, d, pages = gpu_device, 8, 16, 128, (1 << 32) // (8 * 16 * 128) + 40
    kc, vc = (torch.empty(pages, hk, page, d, dtype=torch.int8, device=dev).view(CODES[codes]) for _ in range(2))
    ks, vs = (torch.zeros(pages, hk, 4, device=dev) for _ in range(2))
    scales = dict(k_scale=ks, v_scale=vs)
    places = [pages - 1, 0, pages - 20, 1]
    small = (torch.zeros(5, hk, page, d, dtype=torch.int8).view(CODES[codes]), torch.zeros(5, hk, page, d, dtype=torch.int8).view(CODES[codes]), torch.zeros(5, hk, 4), torch.zeros(5, hk, 4))
    k, v = (torch.randn(64, hk, d, generator=g).to(BF16) for _ in range(2))
    here = torch.arange(64)
    slots = torch.tensor(places).repeat_interleave(page) * page + here % page
    flag_attn.append_to_cache(k.to(dev), v.to(dev), kc, vc, slots.to(dev), **scales)
    small = CO.append(k, v, small[0], small[1], here, small[2], small[3])
    flag_attn.copy_pages(kc, vc, torch.tensor([pages - 20], device=dev), torch.tensor([pages - 3], device=dev), **scales)
    places[2] = pages - 3
    for t, w in zip((kc, vc, ks, vs), small):
        kind = torch.int8 if t.element_size() == 1 else torch.float32
        assert same_numbers(t.view(kind)[torch.tensor(places, device=dev)].view(t.dtype), w[:4])
    table, cu = torch.tensor([places], dtype=torch.int32), torch.tensor([0, 64], dtype=torch.int32)
    for got, c, s in zip(flag_attn.read_cache(kc, vc, table.to(dev), cu.to(dev), 64, **scales), small[:2], small[2:]):
        assert same_numbers(got, CO.read(c, s, torch.arange(4)[None], cu, 64, BF16))
    q = torch.randn(1, 16, d, generator=g).to(BF16)
    o = flag_attn.paged_attention(q.to(dev), kc, vc, table.to(dev), torch.tensor([64], dtype=torch.int32, device=dev), **scales)
    want, _, tol, _ = CO.paged(q, *small, torch.arange(4)[None], [64])
    CO.assert_close(o.cpu(), want, tol)


@pytest.mark.parametrize("tokens", [40, 600])
@pytest.mark.parametrize("blocks", [16, 4, 1])
def test_a_slot_that_occurs_twice(gpu_device, tokens, blocks):
    """Not allowed; all the same every other block is right, and the place holds a row of one of the two."""
    import flag_attn

    g = torch.Generator().manual_seed(44)
    dev, pages = gpu_device, tokens // 16 + 2
    slots = torch.arange(tokens)
    slots[17] = 3
    x, cache, _ = write_case(pages, 2, 16, blocks, 64, INT8, BF16, slots, g)
    kc, vc, ks, vs = (t.to(dev) for t in cache)
    flag_attn.append_to_cache(x[0].to(dev), x[1].to(dev), kc, vc, slots.to(dev), k_scale=ks, v_scale=vs)
    wants = []
    for lost in (3, 17):
        s = slots.clone()
        s[lost] = -1
        wants.append(CO.append(x[0], x[1], cache[0], cache[1], s, cache[2], cache[3]))
    for got, a, b in zip((kc, vc, ks, vs), *wants):
        assert same_numbers(got[1:], a[1:])
        if blocks != 16:
            assert same_numbers(got, a) or same_numbers(got, b)


def test_negative_scales(gpu_device):
    """Scales that a program wrote itself, of either sign and far apart, count as they are."""
    g = torch.Generator().manual_seed(45)
    kc, vc, ks, vs = make_cache(10, 2, 16, 4, 64, INT8, g)
    ks, vs = -ks, vs * torch.where(torch.rand(vs.shape, generator=g) < 0.5, -1.0, 1000.0)
    table, _ = make_table([90, 33], 16, 10, g)
    for dtype in (BF16, FP16):
        check(torch.randn(2, 4, 64, generator=g).to(dtype), (kc, vc, ks, vs), table, [90, 33], gpu_device)


def test_caches_and_lists_without_entries(gpu_device):
    """No pages, no entries of a table, no tokens, no sequences: zero rows, or nothing to do."""
    import flag_attn

    dev = gpu_device

    def cache(pages):
        return [torch.zeros(pages, 2, 16, 64, dtype=INT8, device=dev) for _ in range(2)], dict(k_scale=torch.zeros(pages, 2, 4, device=dev), v_scale=torch.zeros(pages, 2, 4, device=dev))

    q = torch.ones(3, 4, 64, dtype=BF16, device=dev)
    lens = torch.tensor([5, 0, 1], dtype=torch.int32, device=dev)
    for pages, width in ((0, 2), (4, 0), (0, 0)):
        c, s = cache(pages)
        table = torch.zeros(3, width, dtype=torch.int32, device=dev)
        o, norm = flag_attn.paged_attention(q, *c, table, lens, return_log_normalizer=True, **s)
        assert not o.any() and (norm == -math.inf).all()
        k, v = flag_attn.read_cache(*c, table, torch.tensor([0, 5, 5, 6], dtype=torch.int32, device=dev), 6, **s)
        assert k.shape == (6, 2, 64) and not k.any() and not v.any()
    c, s = cache(4)
    row = torch.ones(0, 2, 64, dtype=BF16, device=dev)
    flag_attn.append_to_cache(row, row, *c, torch.zeros(0, dtype=torch.int64, device=dev), **s)
    flag_attn.copy_pages(*c, torch.zeros(0, dtype=torch.int64, device=dev), torch.zeros(0, dtype=torch.int64, device=dev), **s)
    k, v = flag_attn.read_cache(*c, torch.zeros(0, 3, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), 0, **s)
    assert k.shape == (0, 2, 64)
    assert flag_attn.paged_attention(q[:0], *c, torch.zeros(0, 3, dtype=torch.int32, device=dev), lens[:0], **s).shape == (0, 4, 64)


def _prompt_state(codes, g, dev, tokens=700, blocks=2, page=16, hk=2, d=64):
    """A cache, tokens for it in an order of their own, and what an eager program needs to attend over it."""
    pages = tokens // page + 3
    cache = make_cache(pages, hk, page, blocks, d, codes, g)
    now = [t.to(dev) for t in cache]
    b = dict(k=torch.zeros(tokens, hk, d, dtype=BF16, device=dev), v=torch.zeros(tokens, hk, d, dtype=BF16, device=dev), slots=torch.full((tokens,), -1, device=dev),
             q=torch.randn(1, 8, d, generator=g).to(BF16).to(dev), table=torch.zeros(1, 2000, dtype=torch.int32, device=dev), lens=torch.tensor([tokens], dtype=torch.int32, device=dev),
             cu=torch.tensor([0, tokens], dtype=torch.int32, device=dev))
    b["table"][0, :pages] = torch.arange(pages, device=dev)
    return cache, now, b


def _prompt_pass(now, b):
    import flag_attn

    scales = dict(k_scale=now[2], v_scale=now[3])
    flag_attn.append_to_cache(b["k"], b["v"], now[0], now[1], b["slots"], **scales)
    o = flag_attn.paged_attention(b["q"], now[0], now[1], b["table"], b["lens"], **scales)
    return (o, *flag_attn.read_cache(now[0], now[1], b["table"], b["cu"], b["k"].shape[0], **scales))


def test_two_captured_prompts_at_once(gpu_device):
    """Writes through the map, cut attention and reads in two graphs, each with caches of its own, replayed at once on two streams with other
    tokens and slots each time: no workspace is shared."""
    g = torch.Generator().manual_seed(46)
    dev = gpu_device
    sides = []
    for codes in (INT8, E4M3):
        cache, now, b = _prompt_state(codes, g, dev)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _prompt_pass(now, b)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _prompt_pass(now, b)
        sides.append([cache, now, b, stream, graph, out])
    for i in range(4):
        for side in sides:
            cache, b = side[0], side[2]
            slots = torch.randperm(cache[0].shape[0] * 16, generator=g)[:700]
            slots[::9] = -1
            k, v = (torch.randn(700, 2, 64, generator=g).to(BF16) * 2.0 ** (i - 1) for _ in range(2))
            for name, x in (("k", k), ("v", v), ("slots", slots)):
                b[name].copy_(x)
            side[0] = CO.append(k, v, cache[0], cache[1], slots, cache[2], cache[3])
        torch.cuda.synchronize()
        for side in sides:
            with torch.cuda.stream(side[3]):
                for _ in range(3):  # (a write twice is a write once)
                    side[4].replay()
        torch.cuda.synchronize()
        for cache, now, b, _, _, (o, k, v) in sides:
            assert all(same_numbers(x, y) for x, y in zip(now, cache)), i
            want, _, tol, _ = CO.paged(b["q"].cpu(), *cache, b["table"].cpu(), [700])
            CO.assert_close(o.cpu(), want, tol, i)
            for got, c, s in zip((k, v), cache[:2], cache[2:]):
                assert same_numbers(got, CO.read(c, s, b["table"].cpu(), torch.tensor([0, 700]), 700, BF16))
        torch.randn(500, 500, device=dev).sum().item()


def test_two_threads_at_once(gpu_device):
    """Each with a stream and caches of its own; the first calls of a shape and the known ones."""
    import threading

    dev = gpu_device
    failed = []

    def work(seed):
        try:
            g = torch.Generator().manual_seed(seed)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                cache, now, b = _prompt_state(INT8, g, dev, tokens=300 + seed)
                for _ in range(4):
                    slots = torch.randperm(cache[0].shape[0] * 16, generator=g)[:300 + seed]
                    k, v = (torch.randn(300 + seed, 2, 64, generator=g).to(BF16) for _ in range(2))
                    for name, x in (("k", k), ("v", v), ("slots", slots)):
                        b[name].copy_(x)
                    cache = CO.append(k, v, cache[0], cache[1], slots, cache[2], cache[3])
                    o, *_ = _prompt_pass(now, b)
                    stream.synchronize()
                    assert all(same_numbers(x, y) for x, y in zip(now, cache))
                    want, _, tol, _ = CO.paged(b["q"].cpu(), *cache, b["table"].cpu(), [300 + seed])
                    CO.assert_close(o.cpu(), want, tol)
        except Exception as e:  # (an assertion of a thread would be lost)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]
