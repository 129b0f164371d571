"""The serving operators on the GPU against their formulas in 64 bits (oracle/serving_oracle.py, which also derives how far
off a result may be): packed sequences, paged caches, cache writes, page copies, and a run of them together."""
import pytest
import torch

from oracle import serving_oracle as SO

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _cu(lengths, device):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(device)


def _randn(shape, dtype, device, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def _check_varlen(q, k, v, cu_q, cu_k, causal, sm_scale=None):
    import flag_attn

    o, norm = flag_attn.flash_attention_varlen(q, k, v, cu_q, cu_k, causal, sm_scale, return_log_normalizer=True)
    want, want_norm, o_tol, norm_tol = SO.varlen(q, k, v, cu_q, cu_k, causal, sm_scale)
    n = int(cu_q[-1])
    SO.assert_close(o[:n], want[:n], o_tol[:n], "o")
    SO.assert_close(norm[:, :n], want_norm[:, :n], norm_tol[:, :n], "log normalizer")
    alone = flag_attn.flash_attention_varlen(q, k, v, cu_q, cu_k, causal, sm_scale)
    SO.assert_close(alone[:n], want[:n], o_tol[:n], "o without log normalizer")
    return o


LENGTHS = [(1,), (77,), (0, 5, 0, 2), (31, 32, 33, 64, 65), (127, 128, 129, 1), (300, 1, 511), (1500, 40)]
HEADS = [(4, 4), (8, 2), (7, 1), (6, 2)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lengths", LENGTHS)
def test_varlen_lengths(lengths, heads, d, dtype, gpu_device):
    (h, hk), t, dt = heads, sum(lengths), DTYPES[dtype]
    q, k, v = (_randn((t, n, d), dt, gpu_device, i) for i, n in enumerate((h, hk, hk)))
    cu = _cu(lengths, gpu_device)
    for causal in (False, True):
        _check_varlen(q, k, v, cu, cu, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m,n", [((3, 70, 1), (200, 70, 1000)), ((5, 100, 40), (0, 33, 7)), ((64, 0, 9), (1, 50, 8)), ((130,), (1029,))])
def test_varlen_more_or_fewer_keys_than_queries(m, n, d, gpu_device):
    """Chunks of longer prompts; queries that see no key (zero rows, log normalizer -inf)."""
    q = _randn((sum(m), 8, d), torch.bfloat16, gpu_device, 0)
    k, v = (_randn((sum(n), 2, d), torch.bfloat16, gpu_device, i) for i in (1, 2))
    for causal in (False, True):
        _check_varlen(q, k, v, _cu(m, gpu_device), _cu(n, gpu_device), causal)


@pytest.mark.parametrize("h,hk", [(160, 1), (258, 2)])
def test_more_rows_per_token_than_a_block_holds(h, hk, gpu_device):
    """So many query heads for one K/V head that a block, or a workgroup's rows, is less than one token."""
    lengths = (70, 1, 9)
    q, k, v = (_randn((sum(lengths), n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((h, hk, hk)))
    cu = _cu(lengths, gpu_device)
    for causal in (False, True):
        _check_varlen(q, k, v, cu, cu, causal)
    for width in (None, 1500):
        kc, vc, table, lens = _cache(lengths, hk, 16, 64, torch.bfloat16, "NHD", gpu_device, width)
        _check_paged(q[:3], kc, vc, table, lens, "NHD")
        _check_paged(q[:6].view(3, 2, h, 64), kc, vc, table, lens, "NHD")


@pytest.mark.parametrize("seqs", [63, 64, 65, 300, 4097])
def test_varlen_many_sequences(seqs, gpu_device):
    g = torch.Generator().manual_seed(seqs)
    top = 200 if seqs <= 65 else 4
    lengths = torch.randint(0, top, (seqs,), generator=g).tolist()
    q, k, v = (_randn((sum(lengths), n, 64), torch.float16, gpu_device, i) for i, n in enumerate((3, 1, 1)))
    cu = _cu(lengths, gpu_device)
    import flag_attn

    o = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True)
    want, _, tol, _ = SO.varlen(q, k, v, cu, cu, True)
    SO.assert_close(o, want, tol)


@pytest.mark.parametrize("d", [16, 32])
def test_varlen_small_heads_run_padded(d, gpu_device):
    import flag_attn

    lengths = (40, 3, 90)
    q, k, v = (_randn((sum(lengths) + 2, n, d), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 2, 2)))
    cu = _cu(lengths, gpu_device)
    _check_varlen(q, k, v, cu, cu, True)
    out = torch.full_like(q, 7.0)
    o = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, out=out)
    assert o is out and (out[-2:] == 7.0).all()
    SO.assert_close(out[:-2], *(x[:-2] for x in SO.varlen(q, k, v, cu, cu, True)[::2]))


def test_varlen_slices_of_one_projection_and_rows_behind_the_last_sequence(gpu_device):
    """q, k, v as slices of the same rows; further rows hold NaN and are neither read into nor written."""
    import flag_attn

    lengths, h, hk, d = (100, 1, 260), 8, 2, 128
    t = sum(lengths)
    qkv = _randn((t + 13, h + 2 * hk, d), torch.bfloat16, gpu_device, 0)
    qkv[t:] = float("nan")
    q, k, v = qkv.split([h, hk, hk], dim=1)
    cu = _cu(lengths, gpu_device)
    out = torch.full((t + 13, 2 * h, d), 3.0, dtype=torch.bfloat16, device=gpu_device)
    for causal in (False, True):
        res = flag_attn.flash_attention_varlen(q, k, v, cu, causal=causal, out=out[:, ::2])
        assert res.data_ptr() == out.data_ptr()
        want, _, tol, _ = SO.varlen(q[:t], k[:t], v[:t], cu, cu, causal)
        SO.assert_close(out[:t, ::2], want, tol)
        assert (out[t:] == 3.0).all() and (out[:, 1::2] == 3.0).all()


def test_varlen_rows_that_are_not_aligned(gpu_device):
    q, k, v = (_randn((90, n, 65), torch.float16, gpu_device, i)[:, :, 1:] for i, n in enumerate((4, 4, 4)))
    cu = _cu((50, 40), gpu_device)
    _check_varlen(q, k, v, cu, cu, True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_varlen_nonfinite_values_reach_only_the_queries_that_see_them(value, d, dtype, gpu_device):
    lengths, dt = (70, 45, 200), DTYPES[dtype]
    q, k, v = (_randn((sum(lengths), n, d), dt, gpu_device, i) for i, n in enumerate((6, 2, 2)))
    v[69, 0, 5] = value   # the last key of the first sequence
    v[70 + 33, 1, d - 1] = value  # inside the second
    v[115 + 63, 0, 0] = value  # the end of a tile
    v[115 + 130, 0, 33] = -value
    cu = _cu(lengths, gpu_device)
    for causal in (True, False):
        _check_varlen(q, k, v, cu, cu, causal)


def test_varlen_nonfinite_keys_of_the_future(gpu_device):
    """A NaN or infinity in a key makes the rows that see it NaN (or takes their weight), and no other."""
    import flag_attn

    lengths = (40, 100)
    q, k, v = (_randn((140, n, 128), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 2, 2)))
    clean = flag_attn.flash_attention_varlen(q, k, v, _cu(lengths, gpu_device), causal=True)
    k[39] = float("nan")
    k[40 + 77, 0] = float("inf")
    o = flag_attn.flash_attention_varlen(q, k, v, _cu(lengths, gpu_device), causal=True)
    assert torch.equal(o[:39], clean[:39]) and o[39].isnan().all()
    assert torch.equal(o[40:117], clean[40:117]) and torch.equal(o[40:, 2:], clean[40:, 2:])


def test_varlen_scores_that_rise_and_fall(gpu_device):
    """Row maxima that move by hundreds from tile to tile, and rows whose first keys are far above the others."""
    q, k, v = (_randn((700, n, 128), torch.bfloat16, gpu_device, i) for i, n in enumerate((2, 1, 1)))
    gain = torch.linspace(0, 40, 700, device=gpu_device)[:, None, None]
    cu = _cu((300, 400), gpu_device)
    for factor in (gain, 40 - gain):
        _check_varlen(q, (k * factor).to(k.dtype), v, cu, cu, True)
        _check_varlen(q, (k * factor).to(k.dtype), v, cu, cu, False, 0.02)


def test_varlen_offsets_that_lead_nowhere_are_clamped(gpu_device):
    """Offsets past the end or out of order: no access outside, and sequences whose offsets are fine come out right."""
    import flag_attn

    q, k, v = (_randn((64, 2, 64), torch.float16, gpu_device, i) for i in range(3))
    good = torch.tensor([0, 10, 30, 64], dtype=torch.int32, device=gpu_device)
    bad = torch.tensor([0, 10, 30, 9999], dtype=torch.int32, device=gpu_device)
    assert torch.equal(flag_attn.flash_attention_varlen(q, k, v, bad, causal=True), flag_attn.flash_attention_varlen(q, k, v, good, causal=True))
    odd = torch.tensor([-5, 10, 4, 64], dtype=torch.int32, device=gpu_device)
    o = flag_attn.flash_attention_varlen(q, k, v, odd, causal=True)
    want = flag_attn.flash_attention_varlen(q[:10], k[:10], v[:10], _cu((10,), gpu_device), causal=True)
    assert torch.equal(o[:4], want[:4])


def test_varlen_long_sequence(gpu_device):
    q, k, v = (_randn((5000, n, 128), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 1, 1)))
    cu = _cu((4800, 200), gpu_device)
    _check_varlen(q, k, v, cu, cu, True)


def _is_cut(q, k, seqs, causal):
    """Whether a call of these sizes is cut into equal shares."""
    from flagattention_amd import _lib

    p = _lib.VarlenParams()
    for t, x in ((p.q, q), (p.k, k), (p.v, k), (p.out, q)):
        t.ptr, t.stride_h, t.stride_n = x.data_ptr(), x.stride(1), x.stride(0)
    p.cu_seqlens_q = p.cu_seqlens_k = 4096
    p.seqs, p.total_q, p.total_k, p.heads_q, p.heads_kv, p.head_dim = seqs, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]
    p.dtype, p.causal, p.sm_scale = _lib.SAGE_BF16, int(causal), 0.1
    return _lib.load().sage_flash_varlen_workspace_bytes(p) > 0


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (7, 1), (3, 1), (40, 2)])
@pytest.mark.parametrize("m,n", [((100,), (9000,)), ((40, 0, 129, 1), (5000, 7, 3003, 6000)), ((64, 70), (63, 12000)), ((3, 5, 200), (0, 8000, 150))])
def test_varlen_cut_into_shares(m, n, heads, d, dtype, gpu_device):
    """Few queries against many keys: blocks that several workgroups share, shares that hold several blocks, blocks that see
    nothing, sequences without keys or queries."""
    h, hk = heads
    q = _randn((sum(m), h, d), DTYPES[dtype], gpu_device, 0)
    k, v = (_randn((sum(n), hk, d), DTYPES[dtype], gpu_device, i) for i in (1, 2))
    for causal in (False, True):
        assert _is_cut(q, k, len(m), causal)
        _check_varlen(q, k, v, _cu(m, gpu_device), _cu(n, gpu_device), causal)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_varlen_cut_with_nonfinite_values(value, gpu_device):
    m, n = (70, 33), (4000, 5000)
    q = _randn((sum(m), 8, 128), torch.bfloat16, gpu_device, 0)
    k, v = (_randn((sum(n), 2, 128), torch.bfloat16, gpu_device, i) for i in (1, 2))
    v[3999, 0, 5] = value
    v[3970, 1, 100] = -value
    v[4000 + 4980, 1, 0] = value
    assert _is_cut(q, k, 2, True)
    _check_varlen(q, k, v, _cu(m, gpu_device), _cu(n, gpu_device), True)


def _among_many(lengths, seqs=60):
    """The lengths with empty sequences before, between and behind them, `seqs` in all: with 17 K/V heads or more they count as
    enough blocks to run in tiles of 32 keys, with 5 as enough to be sorted."""
    gaps, out = seqs - len(lengths), []
    for i, n in enumerate(lengths):
        out += [0] * (gaps * (i + 1) // (len(lengths) + 1) - gaps * i // (len(lengths) + 1)) + [n]
    return tuple(out + [0] * (seqs - len(out)))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [(17, 17), (40, 20), (119, 17), (5, 5), (24, 8)])
@pytest.mark.parametrize("lengths", [(1,), (0, 5, 0, 2), (31, 32, 33, 64, 65), (127, 128, 129, 1), (300, 1, 511), (161,)])
def test_varlen_many_blocks(lengths, heads, d, dtype, gpu_device):
    (h, hk), t, dt = heads, sum(lengths), DTYPES[dtype]
    q, k, v = (_randn((t, n, d), dt, gpu_device, i) for i, n in enumerate((h, hk, hk)))
    for seqs in (60, 70):  # (in the order of their lengths, in their own order)
        cu = _cu(_among_many(lengths, seqs), gpu_device)
        for causal in (False, True):
            _check_varlen(q, k, v, cu, cu, causal)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("m,n", [((3, 70, 1), (200, 70, 600)), ((5, 100, 40), (0, 33, 7)), ((64, 0, 9), (1, 50, 8)), ((130,), (700,))])
def test_varlen_many_blocks_of_chunks(m, n, d, gpu_device):
    q = _randn((sum(m), 40, d), torch.bfloat16, gpu_device, 0)
    k, v = (_randn((sum(n), 20, d), torch.bfloat16, gpu_device, i) for i in (1, 2))
    for causal in (False, True):
        _check_varlen(q, k, v, _cu(_among_many(m), gpu_device), _cu(_among_many(n), gpu_device), causal)


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_varlen_many_blocks_with_nonfinite_values(value, d, dtype, gpu_device):
    lengths = (70, 45, 200)
    q, k, v = (_randn((sum(lengths), n, d), DTYPES[dtype], gpu_device, i) for i, n in enumerate((34, 17, 17)))
    v[69, 0, 5] = value
    v[70 + 33, 1, d - 1] = value
    v[115 + 31, 0, 0] = value
    v[115 + 130, 16, 33] = -value
    v[115 + 190, 3] = value
    cu = _cu(_among_many(lengths), gpu_device)
    for causal in (True, False):
        _check_varlen(q, k, v, cu, cu, causal)


def test_varlen_many_blocks_leave_other_rows_alone(gpu_device):
    """NaN in a query or a key of the future, slices of one projection, rows behind the last sequence."""
    import flag_attn

    lengths, h, hk, d = (100, 1, 260), 34, 17, 128
    t = sum(lengths)
    qkv = _randn((t + 13, h + 2 * hk, d), torch.bfloat16, gpu_device, 0)
    qkv[t:] = float("nan")
    q, k, v = qkv.split([h, hk, hk], dim=1)
    cu = _cu(_among_many(lengths), gpu_device)
    out = torch.full((t + 13, 2 * h, d), 3.0, dtype=torch.bfloat16, device=gpu_device)
    for causal in (False, True):
        flag_attn.flash_attention_varlen(q, k, v, cu, causal=causal, out=out[:, ::2])
        want, _, tol, _ = SO.varlen(q[:t], k[:t], v[:t], cu, cu, causal)
        SO.assert_close(out[:t, ::2], want, tol)
        assert (out[t:] == 3.0).all() and (out[:, 1::2] == 3.0).all()
    clean = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True)
    q[50, 3], k[99, 5], k[101 + 200] = float("nan"), float("nan"), float("inf")
    o = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True)
    same = torch.ones(t, h, dtype=torch.bool, device=gpu_device)
    same[50, 3], same[99, 10:12], same[301:] = False, False, False
    assert torch.equal(o[:t][same], clean[:t][same]) and o[50, 3].isnan().all() and o[99, 10:12].isnan().all()


@pytest.mark.parametrize("group", [3, 5, 11, 33, 63, 65, 100, 127, 128, 129])
def test_varlen_group_sizes(group, gpu_device):
    """Rows of a block are (query, head) pairs: blocks that begin inside a query, groups around the rows of a block."""
    lengths = (9, 40, 1)
    for hk, seqs in ((1, 3), (17, 60)):  # (few blocks, many)
        q, k, v = (_randn((sum(lengths), n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((group * hk, hk, hk)))
        cu = _cu(_among_many(lengths, seqs), gpu_device)
        for causal in (False, True):
            _check_varlen(q, k, v, cu, cu, causal)


def test_varlen_agrees_with_the_rectangular_forward(gpu_device):
    """Sequences of one length are a batch: the same answers as flash_attention, to the rounding of P and of the output."""
    import flag_attn

    b, m, h, hk, d = 3, 333, 8, 2, 128
    q, k, v = (_randn((b, m, n, d), torch.bfloat16, gpu_device, i) for i, n in enumerate((h, hk, hk)))
    cu = _cu((m,) * b, gpu_device)
    o = flag_attn.flash_attention_varlen(*(x.flatten(0, 1) for x in (q, k, v)), cu, causal=True).view(b, m, h, d)
    dense = flag_attn.flash_attention(*(x.transpose(1, 2) for x in (q, k, v)), True).transpose(1, 2)
    want, _, tol, _ = SO.varlen(*(x.flatten(0, 1) for x in (q, k, v)), cu, cu, True)
    SO.assert_close(o.flatten(0, 1), want, tol)
    SO.assert_close(dense.flatten(0, 1), o.flatten(0, 1).double(), 2 * tol)


# ---- paged

def _cache(lengths, hk, page, d, dtype, layout, device, width=None, seed=0, extra=3):
    """Caches with NaN in every place that belongs to no token, a table in random order with entries behind each sequence's
    pages that are stale, and the lengths."""
    g = torch.Generator().manual_seed(100 + seed)
    used = [-(-n // page) for n in lengths]
    total = sum(used) + extra
    order = torch.randperm(total, generator=g)
    width = max(max(used), 1) + 1 if width is None else width
    table = torch.randint(-3, total + 5, (len(lengths), width), generator=g).to(torch.int32)
    k, v = (torch.full((total, page, hk, d), float("nan"), dtype=dtype) for _ in range(2))
    at = 0
    for s, n in enumerate(lengths):
        mine = order[at:at + used[s]]
        at += used[s]
        table[s, :used[s]] = mine.to(torch.int32)
        for c in (k, v):
            rows = torch.full((used[s] * page, hk, d), float("nan"), dtype=dtype)
            rows[:n] = torch.randn(n, hk, d, generator=g).to(dtype)
            c[mine] = rows.view(used[s], page, hk, d)
    if layout == "HND":
        k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    return k.to(device), v.to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device)


def _check_paged(q, k, v, table, lens, layout, sm_scale=None):
    import flag_attn

    o, norm = flag_attn.paged_attention(q, k, v, table, lens, sm_scale, layout, return_log_normalizer=True)
    want, want_norm, o_tol, norm_tol = SO.paged(q, k, v, table, lens, sm_scale, layout)
    SO.assert_close(o, want, o_tol, "o")
    SO.assert_close(norm, want_norm, norm_tol, "log normalizer")
    alone = flag_attn.paged_attention(q, k, v, table, lens, sm_scale, layout)
    assert torch.equal(alone.view(torch.int16), o.view(torch.int16))  # (NaN among them)
    return o


PAGED_LENGTHS = [(1,), (0, 7, 0), (31, 32, 33), (127, 128, 129, 1, 300), (1000, 5, 260)]


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16"), (128, "fp16"), (64, "bf16")])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (7, 1), (40, 1)])
@pytest.mark.parametrize("page", [16, 1, 24, 48, 128])
@pytest.mark.parametrize("lengths", PAGED_LENGTHS)
def test_paged_lengths(lengths, page, heads, d, dtype, layout, gpu_device):
    """Once with a table as wide as the sequences need (a workgroup per item) and once with a wide one (equal shares)."""
    h, hk = heads
    for width in (None, 1 + 20000 // page):
        k, v, table, lens = _cache(lengths, hk, page, d, DTYPES[dtype], layout, gpu_device, width)
        q = _randn((len(lengths), h, d), DTYPES[dtype], gpu_device, 1)
        _check_paged(q, k, v, table, lens, layout)


@pytest.mark.parametrize("m", [2, 3, 8, 33])
@pytest.mark.parametrize("heads,d", [((4, 4), 64), ((8, 2), 128), ((3, 1), 64)])
def test_paged_several_new_tokens(m, heads, d, gpu_device):
    """Each new token sees the ones before it; sequences shorter than m have rows that see nothing."""
    h, hk = heads
    lengths = (1, m, m + 1, 200, 0, 33, 1030)
    for width in (None, 2000):
        k, v, table, lens = _cache(lengths, hk, 16, d, torch.bfloat16, "HND", gpu_device, width)
        q = _randn((len(lengths), m, h, d), torch.bfloat16, gpu_device, 1)
        _check_paged(q, k, v, table, lens, "HND")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_paged_nonfinite_values_of_new_tokens(value, d, dtype, gpu_device):
    """An infinity or NaN in the value of a new token reaches that token and the ones after it."""
    m, lengths = 5, (70, 5, 300)
    k, v, table, lens = _cache(lengths, 2, 16, d, DTYPES[dtype], "NHD", gpu_device)
    for s, back, ch in ((0, 1, 3), (1, 3, d - 1), (2, 2, 40)):
        t = lengths[s] - back
        v[table[s, t // 16].long(), t % 16, s % 2, ch] = value
    q = _randn((3, m, 6, d), DTYPES[dtype], gpu_device, 1)
    _check_paged(q, k, v, table, lens, "NHD")


def test_paged_items_cut_many_times(gpu_device):
    """Few sequences, long and short, over all compute units; many sequences in shares that hold several."""
    for lengths in ((20000, 3), (9000, 0, 12345, 1, 700), tuple(int(5 + 37 * i % 900) for i in range(150))):
        k, v, table, lens = _cache(lengths, 2, 16, 64, torch.float16, "HND", gpu_device, 1300)
        q = _randn((len(lengths), 8, 64), torch.float16, gpu_device, 1)
        _check_paged(q, k, v, table, lens, "HND")


@pytest.mark.parametrize("seqs", [64, 65, 1000])
def test_paged_many_sequences(seqs, gpu_device):
    lengths = torch.randint(0, 40, (seqs,), generator=torch.Generator().manual_seed(seqs)).tolist()
    k, v, table, lens = _cache(lengths, 1, 8, 64, torch.bfloat16, "HND", gpu_device, 200)
    _check_paged(_randn((seqs, 2, 64), torch.bfloat16, gpu_device, 1), k, v, table, lens, "HND")


def test_paged_entries_that_are_no_page_hide_their_tokens(gpu_device):
    lengths = (100, 300, 64)
    k, v, table, lens = _cache(lengths, 2, 16, 128, torch.bfloat16, "HND", gpu_device)
    table[0, 2] = -1
    table[1, 0] = k.shape[0]
    table[1, 7:11] = 2 ** 31 - 1
    table[2] = -7  # nothing left: a zero row
    o = _check_paged(_randn((3, 8, 128), torch.bfloat16, gpu_device, 1), k, v, table, lens, "HND")
    assert (o[2] == 0).all()
    _check_paged(_randn((3, 3, 8, 128), torch.bfloat16, gpu_device, 1), k, v, table, lens, "HND")


def test_paged_lengths_beyond_the_table_are_clamped(gpu_device):
    k, v, table, lens = _cache((64, 32), 2, 16, 64, torch.float16, "HND", gpu_device)
    table = table[:, :4].contiguous()
    table[1, 2:] = table[1, :2]
    q = _randn((2, 4, 64), torch.float16, gpu_device, 1)
    _check_paged(q, k, v, table, torch.tensor([1 << 30, 64], dtype=torch.int32, device=gpu_device), "HND")
    _check_paged(q, k, v, table, torch.tensor([-4, 64], dtype=torch.int32, device=gpu_device), "HND")


def test_paged_views_and_out(gpu_device):
    """K and V pages interleaved in one tensor, a table that is a slice of a wider one, q and out with strides."""
    import flag_attn

    lengths = (50, 130)
    k, v, table, lens = _cache(lengths, 2, 16, 64, torch.bfloat16, "HND", gpu_device)
    both = torch.stack([k, v], dim=1)
    wide = torch.full((2, table.shape[1] + 9), -1, dtype=torch.int32, device=gpu_device)
    wide[:, 4:4 + table.shape[1]] = table
    q = _randn((2, 16, 64), torch.bfloat16, gpu_device, 1)[:, ::2]
    out = torch.full((2, 16, 64), 3.0, dtype=torch.bfloat16, device=gpu_device)
    o = flag_attn.paged_attention(q, both[:, 0], both[:, 1], wide[:, 4:4 + table.shape[1]], lens, out=out[:, ::2])
    want, _, tol, _ = SO.paged(q, k, v, table, lens)
    SO.assert_close(o, want, tol)
    SO.assert_close(out[:, ::2], want, tol)
    assert (out[:, 1::2] == 3.0).all()


def test_paged_offsets_past_32_bits(gpu_device):
    """A cache of 6 GiB for K and V together as one tensor: pages behind the first 2^31 elements and 2^32 bytes."""
    page, hk, d = 64, 2, 128
    pages = (6 << 30) // (2 * page * hk * d * 2)
    both = torch.zeros((pages, 2, page, hk, d), dtype=torch.bfloat16, device=gpu_device)
    k, v = both[:, 0], both[:, 1]
    table = torch.tensor([[pages - 1, 0, pages // 2 + 1], [pages - 2, pages - 3, 5]], dtype=torch.int32, device=gpu_device)
    lens = torch.tensor([150, 192], dtype=torch.int32, device=gpu_device)
    rows = [(int(p), t) for s in range(2) for p in table[s].tolist() for t in range(page)]
    slots = torch.tensor([p * page + t for p, t in rows], dtype=torch.int64, device=gpu_device)
    new_k, new_v = (_randn((len(rows), hk, d), torch.bfloat16, gpu_device, i) for i in (1, 2))
    import flag_attn

    flag_attn.append_to_cache(new_k, new_v, k, v, slots, "NHD")
    for i, (p, t) in enumerate(rows):
        if i % 37 == 0:
            assert torch.equal(k[p, t], new_k[i]) and torch.equal(v[p, t], new_v[i])
    _check_paged(_randn((2, 8, d), torch.bfloat16, gpu_device, 3), k, v, table, lens, "NHD")
    flag_attn.copy_pages(k, v, table[0, :1], torch.tensor([pages - 9], device=gpu_device))
    assert torch.equal(k[pages - 9], k[pages - 1]) and torch.equal(v[pages - 9], v[pages - 1])


# ---- the cache's movements

@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,hk,page,d", [(1, 1, 1, 8), (5, 3, 16, 64), (700, 8, 16, 128), (33, 2, 24, 40)])
def test_append(tokens, hk, page, d, dtype, layout, gpu_device):
    import flag_attn

    pages = tokens // page + 4
    g = torch.Generator().manual_seed(tokens)
    for wide in (torch.int32, torch.int64):
        kc, vc = (_randn((pages, hk, page, d) if layout == "HND" else (pages, page, hk, d), dtype, gpu_device, i) for i in (5, 6))
        want_k, want_v = kc.clone(), vc.clone()
        slots = torch.randperm(pages * page, generator=g)[:tokens]
        if tokens > 3:
            slots[1], slots[2], slots[3] = -1, pages * page, -(1 << 31)
        rows = _randn((tokens, 4 * hk, d), dtype, gpu_device, 7)
        k, v = rows[:, hk:2 * hk], rows[:, 3 * hk:]
        flag_attn.append_to_cache(k, v, kc, vc, slots.to(wide).to(gpu_device), layout)
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                at = (s // page, slice(None), s % page) if layout == "HND" else (s // page, s % page)
                want_k[at], want_v[at] = k[t], v[t]
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_append_rows_that_are_not_aligned(gpu_device):
    import flag_attn

    rows = _randn((9, 2, 65), torch.bfloat16, gpu_device, 0)[:, :, 1:]
    kc, vc = (torch.zeros(3, 2, 4, 64, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    flag_attn.append_to_cache(rows, -rows, kc, vc, torch.arange(2, 11, device=gpu_device))
    flat = kc.transpose(1, 2).reshape(12, 2, 64)
    assert torch.equal(flat[2:11], rows) and (flat[:2] == 0).all() and (flat[11:] == 0).all()
    assert torch.equal(vc, -kc)


@pytest.mark.parametrize("layers", [0, 1, 3])
@pytest.mark.parametrize("count,page,d", [(1, 1, 8), (7, 16, 64), (200, 16, 128), (3, 128, 128)])
def test_copy_pages(count, page, d, layers, gpu_device):
    import flag_attn

    pages = 2 * count + 5
    shape = ((layers,) if layers else ()) + (pages, 2, page, d)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(count))
    src, dst = order[:count].clone(), order[count:2 * count].clone()
    real = torch.ones(count, dtype=torch.bool)
    if count > 3:
        src[1], dst[2], src[3] = -1, pages, 1 << 30
        real[1:4] = False
    for a, b in ((torch.int32, torch.int64), (torch.int64, torch.int32)):
        k, v = (_randn(shape, torch.bfloat16, gpu_device, i) for i in (1, 2))
        want = [k.clone(), v.clone()]
        for w in want:
            x = w if layers else w[None]
            x[:, dst[real].to(gpu_device)] = x[:, src[real].to(gpu_device)]
        flag_attn.copy_pages(k, v, src.to(a).to(gpu_device), dst.to(b).to(gpu_device))
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copy_more_pages_than_a_grid_dimension_holds(gpu_device):
    import flag_attn

    count = 70001
    k, v = (_randn((2 * count, 1, 1, 8), torch.float16, gpu_device, i) for i in (1, 2))
    src, dst = torch.arange(count, device=gpu_device), torch.arange(count, 2 * count, device=gpu_device).flip(0)
    want = [torch.cat([x[:count], x[:count].flip(0)]) for x in (k, v)]
    flag_attn.copy_pages(k, v, src, dst)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copy_pages_of_views(gpu_device):
    """K and V pages interleaved in one tensor; pages whose dimensions lie in another order."""
    import flag_attn

    both = _randn((9, 2, 3, 8, 16), torch.float16, gpu_device, 0)
    before = both.clone()
    src, dst = (torch.tensor(x, device=gpu_device) for x in ([1, 4], [8, 0]))
    flag_attn.copy_pages(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), src, dst)
    before[dst] = before[src]
    assert torch.equal(both, before)


# ---- together


def test_prompt_then_new_tokens_then_a_split(gpu_device):
    """Prompts through flash_attention_varlen and into the cache; new tokens one by one against it; one sequence splits in
    two (its last page is copied, the full ones are shared) and both go on with different tokens."""
    import flag_attn

    h, hk, d, page = 4, 2, 64, 16
    prompts = [37, 5, 64]
    kc, vc = (torch.full((40, hk, page, d), float("nan"), dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    free = list(range(39, -1, -1))
    tables = [[free.pop() for _ in range(-(-n // page))] for n in prompts]
    rows = [[_randn((n, x, d), torch.bfloat16, gpu_device, 10 * i + j) for j, x in enumerate((h, hk, hk))] for i, n in enumerate(prompts)]
    q, k, v = (torch.cat([r[j] for r in rows]) for j in range(3))
    cu = _cu(prompts, gpu_device)
    o = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True)
    SO.assert_close(o, *SO.varlen(q, k, v, cu, cu, True)[::2])
    slots = [tables[i][t // page] * page + t % page for i, n in enumerate(prompts) for t in range(n)]
    flag_attn.append_to_cache(k, v, kc, vc, torch.tensor(slots, device=gpu_device))
    history = [[r[1], r[2]] for r in rows]

    def step(seed):
        s = len(tables)
        new = [_randn((s, x, d), torch.bfloat16, gpu_device, seed + j) for j, x in enumerate((h, hk, hk))]
        slots, lens = [], []
        for i in range(s):
            n = history[i][0].shape[0]
            if n % page == 0:
                tables[i].append(free.pop())
            slots.append(tables[i][n // page] * page + n % page)
            history[i] = [torch.cat([history[i][0], new[1][i:i + 1]]), torch.cat([history[i][1], new[2][i:i + 1]])]
            lens.append(n + 1)
        flag_attn.append_to_cache(new[1], new[2], kc, vc, torch.tensor(slots, device=gpu_device))
        width = max(map(len, tables))
        table = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32, device=gpu_device)
        o = flag_attn.paged_attention(new[0], kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=gpu_device))
        for i in range(s):
            want, _, tol, _ = SO.attend(new[0][i][None], *history[i], True, d ** -0.5)
            SO.assert_close(o[i][None], want, tol, (seed, i))

    for i in range(3):
        step(100 + 10 * i)
    last = free.pop()
    flag_attn.copy_pages(kc, vc, torch.tensor([tables[0][-1]], device=gpu_device), torch.tensor([last], device=gpu_device))
    tables.append(tables[0][:-1] + [last])
    history.append(list(history[0]))
    for i in range(12):
        step(200 + 10 * i)


def test_captured_step_follows_the_present_lengths(gpu_device):
    """A step of all four operators, captured once; lengths, tables, slots and data change between the replays, with eager work
    in between; every replay equals the eager calls."""
    import flag_attn

    h, hk, d, page, s = 8, 2, 128, 16, 6
    kc, vc = (torch.zeros(200, hk, page, d, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    kc.normal_(generator=torch.Generator(device=gpu_device).manual_seed(1))
    vc.normal_(generator=torch.Generator(device=gpu_device).manual_seed(2))
    q, k, v = (torch.empty(s, n, d, dtype=torch.bfloat16, device=gpu_device) for n in (h, hk, hk))
    pq, pk, pv = (torch.empty(300, n, d, dtype=torch.bfloat16, device=gpu_device) for n in (h, hk, hk))
    cu = torch.zeros(5, dtype=torch.int32, device=gpu_device)
    table = torch.zeros(s, 90, dtype=torch.int32, device=gpu_device)  # (wide: the shares are planned for 1440 tokens)
    lens = torch.zeros(s, dtype=torch.int32, device=gpu_device)
    slots = torch.full((s,), -1, dtype=torch.int64, device=gpu_device)
    src, dst = (torch.full((2,), -1, dtype=torch.int32, device=gpu_device) for _ in range(2))

    def work():
        flag_attn.copy_pages(kc, vc, src, dst)
        flag_attn.append_to_cache(k, v, kc, vc, slots)
        o = flag_attn.paged_attention(q, kc, vc, table, lens, return_log_normalizer=True)
        return (*o, flag_attn.flash_attention_varlen(pq, pk, pv, cu, causal=True, out=prompt_out))

    prompt_out = torch.zeros(300, h, d, dtype=torch.bfloat16, device=gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        for x in (q, k, v, pq, pk, pv):
            x.copy_(torch.randn(x.shape, generator=g))
        n = torch.randint(0, 1400 if i else 30, (s,), generator=g)
        n[i] = 0
        lens.copy_(n)
        table.copy_(torch.randperm(150, generator=g)[:90].expand(s, 90))
        slots.copy_(torch.tensor([150 * page + 7 * j if j % 2 else -1 for j in range(s)]))
        src.copy_(torch.tensor([3, -1]))
        dst.copy_(torch.tensor([160 + i, 5]))
        cu.copy_(torch.tensor([0, 10 * i, 10 * i, 100 + i, 300 - i]))
        prompt_out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in captured]
        cache = kc.clone(), vc.clone()
        prompt_out.fill_(5.0)
        for a, b in zip(got, work()):
            assert torch.equal(a, b), i
        assert torch.equal(kc, cache[0]) and torch.equal(vc, cache[1])
        want, want_norm, tol, norm_tol = SO.paged(q, kc, vc, table, lens)
        SO.assert_close(got[0], want, tol)
        SO.assert_close(got[1], want_norm, norm_tol)


def test_calls_of_a_known_shape_take_the_present_arguments(gpu_device):
    """A second call of the same sizes and strides with other tensors, the same call with other flags, and errors after it."""
    import flag_attn

    k, v, table, lens = _cache((300, 100), 2, 16, 64, torch.bfloat16, "HND", gpu_device)
    for seed in range(3):
        q = _randn((2, 8, 64), torch.bfloat16, gpu_device, seed)
        lens2 = lens - 7 * seed
        _check_paged(q, k, v, table.clone(), lens2, "HND", None if seed < 2 else 0.3)
        p = [_randn((130, n, 64), torch.bfloat16, gpu_device, seed + i) for i, n in enumerate((4, 2, 2))]
        cu = _cu((50 + seed, 80 - seed), gpu_device)
        for causal in (True, False):
            _check_varlen(*p, cu, cu, causal, None if seed < 2 else 0.3)
        kc, vc = (_randn((5, 2, 16, 64), torch.bfloat16, gpu_device, seed + 7 + i) for i in range(2))
        slots = torch.arange(7, device=gpu_device) + seed
        flag_attn.append_to_cache(p[1][:7], p[2][:7], kc, vc, slots)
        assert torch.equal(kc[0, :, seed:seed + 7].transpose(0, 1), p[1][:7]) and torch.equal(vc[0, :, seed:seed + 7].transpose(0, 1), p[2][:7])
        flag_attn.copy_pages(kc, vc, slots[:1], slots[1:2])
        assert torch.equal(kc[seed], kc[seed + 1]) and torch.equal(vc[seed], vc[seed + 1])
    with pytest.raises(NotImplementedError):
        flag_attn.flash_attention_varlen(p[0].requires_grad_(), p[1], p[2], cu)
    with pytest.raises(ValueError):
        flag_attn.paged_attention(q, k, v, table[:1], lens)
    with pytest.raises(RuntimeError, match="seq_lens is on cpu"):
        flag_attn.paged_attention(q, k, v, table, lens.cpu())


def test_calls_on_another_stream(gpu_device):
    import flag_attn

    k, v, table, lens = _cache((3000, 100), 2, 16, 64, torch.bfloat16, "HND", gpu_device, 400)
    q = _randn((2, 8, 64), torch.bfloat16, gpu_device, 1)
    p = [_randn((500, n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 2, 2))]
    cu = _cu((200, 300), gpu_device)
    want = flag_attn.paged_attention(q, k, v, table, lens), flag_attn.flash_attention_varlen(*p, cu, causal=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [(flag_attn.paged_attention(q, k, v, table, lens), flag_attn.flash_attention_varlen(*p, cu, causal=True)) for _ in range(3)]
    here = [(flag_attn.paged_attention(q, k, v, table, lens), flag_attn.flash_attention_varlen(*p, cu, causal=True)) for _ in range(3)]
    torch.cuda.synchronize()
    for a, b in got + here:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
