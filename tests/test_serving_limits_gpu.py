"""The serving operators at the ends of their ranges on the GPU, against their formulas in 64 bits."""
import pytest
import torch

from oracle import serving_oracle as SO

pytestmark = pytest.mark.gpu


def _cu(lengths, device):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(device)


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


@pytest.mark.parametrize("n", [2965900, 2965940, 5931900])
def test_varlen_a_chunk_against_millions_of_keys(n, gpu_device):
    """The steps that a block of such a sequence counts from the first key on pass 2^31.  All keys but 400 have scores 64 below the
    others' (their weights sum up to less than 10^-20), so that a row is the mean of the values of those that it sees."""
    import flag_attn

    m, h, d = 200, 2, 64
    g = torch.Generator(device=gpu_device).manual_seed(n)
    at = torch.randperm(n - m, generator=g, device=gpu_device)[:300].sort().values
    at = torch.cat([at, torch.arange(n - m, n, 2, device=gpu_device)])  # some of them along the diagonal
    q = torch.zeros(m, h, d, dtype=torch.bfloat16, device=gpu_device)
    k, v = (torch.zeros(n, 1, d, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    q[:, :, 3] = k[at, :, 3] = 8.0
    v.normal_(generator=g)
    assert _is_cut(q, k, 1, True)
    out = torch.full_like(q, float("nan"))
    o, norm = flag_attn.flash_attention_varlen(q, k, v, _cu((m,), gpu_device), _cu((n,), gpu_device), True, 1.0, True, out=out)
    sees = at[None, :] <= torch.arange(n - m, n, device=gpu_device)[:, None]
    count, values = sees.sum(1, keepdim=True), v[at, 0].double()
    want, size = sees.double() @ values / count, sees.double() @ values.abs() / count
    # P and the output are rounded by half a step; 400 weights are added up in fp32 (400 2^-24 at worst), to a maximum of 92 in base 2
    # (four roundings of 2^-18 each)
    tol, norm_tol = 2.0 ** -8 * (want.abs() + size) + 2.0 ** -14 * size, torch.full((m,), 2.0 ** -14, dtype=torch.float64, device=gpu_device)
    for i in range(h):
        SO.assert_close(o[:, i], want, tol, i)
        SO.assert_close(norm[i], 64.0 + count[:, 0].double().log(), norm_tol, i)


def _randn(shape, dtype, device, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def _odd(t, offset=1):
    """The tensor, contiguous, `offset` elements behind a 16-byte boundary."""
    buf = torch.zeros(t.numel() + offset, dtype=t.dtype, device=t.device)
    return buf[offset:].view(t.shape).copy_(t)


def _lone(t, dim, stride):
    """The tensor, one entry long in `dim`, with an odd stride there."""
    strides = list(t.stride())
    strides[dim] = stride
    return torch.as_strided(t, t.shape, strides, t.storage_offset())


@pytest.mark.parametrize("d", [16, 64, 128])
def test_contiguous_tensors_at_odd_offsets(d, gpu_device):
    import flag_attn

    q, k, v = (_odd(_randn((70, n, d), torch.float16, gpu_device, i), 1 + 2 * i) for i, n in enumerate((4, 2, 2)))
    cu = _cu((50, 20), gpu_device)
    for _ in range(2):  # (and once more as a call of a known shape)
        o, norm = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, return_log_normalizer=True)
        want, want_norm, tol, norm_tol = SO.varlen(q, k, v, cu, cu, True)
        SO.assert_close(o, want, tol)
        SO.assert_close(norm, want_norm, norm_tol)
    aligned = [x.clone() for x in (q, k, v)]  # (a plan of aligned tensors of these sizes serves no others)
    assert torch.equal(flag_attn.flash_attention_varlen(*aligned, cu, causal=True), o)
    assert torch.equal(flag_attn.flash_attention_varlen(q, k, v, cu, causal=True), o)
    with pytest.raises(ValueError, match="out: rows"):
        flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, out=_odd(torch.zeros_like(q)))
    kc, vc = (torch.zeros(5, 2, 16, d, dtype=torch.float16, device=gpu_device) for _ in range(2))
    flag_attn.append_to_cache(k, v, kc, vc, torch.arange(70, device=gpu_device))
    assert torch.equal(kc.transpose(1, 2).reshape(80, 2, d)[:70], k) and torch.equal(vc.transpose(1, 2).reshape(80, 2, d)[:70], v)
    if d == 16:
        return
    table, lens = torch.arange(5, dtype=torch.int32, device=gpu_device)[None].repeat(3, 1), torch.tensor([70, 3, 17], dtype=torch.int32, device=gpu_device)
    p = _odd(q[:3].clone())
    want, _, tol, _ = SO.paged(p, kc, vc, table, lens)
    SO.assert_close(flag_attn.paged_attention(p, kc, vc, table, lens), want, tol)


def test_strides_of_dimensions_with_one_entry(gpu_device):
    """One token, one head, one sequence, one page: what a tensor's stride is there does not matter, 2^40 neither."""
    import flag_attn

    for stride in (3, 1 << 40):
        for h, hk, t in ((4, 2, 1), (1, 1, 5), (1, 1, 1)):
            q, k, v = (_randn((t, n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((h, hk, hk)))
            cu = _cu((t,), gpu_device)
            want, _, tol, _ = SO.varlen(q, k, v, cu, cu, True)
            out = torch.zeros_like(q)
            dims = [i for i, n in ((0, t), (1, h)) if n == 1]
            for dim in dims:
                q, out = _lone(q, dim, stride), _lone(out, dim, stride)
            for dim in [i for i, n in ((0, t), (1, hk)) if n == 1]:
                k, v = _lone(k, dim, stride), _lone(v, dim, stride)
            SO.assert_close(flag_attn.flash_attention_varlen(q, k, v, cu, causal=True), want, tol)
            flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, out=out)
            SO.assert_close(out, want, tol)
        for layout in ("HND", "NHD"):
            # one page of one head, one sequence of one new token
            kc, vc = (_lone(_lone(torch.zeros((1, 1, 16, 64) if layout == "HND" else (1, 16, 1, 64), dtype=torch.bfloat16, device=gpu_device), 0, stride),
                            1 if layout == "HND" else 2, stride) for _ in range(2))
            k, v = (_randn((9, 1, 64), torch.bfloat16, gpu_device, i) for i in (5, 6))
            flag_attn.append_to_cache(_lone(k, 1, stride), _lone(v, 1, stride), kc, vc, torch.arange(9, device=gpu_device), layout)
            assert torch.equal(kc.reshape(16, 1, 64)[:9], k) and torch.equal(vc.reshape(16, 1, 64)[:9], v)
            q = _randn((1, 1, 1, 64), torch.bfloat16, gpu_device, 7)
            table, lens = torch.zeros(1, 1, dtype=torch.int32, device=gpu_device), torch.tensor([9], dtype=torch.int32, device=gpu_device)
            want, _, tol, _ = SO.paged(q, kc, vc, table, lens, layout=layout)
            for dim in range(3):
                q = _lone(q, dim, stride)
            SO.assert_close(flag_attn.paged_attention(q, kc, vc, _lone(table, 1, 3), lens, tensor_layout=layout), want, tol)
        both = [_lone(_randn((1, 2, 3, 8), torch.float32, gpu_device, i)[None], 0, stride) for i in (8, 9)]
        both = [torch.as_strided(x, (1, 1, 2, 3, 8), (stride, stride, 24, 8, 1)) for x in both]
        before = [x.clone() for x in both]
        flag_attn.copy_pages(*both, torch.zeros(1, dtype=torch.int32, device=gpu_device), torch.zeros(1, dtype=torch.int32, device=gpu_device))
        assert all(torch.equal(x, y) for x, y in zip(both, before))


@pytest.mark.parametrize("pages,width", [(6, 0), (0, 3), (0, 0)])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_paged_without_a_place_for_a_key(layout, pages, width, gpu_device):
    """All slots idle and a table as wide as the longest sequence needs; a cache that has no pages yet."""
    import flag_attn

    kc, vc = (torch.zeros((pages, 2, 16, 64) if layout == "HND" else (pages, 16, 2, 64), dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    table, lens = torch.zeros(3, width, dtype=torch.int32, device=gpu_device), torch.tensor([0, 5, 0], dtype=torch.int32, device=gpu_device)
    for shape in ((3, 4, 64), (3, 2, 4, 64)):
        q = _randn(shape, torch.bfloat16, gpu_device, 1)
        o, norm = flag_attn.paged_attention(q, kc, vc, table, lens, tensor_layout=layout, return_log_normalizer=True)
        assert o.shape == q.shape and (o == 0).all()
        assert norm.shape == ((3, 4) if len(shape) == 3 else (3, 4, 2)) and (norm == float("-inf")).all()
        wide = torch.full((*shape[:-1], 128), 7.0, dtype=torch.bfloat16, device=gpu_device)
        assert flag_attn.paged_attention(q, kc, vc, table, lens, tensor_layout=layout, out=wide[..., :64]).data_ptr() == wide.data_ptr()
        assert (wide[..., :64] == 0).all() and (wide[..., 64:] == 7.0).all()
    with pytest.raises(ValueError):
        flag_attn.paged_attention(q, kc, vc, table[:2], lens, tensor_layout=layout)


# Scores so far from 0 that their rounding to 24 bits is worth many powers of two: the weights are 0 or 1 then (or equal, for equal keys).

def _means(q, k, v, causal):
    """softmax(q k^T) v for q, k whose rows are multiples of the vector of ones, in 64 bits; the mean of |v| under the weights; the
    log normalizer [H, M]."""
    m, h, d = q.shape
    n, hk = k.shape[:2]
    s = q[:, :, :1].double() * k[:, :, :1].double().repeat_interleave(h // hk, 1).permute(2, 1, 0) * d  # [M, H, N]
    if causal:
        s = s.masked_fill((torch.arange(n, device=q.device)[None] > torch.arange(m, device=q.device)[:, None] + n - m)[:, None], float("-inf"))
    w, vv = torch.softmax(s, -1), v.double().repeat_interleave(h // hk, 1)
    return torch.einsum("mhn,nhd->mhd", w, vv), torch.einsum("mhn,nhd->mhd", w, vv.abs()), torch.logsumexp(s, -1).t()


def _check_means(o, norm, want, half_step):
    """P and o are rounded by half a step; weights are added up in fp32, 300 at most that are not 0; a score is the sum of at most 128
    products in fp32, times a scale."""
    o_want, size, norm_want = want
    SO.assert_close(o, o_want, half_step * (o_want.abs() + size) + 300 * 2.0 ** -24 * size)
    SO.assert_close(norm, norm_want, 140 * 2.0 ** -24 * norm_want.abs() + 300 * 2.0 ** -24)


@pytest.mark.parametrize("heads,seqs", [((4, 2), 1), ((34, 17), 60)])  # (few blocks, many)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 2000.0), (torch.float16, 4000.0), (torch.float16, 60000.0),
                                        (torch.bfloat16, 16000.0), (torch.bfloat16, 2.0 ** 56)])
def test_varlen_huge_scores(dtype, size, d, heads, seqs, gpu_device):
    import flag_attn

    (h, hk), n = heads, 300
    g = torch.Generator().manual_seed(0)
    keys = (1 - torch.randperm(n, generator=g) / 512).to(gpu_device)
    v = _randn((n, hk, d), dtype, gpu_device, 1)
    cu = torch.tensor([0] * seqs + [n], dtype=torch.int32, device=gpu_device)
    for sign in (1, -1):
        q = torch.full((n, h, d), sign * size, dtype=dtype, device=gpu_device)
        k = (size * keys)[:, None, None].expand(n, hk, d).to(dtype).contiguous()
        for causal in (True, False):
            o, norm = flag_attn.flash_attention_varlen(q, k, v, cu, causal=causal, sm_scale=1.0, return_log_normalizer=True)
            _check_means(o, norm, _means(q, k, v, causal), torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("heads,seqs", [((4, 2), 1), ((34, 17), 60)])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 2000.0), (torch.bfloat16, 16000.0), (torch.bfloat16, 2.0 ** 56)])
def test_varlen_scores_that_rise_from_far_below(dtype, size, heads, seqs, gpu_device):
    """Keys whose weights are infinite against the first reference point, and 0 against the one of the rows that see more; a
    query among them that is NaN, and stays alone."""
    import flag_attn

    (h, hk), n, d = heads, 300, 128
    q = torch.full((n, h, d), size, dtype=dtype, device=gpu_device)
    k = torch.zeros(n, hk, d, dtype=dtype, device=gpu_device)
    k[:100] = (-size * (1 - torch.arange(100, device=gpu_device) / 512))[:, None, None]
    v = _randn((n, hk, d), dtype, gpu_device, 1)
    cu = torch.tensor([0] * seqs + [n], dtype=torch.int32, device=gpu_device)
    for causal in (True, False):
        clean = flag_attn.flash_attention_varlen(q, k, v, cu, causal=causal, sm_scale=1.0, return_log_normalizer=True)
        _check_means(*clean, _means(q, k, v, causal), torch.finfo(dtype).eps / 2)
    clean = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, sm_scale=1.0)
    q[150, 1] = float("nan")
    o = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, sm_scale=1.0)
    bad = torch.zeros(n, h, dtype=torch.bool, device=gpu_device)
    bad[150, 1] = True
    assert o[bad].isnan().all() and torch.equal(o[~bad], clean[~bad])


@pytest.mark.parametrize("dtype,size", [(torch.float16, 4000.0), (torch.bfloat16, 16000.0)])
def test_varlen_huge_scores_in_shares(dtype, size, gpu_device):
    import flag_attn

    m, n, h, hk, d = 70, 9000, 4, 2, 128
    g = torch.Generator().manual_seed(0)
    keys = 0.5 + torch.rand(n, generator=g) / 4
    keys[777] = 1.0
    q = torch.full((m, h, d), size, dtype=dtype, device=gpu_device)
    k = (size * keys.to(gpu_device))[:, None, None].expand(n, hk, d).to(dtype).contiguous()
    v = _randn((n, hk, d), dtype, gpu_device, 1)
    assert _is_cut(q, k, 1, True)
    for causal in (True, False):
        o, norm = flag_attn.flash_attention_varlen(q, k, v, _cu((m,), gpu_device), _cu((n,), gpu_device), causal, 1.0, True)
        _check_means(o, norm, _means(q, k, v, causal), torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("width", [20, 600])  # (a workgroup per item, equal shares)
@pytest.mark.parametrize("dtype,size", [(torch.float16, 4000.0), (torch.bfloat16, 16000.0), (torch.bfloat16, 2.0 ** 56)])
def test_paged_huge_scores(dtype, size, width, gpu_device):
    import flag_attn

    n, m, h, hk, d = 300, 3, 8, 2, 128
    g = torch.Generator().manual_seed(0)
    keys = 0.5 + torch.rand(320, generator=g) / 4
    keys[:5], keys[77] = -1.0, 1.0
    kc = (size * keys.to(gpu_device))[:, None, None].expand(320, hk, d).to(dtype).contiguous().view(20, 16, hk, d)
    vc = _randn((20, 16, hk, d), dtype, gpu_device, 1)
    q = torch.full((1, m, h, d), size, dtype=dtype, device=gpu_device)
    table = torch.full((1, width), -1, dtype=torch.int32, device=gpu_device)
    table[0, :20] = torch.arange(20)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu_device)
    o, norm = flag_attn.paged_attention(q, kc, vc, table, lens, 1.0, "NHD", True)
    want = _means(q[0], kc.view(320, hk, d)[:n], vc.view(320, hk, d)[:n], True)
    _check_means(o[0], norm[0], want, torch.finfo(dtype).eps / 2)


def test_tangents_raise_in_calls_of_a_known_shape_too(gpu_device):
    import flag_attn
    from torch.autograd import forward_ad

    q, k, v = (_randn((30, n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 2, 2)))
    kc, vc = (torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
    cu, slots = _cu((30,), gpu_device), torch.arange(30, device=gpu_device)
    table, lens = torch.arange(4, dtype=torch.int32, device=gpu_device)[None], torch.tensor([30], dtype=torch.int32, device=gpu_device)
    pages = slots[:1], slots[3:4]
    calls = [lambda x: flag_attn.flash_attention_varlen(x(q), k, v, cu), lambda x: flag_attn.append_to_cache(k, x(v), kc, vc, slots),
             lambda x: flag_attn.paged_attention(q[:1], kc, x(vc), table, lens), lambda x: flag_attn.copy_pages(x(kc), vc, *pages)]
    for _ in range(2):
        for call in calls:
            call(lambda t: t)
    with forward_ad.dual_level():
        for call in calls:
            call(lambda t: t)
            with pytest.raises(NotImplementedError, match="tangents"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))


def test_autograd_knows_what_was_written(gpu_device):
    """A graph that keeps a cache or an output for its backward pass raises once the operators have changed it, in first calls and in
    calls of a known shape; tensors made in inference mode are written as well."""
    import flag_attn

    q, k, v = (_randn((30, n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 2, 2)))
    cu, slots = _cu((30,), gpu_device), torch.arange(30, device=gpu_device)
    table, lens = torch.arange(4, dtype=torch.int32, device=gpu_device)[None], torch.tensor([30], dtype=torch.int32, device=gpu_device)
    w = torch.ones(1, device=gpu_device, requires_grad=True)
    for i in range(3):
        kc, vc = (torch.ones(4, 2, 16, 64, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
        out, out1 = torch.ones_like(q), torch.ones_like(q[:1])
        writes = [((kc, vc), lambda: flag_attn.append_to_cache(k, v, kc, vc, slots)), ((kc, vc), lambda: flag_attn.copy_pages(kc, vc, slots[:1], slots[3:4])),
                  ((out,), lambda: flag_attn.flash_attention_varlen(q, k, v, cu, out=out)),
                  ((out1,), lambda: flag_attn.paged_attention(q[:1], kc, vc, table, lens, out=out1))]
        for kept, write in writes:
            for x in kept:
                y, version = (w * x.float()).sum() + (w * x).sum(), x._version
                write()
                assert x._version > version
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.backward()
        with torch.inference_mode():
            kc, vc = (torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=gpu_device) for _ in range(2))
        for _ in range(2):
            flag_attn.append_to_cache(k, v, kc, vc, slots)
            flag_attn.copy_pages(kc, vc, slots[:1], slots[3:4])
        assert torch.equal(kc.transpose(1, 2).reshape(64, 2, 64)[:30], k) and torch.equal(vc[3], vc[0])


def test_expanded_tensors_are_read_and_not_written(gpu_device):
    import flag_attn

    q, k, v = (_randn((30, n, 64), torch.bfloat16, gpu_device, i) for i, n in enumerate((4, 2, 2)))
    cu, slots = _cu((30,), gpu_device), torch.arange(30, device=gpu_device)
    table, lens = torch.arange(4, dtype=torch.int32, device=gpu_device)[None], torch.tensor([30], dtype=torch.int32, device=gpu_device)
    kc, vc = (_randn((4, 2, 16, 64), torch.bfloat16, gpu_device, i) for i in (5, 6))
    # one K/V head, one page, one table row for all: the answers are those of the copies
    for x, y in ((k[:, :1].expand(30, 2, 64), v), (k, v[:1].expand(30, 2, 64))):
        assert torch.equal(flag_attn.flash_attention_varlen(q, x, y, cu), flag_attn.flash_attention_varlen(q, x.contiguous(), y.contiguous(), cu))
    for x in (vc[:1].expand_as(vc), vc[:, :1].expand_as(vc), vc[:, :, :1].expand_as(vc)):
        assert torch.equal(flag_attn.paged_attention(q[:1], kc, x, table, lens), flag_attn.paged_attention(q[:1], kc, x.contiguous(), table, lens))
        with pytest.raises(ValueError, match="share memory"):
            flag_attn.append_to_cache(k, v, kc, x, slots)
        with pytest.raises(ValueError):
            flag_attn.copy_pages(kc, x, slots[:1], slots[3:4])
    both = flag_attn.paged_attention(q[:1].expand(3, 4, 64), kc, vc, table.expand(3, 4), lens.expand(3))
    assert all(torch.equal(row, flag_attn.paged_attention(q[:1], kc, vc, table, lens)[0]) for row in both)
    for out in (q[:1].clone().expand_as(q), q[:, :1].clone().expand_as(q)):
        with pytest.raises(ValueError, match="share memory"):
            flag_attn.flash_attention_varlen(q, k, v, cu, out=out)
    with pytest.raises(ValueError, match="share memory"):
        flag_attn.paged_attention(q[:3], kc, vc, table.expand(3, 4), lens.expand(3), out=q[:1].clone().expand(3, 4, 64))
    with pytest.raises(ValueError, match="share memory"):
        flag_attn.copy_pages(kc[None].expand(3, 4, 2, 16, 64), vc[None].expand(3, 4, 2, 16, 64), slots[:1], slots[3:4])


@pytest.mark.parametrize("heads,seqs", [((4, 2), 1), ((34, 17), 60)])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_varlen_rows_that_are_nan_throughout(d, dtype, heads, seqs, gpu_device):
    """All values NaN from some token on, of one head or of all: the rows that see one are NaN in every channel, whatever their log
    normalizer; those before are as ever."""
    import flag_attn

    (h, hk), n = heads, 400
    q, k, v = (_randn((n, x, d), dtype, gpu_device, i) for i, x in enumerate((h, hk, hk)))
    cu = torch.tensor([0] * seqs + [150, n], dtype=torch.int32, device=gpu_device)
    v[77:100, 1] = float("nan")
    v[150 + 201:] = float("nan")
    o, norm = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True, return_log_normalizer=True)
    want, want_norm, tol, norm_tol = SO.varlen(q, k, v, cu, cu, True)
    SO.assert_close(o, want, tol)
    SO.assert_close(norm, want_norm, norm_tol)
    alone = flag_attn.flash_attention_varlen(q, k, v, cu, causal=True)
    SO.assert_close(alone, want, tol)
    lost = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    o, norm = flag_attn.flash_attention_varlen(*lost, cu, causal=True, return_log_normalizer=True)
    assert o.isnan().all() and norm.isnan().all()


def test_varlen_parts_that_are_nan_throughout(gpu_device):
    import flag_attn

    m, n = (70, 33), (4000, 5000)
    q = _randn((sum(m), 8, 128), torch.bfloat16, gpu_device, 0)
    k, v = (_randn((sum(n), 2, 128), torch.bfloat16, gpu_device, i) for i in (1, 2))
    assert _is_cut(q, k, 2, True)
    v[3960:4000, 0] = float("nan")
    v[4000 + 4990:, 1] = float("nan")
    cu_q, cu_k = _cu(m, gpu_device), _cu(n, gpu_device)
    o, norm = flag_attn.flash_attention_varlen(q, k, v, cu_q, cu_k, True, return_log_normalizer=True)
    want, want_norm, tol, norm_tol = SO.varlen(q, k, v, cu_q, cu_k, True)
    SO.assert_close(o, want, tol)
    SO.assert_close(norm, want_norm, norm_tol)
