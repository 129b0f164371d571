"""Forms of the serving operators' kernels that only certain sizes together reach: several new tokens in pages that are no multiple
of 16, missing pages among those, cut launches of more sequences than a wave has lanes."""
import pytest
import torch

from oracle import serving_oracle as SO

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _cu(lengths, device):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32).to(device)


def _randn(shape, dtype, device, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device)


def _cache(lengths, hk, page, d, dtype, layout, device, width=None, extra=3):
    """Caches with NaN in every place that belongs to no token, a table in random order whose entries behind a sequence's pages
    are stale, and the lengths."""
    g = torch.Generator().manual_seed(7)
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


def _check_paged(q, k, v, table, lens, layout):
    import flag_attn

    o, norm = flag_attn.paged_attention(q, k, v, table, lens, None, layout, return_log_normalizer=True)
    want, want_norm, o_tol, norm_tol = SO.paged(q, k, v, table, lens, None, layout)
    SO.assert_close(o, want, o_tol, "o")
    SO.assert_close(norm, want_norm, norm_tol, "log normalizer")
    return o


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (64, "fp16"), (128, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("page", [1, 8, 24, 100])
@pytest.mark.parametrize("m,heads", [(2, (4, 4)), (7, (8, 2)), (3, (14, 2)), (33, (3, 1))])
def test_several_new_tokens_in_pages_of_any_size(m, heads, page, d, dtype, gpu_device):
    h, hk = heads
    lengths = (1, m, m + 1, 200, 0, 33, 777)
    for width in (None, 1 + 20000 // page):  # (a workgroup per item, equal shares)
        for layout in ("HND", "NHD"):
            k, v, table, lens = _cache(lengths, hk, page, d, DTYPES[dtype], layout, gpu_device, width)
            _check_paged(_randn((len(lengths), m, h, d), DTYPES[dtype], gpu_device, 1), k, v, table, lens, layout)


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (64, "fp16"), (128, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("page", [1, 24])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_values_of_new_tokens_in_pages_of_any_size(value, page, d, dtype, gpu_device):
    m, lengths = 5, (70, 5, 300)
    for width in (None, 1 + 20000 // page):
        k, v, table, lens = _cache(lengths, 2, page, d, DTYPES[dtype], "NHD", gpu_device, width)
        for s, back, ch in ((0, 1, 3), (1, 3, d - 1), (2, 2, 40), (2, 5, 41)):
            t = lengths[s] - back
            v[table[s, t // page].long(), t % page, s % 2, ch] = value
        _check_paged(_randn((3, m, 6, d), DTYPES[dtype], gpu_device, 1), k, v, table, lens, "NHD")


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("page", [1, 8, 24])
def test_entries_that_are_no_page_among_pages_of_any_size(page, d, dtype, gpu_device):
    lengths = (100, 300, 64, 301)
    for width in (None, 1 + 20000 // page):
        k, v, table, lens = _cache(lengths, 2, page, d, DTYPES[dtype], "HND", gpu_device, width)
        table[0, 32 // page] = -1
        table[1, 0] = k.shape[0]
        table[1, 112 // page:176 // page] = 2 ** 31 - 1
        table[2] = -7  # nothing left: zero rows
        table[3, -(-301 // page) - 1] = -2 ** 31  # the last page, with the newest tokens
        for shape in ((4, 8, d), (4, 3, 8, d), (4, 9, 8, d)):
            o = _check_paged(_randn(shape, DTYPES[dtype], gpu_device, 1), k, v, table, lens, "HND")
            assert (o[2] == 0).all()


@pytest.mark.parametrize("seqs", [64, 65, 130, 300])
@pytest.mark.parametrize("heads,d,dtype", [((2, 1), 64, "fp16"), ((5, 1), 128, "bf16")])
def test_cut_launches_of_many_sequences(heads, d, dtype, seqs, gpu_device):
    """Few queries of many sequences, some without queries or keys, against long histories."""
    import flag_attn
    from flagattention_amd import _lib

    h, hk = heads
    g = torch.Generator().manual_seed(seqs)
    m = torch.randint(0, 4, (seqs,), generator=g)
    n = torch.randint(0, 7000, (seqs,), generator=g)
    n[::7] = 0
    n[3::11] = 1
    q = _randn((int(m.sum()), h, d), DTYPES[dtype], gpu_device, 0)
    gk = torch.Generator(device=gpu_device).manual_seed(seqs)
    k, v = (torch.randn((int(n.sum()), hk, d), generator=gk, device=gpu_device).to(DTYPES[dtype]) for _ in range(2))
    p = _lib.VarlenParams()
    for t, x in ((p.q, q), (p.k, k), (p.v, v), (p.out, q)):
        t.ptr, t.stride_h, t.stride_n = x.data_ptr(), x.stride(1), x.stride(0)
    p.cu_seqlens_q = p.cu_seqlens_k = 4096
    p.seqs, p.total_q, p.total_k, p.heads_q, p.heads_kv, p.head_dim = seqs, q.shape[0], k.shape[0], h, hk, d
    p.dtype, p.sm_scale = _lib.SAGE_BF16, 0.1
    cu_q, cu_k = _cu(m.tolist(), gpu_device), _cu(n.tolist(), gpu_device)
    for causal in (False, True):
        p.causal = int(causal)
        assert _lib.load().sage_flash_varlen_workspace_bytes(p) > 0
        o, norm = flag_attn.flash_attention_varlen(q, k, v, cu_q, cu_k, causal, return_log_normalizer=True)
        want, want_norm, tol, norm_tol = SO.varlen(q, k, v, cu_q, cu_k, causal)
        SO.assert_close(o, want, tol)
        SO.assert_close(norm, want_norm, norm_tol)


def _work(seed, device):
    """A cut packed call and a paged call in shares, on inputs of their own: a function without arguments, and its tensors."""
    import flag_attn

    q, k, v = (_randn((t, n, 128), torch.bfloat16, device, seed + i) for i, (t, n) in enumerate(((70, 8), (9000, 2), (9000, 2))))
    cu_q, cu_k = _cu((40, 30), device), _cu((3000, 6000), device)
    kc, vc, table, lens = _cache((5000 + seed, 900), 2, 16, 128, torch.bfloat16, "HND", device, 1300)
    q1 = _randn((2, 8, 128), torch.bfloat16, device, seed + 9)

    def work():
        return (flag_attn.flash_attention_varlen(q, k, v, cu_q, cu_k, True), flag_attn.paged_attention(q1, kc, vc, table, lens))

    return work, (q, q1)


def test_two_graphs_at_once(gpu_device):
    """Two captured graphs, each with partial results of its own, replayed at the same time on two streams, with eager calls between."""
    works = [_work(10 * i, gpu_device) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in works]
    for work, _ in works:
        work()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for work, _ in works:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work())
        graphs.append(g)
    for turn in range(4):
        for i, (work, inputs) in enumerate(works):
            for x in inputs:
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(100 * turn + i)))
        torch.cuda.synchronize()
        for _ in range(5):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        eager = [work() for work, _ in works]  # (beside the replays)
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_two_threads_at_once(gpu_device):
    """Calls of the same and of other shapes from two threads, a stream each."""
    import threading

    works = [_work(20 * i, gpu_device) for i in range(2)]
    want = [work() for work, _ in works]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got[i].append(works[i][0]())
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))
