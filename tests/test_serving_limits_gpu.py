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
