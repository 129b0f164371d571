"""The serving operators without a GPU: refusals of the Python functions and of the C ABI, the layout of its structs, the workspace
of the paged attention, and the one use of m0 in the kernels that load straight into LDS."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sage_attention_hip.h")


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _varlen(**change):
    a = dict(q=_bf16(10, 4, 64), k=_bf16(12, 2, 64), v=_bf16(12, 2, 64), cu_seqlens_q=torch.tensor([0, 10], dtype=torch.int32),
             cu_seqlens_k=torch.tensor([0, 12], dtype=torch.int32))
    a.update(change)
    return a


def _paged(**change):
    a = dict(q=_bf16(3, 4, 64), k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64),
             block_table=torch.zeros(3, 4, dtype=torch.int32), seq_lens=torch.ones(3, dtype=torch.int32))
    a.update(change)
    return a


def _append(**change):
    a = dict(k=_bf16(7, 2, 64), v=_bf16(7, 2, 64), k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64), slots=torch.arange(7))
    a.update(change)
    return a


def _copy(**change):
    a = dict(k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64), src=torch.tensor([0]), dst=torch.tensor([1]))
    a.update(change)
    return a


REFUSALS = [
    # what, arguments, error, message
    ("flash_attention_varlen", _varlen(q=_bf16(1, 10, 4, 64)), ValueError, "tokens, heads"),
    ("flash_attention_varlen", _varlen(k=_bf16(12, 2, 128)), ValueError, "feature size"),
    ("flash_attention_varlen", _varlen(v=_bf16(12, 1, 64)), ValueError, "num of heads"),
    ("flash_attention_varlen", _varlen(q=_bf16(10, 5, 64)), ValueError, "multiple"),
    ("flash_attention_varlen", _varlen(v=_bf16(11, 2, 64)), ValueError, "number of tokens"),
    ("flash_attention_varlen", _varlen(q=_bf16(10, 4, 96), k=_bf16(12, 2, 96), v=_bf16(12, 2, 96)), NotImplementedError, "head_dim 96"),
    ("flash_attention_varlen", _varlen(q=_bf16(10, 4, 64).float()), TypeError, "float16"),
    ("flash_attention_varlen", _varlen(k=_bf16(12, 2, 64).half()), TypeError, "float16"),
    ("flash_attention_varlen", _varlen(cu_seqlens_q=torch.tensor([0, 10])), TypeError, "cu_seqlens_q must be an int32"),
    ("flash_attention_varlen", _varlen(cu_seqlens_k=torch.tensor([0, 5, 12], dtype=torch.int32)), ValueError, "one entry more"),
    ("flash_attention_varlen", _varlen(cu_seqlens_k=torch.tensor([[0, 12]], dtype=torch.int32)), ValueError, "dimension"),
    ("flash_attention_varlen", _varlen(q=_bf16(10, 4, 64).requires_grad_()), NotImplementedError, "no backward pass"),
    ("flash_attention_varlen", _varlen(), RuntimeError, "no CPU fallback"),
    ("paged_attention", _paged(q=_bf16(3, 64)), ValueError, "q must be"),
    ("paged_attention", _paged(k_cache=_bf16(5, 2, 16, 128)), ValueError, "same shape"),
    ("paged_attention", _paged(q=_bf16(3, 4, 128)), ValueError, "feature size"),
    ("paged_attention", _paged(q=_bf16(3, 3, 64)), ValueError, "multiple"),
    ("paged_attention", _paged(q=_bf16(3, 4, 32), k_cache=_bf16(5, 2, 16, 32), v_cache=_bf16(5, 2, 16, 32)), NotImplementedError, "head_dim 32"),
    ("paged_attention", _paged(q=_bf16(3, 4, 64).half()), TypeError, "float16"),
    ("paged_attention", _paged(block_table=torch.zeros(3, 4, dtype=torch.int64)), TypeError, "block_table must be an int32"),
    ("paged_attention", _paged(seq_lens=torch.ones(3, dtype=torch.int64)), TypeError, "seq_lens must be an int32"),
    ("paged_attention", _paged(block_table=torch.zeros(2, 4, dtype=torch.int32)), ValueError, "row for every sequence"),
    ("paged_attention", _paged(k_cache=_bf16(5, 2, 16, 65)[..., 1:], v_cache=_bf16(5, 2, 16, 65)[..., 1:]), ValueError, "not copied"),
    ("paged_attention", _paged(tensor_layout="NDH"), ValueError, "Unknown tensor layout"),
    ("paged_attention", _paged(q=_bf16(3, 4, 64).requires_grad_()), NotImplementedError, "no backward pass"),
    ("paged_attention", _paged(), RuntimeError, "no CPU fallback"),
    ("append_to_cache", _append(v=_bf16(6, 2, 64)), ValueError, "same shape"),
    ("append_to_cache", _append(k=_bf16(7, 1, 64), v=_bf16(7, 1, 64)), ValueError, "heads and head_dim"),
    ("append_to_cache", _append(k=_bf16(7, 2, 64).half()), TypeError, "share one"),
    ("append_to_cache", _append(slots=torch.arange(6)), ValueError, "entry for every token"),
    ("append_to_cache", _append(slots=torch.zeros(7)), TypeError, "int32 or int64"),
    ("append_to_cache", _append(slots=torch.zeros(7, 1, dtype=torch.int64)), ValueError, "one dimension"),
    ("append_to_cache", _append(k=_bf16(7, 2, 64).requires_grad_()), NotImplementedError, "no backward pass"),
    ("append_to_cache", _append(), RuntimeError, "no CPU fallback"),
    ("copy_pages", _copy(v_cache=_bf16(4, 2, 16, 64)), ValueError, "same shape"),
    ("copy_pages", _copy(k_cache=_bf16(5, 64), v_cache=_bf16(5, 64)), ValueError, "pages, "),
    ("copy_pages", _copy(dst=torch.tensor([1, 2])), ValueError, "same number"),
    ("copy_pages", _copy(src=torch.tensor([0.0])), TypeError, "src must be"),
    ("copy_pages", _copy(), RuntimeError, "no CPU fallback"),
]


@pytest.mark.parametrize("name,args,error,message", REFUSALS, ids=[f"{r[0]}-{i}" for i, r in enumerate(REFUSALS)])
def test_refusals(name, args, error, message):
    import flag_attn

    with pytest.raises(error, match=message):
        getattr(flag_attn, name)(**args)


def test_pages_in_one_piece():
    from flagattention_amd.serving import _page_bytes

    x = _bf16(5, 2, 16, 64)
    assert _page_bytes(x) == _page_bytes(x.transpose(1, 2)) == _page_bytes(x[::2]) == 2 * 16 * 64 * 2
    assert _page_bytes(x[:, :1]) == 16 * 64 * 2
    assert _page_bytes(x[:, :, ::2]) is None and _page_bytes(x[..., :32]) is None


def test_struct_layouts_match_header(tmp_path):
    from flagattention_amd import _lib

    if shutil.which("gcc") is None:
        pytest.skip("needs gcc for the offsetof check")
    structs = {"sage_varlen_params": _lib.VarlenParams, "sage_paged_params": _lib.PagedParams,
               "sage_append_params": _lib.AppendParams, "sage_copy_params": _lib.CopyParams}
    lines = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{n} %zu\\n", offsetof({cname}, {n}));' for n, _ in cls._fields_]
    src = tmp_path / "off.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "off"), str(src)], check=True)
    out = subprocess.run([str(tmp_path / "off")], capture_output=True, text=True, check=True).stdout
    seen = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for cname, cls in structs.items():
        assert int(seen[cname]) == ctypes.sizeof(cls)
        for n, _ in cls._fields_:
            assert int(seen[f"{cname}.{n}"]) == getattr(cls, n).offset, (cname, n)


def test_lines_of_steps(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-o", exe, os.path.join(ROOT, "tests", "csrc", "step_lines_check.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout


def _varlen_params():
    from flagattention_amd import _lib

    p = _lib.VarlenParams()
    for t, heads in ((p.q, 8), (p.k, 2), (p.v, 2), (p.out, 8)):
        t.ptr, t.stride_h, t.stride_n = 4096, 128, heads * 128
    p.cu_seqlens_q = p.cu_seqlens_k = 4096
    p.seqs, p.total_q, p.total_k, p.heads_q, p.heads_kv, p.head_dim = 2, 100, 100, 8, 2, 128
    p.dtype, p.sm_scale = _lib.SAGE_BF16, 0.1
    return p


def _paged_params(seqs=4, width=1000, page=16):
    from flagattention_amd import _lib

    p = _lib.PagedParams()
    for t in (p.q, p.out, p.k_cache, p.v_cache):
        t.ptr, t.stride_b, t.stride_h, t.stride_n = 4096, 8 * page * 128, page * 128, 128
    p.block_table = p.seq_lens = 4096
    p.table_stride = p.table_width = width
    p.seqs, p.new_tokens, p.heads_q, p.heads_kv, p.head_dim = seqs, 1, 32, 8, 128
    p.pages, p.page_size, p.dtype, p.sm_scale = 10000, page, _lib.SAGE_BF16, 0.1
    return p


@pytest.mark.parametrize("field,value,status,message", [
    ("head_dim", 96, -2, b"head_dim 96"), ("heads_kv", 3, -1, b"multiple of heads_kv"), ("dtype", 2, -2, b"fp16 or bf16"),
    ("sm_scale", 0.0, -1, b"sm_scale"), ("sm_scale", float("nan"), -1, b"sm_scale"), ("total_q", -1, -1, b"negative"),
    ("cu_seqlens_q", None, -1, b"null"), ("total_q", 1 << 29, -2, b"2^30"), ("seqs", 1 << 30, -2, b"2^30")])
def test_varlen_validation(field, value, status, message):
    from flagattention_amd import _lib

    lib, p = _lib.load(), _varlen_params()
    setattr(p, field, value)
    assert lib.sage_flash_varlen_fwd(p, None, 0, None) == status and message in lib.sage_hip_last_error()
    assert lib.sage_flash_varlen_fwd(None, None, 0, None) == -1


def test_varlen_validation_of_rows():
    from flagattention_amd import _lib

    lib = _lib.load()
    for name, part, value, status in (("q", "ptr", 4104, -1), ("out", "stride_h", 100, -1), ("k", "stride_n", 4, -1),
                                      ("v", "stride_n", 1 << 24, -2), ("v", "ptr", None, -1)):
        p = _varlen_params()
        setattr(getattr(p, name), part, value)
        assert lib.sage_flash_varlen_fwd(p, None, 0, None) == status, (name, part)
    for empty in ("seqs", "total_q"):  # nothing to compute, nothing launched
        p = _varlen_params()
        setattr(p, empty, 0)
        assert lib.sage_flash_varlen_fwd(p, None, 0, None) == 0


@pytest.mark.parametrize("field,value,status,message", [
    ("head_dim", 32, -2, b"head_dim 32"), ("page_size", 0, -1, b"page_size"), ("pages", 0, -1, b"without pages"),
    ("table_width", 0, -1, b"without"), ("new_tokens", -1, -1, b"negative"), ("block_table", None, -1, b"null"),
    ("pages", 1 << 30, -2, b"2^30"), ("new_tokens", 1 << 29, -2, b"2^30")])
def test_paged_validation(field, value, status, message):
    from flagattention_amd import _lib

    lib, p = _lib.load(), _paged_params()
    setattr(p, field, value)
    assert lib.sage_paged_attn(p, None, 0, None) == status and message in lib.sage_hip_last_error()
    assert lib.sage_paged_attn_workspace_bytes(p) == -1


def test_paged_validation_of_rows():
    from flagattention_amd import _lib

    lib = _lib.load()
    for name, part, value, status in (("q", "ptr", 4104, -1), ("out", "stride_b", 100, -1), ("k_cache", "stride_b", 4, -1),
                                      ("v_cache", "stride_n", 1 << 27, -2), ("v_cache", "ptr", None, -1)):
        p = _paged_params()
        setattr(getattr(p, name), part, value)
        assert lib.sage_paged_attn(p, None, 0, None) == status, (name, part)


def test_paged_workspace():
    """Long tables share their keys out and need room for two partial results per workgroup; short ones need none."""
    from flagattention_amd import _lib

    lib = _lib.load()
    assert lib.sage_paged_attn_workspace_bytes(_paged_params(width=8)) == 0
    n = lib.sage_paged_attn_workspace_bytes(_paged_params())
    assert n > 0 and n % (4 * (128 + 1) * 4) == 0  # four rows of 128 channels and a log-sum-exp each
    assert lib.sage_paged_attn_workspace_bytes(_paged_params(seqs=90)) == lib.sage_paged_attn_workspace_bytes(_paged_params(seqs=40))
    assert lib.sage_paged_attn_workspace_bytes(_paged_params(seqs=4000)) == 0  # (enough of them for a workgroup each)
    p = _paged_params()
    assert lib.sage_paged_attn(p, None, 16, None) == -1 and lib.sage_paged_attn(p, 4100, n, None) == -1
    p.seqs = 0
    assert lib.sage_paged_attn(p, None, 0, None) == 0 and lib.sage_paged_attn_workspace_bytes(p) == 0


def test_varlen_workspace():
    """Few blocks against many keys are cut into equal shares: two partial results of 128 rows for each of 512 workgroups."""
    from flagattention_amd import _lib

    lib, p = _lib.load(), _varlen_params()
    assert lib.sage_flash_varlen_workspace_bytes(p) == 0
    p.total_q, p.total_k, p.seqs = 512, 17000, 1
    assert lib.sage_flash_varlen_workspace_bytes(p) == 2 * 512 * 128 * (128 + 1) * 4
    assert lib.sage_flash_varlen_fwd(p, None, 16, None) == -1 and lib.sage_flash_varlen_fwd(p, 4100, 1 << 30, None) == -1
    p.total_q = 17000
    assert lib.sage_flash_varlen_workspace_bytes(p) == 0
    p.heads_q, p.heads_kv, p.total_q = 256, 1, 512  # (a query's rows do not fit a block)
    assert lib.sage_flash_varlen_workspace_bytes(p) == 0
    p.head_dim = 96
    assert lib.sage_flash_varlen_workspace_bytes(p) == -1


def test_launches_too_large():
    """Calls whose workgroups would need more than 2^32 threads are refused before any launch."""
    from flagattention_amd import _lib

    lib = _lib.load()
    p = _varlen_params()
    p.seqs, p.total_q, p.total_k, p.heads_kv, p.heads_q = 5, 1 << 29, 1 << 29, 32, 32
    assert lib.sage_flash_varlen_fwd(p, None, 0, None) == -2 and b"too many workgroups" in lib.sage_hip_last_error()
    p = _paged_params(seqs=1 << 22)
    assert lib.sage_paged_attn_workspace_bytes(p) == 0
    assert lib.sage_paged_attn(p, None, 0, None) == -2 and b"too many workgroups" in lib.sage_hip_last_error()
    p.seqs, p.new_tokens = 1 << 29, 1 << 20
    assert lib.sage_paged_attn(p, None, 0, None) == -2 and b"2^40" in lib.sage_hip_last_error()
    p = _lib.AppendParams()
    for t in (p.k, p.v, p.k_cache, p.v_cache):
        t.ptr, t.stride_b, t.stride_h, t.stride_n = 4096, 1024, 64, 128
    p.page_size, p.tokens, p.heads_kv, p.head_dim, p.pages, p.slots = 16, 1 << 29, 1 << 16, 128, 4, 4096
    p.dtype = _lib.SAGE_BF16
    assert lib.sage_cache_append(p, None) == -2 and b"too many rows" in lib.sage_hip_last_error()


def test_cache_movement_validation():
    from flagattention_amd import _lib

    lib = _lib.load()
    p = _lib.AppendParams()
    assert lib.sage_cache_append(None, None) == -1 and lib.sage_cache_append(p, None) == -1  # (page_size 0)
    for t in (p.k, p.v, p.k_cache, p.v_cache):
        t.ptr, t.stride_b, t.stride_h, t.stride_n = 4096, 1024, 64, 128
    p.page_size, p.tokens, p.heads_kv, p.head_dim, p.pages, p.slots = 16, 0, 2, 64, 4, 4096
    assert lib.sage_cache_append(p, None) == 0
    p.tokens, p.head_dim = 3, 60
    assert lib.sage_cache_append(p, None) == -1 and b"16 bytes" in lib.sage_hip_last_error()
    p.head_dim, p.slots = 64, None
    assert lib.sage_cache_append(p, None) == -1 and b"null" in lib.sage_hip_last_error()
    c = _lib.CopyParams()
    assert lib.sage_cache_copy_pages(None, None) == -1 and lib.sage_cache_copy_pages(c, None) == 0
    c.count = c.layers = c.pages = 1
    c.page_bytes = 24
    c.k_cache = c.v_cache = c.src = c.dst = 4096
    assert lib.sage_cache_copy_pages(c, None) == -1 and b"16 bytes" in lib.sage_hip_last_error()
    c.page_bytes, c.src = 32, None
    assert lib.sage_cache_copy_pages(c, None) == -1 and b"null" in lib.sage_hip_last_error()


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
@pytest.mark.parametrize("causal", [False, True])
def test_the_oracle_agrees_with_torch_in_64_bits(causal):
    """The formulas that the GPU tests compare with, against torch's attention sequence by sequence, packed and in pages."""
    from oracle import serving_oracle as SO

    m, n, h, hk, d, page = (5, 0, 17), (9, 3, 17), 6, 2, 16, 4
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(t, heads, d, generator=g).to(torch.bfloat16) for t, heads in ((sum(m), h), (sum(n), hk), (sum(n), hk)))
    cu_q, cu_k = (torch.tensor([0] + list(x)).cumsum(0).to(torch.int32) for x in (m, n))
    o, norm, _, _ = SO.varlen(q, k, v, cu_q, cu_k, causal)
    for s in range(len(m)):
        qs, ks, vs = (x[cu[s]:cu[s + 1]].double().transpose(0, 1) for x, cu in ((q, cu_q), (k, cu_k), (v, cu_k)))
        ks, vs = (x.repeat_interleave(h // hk, 0) for x in (ks, vs))
        sees = torch.ones(m[s], n[s], dtype=torch.bool).tril(n[s] - m[s]) if causal else torch.ones(m[s], n[s], dtype=torch.bool)
        want = torch.nn.functional.scaled_dot_product_attention(qs[None], ks[None], vs[None], attn_mask=sees)[0].transpose(0, 1)
        logits = (qs @ ks.transpose(1, 2) * d ** -0.5).masked_fill(~sees, float("-inf"))
        rows = slice(cu_q[s], cu_q[s + 1])
        assert torch.allclose(o[rows], want, rtol=1e-12, atol=1e-12)
        assert torch.allclose(norm[:, rows], torch.logsumexp(logits, -1), rtol=1e-12, atol=1e-12)
        if not causal or m[s] == 0:
            continue
        # the same keys in pages, in an order of their own
        table = torch.randperm(8, generator=g)[: -(-n[s] // page)].to(torch.int32)
        caches = [torch.full((8, page, hk, d), float("nan"), dtype=torch.bfloat16) for _ in range(2)]
        for c, x in zip(caches, (k, v)):
            for j in range(n[s]):
                c[table[j // page], j % page] = x[cu_k[s] + j]
        paged = SO.paged(q[rows][None], *caches, table[None], torch.tensor([n[s]]), layout="NHD")
        assert torch.allclose(paged[0][0], want, rtol=1e-12, atol=1e-12) and torch.allclose(paged[1][0], norm[:, rows])


def test_only_the_lds_load_sequence_touches_m0(tmp_path):
    """The packed forward sets m0 in inline assembly, which the compiler cannot be told about: in its assembly m0 appears
    only as the destination of the move that precedes each direct-to-LDS load."""
    out = tmp_path / "varlen.s"
    subprocess.run(["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950", "-ffp-contract=off", "-Xclang", "-target-feature",
                    "-Xclang", "-packed-fp32-ops", "-S", "--cuda-device-only", "-o", str(out),
                    os.path.join(ROOT, "flagattention_amd", "csrc", "flash_varlen.hip")], check=True, capture_output=True, timeout=600)
    lines = [ln.split(";")[0].strip() for ln in out.read_text().splitlines()]
    lines = [ln for ln in lines if ln and not ln.startswith((".", "s_nop"))]
    mentions = [ln for ln in lines if re.search(r"\bm0\b", ln)]
    loads = [i for i, ln in enumerate(lines) if ln.startswith("global_load_lds_")]
    assert loads and len(loads) == len(mentions)
    for i in loads:
        assert re.fullmatch(r"s_mov_b32 m0, s\d+", lines[i - 1]), lines[i - 1]
