"""The serving operators at the ends of their ranges, without a GPU."""
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHECKED = ("-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined")


def _run_check(name, flags, tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "check")
    subprocess.run(["g++", *flags, "-std=c++17", "-o", exe, os.path.join(ROOT, "tests", "csrc", name)], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


@pytest.mark.parametrize("flags", [("-O2",), CHECKED], ids=["plain", "checked"])
def test_lines_of_steps_of_long_sequences(flags, tmp_path):
    _run_check("long_lines_check.cpp", flags, tmp_path)


def test_steps_outside_a_line_belong_to_its_ends(tmp_path):
    """Offsets of packed sequences that overlap: what a kernel reads for a step that is not on its line has to exist."""
    _run_check("shares_check.cpp", CHECKED, tmp_path)


def test_rows_are_aligned_or_copied():
    """Contiguous tensors at odd storage offsets are copied; strides of dimensions with one entry are no strides."""
    from flagattention_amd import serving as S

    buf = torch.zeros(4 * 64 * 10 + 8, dtype=torch.bfloat16)
    t = buf[1:-7].view(10, 4, 64)
    assert t.is_contiguous() and t.data_ptr() % 16 == 2 and not S._aligned(t)
    c = S._rows16(t)
    assert c.data_ptr() % 16 == 0 and c.is_contiguous() and c.shape == t.shape
    one = torch.as_strided(buf, (1, 4, 64), (261, 64, 1))
    assert S._aligned(one) and S._rows16(one) is one
    d = S._token_desc(one)
    assert (d.stride_b, d.stride_h, d.stride_n) == (0, 64, 0)
    assert S._token_desc(torch.as_strided(buf, (3, 1, 64), (64, 3, 1))).stride_h == 0
    page = torch.as_strided(buf, (1, 1, 4, 64), (3, 5, 64, 1))
    assert S._aligned(page)
    for hnd, want in ((True, (0, 0, 64)), (False, (0, 64, 0))):
        d = S._cache_desc(page, hnd)
        assert (d.stride_b, d.stride_h, d.stride_n) == want
    assert not S._aligned(torch.as_strided(buf, (2, 4, 64), (260, 64, 1)))
    assert not S._aligned(torch.as_strided(buf, (2, 4, 64), (256, 64, 2)))
    assert S._aligned(torch.zeros(0, 4, 64)) and S._aligned(torch.zeros(3, 0, 64))


@pytest.mark.parametrize("causal", [False, True])
def test_the_oracle_is_torchs_attention(causal):
    """What the GPU tests compare with, against torch's attention in 64 bits (needs no compiler)."""
    from oracle import serving_oracle as SO

    m, n, h, hk, d = (1, 12, 0, 20), (30, 5, 4, 20), 4, 2, 8
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(sum(x), heads, d, generator=g).to(torch.float16) for x, heads in ((m, h), (n, hk), (n, hk)))
    cu_q, cu_k = (torch.tensor([0] + list(x)).cumsum(0) for x in (m, n))
    o, norm, _, _ = SO.varlen(q, k, v, cu_q, cu_k, causal)
    for s in range(len(m)):
        rows = slice(cu_q[s], cu_q[s + 1])
        qs, ks, vs = (x.double().transpose(0, 1) for x in (q[rows], k[cu_k[s]:cu_k[s + 1]], v[cu_k[s]:cu_k[s + 1]]))
        ks, vs = (x.repeat_interleave(h // hk, 0) for x in (ks, vs))
        sees = torch.ones(m[s], n[s], dtype=torch.bool).tril(n[s] - m[s]) if causal else torch.ones(m[s], n[s], dtype=torch.bool)
        want = torch.nn.functional.scaled_dot_product_attention(qs, ks, vs, attn_mask=sees).transpose(0, 1)
        want = torch.where(sees.any(1)[:, None, None], want, 0.0)  # (rows that see nothing are zeros here)
        logits = (qs @ ks.transpose(1, 2) * d ** -0.5).masked_fill(~sees, float("-inf"))
        assert torch.allclose(o[rows], want, rtol=1e-12, atol=1e-12)
        assert torch.allclose(norm[:, rows], torch.logsumexp(logits, -1), rtol=1e-12, atol=1e-12)


def _calls(grad=(), tangent=()):
    """A call of each operator on CPU tensors, those named with a gradient or a tangent: (function, arguments)."""
    import flag_attn
    from torch.autograd import forward_ad

    def t(name, *shape):
        x = torch.zeros(shape, dtype=torch.bfloat16)
        if name in tangent:
            x = forward_ad.make_dual(x, torch.ones_like(x))
        return x.requires_grad_() if name in grad else x

    cu, lens = torch.tensor([0, 5], dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    caches = {n: t(n, 4, 2, 16, 64) for n in ("k_cache", "v_cache")}
    return [
        (flag_attn.flash_attention_varlen, dict(q=t("q", 5, 4, 64), k=t("k", 5, 2, 64), v=t("v", 5, 2, 64), cu_seqlens_q=cu, out=t("out", 5, 4, 64))),
        (flag_attn.paged_attention, dict(q=t("q", 3, 4, 64), **caches, block_table=torch.zeros(3, 2, dtype=torch.int32), seq_lens=lens, out=t("out", 3, 4, 64))),
        (flag_attn.append_to_cache, dict(k=t("k", 5, 2, 64), v=t("v", 5, 2, 64), **caches, slots=torch.arange(5))),
        (flag_attn.copy_pages, dict(**caches, src=torch.tensor([0]), dst=torch.tensor([1]))),
    ]


@pytest.mark.parametrize("name", ["q", "k", "v", "k_cache", "v_cache", "out"])
def test_gradients_and_tangents_raise(name):
    """Nothing that takes part in differentiation, in either mode, is taken and dropped."""
    from torch.autograd import forward_ad

    for f, args in _calls(grad=(name,)):
        if name in args:
            with pytest.raises(NotImplementedError, match="no backward pass"):
                f(**args)
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
                f(**args)
    with forward_ad.dual_level():
        for f, args in _calls(tangent=(name,)):
            if name in args:
                with pytest.raises(NotImplementedError, match="tangents"):
                    f(**args)
        for f, args in _calls():
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                f(**args)
