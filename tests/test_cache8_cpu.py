"""The cache of 8-bit codes without a GPU: refusals of the Python functions and of the C ABI, the layout of its structs, its workspaces, and the
oracle that the GPU tests compare with."""
import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

from oracle import cache8_oracle as CO

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "sage_attention_hip.h")


def _codes(*shape):
    return torch.zeros(shape, dtype=torch.int8)


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _scales(**change):
    return {**dict(k_scale=torch.zeros(5, 2, 4), v_scale=torch.zeros(5, 2, 4)), **change}


def _paged(**change):
    a = dict(q=_bf16(3, 4, 64), k_cache=_codes(5, 2, 16, 64), v_cache=_codes(5, 2, 16, 64),
             block_table=torch.zeros(3, 4, dtype=torch.int32), seq_lens=torch.ones(3, dtype=torch.int32), **_scales())
    return {**a, **change}


def _append(**change):
    a = dict(k=_bf16(7, 2, 64), v=_bf16(7, 2, 64), k_cache=_codes(5, 2, 16, 64), v_cache=_codes(5, 2, 16, 64), slots=torch.arange(7), **_scales())
    return {**a, **change}


def _read(**change):
    a = dict(k_cache=_codes(5, 2, 16, 64), v_cache=_codes(5, 2, 16, 64), block_table=torch.zeros(3, 4, dtype=torch.int32),
             cu_seqlens=torch.zeros(4, dtype=torch.int32), total=9, **_scales())
    return {**a, **change}


def _copy(**change):
    a = dict(k_cache=_codes(5, 2, 16, 64), v_cache=_codes(5, 2, 16, 64), src=torch.tensor([0]), dst=torch.tensor([1]), **_scales())
    return {**a, **change}


REFUSALS = [
    ("paged_attention", _paged(k_scale=None), ValueError, "go together"),
    ("paged_attention", _paged(k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64)), TypeError, "int8 / torch.float8_e4m3fn"),
    ("paged_attention", _paged(v_cache=_codes(5, 2, 16, 64).view(torch.float8_e4m3fn)), TypeError, "share one"),
    ("paged_attention", _paged(k_scale=None, v_scale=None), TypeError, "share one of torch.float16"),
    ("paged_attention", _paged(q=torch.zeros(3, 4, 64)), TypeError, "float16"),
    ("paged_attention", _paged(k_scale=torch.zeros(5, 2, 4).half()), TypeError, "k_scale must be a float32"),
    ("paged_attention", _paged(v_scale=torch.zeros(5, 1, 4)), ValueError, "v_scale must be"),
    ("paged_attention", _paged(**_scales(k_scale=torch.zeros(5, 2, 3), v_scale=torch.zeros(5, 2, 3))), ValueError, "divisor of the page size"),
    ("paged_attention", _paged(v_scale=torch.zeros(5, 2, 8)), ValueError, "as many blocks"),
    ("paged_attention", _paged(**_scales(k_scale=torch.zeros(5, 2, 0), v_scale=torch.zeros(5, 2, 0))), ValueError, "divisor of the page size"),
    ("paged_attention", _paged(q=_bf16(3, 4, 32), k_cache=_codes(5, 2, 16, 32), v_cache=_codes(5, 2, 16, 32)), NotImplementedError, "head_dim 32"),
    ("paged_attention", _paged(k_cache=_codes(5, 2, 16, 72)[..., :64], v_cache=_codes(5, 2, 16, 72)[..., :64]), ValueError, "not copied"),
    ("paged_attention", _paged(k_scale=torch.zeros(5, 2, 4, requires_grad=True)), NotImplementedError, "no backward pass"),
    ("paged_attention", _paged(), RuntimeError, "no CPU fallback"),
    ("append_to_cache", _append(v_scale=None), ValueError, "go together"),
    ("append_to_cache", _append(k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64)), TypeError, "int8 / torch.float8_e4m3fn"),
    ("append_to_cache", _append(k=_bf16(7, 2, 64).half()), TypeError, "k and v must share"),
    ("append_to_cache", _append(k=_codes(7, 2, 64), v=_codes(7, 2, 64)), TypeError, "k and v must share"),
    ("append_to_cache", _append(k_scale=torch.zeros(5, 2, 1).expand(5, 2, 4)), ValueError, "k_scale: entries share memory"),
    ("append_to_cache", _append(k_scale=torch.zeros(5, 3, 4)), ValueError, "k_scale must be"),
    ("append_to_cache", _append(v_scale=torch.zeros(5, 2, 4, requires_grad=True)), NotImplementedError, "no backward pass"),
    ("append_to_cache", _append(), RuntimeError, "no CPU fallback"),
    ("read_cache", _read(v_scale=None), ValueError, "go together"),
    ("read_cache", _read(dtype=torch.int8), TypeError, "dtype must be"),
    ("read_cache", _read(k_scale=None, v_scale=None, k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64), dtype=torch.float16), TypeError, "dtype that is asked for"),
    ("read_cache", _read(k_scale=None, v_scale=None), TypeError, "dtype must be"),
    ("read_cache", _read(cu_seqlens=torch.zeros(3, dtype=torch.int32)), ValueError, "one entry more"),
    ("read_cache", _read(cu_seqlens=torch.zeros(4, dtype=torch.int64)), TypeError, "cu_seqlens must be an int32"),
    ("read_cache", _read(total=-1), ValueError, "number of rows"),
    ("read_cache", _read(total=2.0), ValueError, "number of rows"),
    ("read_cache", _read(out=_bf16(9, 2, 64)), ValueError, "pair"),
    ("read_cache", _read(k_cache=_codes(5, 2, 0, 64), v_cache=_codes(5, 2, 0, 64)), ValueError, "page_size"),
    ("read_cache", _read(), RuntimeError, "no CPU fallback"),
    ("copy_pages", _copy(k_scale=None), ValueError, "go together"),
    ("copy_pages", _copy(k_cache=_bf16(5, 2, 16, 64), v_cache=_bf16(5, 2, 16, 64)), TypeError, "int8 / torch.float8_e4m3fn"),
    ("copy_pages", _copy(k_scale=torch.zeros(4, 2, 4)), ValueError, "k_scale must be"),
    ("copy_pages", _copy(v_scale=torch.zeros(5, 2, 8)), ValueError, "v_scale must be"),
    ("copy_pages", _copy(k_scale=torch.zeros(5, 2, 4).double()), TypeError, "float32"),
    ("copy_pages", _copy(), RuntimeError, "no CPU fallback"),
]


@pytest.mark.parametrize("name,args,error,message", REFUSALS, ids=[f"{r[0]}-{i}" for i, r in enumerate(REFUSALS)])
def test_refusals(name, args, error, message):
    import flag_attn

    with pytest.raises(error, match=re.escape(message)):
        getattr(flag_attn, name)(**args)


def test_struct_layouts_match_header(tmp_path):
    from flagattention_amd import _lib

    if shutil.which("gcc") is None:
        pytest.skip("needs gcc for the offsetof check")
    structs = {"sage_cache_scales": _lib.CacheScales, "sage_paged8_params": _lib.Paged8Params, "sage_append8_params": _lib.Append8Params,
               "sage_read_params": _lib.ReadParams, "sage_copy8_params": _lib.Copy8Params}
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


def _fill_scales(s, blocks=4):
    s.k = s.v = 4096
    s.k_stride_page = s.v_stride_page = 2 * blocks
    s.k_stride_head = s.v_stride_head = blocks
    s.k_stride_block = s.v_stride_block = 1
    s.blocks, s.codes = blocks, 0


def _paged_params(seqs=4, width=1000, page=16):
    from flagattention_amd import _lib

    p8 = _lib.Paged8Params()
    p = p8.paged
    for t in (p.q, p.out, p.k_cache, p.v_cache):
        t.ptr, t.stride_b, t.stride_h, t.stride_n = 4096, 8 * page * 128, page * 128, 128
    p.block_table = p.seq_lens = 4096
    p.table_stride = p.table_width = width
    p.seqs, p.new_tokens, p.heads_q, p.heads_kv, p.head_dim = seqs, 1, 32, 8, 128
    p.pages, p.page_size, p.dtype, p.sm_scale = 10000, page, _lib.SAGE_BF16, 0.1
    _fill_scales(p8.scales)
    return p8


@pytest.mark.parametrize("field,value,status,message", [
    ("codes", 2, -1, b"unknown kind"), ("codes", -1, -1, b"unknown kind"), ("blocks", 0, -1, b"divide"), ("blocks", 3, -1, b"divide"),
    ("k", None, -1, b"null scales"), ("v", None, -1, b"null scales"), ("k_stride_page", -1, -2, b"strides"), ("v_stride_block", 1 << 31, -2, b"strides")])
def test_scales_are_checked(field, value, status, message):
    from flagattention_amd import _lib

    lib = _lib.load()
    p = _paged_params()
    setattr(p.scales, field, value)
    assert lib.sage_paged8_attn(p, None, 0, None) == status and message in lib.sage_hip_last_error()
    assert lib.sage_paged8_attn_workspace_bytes(p) == -1
    a = _append_params()
    setattr(a.scales, field, value)
    assert lib.sage_cache8_append(a, None, 0, None) == status and message in lib.sage_hip_last_error()
    if field != "codes" or value != -1:  # (a cache without scales)
        r = _read_params()
        setattr(r.scales, field, value)
        assert lib.sage_cache_read(r, None) == status and message in lib.sage_hip_last_error()


def test_paged_checks():
    from flagattention_amd import _lib

    lib = _lib.load()
    for name, part, value, status in (("q", "ptr", 4104, -1), ("k_cache", "stride_n", 8, -1), ("k_cache", "stride_b", 16 * 128 + 8, -1),
                                      ("v_cache", "stride_n", 1 << 27, -2), ("v_cache", "ptr", None, -1)):
        p = _paged_params()
        setattr(getattr(p.paged, name), part, value)
        assert lib.sage_paged8_attn(p, None, 0, None) == status, (name, part)
    for field, value, status in (("head_dim", 32, -2), ("pages", 0, -1), ("page_size", 0, -1), ("seqs", -1, -1), ("dtype", 2, -2)):
        p = _paged_params()
        setattr(p.paged, field, value)
        assert lib.sage_paged8_attn(p, None, 0, None) == status, field
    assert lib.sage_paged8_attn(None, None, 0, None) == -1
    assert lib.sage_paged8_attn_workspace_bytes(_paged_params(width=8)) == 0
    n = lib.sage_paged8_attn_workspace_bytes(_paged_params())
    assert n > 0 and n % (4 * (128 + 1) * 4) == 0
    p = _paged_params()
    assert lib.sage_paged8_attn(p, None, 16, None) == -1 and lib.sage_paged8_attn(p, 4100, n, None) == -1
    p = _paged_params(seqs=1 << 22)
    assert lib.sage_paged8_attn(p, None, 0, None) == -2 and b"too many workgroups" in lib.sage_hip_last_error()
    p.paged.seqs = 0
    assert lib.sage_paged8_attn(p, None, 0, None) == 0 and lib.sage_paged8_attn_workspace_bytes(p) == 0


def _append_params(tokens=3, blocks=4, pages=4):
    from flagattention_amd import _lib

    p8 = _lib.Append8Params()
    p = p8.append
    for t in (p.k, p.v, p.k_cache, p.v_cache):
        t.ptr, t.stride_b, t.stride_h, t.stride_n = 4096, 1024, 64, 128
    p.page_size, p.tokens, p.heads_kv, p.head_dim, p.pages, p.slots, p.dtype = 16, tokens, 2, 64, pages, 4096, _lib.SAGE_BF16
    _fill_scales(p8.scales, blocks)
    return p8


def test_append_checks():
    from flagattention_amd import _lib

    lib = _lib.load()
    assert lib.sage_cache8_append(None, None, 0, None) == -1
    for field, value, status, message in (("head_dim", 72, -1, b"16 bytes"), ("head_dim", 528, -2, b"512"), ("slots", None, -1, b"null"), ("tokens", -1, -1, b"negative"),
                                          ("pages", 1 << 30, -2, b"2^30"), ("dtype", 7, -1, b"dtype"), ("page_size", 0, -1, b"page_size")):
        p = _append_params()
        setattr(p.append, field, value)
        assert lib.sage_cache8_append(p, None, 0, None) == status and message in lib.sage_hip_last_error(), field
    p = _append_params()
    p.append.page_size, p.scales.blocks = 4096, 2
    assert lib.sage_cache8_append(p, None, 0, None) == -2 and b"1024" in lib.sage_hip_last_error()
    # few tokens, or a scale for each: no workspace; many: a word for every slot of the cache, and a refusal without
    assert lib.sage_cache8_append_workspace_bytes(_append_params(tokens=256)) == 0
    assert lib.sage_cache8_append_workspace_bytes(_append_params(tokens=100000, blocks=16)) == 0
    p = _append_params(tokens=257)
    assert lib.sage_cache8_append_workspace_bytes(p) == 4 * 16 * 4
    assert lib.sage_cache8_append(p, None, 0, None) == -1 and b"workspace" in lib.sage_hip_last_error()
    assert lib.sage_cache8_append(p, 4096, 128, None) == -1 and b"needs a workspace" in lib.sage_hip_last_error()
    p = _append_params(tokens=257, pages=(1 << 28) + 1)
    assert lib.sage_cache8_append_workspace_bytes(p) == -1 and b"2^32" in lib.sage_hip_last_error()
    p = _append_params(tokens=1 << 29, blocks=16)
    p.append.heads_kv = 1 << 16
    assert lib.sage_cache8_append(p, None, 0, None) == -2 and b"too many rows" in lib.sage_hip_last_error()
    p = _append_params(tokens=0)
    assert lib.sage_cache8_append(p, None, 0, None) == 0


def _read_params():
    from flagattention_amd import _lib

    p = _lib.ReadParams()
    for t in (p.k_cache, p.v_cache, p.k_out, p.v_out):
        t.ptr, t.stride_b, t.stride_h, t.stride_n = 4096, 2048, 64, 128
    p.block_table = p.cu_seqlens = 4096
    p.table_stride = p.table_width = 8
    p.seqs, p.total, p.heads_kv, p.head_dim, p.pages, p.page_size, p.out_dtype = 2, 50, 2, 64, 10, 16, _lib.SAGE_BF16
    _fill_scales(p.scales)
    return p


def test_read_and_copy_checks():
    from flagattention_amd import _lib

    lib = _lib.load()
    assert lib.sage_cache_read(None, None) == -1
    for field, value, status in (("total", -1, -1), ("page_size", 0, -1), ("out_dtype", 9, -1), ("head_dim", 56, -1), ("block_table", None, -1), ("cu_seqlens", None, -1),
                                 ("total", 1 << 30, -2), ("head_dim", 8192, -2)):
        p = _read_params()
        setattr(p, field, value)
        assert lib.sage_cache_read(p, None) == status, field
    for name, part, value in (("k_cache", "stride_n", 72), ("k_out", "stride_h", 4), ("v_out", "ptr", 4104), ("v_out", "ptr", None)):
        p = _read_params()
        setattr(getattr(p, name), part, value)
        assert lib.sage_cache_read(p, None) == -1, (name, part)
    p = _read_params()
    p.total = 0
    assert lib.sage_cache_read(p, None) == 0
    c = _lib.Copy8Params()
    assert lib.sage_cache8_copy_pages(None, None) == -1 and lib.sage_cache8_copy_pages(c, None) == 0
    c.copy.count = c.copy.layers = c.copy.pages = 1
    c.copy.page_bytes = 32
    c.copy.k_cache = c.copy.v_cache = c.copy.src = c.copy.dst = 4096
    assert lib.sage_cache8_copy_pages(c, None) == -1 and b"null scales" in lib.sage_hip_last_error()
    c.scale_words = -1
    assert lib.sage_cache8_copy_pages(c, None) == -1 and b"negative" in lib.sage_hip_last_error()


# ---- the oracle

def test_the_numbers_of_e4m3():
    bits = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert torch.equal(bits.float().double(), CO.e4m3_numbers())


def test_nearest_codes():
    """Against all codes, by distance and then evenness."""
    g = torch.Generator().manual_seed(0)
    grid = CO.e4m3_numbers()
    x = torch.cat([torch.randn(4000, generator=g).double() * 100, (grid[:-1] + grid[1:]) / 2, grid, torch.randn(1000, generator=g).double() * 2.0 ** -8]).clamp(-448, 448)
    codes = torch.cat([grid, -grid[1:]])
    even = torch.cat([torch.arange(127), torch.arange(1, 127)]) % 2 == 0
    away = (x[:, None] - codes).abs()
    best = away.min(dim=1, keepdim=True).values
    pick = torch.where((away == best) & even, 2, (away == best).long()).argmax(dim=1)  # of those as near, an even one
    assert torch.equal(CO.nearest(x, torch.float8_e4m3fn).abs(), codes[pick].abs())
    assert CO.nearest(torch.tensor([0.5, 1.5, -2.5, 126.5]).double(), torch.int8).tolist() == [0, 2, -2, 126]


@pytest.mark.parametrize("codes,top", [(torch.int8, 127), (torch.float8_e4m3fn, 448)])
def test_append_of_the_oracle(codes, top):
    """By hand: a block begun, one that goes on with a larger token, one with a smaller one; what a code stands for is off by half a step."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 1, 16, generator=g)
    x[0] *= 4 / x[0].abs().max()
    x[1] *= 1 / x[1].abs().max()
    x[2] *= 8 / x[2].abs().max()
    empty = (torch.zeros(1, 1, 4, 16, dtype=torch.int8).view(codes), torch.zeros(1, 1, 4, 16, dtype=torch.int8).view(codes), torch.full((1, 1, 1), 99.0), torch.full((1, 1, 1), 99.0))
    state = empty
    for i, largest in ((0, 4), (1, 4), (2, 8)):
        state = CO.append(x[i:i + 1], -x[i:i + 1], state[0], state[1], torch.tensor([i]), state[2], state[3])
        assert float(state[2]) == float(torch.tensor(largest / top, dtype=torch.float64).float()) == float(state[3])
        step = float(state[2]) if codes == torch.int8 else largest / 14  # e4m3: 32 / 448 of the largest
        for j in range(i + 1):
            off = (CO.values(state[0], state[2])[0, j, 0] - x[j, 0].double()).abs().max()
            assert off <= (1.01 if j < i else 0.51) * step
    again = CO.append(x[1:2], x[1:2], state[0], state[1], torch.tensor([0]), state[2], state[3])
    assert float(again[2]) == float(torch.tensor(1 / top, dtype=torch.float64).float()) and not CO.numbers(again[0])[0, 0, 1:].any()
    bad = CO.append(torch.full((1, 1, 16), math.inf), x[1:2], state[0], state[1], torch.tensor([3]), state[2], state[3])
    assert torch.isnan(bad[2]).all() and not torch.isnan(bad[3]).any()


def test_attention_of_the_oracle():
    """With scales of one and small codes, the oracle of 16-bit caches."""
    from oracle import serving_oracle as SO

    g = torch.Generator().manual_seed(2)
    k, v = (torch.randint(-3, 4, (4, 2, 8, 16), generator=g).to(torch.int8) for _ in range(2))
    ones = torch.ones(4, 2, 2)
    q = torch.randn(2, 3, 4, 16, generator=g).half()
    table, lens = torch.tensor([[2, 0, 1], [3, 7, 0]], dtype=torch.int32), torch.tensor([20, 12])
    a = CO.paged(q, k, v, ones, ones, table, lens)
    b = SO.paged(q, k.half(), v.half(), table, lens)
    assert torch.allclose(a[0], b[0], rtol=1e-12, atol=1e-12) and torch.allclose(a[1], b[1], rtol=1e-12)
    half = CO.paged(q, k, v, ones / 2, ones * 3, table, lens, sm_scale=0.5)
    same = SO.paged(q, k.half(), v.half() * 3, table, lens, sm_scale=0.25)
    assert torch.allclose(half[0], same[0], rtol=1e-12, atol=1e-12)


# ---- the line of shares with units before an item's chunks (the arithmetic of paged_common.h, restated)

def _shares_of(chunks, per_seq, shares, start):
    """Every chunk of every item is in one piece, pieces of cut items have slots of their own, and the joining kernel looks for
    them where they are; one cut is responsible for each cut item."""
    units = [start + c for c in chunks]
    total = sum(units) * per_seq
    base, rest = divmod(total, shares)

    def begin_of(w):
        return w * base + min(w, rest)

    def owner(pos):
        pos = max(min(pos, total - 1), 0)
        longer = rest * (base + 1)
        return pos // (base + 1) if pos < longer else rest + (pos - longer) // base

    slots, pieces = {}, {}
    for w in range(shares):
        pos, end = begin_of(w), begin_of(w + 1)
        if pos >= end:
            continue
        share_begin, seq, seq_begin = pos, 0, 0
        while seq_begin + units[seq] * per_seq <= pos:
            seq_begin += units[seq] * per_seq
            seq += 1
        while pos < end:
            s, u = seq, units[seq]
            item = (pos - seq_begin) // u
            begin = seq_begin + item * u
            to = min(begin + u, end)
            first = max(pos - begin - start, 0)
            n = max(to - begin - start, 0) - first
            pos = to
            if pos - seq_begin == u * per_seq:
                seq_begin, seq = pos, seq + 1
            if n == 0:
                continue
            pieces.setdefault((s, item), []).append((first, n))
            if n != chunks[s]:
                slot = 2 * w + (begin > share_begin)
                assert slot not in slots
                slots[slot] = (s, item)
    begin, joined = 0, set()
    for s, u in enumerate(units):
        for item in range(per_seq):
            got = pieces[s, item]
            assert got[0][0] == 0 and sum(n for _, n in got) == chunks[s] and all(a[0] + a[1] == b[0] for a, b in zip(got, got[1:]))
            first, last = owner(begin + start), owner(begin + u - 1)
            assert (first == last) == (len(got) == 1)
            if first != last:
                for w in range(first, last + 1):
                    slot = 2 * w + (w == first and begin > begin_of(w))
                    assert slots[slot] == (s, item)
                    joined.add(slot)
                cuts = [w for w in range(shares - 1) if begin_of(w + 1) < begin_of(w + 2) and begin <= begin_of(w + 1) < begin + u and first == w]
                assert len(cuts) == 1
            begin += u
    assert joined == set(slots)


def test_shares_with_units_before_chunks():
    import random

    r = random.Random(0)
    for _ in range(1500):
        chunks = [max(1, int(r.choice([0, 1, 2, 5, 20]) * r.random())) for _ in range(r.randint(1, 12))]
        _shares_of(chunks, r.choice([1, 2, 8]), r.randint(1, 40), r.choice([0, 1, 2, 3, 5]))


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_kernels_spill_no_vector_registers():
    """A kernel with scratch memory costs several microseconds a launch."""
    csrc = os.path.join(ROOT, "flagattention_amd", "csrc")
    flags = ["-O3", "-std=c++17", "--offload-arch=gfx950", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-Rpass-analysis=kernel-resource-usage", "-c", "--cuda-device-only", "-o", os.devnull]
    runs = [subprocess.Popen(["/opt/rocm/bin/hipcc", *flags, os.path.join(csrc, unit)], stderr=subprocess.PIPE, text=True)
            for unit in ("paged8_attn.hip", "cache8_ops.hip")]
    for run, kernels in zip(runs, (32, 100)):
        said = run.communicate(timeout=600)[1]
        found = re.findall(r"Function Name: (\S+).*?VGPRs Spill: (\d+)", said, re.S)
        assert run.returncode == 0 and len(found) >= kernels and all(int(n) == 0 for _, n in found), [x for x in found if int(x[1])]
