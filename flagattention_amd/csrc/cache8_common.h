// Caches of 8-bit codes (paged8_attn.hip, cache8_ops.hip): how codes become numbers.  A block of tokens of a page and a head share a
// scale in fp32; a value is code * scale.  Codes are exact in fp16 (int8: 7 bits and a sign, e4m3: 4 bits from 2^-9 to 448), so that
// they go to the 16-bit matrix instructions as they are, and scales meet scores and weights in fp32.
#pragma once
#include "attn_common.h"

namespace sage {
namespace attn {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef int v2i __attribute__((ext_vector_type(2)));

struct Int8 {
    static constexpr float kLargest = 127.0f;
    static constexpr bool kHasNan = false;
    // Four codes.  Byte u = code + 128 below the exponent of 1024 is 1024 + u in fp16: two instructions for two codes, and one
    // to flip the signs of four.
    static __device__ __forceinline__ v2i halves(unsigned w) {
        w ^= 0x80808080u;
        const v2h off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const v2h lo = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
        const v2h hi = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
        return v2i{__builtin_bit_cast(int, lo), __builtin_bit_cast(int, hi)};
    }
};

struct E4m3 {
    static constexpr float kLargest = 448.0f;
    static constexpr bool kHasNan = true;
    static __device__ __forceinline__ v2i halves(unsigned w) {
        const v2h lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
        return v2i{__builtin_bit_cast(int, lo), __builtin_bit_cast(int, hi)};
    }
    // Marks (bit 7 of its byte) the codes that are NaN: all bits but the sign are ones.
    static __device__ __forceinline__ unsigned nan_bytes(unsigned w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
};

// Eight codes as the operand of a matrix instruction.
template <typename Code>
__device__ __forceinline__ f16x8 to_f16(v2i w) {
    const v2i a = Code::halves((unsigned)w[0]), b = Code::halves((unsigned)w[1]);
    return __builtin_bit_cast(f16x8, v4i{a[0], a[1], b[0], b[1]});
}

}  // namespace
}  // namespace attn

// The scales of a cache's blocks, strides in elements; tokens of a page: block of them to a scale.
struct BlockScales {
    float* k;
    float* v;
    int64_t k_p, k_h, k_b, v_p, v_h, v_b;
    int32_t block, shift;  // shift: log2 of block, -1: it has none
    __device__ __forceinline__ int of(int place) const { return shift >= 0 ? place >> shift : place / block; }
};

inline BlockScales block_scales(const sage_cache_scales& s, int64_t page_size) {
    BlockScales r{};
    r.k = s.k; r.v = s.v;
    r.k_p = s.k_stride_page; r.k_h = s.k_stride_head; r.k_b = s.k_stride_block;
    r.v_p = s.v_stride_page; r.v_h = s.v_stride_head; r.v_b = s.v_stride_block;
    r.block = s.blocks > 0 ? (int)(page_size / s.blocks) : 1;
    r.shift = (r.block & (r.block - 1)) == 0 ? __builtin_ctz((unsigned)r.block) : -1;
    return r;
}

}  // namespace sage
