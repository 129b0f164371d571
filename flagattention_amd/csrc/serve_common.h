// Device helpers of the kernels for packed sequences (flash_varlen.hip) and paged caches (paged_attn.hip), gfx950.
#pragma once
#include <type_traits>

#include "attn_common.h"
#include "step_lines.h"

namespace sage {
namespace attn {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

// Inclusive scan over the lanes of a wave (0: what joins nothing), by lane moves inside the vector unit.
template <typename Join>
__device__ __forceinline__ int wave_scan(int x, Join&& join) {
    auto step = [&](auto ctrl, auto rows) {
        x = join(x, __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    };
    step(IC<0x111>{}, IC<0xf>{});  // from 1, 2, 4, 8 lanes below, within rows of 16
    step(IC<0x112>{}, IC<0xf>{});
    step(IC<0x114>{}, IC<0xf>{});
    step(IC<0x118>{}, IC<0xf>{});
    step(IC<0x142>{}, IC<0xa>{});  // the last lane of a row into the next one: rows 1 and 3
    step(IC<0x143>{}, IC<0xc>{});  // lane 31 into rows 2 and 3
    return x;
}
__device__ __forceinline__ int wave_scan(int x) { return wave_scan(x, [](int a, int b) { return a + b; }); }
// Over all lanes, the same in each of them: the sum, the largest of numbers that are not negative.
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
__device__ __forceinline__ int wave_max(int x) { return __builtin_amdgcn_readlane(wave_scan(x, [](int a, int b) { return max(a, b); }), 63); }

// Which of n consecutive runs, run i count(i) >= 0 entries long, holds entry `at`, and where that run begins; false: all of
// them end before `at`.  Every wave finds it for itself: lane after lane takes an equal stretch of the runs, a scan says
// which stretch, a second one which run of it.  `at` is uniform, and so are the results.
template <typename Count>
__device__ __forceinline__ bool find_run(int n, int at, Count&& count, int& run, int& begin) {
    const int lane = threadIdx.x & 63;
    const int per_lane = (n + 63) / 64;
    const int mine = per_lane * lane;
    int sum = 0;
    for (int i = 0; i < per_lane; i++) sum += mine + i < n ? count(mine + i) : 0;
    const int incl = wave_scan(sum);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(incl > at);
    if (past == 0) return false;
    const int owner = __builtin_ctzll(past);
    run = per_lane * owner;
    begin = __builtin_amdgcn_readlane(incl - sum, owner);
    while (per_lane > 1) {
        if (run >= n) return false;
        const int i = run + lane;
        const int c = lane < per_lane && i < n ? count(i) : 0;
        const int s = begin + wave_scan(c);
        const unsigned long long hit = __builtin_amdgcn_ballot_w64(s > at);
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            run += l;
            begin = __builtin_amdgcn_readlane(s - c, l);
            break;
        }
        run += 64;
        begin = __builtin_amdgcn_readlane(s, 63);
    }
    return true;
}

// Marks (bit 15 of its half) the 16-bit numbers of a word that are an infinity or NaN: their exponent field is all ones.
template <typename VT>
__device__ __forceinline__ unsigned nonfinite_halves(unsigned w) {
    constexpr unsigned field = std::is_same<VT, __bf16>::value ? 0x7f807f80u : 0x7c007c00u;
    const unsigned t = ~w & field;  // zero in such a half
    return (t - 0x00010001u) & ~t & 0x80008000u;
}

// (paged_attn.hip) The eight numbers with zeros for infinities and NaN.
template <typename VT>
__device__ __forceinline__ v4i finite_only(v4i x) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned z = nonfinite_halves<VT>((unsigned)x[i]);
        x[i] = (int)((unsigned)x[i] & ~(z | (z - (z >> 15))));
    }
    return x;
}

// (paged_attn.hip) What the infinities and NaN of a 32-key V tile in LDS add to the outputs of a lane's row (16x16 layout: accumulator i
// of tile ct is channel 16 ct + 4 quad + i): for every key j < see_end of the tile and every channel that the lane holds.  p: the
// lane's P of the keys 16 (e / 4) + 4 quad + e % 4.  V row j, chunk c lies at row j * 2 D + 16 (c ^ swizzle(j)).  Slow, and hardly ever
// called.
template <int D, typename VT, typename Swizzle>
__device__ __forceinline__ void add_nonfinite(const unsigned char* vtile, Swizzle&& swizzle, typename PV<VT>::vec p, int see_end, v4f (&acc)[D / 16]) {
    const int lane = threadIdx.x & 63, quad = lane >> 4;
    const v4i words = __builtin_bit_cast(v4i, p);
#pragma unroll 1
    for (int j = 0; j < 32; j++) {
        const int owner = (j >> 2) & 3, e = 4 * (j >> 4) + (j & 3);  // P of key j: number e of the lane of that quad
        unsigned pair = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int w = words[i];
            pair = i == e >> 1 ? (unsigned)w : pair;
        }
        const float mine = (float)__builtin_bit_cast(VT, (unsigned short)(e & 1 ? pair >> 16 : pair));
        const float pj = __shfl(mine, 16 * owner + (lane & 15));
        const bool sees = j < see_end;
#pragma unroll
        for (int ct = 0; ct < D / 16; ct++) {
            typedef unsigned v2u __attribute__((ext_vector_type(2)));
            const v2u w = *reinterpret_cast<const v2u*>(vtile + j * (2 * D) + 16 * ((2 * ct + (quad >> 1)) ^ swizzle(j)) + 8 * (quad & 1));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const unsigned word = w[i >> 1];
                const unsigned z = nonfinite_halves<VT>(word);
                const float v = (float)__builtin_bit_cast(VT, (unsigned short)(word >> (16 * (i & 1))));
                const bool odd = (z >> (15 + 16 * (i & 1))) & 1;
                acc[ct][i] = sees && odd ? __builtin_fmaf(pj, v, acc[ct][i]) : acc[ct][i];
            }
            __builtin_amdgcn_sched_barrier(0);  // (a few registers at a time)
        }
    }
}

// Four fp32 numbers, rounded, to a 16-bit output.
template <typename VT>
__device__ __forceinline__ void store_rounded(VT* to, v4f x) {
    typedef VT v4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<v4*>(to) = v4{(VT)x[0], (VT)x[1], (VT)x[2], (VT)x[3]};
}

}  // namespace
}  // namespace attn
}  // namespace sage
