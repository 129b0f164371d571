// A paged cache of 8-bit codes for gfx950: rows of new tokens quantized into it, tokens read back into packed rows, pages copied with
// their scales.  All are bound by bytes, and short calls by a launch and a chain of loads (slot, the block's other tokens, rows).
// Measured: 16384 tokens of 8 heads, D128, bf16 into int8, a scale for 16 tokens 27 us = 3.7 TB/s (2 to 5 of them the map), a scale a token 24 us; 2900 of
// 16 heads, D64, fp16 into e4m3, a scale a token 8.5 us; a step of 28 tokens 6.0; 17700 tokens read 20 to 23 us = 4.8 to 5.4 TB/s, 500 of them 5.7; 700 pages of
// 8 layers copied 76 us = 5.0 TB/s, 12 pages 4.3.
//
// Quantizing.  A block's scale is s = a / L, a the largest |x| of the call's tokens for it and head (at least 2^-100), L = 127 or 448, or
// the size of what it was where that is more and the block goes on; codes are x / s to the nearest, ties to even.  x / s is x times the rounded
// 1 / s first, off by at most 2^-22 of itself; only where that lies next to the middle between two codes (a wave in sixteen) the
// remainder x - c s, which is exact in an fma, decides.  Codes that stay when a scale grows are c s_old / s, decided by a remainder in 64 bits.
#include "cache8_common.h"

namespace sage {
namespace {

using namespace attn;

constexpr int kOpThreads = 256;
constexpr int kMostBlock = 1024;     // tokens that share a scale
// Calls of up to so many tokens look their slots over instead of mapping them, which is a launch of its own (500 tokens, blocks of 8, 16 heads, D64:
// 10.4 us by looking, 7.8 through the map).  Tokens that go to blocks of their own cost more beyond (8 heads, D128, blocks of 16: 256 7.3 us, 257 48.7), since a
// workgroup then looks at as many as fill its waves' blocks.
constexpr int kScanTokens = 256;
// Workgroups that a write of blocks makes where it can (16384 tokens of 8 heads, D128, bf16, blocks of 16 and 32: 512 32 and 34 us, 1024 26.4 and 34,
// 2048 28.7 and 36, 4096 30.6 and 42: a wave that goes through more heads looks its tokens up less often).
constexpr int kWriteWorkgroups = 1024;
constexpr float kSmallest = 0x1p-100f;

__device__ __forceinline__ int64_t index_at(const void* list, int wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(list)[i] : (int64_t) static_cast<const int32_t*>(list)[i];
}

// x / d for x >= 0, in 32 bits where x has no more (a division in 64 costs about 150 instructions); shift: log2 of d, -1: it has none
__device__ __forceinline__ int64_t quotient(int64_t x, int d, int shift) {
    if (shift >= 0) return x >> shift;
    return (x >> 32) == 0 ? (int64_t)((unsigned)x / (unsigned)d) : x / d;
}

// Sixteen entries of a row.
template <typename T> struct Row16;
template <typename T> struct Row16_16 {
    v4i w[2];
    __device__ __forceinline__ void load(const unsigned char* p) {
        w[0] = reinterpret_cast<const v4i*>(p)[0];
        w[1] = reinterpret_cast<const v4i*>(p)[1];
    }
    __device__ __forceinline__ void clear() { w[0] = w[1] = v4i{0, 0, 0, 0}; }
    __device__ __forceinline__ float at(int i) const {
        const unsigned x = (unsigned)w[i / 8][i % 8 / 2];
        return (float)__builtin_bit_cast(T, (unsigned short)(i & 1 ? x >> 16 : x));
    }
    // the largest absolute value, as the bits of |x| in T: NaN above infinity above the finite ones
    __device__ __forceinline__ unsigned top(unsigned so_far) const {
        typedef unsigned short v2s __attribute__((ext_vector_type(2)));
        v2s m = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2s, (unsigned)w[i / 4][i % 4] & 0x7fff7fffu));
        return max(so_far, max((unsigned)m[0], (unsigned)m[1]));
    }
    static __device__ __forceinline__ float size(unsigned top) { return (float)__builtin_bit_cast(T, (unsigned short)top); }
};
template <> struct Row16<__bf16> : Row16_16<__bf16> {};
template <> struct Row16<_Float16> : Row16_16<_Float16> {};
template <> struct Row16<float> {
    v4f w[4];
    __device__ __forceinline__ void load(const unsigned char* p) {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = reinterpret_cast<const v4f*>(p)[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ float at(int i) const { return w[i / 4][i % 4]; }
    __device__ __forceinline__ unsigned top(unsigned so_far) const {
#pragma unroll
        for (int i = 0; i < 16; i++) so_far = max(so_far, __builtin_bit_cast(unsigned, at(i)) & 0x7fffffffu);
        return so_far;
    }
    static __device__ __forceinline__ float size(unsigned top) { return __builtin_bit_cast(float, top); }
};

// The scale that new rows, whose largest entry has the size `top`, ask for.
template <typename Code>
__device__ __forceinline__ float scale_for(float top) {
    return top < INFINITY ? fmaxf(top, kSmallest) / Code::kLargest : NAN;
}

// x / s to the nearest integer, ties to even, for |x| <= 127.5 s (codes of int8) or |x| <= 16 s (an e4m3 number in steps of its own): n is
// next to it or it, and the remainder x - n s exact, a multiple of the last place of s or of x and no larger than s.
__device__ __forceinline__ float settle(float x, float s, float n) {
    const float r = __builtin_fmaf(-n, s, x), h = 0.5f * s;
    const bool odd = ((int)n & 1) != 0;
    if (r > h || (r == h && odd)) n += 1.0f;
    if (r < -h || (r == -h && odd)) n -= 1.0f;
    return n;
}
// The same with 64 bits, where x is code * old scale, 31 bits.
__device__ __forceinline__ double settle(double x, double s, double n) {
    const double r = __builtin_fma(-n, s, x), h = 0.5 * s;
    const bool odd = ((int)n & 1) != 0;
    if (r > h || (r == h && odd)) n += 1.0;
    if (r < -h || (r == -h && odd)) n -= 1.0;
    return n;
}

template <typename Code> struct Rounding;
template <> struct Rounding<Int8> {
    // Sixteen codes of x, s > 0 (or inv = 0: codes 0).  x inv + 1.5 2^23 is an integer in its low bits.
    template <typename Row>
    static __device__ __forceinline__ v4i codes(const Row& x, float s, float inv) {
        constexpr float magic = 12582912.0f, near = 0.5f - 0x1p-15f;
        auto off = [&](int i, float z) { return __builtin_fabsf(__builtin_fmaf(x.at(i), inv, -(z - magic))); };
        float z[16], far = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            z[i] = __builtin_fmaf(x.at(i), inv, magic);
            far = fmaxf(far, off(i, z[i]));
        }
        if (__builtin_amdgcn_ballot_w64(far > near) != 0) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (__builtin_amdgcn_ballot_w64(off(i, z[i]) > near) != 0) z[i] = settle(x.at(i), s, z[i] - magic) + magic;
        }
        v4i w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned lo = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, z[4 * i + 1]), __builtin_bit_cast(unsigned, z[4 * i]), 0x0c0c0400u);
            const unsigned hi = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, z[4 * i + 3]), __builtin_bit_cast(unsigned, z[4 * i + 2]), 0x04000c0cu);
            w[i] = (int)(lo | hi);
        }
        return w;
    }
    // A word of codes that stand for numbers in units of `was`, in units of s >= |was|.  (-128, which no write makes, may change its sign: 127)
    static __device__ __forceinline__ unsigned again(unsigned w, double was, double s) {
        const double ratio = was / s;
        unsigned to = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double c = (double)(int8_t)(w >> (8 * i));
            const double n = __builtin_fmin(settle(c * was, s, __builtin_rint(c * ratio)), 127.0);
            to |= ((unsigned)(int)n & 255u) << (8 * i);
        }
        return to;
    }
};
template <> struct Rounding<E4m3> {
    // The step between e4m3 numbers around y: 2^-3 of its power of two, at least 2^-9.
    static __device__ __forceinline__ float step(float y) {
        return __builtin_amdgcn_ldexpf(1.0f, max(__builtin_amdgcn_frexp_expf(y) - 1, -6) - 3);
    }
    template <typename Row>
    static __device__ __forceinline__ v4i codes(const Row& x, float s, float inv) {
        // Next to the middle between two numbers: the 20 bits that are rounded away are 2^19, or up to 8 less or more; or among the small
        // numbers, below 2^-6, whose steps are all the same, and not zero.
        auto middle = [](float y) { return (__builtin_bit_cast(unsigned, y) << 12) + ((0x80000u + 8) << 12); };
        auto small = [](float y) { return (__builtin_bit_cast(unsigned, y) << 1) - 1; };
        auto close = [](unsigned middle, unsigned small) { return middle <= (16u << 12) || small < (0x3c800000u << 1) - 1; };
        float y[16];
        unsigned least_middle = ~0u, least_small = ~0u;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            y[i] = x.at(i) * inv;
            least_middle = min(least_middle, middle(y[i]));
            least_small = min(least_small, small(y[i]));
        }
        if (__builtin_amdgcn_ballot_w64(close(least_middle, least_small)) != 0) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (__builtin_amdgcn_ballot_w64(close(middle(y[i]), small(y[i]))) != 0) {
                    const float u = step(y[i]);
                    y[i] = inv != 0.0f ? settle(x.at(i), s * u, __builtin_rintf(y[i] / u)) * u : 0.0f;
                }
        }
        v4i w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int z = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
            w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], z, true);
        }
        return w;
    }
    static __device__ __forceinline__ unsigned again(unsigned w, double was, double s) {
        const double ratio = was / s;
        const v2i h = E4m3::halves(w);
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double c = (double)__builtin_bit_cast(_Float16, (unsigned short)((unsigned)h[i / 2] >> (16 * (i & 1))));
            const double u = step((float)(c * ratio));
            y[i] = (float)(settle(c * was, s * u, __builtin_rint(c * ratio / u)) * u);
        }
        int z = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], z, true);
    }
};

struct WriteArgs {
    const unsigned char* src[2];  // k, v
    unsigned char* dst[2];        // caches
    int64_t ss_t[2], ss_h[2], ds_p[2], ds_h[2], ds_n[2];  // bytes
    BlockScales scales;
    const void* slots;
    int32_t* map;  // [slots of the cache]: token that goes there, where that token's slot says so too; null: few tokens
    int64_t slot_limit, rows;  // rows: tokens * heads
    int32_t wide, tokens, page_size, page_shift, heads, head_shift, pieces, group, span;  // pieces: of 16 entries, of a row; group: tokens a workgroup looks at; span: lanes of a block
};

__device__ __forceinline__ float& scale_of(const WriteArgs& a, int x, int64_t page, int h, int block) {
    return x ? a.scales.v[page * a.scales.v_p + h * a.scales.v_h + block * a.scales.v_b]
             : a.scales.k[page * a.scales.k_p + h * a.scales.k_h + block * a.scales.k_b];
}

// A scale for every token: LPR lanes take a row of k and the same one of v, 16 entries each.  The rows are requested before it is known
// where they go.
template <int LPR, typename T, typename Code>
__global__ __launch_bounds__(kOpThreads) void cache8_write_rows_kernel(WriteArgs a) {
    const int64_t row = (int64_t)blockIdx.x * (kOpThreads / LPR) + threadIdx.x / LPR;
    const int c = threadIdx.x % LPR;
    const int64_t t = quotient(min(row, a.rows - 1), a.heads, a.head_shift);
    const int h = (int)(min(row, a.rows - 1) - t * a.heads);
    const int64_t slot = index_at(a.slots, a.wide, t);
    Row16<T> x[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (c < a.pieces) x[i].load(a.src[i] + t * a.ss_t[i] + h * a.ss_h[i] + c * (16 * (int)sizeof(T)));
        else x[i].clear();
    }
    const bool ok = row < a.rows && slot >= 0 && slot < a.slot_limit, mine = ok && c < a.pieces;
    const int64_t page = ok ? quotient(slot, a.page_size, a.page_shift) : 0;
    const int place = ok ? (int)(slot - page * a.page_size) : 0;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        unsigned top = x[i].top(0);
#pragma unroll
        for (int d = 1; d < LPR; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
        const float s = scale_for<Code>(Row16<T>::size(top));
        const float inv = s < INFINITY ? 1.0f / s : 0.0f;
        if (!(s < INFINITY)) x[i].clear();  // (NaN: an entry was not finite)
        const v4i w = Rounding<Code>::codes(x[i], s, inv);
        if (mine) *reinterpret_cast<v4i*>(a.dst[i] + page * a.ds_p[i] + h * a.ds_h[i] + place * a.ds_n[i] + 16 * c) = w;
        if (mine && c == 0) scale_of(a, i, page, h, place) = s;
    }
}

__global__ __launch_bounds__(kOpThreads) void cache8_map_kernel(WriteArgs a) {
    const int t = blockIdx.x * kOpThreads + threadIdx.x;
    if (t >= a.tokens) return;
    const int64_t slot = index_at(a.slots, a.wide, t);
    if (slot >= 0 && slot < a.slot_limit) a.map[slot] = t;
}

// Blocks of several tokens.  Of the call's tokens that go to a block, the one with the lowest place takes care of it.  A workgroup looks at
// `group` tokens, at most 64, and leaves out at once those that follow another one of their block from the place before their own.
// The tokens of a block are looked for among all of the call's (SCAN) or through the map, which is not cleared before, since an
// entry counts only where its token's slot leads back to it.
struct Candidates {
    int64_t base;   // of the lane's token: slot of its block's first place
    int place;      // in the block
    unsigned long long todo;  // tokens left (the same in every lane)
};
__device__ __forceinline__ Candidates look(const WriteArgs& a) {
    Candidates r{0, 0, 0};
    const int lane = threadIdx.x & 63;
    bool candidate = false;
    const int64_t t = (int64_t)blockIdx.x * a.group + lane;
    if (lane < a.group && t < a.tokens) {
        const int64_t slot = index_at(a.slots, a.wide, t);
        const int64_t before = t > 0 ? index_at(a.slots, a.wide, t - 1) : -1;
        if (slot >= 0 && slot < a.slot_limit) {
            const int place = (int)(slot - quotient(slot, a.page_size, a.page_shift) * a.page_size);
            r.place = place - a.scales.of(place) * a.scales.block;
            r.base = slot - r.place;
            candidate = r.place == 0 || before != slot - 1;
        }
    }
    r.todo = __builtin_amdgcn_ballot_w64(candidate);
    return r;
}
__device__ __forceinline__ int64_t lane_value(int64_t x, int lane) {
    return ((int64_t)__shfl((int)(x >> 32), lane) << 32) | (unsigned)__shfl((int)(unsigned)x, lane);
}
__device__ __forceinline__ int mapped(const WriteArgs& a, int64_t slot) {
    const int who = a.map[slot];
    return who >= 0 && who < a.tokens && index_at(a.slots, a.wide, who) == slot ? who : -1;
}

// The scale of a block that had `was`, of either sign, and gets rows whose largest entry has the size `top`.  One that is not finite stays.
template <typename Code>
__device__ __forceinline__ float next_scale(float was, float top) {
    const float asked = scale_for<Code>(top), size = __builtin_fabsf(was);
    if (was != was) return was;
    return !(size >= asked) ? asked : size < INFINITY ? size : was;
}
// Sixteen codes that stay when a scale changes.
template <typename Code>
__device__ __forceinline__ void convert(unsigned char* at, float was, float s) {
    v4i w = *reinterpret_cast<v4i*>(at);
#pragma unroll 1
    for (int i = 0; i < 4; i++) {
        const unsigned now = Rounding<Code>::again((unsigned)w[0], was, s);
        w = v4i{w[1], w[2], w[3], (int)now};
    }
    *reinterpret_cast<v4i*>(at) = w;
}

constexpr int kKeep = 2;  // steps of 64 / LPR rows that a wave keeps in registers
constexpr int kScanGroup = 4;

// Blocks whose rows a wave keeps in registers.  A wave takes a block (blocks of 2, 4 or 8 tokens through the map: as many as fit its
// lanes, `span` of them each) and goes through heads of K and V, the next one's rows on their way.
template <int LPR, typename T, typename Code, bool SCAN>
__global__ __launch_bounds__(kOpThreads, 4) void cache8_write_blocks_kernel(WriteArgs a) {
    constexpr int ROWS = 64 / LPR, WAVES = kOpThreads / 64;
    __shared__ int found[SCAN ? kScanGroup * 64 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int block = a.scales.block, span = a.span, sub = lane / span, c = lane % LPR;
    constexpr int EACH = SCAN ? kScanTokens / kOpThreads : 1;
    int64_t slot[EACH];  // (requested beside those that look() asks for)
    if constexpr (SCAN) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int i = e * kOpThreads + threadIdx.x;
            slot[e] = i < a.tokens ? index_at(a.slots, a.wide, i) : -1;
        }
        found[threadIdx.x] = -1;
    }
    Candidates cand = look(a);
    if constexpr (SCAN) {
        __syncthreads();
        int n = 0;
        for (unsigned long long todo = cand.todo; todo != 0; todo &= todo - 1, n++) {
            const int64_t begin = lane_value(cand.base, __builtin_ctzll(todo));
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const int64_t d = slot[e] - begin;
                if (slot[e] >= 0 && d >= 0 && d < block) atomicMax(&found[n * 64 + d], e * kOpThreads + (int)threadIdx.x);  // (slots that occur twice: the last one)
            }
        }
        __syncthreads();
    }
    for (int nth = 0; cand.todo != 0; nth++) {
        int looker = -1;
        for (int j = 0; j < 64 / span && cand.todo != 0; j++) {
            if (sub == j) looker = __builtin_ctzll(cand.todo);
            cand.todo &= cand.todo - 1;
        }
        if (nth % WAVES != wave) continue;
        const int64_t begin = lane_value(cand.base, looker & 63);
        const int t = (int)((int64_t)blockIdx.x * a.group + looker), place = __shfl(cand.place, looker & 63);
        int who[kKeep];  // tokens of the lane's rows, -1: none, -2: no such place
        bool other = looker < 0, first = false;
#pragma unroll
        for (int e = 0; e < kKeep; e++) {
            const int p = e * ROWS + lane % span / LPR;
            who[e] = -2;
            if (p < block && looker >= 0) {
                who[e] = SCAN ? found[nth * 64 + p] : mapped(a, begin + p);
                other |= (who[e] >= 0 && p < place) || (p == place && who[e] != t);
                first |= p == 0 && who[e] >= 0;
            }
        }
        // (bit masks of the lanes of this block)
        const unsigned long long lanes = span == 64 ? ~0ull : ((1ull << span) - 1) << (sub * span);
        const bool mine = (__builtin_amdgcn_ballot_w64(other) & lanes) == 0, begun = (__builtin_amdgcn_ballot_w64(first) & lanes) != 0;
        if (__builtin_amdgcn_ballot_w64(mine) == 0) continue;
        if (!mine || c >= a.pieces) {
#pragma unroll
            for (int e = 0; e < kKeep; e++) who[e] = -2;
        }
        const int64_t page = mine ? quotient(begin, a.page_size, a.page_shift) : 0;
        const int at = mine ? (int)(begin - page * a.page_size) : 0, b = a.scales.of(at);
        Row16<T> rows[kKeep];
        auto load = [&](int unit) {
            const int x = unit & 1, h = unit >> 1;
            const unsigned char* src = a.src[x] + h * a.ss_h[x] + c * (16 * (int)sizeof(T));
#pragma unroll
            for (int e = 0; e < kKeep; e++) {
                if (who[e] >= 0) rows[e].load(src + who[e] * a.ss_t[x]);
                else rows[e].clear();
            }
        };
        int unit = blockIdx.y;
        if (unit < 2 * a.heads) load(unit);
        for (; unit < 2 * a.heads; unit += gridDim.y) {
            const int x = unit & 1, h = unit >> 1;
            unsigned char* dst = a.dst[x] + page * a.ds_p[x] + h * a.ds_h[x] + (at + lane % span / LPR) * a.ds_n[x] + 16 * c;
            const float was = begun || !mine ? 0.0f : scale_of(a, x, page, h, b);
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < kKeep; e++) top = rows[e].top(top);
            for (int d = 1; d < span; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
            const float s = next_scale<Code>(was, Row16<T>::size(top));
            const float inv = __builtin_fabsf(s) < INFINITY ? 1.0f / s : 0.0f;
#pragma unroll
            for (int e = 0; e < kKeep; e++) {
                if (e * ROWS >= block) break;
                if (!(__builtin_fabsf(s) < INFINITY)) rows[e].clear();  // (NaN: an entry was not finite)
                const v4i w = Rounding<Code>::codes(rows[e], s, inv);
                if (who[e] >= 0 || (who[e] == -1 && begun))  // (zeros where a block begins)
                    *reinterpret_cast<v4i*>(dst + e * ROWS * a.ds_n[x]) = w;
            }
            if (unit + (int)gridDim.y < 2 * a.heads) load(unit + gridDim.y);
            if (s != was && s == s && !begun) {
                for (int e = 0; e < kKeep; e++)
                    if (who[e] == -1) convert<Code>(dst + e * ROWS * a.ds_n[x], was, s);
            }
            if (mine && lane % span == 0) scale_of(a, x, page, h, b) = s;
        }
    }
}

// Longer blocks: a workgroup takes a block and goes through heads of K and V, its waves sharing the rows; it goes over them twice where they are
// more than it keeps in registers (128 of them at D128, 256 at D64).
template <int LPR, typename T, typename Code, bool SCAN>
__global__ __launch_bounds__(kOpThreads, sizeof(T) == 4 ? 3 : 4) void cache8_write_long_blocks_kernel(WriteArgs a) {
    constexpr int ROWS = 64 / LPR, KEEP = 4, WAVES = kOpThreads / 64, PASS = KEEP * WAVES * ROWS;
    __shared__ int token[kMostBlock];
    __shared__ int lowest;
    __shared__ unsigned tops[2][WAVES];  // in turn, so that a barrier a unit is enough
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int block = a.scales.block;
    const int my_row = wave * ROWS + lane / LPR, c = lane % LPR;
    Candidates cand = look(a);
    for (; cand.todo != 0; cand.todo &= cand.todo - 1) {
        const int looker = __builtin_ctzll(cand.todo);
        const int t = (int)((int64_t)blockIdx.x * a.group + looker);
        const int64_t begin = lane_value(cand.base, looker);
        __syncthreads();  // (the tokens of the block before have been read)
        if (tid == 0) lowest = block;
        for (int p = tid; p < block; p += kOpThreads) token[p] = SCAN ? -1 : mapped(a, begin + p);
        __syncthreads();
        if (SCAN) {
            for (int i = tid; i < a.tokens; i += kOpThreads) {
                const int64_t d = index_at(a.slots, a.wide, i) - begin;
                if (d >= 0 && d < block) atomicMax(&token[d], i);  // (slots that occur twice: the last one)
            }
            __syncthreads();
        }
        for (int p = tid; p < block; p += kOpThreads)
            if (token[p] >= 0) atomicMin(&lowest, p);
        __syncthreads();
        if (token[lowest] != t) continue;
        const bool begun = lowest == 0;
        const int64_t page = quotient(begin, a.page_size, a.page_shift);
        const int at = (int)(begin - page * a.page_size), b = a.scales.of(at);
        for (int unit = blockIdx.y, turn = 0; unit < 2 * a.heads; unit += gridDim.y, turn ^= 1) {
            const int x = unit & 1, h = unit >> 1;
            const unsigned char* src = a.src[x] + h * a.ss_h[x] + c * (16 * (int)sizeof(T));
            unsigned char* dst = a.dst[x] + page * a.ds_p[x] + h * a.ds_h[x] + at * a.ds_n[x] + 16 * c;
            const float was = begun ? 0.0f : scale_of(a, x, page, h, b);
            Row16<T> rows[KEEP];
            int who[KEEP];
            auto load = [&](int p0) {  // rows of places p0 ..; who: their tokens, -1: none, -2: no such place
#pragma unroll
                for (int e = 0; e < KEEP; e++) {
                    const int p = p0 + e * (WAVES * ROWS) + my_row;
                    who[e] = p < block && c < a.pieces ? token[p] : -2;
                    if (who[e] >= 0) rows[e].load(src + who[e] * a.ss_t[x]);
                    else rows[e].clear();
                }
            };
            unsigned top = 0;
            for (int p0 = 0; p0 < block; p0 += PASS) {
                load(p0);
#pragma unroll
                for (int e = 0; e < KEEP; e++) top = rows[e].top(top);
            }
#pragma unroll
            for (int d = 1; d < 64; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
            if (lane == 0) tops[turn][wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; w++) top = max(top, tops[turn][w]);
            const float s = next_scale<Code>(was, Row16<T>::size(top));
            const float inv = __builtin_fabsf(s) < INFINITY ? 1.0f / s : 0.0f;
            for (int p0 = 0; p0 < block; p0 += PASS) {
                if (block > PASS) load(p0);
#pragma unroll
                for (int e = 0; e < KEEP; e++) {
                    if (p0 + e * (WAVES * ROWS) >= block) break;
                    if (!(__builtin_fabsf(s) < INFINITY)) rows[e].clear();  // (NaN: an entry was not finite)
                    const v4i w = Rounding<Code>::codes(rows[e], s, inv);
                    if (who[e] >= 0 || (who[e] == -1 && begun))  // (zeros where a block begins)
                        *reinterpret_cast<v4i*>(dst + (p0 + e * (WAVES * ROWS) + my_row) * a.ds_n[x]) = w;
                }
            }
            if (s != was && s == s && !begun)
                for (int p = my_row; p < block; p += WAVES * ROWS)
                    if (c < a.pieces && token[p] < 0) convert<Code>(dst + p * a.ds_n[x], was, s);
            if (tid == 0) scale_of(a, x, page, h, b) = s;
        }
    }
}

// Packed rows of sequences from the pages of a cache.  A workgroup takes some rows, about 1024 pieces of K and as many of V: one search over the
// sequences for the first row, the others go on from there.
constexpr int kMostReadRows = 32;

struct ReadArgs {
    const unsigned char* src[2];  // caches
    unsigned char* dst[2];
    int64_t ss_p[2], ss_h[2], ss_n[2], ds_t[2], ds_h[2];  // bytes
    BlockScales scales;
    const int32_t* table;
    const int32_t* cu;
    int64_t table_stride, capacity;
    int32_t seqs, total, page_size, page_shift, pages, heads, pieces, rows;  // pieces: of 8 codes, or 16 bytes, of a row; rows: of a workgroup
};

// OutT: codes become numbers of it; Code void: 16 bytes of a row are copied.
template <typename OutT, typename Code>
__global__ __launch_bounds__(kOpThreads) void cache_read_kernel(ReadArgs a) {
    __shared__ int page_of[kMostReadRows], place_of[kMostReadRows], block_of[kMostReadRows];  // page -1: a row of zeros, -2: no row
    __shared__ int ends;
    const int tid = threadIdx.x, t0 = blockIdx.x * a.rows;
    if (tid == 0) ends = 0;
    __syncthreads();
    int before = 0;  // sequences that end at or before row t0
    for (int s = tid; s < a.seqs; s += kOpThreads) before += a.cu[s + 1] <= t0 ? 1 : 0;
    if (before) atomicAdd(&ends, before);
    __syncthreads();
    if (tid < a.rows) {
        const int t = t0 + tid;
        int seq = ends;
        while (seq < a.seqs && a.cu[seq + 1] <= t) seq++;
        int page = -2, place = 0;
        if (t < a.total && seq < a.seqs) {
            const int64_t pos = (int64_t)t - a.cu[seq];
            page = pos >= 0 ? -1 : -2;
            if (pos >= 0 && pos < a.capacity) {
                const int64_t e = quotient(pos, a.page_size, a.page_shift);
                place = (int)(pos - e * a.page_size);
                const int p = a.table[seq * a.table_stride + e];
                if (p >= 0 && p < a.pages) page = p;
            }
        }
        page_of[tid] = page;
        place_of[tid] = place;
        if (!std::is_same<Code, void>::value) block_of[tid] = a.scales.of(place);
    }
    __syncthreads();
    // pieces of the rows, a few of them on their way together
    const int per_row = a.heads * a.pieces, all = a.rows * per_row;
    constexpr int BATCH = 4;
    constexpr bool CODED = !std::is_same<Code, void>::value;
    typedef typename std::conditional<CODED, v2i, v4i>::type piece;  // eight codes, or 16 bytes
    for (int i0 = tid; i0 < all; i0 += BATCH * kOpThreads) {
        piece w[BATCH][2];
        float s[BATCH][2];
        int row[BATCH], head[BATCH], part[BATCH];
        bool write[BATCH];
#pragma unroll
        for (int e = 0; e < BATCH; e++) {
            const int i = i0 + e * kOpThreads;
            const int r = i < all ? i / per_row : 0, q = i - r * per_row;
            row[e] = r; head[e] = q / a.pieces; part[e] = q - head[e] * a.pieces;
            const int page = page_of[r], place = place_of[r];
            write[e] = i < all && page != -2;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                w[e][x] = piece{};
                s[e][x] = 0.0f;
                if (i < all && page >= 0) {
                    w[e][x] = *reinterpret_cast<const piece*>(a.src[x] + page * a.ss_p[x] + head[e] * a.ss_h[x] + place * a.ss_n[x] + (int)sizeof(piece) * part[e]);
                    if constexpr (CODED) {
                        const BlockScales& b = a.scales;
                        s[e][x] = x ? b.v[page * b.v_p + head[e] * b.v_h + block_of[r] * b.v_b] : b.k[page * b.k_p + head[e] * b.k_h + block_of[r] * b.k_b];
                    }
                }
            }
        }
#pragma unroll
        for (int e = 0; e < BATCH; e++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                if (!write[e]) continue;
                unsigned char* to = a.dst[x] + (int64_t)(t0 + row[e]) * a.ds_t[x] + head[e] * a.ds_h[x];
                if constexpr (CODED) {
                    typedef OutT v8 __attribute__((ext_vector_type(8)));
                    const f16x8 codes = to_f16<Code>(w[e][x]);
                    v8 out;
#pragma unroll
                    for (int j = 0; j < 8; j++) out[j] = (OutT)((float)codes[j] * s[e][x]);
                    *reinterpret_cast<v8*>(to + 8 * (int)sizeof(OutT) * part[e]) = out;
                } else {
                    *reinterpret_cast<v4i*>(to + 16 * part[e]) = w[e][x];
                }
            }
    }
}

struct Copy8Args {
    unsigned char* cache[2];
    float* scale[2];
    int64_t stride_l[2], stride_p[2];    // bytes
    int64_t sstride_l[2], sstride_p[2];  // floats
    const void* src;
    const void* dst;
    int64_t pages;
    int32_t src_wide, dst_wide, page_pieces, count, words;
};

constexpr int kCopyPieces = 4;  // per thread, on their way together

// blockIdx: part of a page, pair, layer * 2 + cache; the first part of a page copies its scales too
__global__ __launch_bounds__(kOpThreads) void cache8_copy_kernel(Copy8Args a) {
    const int which = blockIdx.z & 1;
    const int64_t layer = blockIdx.z >> 1;
    const int first = blockIdx.x * (kOpThreads * kCopyPieces) + threadIdx.x;
    for (int i = blockIdx.y; i < a.count; i += gridDim.y) {
        const int64_t from = index_at(a.src, a.src_wide, i), to = index_at(a.dst, a.dst_wide, i);
        if (from < 0 || from >= a.pages || to < 0 || to >= a.pages) continue;
        unsigned char* base = a.cache[which] + layer * a.stride_l[which];
        const v4i* s = reinterpret_cast<const v4i*>(base + from * a.stride_p[which]);
        v4i* d = reinterpret_cast<v4i*>(base + to * a.stride_p[which]);
        v4i x[kCopyPieces];
#pragma unroll
        for (int e = 0; e < kCopyPieces; e++)
            if (first + e * kOpThreads < a.page_pieces) x[e] = s[first + e * kOpThreads];
        if (blockIdx.x == 0) {
            float* scale = a.scale[which] + layer * a.sstride_l[which];
            for (int w = threadIdx.x; w < a.words; w += kOpThreads) scale[to * a.sstride_p[which] + w] = scale[from * a.sstride_p[which] + w];
        }
#pragma unroll
        for (int e = 0; e < kCopyPieces; e++)
            if (first + e * kOpThreads < a.page_pieces) d[first + e * kOpThreads] = x[e];
    }
}

int log2_or_none(int64_t n) { return (n & (n - 1)) == 0 ? __builtin_ctzll((unsigned long long)n) : -1; }

bool maps_tokens(const sage_append8_params& p) { return p.scales.blocks != p.append.page_size && p.append.tokens > kScanTokens; }

}  // namespace

int64_t append8_workspace_bytes(const sage_append8_params& p) { return maps_tokens(p) ? p.append.pages * p.append.page_size * (int64_t)sizeof(int32_t) : 0; }

template <int LPR, typename T, typename Code>
static int launch_write(WriteArgs a, hipStream_t stream) {
    if (a.scales.block == 1) {
        const int64_t wgs = (a.rows * LPR + kOpThreads - 1) / kOpThreads;
        if (wgs > kMaxThreads / kOpThreads) return fail(SAGE_E_UNSUPPORTED, "sage_cache8_append: too many rows for one launch");
        hipLaunchKernelGGL((cache8_write_rows_kernel<LPR, T, Code>), dim3((unsigned)wgs), dim3(kOpThreads), 0, stream, a);
        return check_launch("cache8_write_rows_kernel");
    }
    // A wave goes through heads where the blocks fill the chip, and takes one where there are few.
    constexpr int ROWS = 64 / LPR;
    const int block = a.scales.block;
    const bool longer = block > kKeep * ROWS;
    a.span = a.map && block <= ROWS && a.scales.shift >= 0 ? LPR * block : 64;
    const int per_workgroup = kOpThreads / a.span * block;  // tokens of the blocks that its waves take at a time
    a.group = longer ? (a.map ? block < 64 ? block : 64 : 1) : a.map ? per_workgroup < 64 ? per_workgroup : 64 : kScanGroup;
    const int64_t groups = (a.tokens + a.group - 1) / a.group;
    if (groups > kMaxThreads / kOpThreads) return fail(SAGE_E_UNSUPPORTED, "sage_cache8_append: too many rows for one launch");
    const int units = 2 * a.heads;
    const int64_t most = kWriteWorkgroups / groups;
    const dim3 grid((unsigned)groups, (unsigned)(most < 1 ? 1 : most < units ? most : units)), threads(kOpThreads);
    if (a.map) {
        hipLaunchKernelGGL(cache8_map_kernel, dim3((unsigned)((a.tokens + kOpThreads - 1) / kOpThreads)), threads, 0, stream, a);
        if (int rc = check_launch("cache8_map_kernel")) return rc;
        if (longer) hipLaunchKernelGGL((cache8_write_long_blocks_kernel<LPR, T, Code, false>), grid, threads, 0, stream, a);
        else hipLaunchKernelGGL((cache8_write_blocks_kernel<LPR, T, Code, false>), grid, threads, 0, stream, a);
    } else {
        if (longer) hipLaunchKernelGGL((cache8_write_long_blocks_kernel<LPR, T, Code, true>), grid, threads, 0, stream, a);
        else hipLaunchKernelGGL((cache8_write_blocks_kernel<LPR, T, Code, true>), grid, threads, 0, stream, a);
    }
    return check_launch("cache8_write_blocks_kernel");
}

template <typename T, typename Code>
static int launch_write(const WriteArgs& a, hipStream_t stream) {
    if (a.pieces <= 4) return launch_write<4, T, Code>(a, stream);
    if (a.pieces <= 8) return launch_write<8, T, Code>(a, stream);
    if (a.pieces <= 16) return launch_write<16, T, Code>(a, stream);
    return launch_write<32, T, Code>(a, stream);
}

template <typename Code>
static int launch_write(const WriteArgs& a, int dtype, hipStream_t stream) {
    return dtype == SAGE_BF16 ? launch_write<__bf16, Code>(a, stream) : dtype == SAGE_F16 ? launch_write<_Float16, Code>(a, stream)
                                                                                          : launch_write<float, Code>(a, stream);
}

int launch_cache8_append(const sage_append8_params& p8, void* workspace, hipStream_t stream) {
    const sage_append_params& p = p8.append;
    WriteArgs a{};
    const sage_tensor* src[2] = {&p.k, &p.v};
    const sage_tensor* dst[2] = {&p.k_cache, &p.v_cache};
    const int64_t e = dtype_bytes(p.dtype);
    for (int x = 0; x < 2; x++) {
        a.src[x] = (const unsigned char*)src[x]->ptr; a.ss_t[x] = e * src[x]->stride_n; a.ss_h[x] = e * src[x]->stride_h;
        a.dst[x] = (unsigned char*)dst[x]->ptr; a.ds_p[x] = dst[x]->stride_b; a.ds_h[x] = dst[x]->stride_h; a.ds_n[x] = dst[x]->stride_n;
    }
    a.scales = block_scales(p8.scales, p.page_size);
    a.slots = p.slots; a.wide = p.slots_int64 ? 1 : 0;
    a.map = maps_tokens(p8) ? (int32_t*)workspace : nullptr;
    a.slot_limit = p.pages * p.page_size; a.rows = p.tokens * p.heads_kv;
    a.page_shift = log2_or_none(p.page_size); a.head_shift = log2_or_none(p.heads_kv);
    a.tokens = (int)p.tokens; a.page_size = (int)p.page_size; a.heads = (int)p.heads_kv; a.pieces = (int)(p.head_dim / 16);
    return p8.scales.codes == SAGE_CODE_INT8 ? launch_write<Int8>(a, p.dtype, stream) : launch_write<E4m3>(a, p.dtype, stream);
}

template <typename Code>
static void launch_read(const ReadArgs& a, int dtype, dim3 grid, hipStream_t stream) {
    if (dtype == SAGE_BF16) hipLaunchKernelGGL((cache_read_kernel<__bf16, Code>), grid, dim3(kOpThreads), 0, stream, a);
    else if (dtype == SAGE_F16) hipLaunchKernelGGL((cache_read_kernel<_Float16, Code>), grid, dim3(kOpThreads), 0, stream, a);
    else hipLaunchKernelGGL((cache_read_kernel<float, Code>), grid, dim3(kOpThreads), 0, stream, a);
}

int launch_cache_read(const sage_read_params& p, hipStream_t stream) {
    ReadArgs a{};
    const sage_tensor* src[2] = {&p.k_cache, &p.v_cache};
    const sage_tensor* dst[2] = {&p.k_out, &p.v_out};
    const bool coded = p.scales.codes != SAGE_CODE_NONE;
    const int64_t e = dtype_bytes(p.out_dtype), ce = coded ? 1 : e;
    for (int x = 0; x < 2; x++) {
        a.src[x] = (const unsigned char*)src[x]->ptr; a.ss_p[x] = ce * src[x]->stride_b; a.ss_h[x] = ce * src[x]->stride_h; a.ss_n[x] = ce * src[x]->stride_n;
        a.dst[x] = (unsigned char*)dst[x]->ptr; a.ds_t[x] = e * dst[x]->stride_n; a.ds_h[x] = e * dst[x]->stride_h;
    }
    if (coded) a.scales = block_scales(p.scales, p.page_size);
    a.table = p.block_table; a.cu = p.cu_seqlens; a.table_stride = p.table_stride;
    a.capacity = p.pages > 0 ? p.table_width * p.page_size : 0;
    a.page_shift = log2_or_none(p.page_size);
    a.seqs = (int)p.seqs; a.total = (int)p.total; a.page_size = (int)p.page_size; a.pages = (int)p.pages; a.heads = (int)p.heads_kv;
    a.pieces = (int)(coded ? p.head_dim / 8 : p.head_dim * e / 16);
    // (8 heads, D128: 8 rows 20.3 us for 17700 tokens, 16 rows 22; 1 head: 16 rows 12, 8 rows 16)
    for (a.rows = 4; a.rows < kMostReadRows && a.rows * a.heads * a.pieces < 1024;) a.rows *= 2;
    const dim3 grid((unsigned)((p.total + a.rows - 1) / a.rows));
    if ((int64_t)grid.x > kMaxThreads / kOpThreads) return fail(SAGE_E_UNSUPPORTED, "sage_cache_read: too many rows for one launch");
    if (p.scales.codes == SAGE_CODE_INT8) launch_read<Int8>(a, p.out_dtype, grid, stream);
    else if (coded) launch_read<E4m3>(a, p.out_dtype, grid, stream);
    else hipLaunchKernelGGL((cache_read_kernel<float, void>), grid, dim3(kOpThreads), 0, stream, a);
    return check_launch("cache_read_kernel");
}

int launch_cache8_copy(const sage_copy8_params& p8, hipStream_t stream) {
    const sage_copy_params& p = p8.copy;
    Copy8Args a{};
    a.cache[0] = (unsigned char*)p.k_cache; a.cache[1] = (unsigned char*)p.v_cache;
    a.stride_l[0] = p.k_stride_layer; a.stride_l[1] = p.v_stride_layer;
    a.stride_p[0] = p.k_stride_page; a.stride_p[1] = p.v_stride_page;
    a.scale[0] = p8.k_scale; a.scale[1] = p8.v_scale;
    a.sstride_l[0] = p8.k_scale_stride_layer; a.sstride_l[1] = p8.v_scale_stride_layer;
    a.sstride_p[0] = p8.k_scale_stride_page; a.sstride_p[1] = p8.v_scale_stride_page;
    a.src = p.src; a.dst = p.dst; a.src_wide = p.src_int64 ? 1 : 0; a.dst_wide = p.dst_int64 ? 1 : 0;
    a.pages = p.pages; a.page_pieces = (int)(p.page_bytes / 16); a.count = (int)p.count; a.words = (int)p8.scale_words;
    const int parts = (a.page_pieces + kOpThreads * kCopyPieces - 1) / (kOpThreads * kCopyPieces);
    const unsigned pairs = (unsigned)(p.count < 65535 ? p.count : 65535);
    hipLaunchKernelGGL(cache8_copy_kernel, dim3((unsigned)parts, pairs, (unsigned)(2 * p.layers)), dim3(kOpThreads), 0, stream, a);
    return check_launch("cache8_copy_kernel");
}

}  // namespace sage
