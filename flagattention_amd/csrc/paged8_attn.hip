// Dense attention of the newest tokens of every sequence over a paged cache of 8-bit codes (int8 or e4m3), for gfx950.
//
// As paged_attn.hip, with keys ks_j c_j and values vs_j d_j for codes c, d and the scales of their blocks:
//     o = sum_j p_j vs_j d_j / l,   l = sum_j p_j,   p_j = 2^(x_j - m),   x_j = sm_scale log2(e) ks_j (q . c_j).
// Codes are exact in fp16, so both products run on the 16-bit matrix instructions without another rounding of K or V; a score is
// multiplied by its key's scale in fp32, and a weight by its value's before the weights are rounded.
//   * Queries in bf16 become fp16 by a power of two of their row's own, 2^(15 - e) with the row's largest entry below 2^e: the entries
//     above 2^-29 of it keep all their bits, the others are off by at most 2^-39 of it (half of fp16's least step, 2^-25, against 2^14).  Scores stay in that unit, and the
//     exponent's fma takes them out of it.
//   * Weights w_j = p_j vs_j are rounded to fp16 (off by 2^-11 of themselves at most) in a unit of their row's own, a power of two in which the
//     largest |w| of the keys that the wave has seen lies between kUnitLow and kUnitTop: weights down to 2^-24 of it keep all 11 bits, smaller ones
//     are off by at most 2^-35 of it.  (The largest |vs| says nothing about it: it may belong to a key of no weight.)  A row's unit changes with
//     its accumulators, as its reference m does.
//
// Bound by the bytes of the codes: half of a 16-bit cache's.  The layout of the work is paged_attn.hip's.  K rows go to the operand
// registers 16 codes a lane, so that a load holds two steps of channels, and Q's channels lie in the same order; V tiles go through
// the wave's slice of LDS as codes, from where they are read transposed, eight keys of a channel a lane, and become fp16 after that.
// The 64 scales of a tile are one load, a lane each, and go through LDS to the lanes that hold their keys' scores.
//
// A beginning and an end cost about what two or three chunks do, and a share may begin several short items: each takes kPaged8Start units of
// the line besides its chunks.  Registers are left for as many workgroups as run without spilling: scratch memory costs 3 to
// 10 us a launch (three workgroups on a compute unit at D128, two registers spilled: 38 us instead of 35).
//
// Measured (inputs that change from pass to pass; the slope over the length is 5.95 TB/s): 128 sequences of 512 to 2048 tokens, 16 heads,
// D64, fp16, int8 66 us = 4.4 TB/s; 32 of up to 8192, H32/8, D128, bf16, int8 34 us = 3.6 TB/s, 5 of them the second kernel; 2 of 50000 to 65536,
// H32/4, e4m3, a scale a token 36 us = 3.4 TB/s, 6 of them the second kernel; 24 of up to 5000 with 4 new tokens each 25.6 us; one of 300
// tokens 10.3 us.  The launch, the chain of loads before the first product, the last outputs and the second kernel take 12 us of a call in shares.
#include "cache8_common.h"
#include "paged_common.h"

namespace sage {
namespace {

// Two workgroups on each compute unit (32 sequences of 2048 tokens, H32/8, D128: 256 shares 39 us, 512 38, 768 42, 1024 45).
constexpr int kPaged8Shares = 512;
// Chunks that an item's beginning and end cost (32 sequences of 200 to 8192 tokens, 24 of 100 to 5000 with 4 new tokens each: 0 44.5 and 38.1 us, 1 38.5
// and 29.0, 2 36.9 and 27.5, 3 35.9 and 26.5, 4 36.8 and 26.9).
constexpr int kPaged8Start = 3;
// A row's largest weight in its unit.  fp16 ends at 65504; the lower end is 2^3 to 2^4 below a new unit's largest weight, so that units change rarely after a
// wave's first tiles (the cases take the same time as with one unit for all rows: 34.2 and 34.7 us, 36.0 and 35.5, 66 and 66, 25.6 and 25.1, 10.3 and 10.8).
constexpr float kUnitLow = 1024.0f, kUnitTop = 32768.0f;
constexpr int kUnitBits = 14;      // a new unit makes the largest weight so far less than 2^14, and at least half of that
constexpr int kUnitLeast = -112;   // weights below 2^-112 get the unit of that: 2^126

// V tiles in LDS: 16-byte chunk c of row r lies at chunk c ^ paged8_v_swizzle(r), so that the sixteen rows that half a wave's
// transposed read touches, 16 bytes each, lie on different banks.
template <int D> __device__ __forceinline__ int paged8_v_swizzle(int row) {
    return D == 128 ? ((row >> 1) & 3) | ((row >> 2) & 4) : ((row >> 2) & 1) | ((row >> 3) & 2);
}

// Of a row in a cache.  (strides below 2^32: a product of 64-bit numbers costs three times as many instructions)
__device__ __forceinline__ int64_t row_offset(int page, int place, int64_t stride_p, int64_t stride_n) {
    return (int64_t)((uint64_t)(unsigned)page * (unsigned)stride_p + (uint64_t)(unsigned)place * (unsigned)stride_n);
}

template <int D, typename QT, typename Code, bool SEVERAL, bool PAGE16>
__global__ __launch_bounds__(kPagedThreads, D == 128 ? 2 : SEVERAL || !PAGE16 ? 3 : 4) void paged8_attn_kernel(PagedArgs a, BlockScales bs) {
    using F16 = PV<_Float16>;
    constexpr int KLOADS = D / 64;        // 64 codes of a row each
    constexpr int CT = D / 16;            // 16-channel tiles
    constexpr int VCPR = D / 16;          // 16-byte chunks per V row
    constexpr int VLOADS = kTileKeys * VCPR / 64;
    constexpr int VSTEP = 64 / VCPR;      // rows of a V load
    constexpr int V_TILE = kTileKeys * D;
    constexpr int WAVE_LDS = V_TILE + 64 * 4;  // and the scales of K and V
    constexpr int SL_RS = D + 4;          // floats per row of the buffer in which the waves' results meet, sixteen rows at a time
    constexpr int SLICE = kPagedWaves * 16 * SL_RS * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[kPagedWaves * WAVE_LDS > SLICE ? kPagedWaves * WAVE_LDS : SLICE];
    __shared__ float row_m[kPagedWaves][16], row_l[kPagedWaves][16];

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Waves share the rows of an item, sixteen each, and then its key tiles.
    const int row_waves = a.row_waves, key_waves = kPagedWaves / row_waves, row_wave = wave % row_waves;
    const int kstep = kTileKeys * key_waves;
    const int per_seq = a.Hkv * a.row_tiles;  // items of a sequence
    const int rows = a.groups * a.M;
    int seq, pos, end, seq_begin;  // share of the line; where the sequence begins on it
    if (a.shares == 0) {
        seq = blockIdx.x / per_seq;
        seq_begin = pos = 0;
        end = seq_chunks(a, seq);
    } else {
        const EqualShares line(line_total(a), a.shares);
        pos = line.begin(blockIdx.x);
        end = line.begin(blockIdx.x + 1);
        if (pos >= end) return;
        if (!find_run(a.seqs, pos, [&](int s) { return seq_units(a, s) * per_seq; }, seq, seq_begin)) return;
    }
    const int share_begin = pos;

    const int vr0 = lane / VCPR, vchunk = lane % VCPR;  // V load e of a lane: row vr0 + VSTEP e, this chunk
    unsigned char* vlds = smem + wave * WAVE_LDS;
    float* slds = reinterpret_cast<float*>(vlds + V_TILE);
    // ds_read_b64_tr_b8: in each group of 16 lanes, lane 2 s + c supplies channels 8 c .. of key row s, and lane i receives channel i
    // of the eight rows.  Group g reads keys 4 g .. and 16 + 4 g .. of the tile, where the lane's P come from.
    const int vkey = 16 * ((l16 >> 3) & 1) + 4 * quad + ((l16 >> 1) & 3);
    const int vtr = vkey * D + 16 * paged8_v_swizzle<D>(vkey) + 8 * (lane & 1);
    static_assert(D == 64 || D == 128, "swizzle periods");

    while (pos < end) {
        // ---- the piece: chunks `first` .. of an item
        const int len = seq_len(a, seq), chunks = seq_chunks(a, seq), units = a.start + chunks;
        // (a workgroup per item: all items at once may be more than 31 bits of chunks)
        int item = blockIdx.x % per_seq, first = 0, n = chunks, before = 0;  // before: other pieces of the share
        const int oseq = seq;
        if (a.shares != 0) {
            item = (pos - seq_begin) / units;
            const int begin = seq_begin + item * units, to = min(begin + units, end);
            before = begin > share_begin ? 1 : 0;
            first = max(pos - begin - a.start, 0);
            n = max(to - begin - a.start, 0) - first;
            pos = to;
            if (pos - seq_begin == units * per_seq) {
                seq_begin = pos;
                seq++;
            }
            if (n == 0) continue;  // (nothing but units before its chunks)
        } else {
            pos = end;
        }
        const int hk = item / a.row_tiles, row0 = item % a.row_tiles * (16 * row_waves);
        const bool whole = n == chunks;
        const int slot = 2 * (int)blockIdx.x + before;
        const int kbeg = first * kChunk, kend = min((first + n) * kChunk, len);

        // this lane's row; rows past the last one multiply a copy of it
        const int wrow0 = row0 + 16 * row_wave, r = min(wrow0 + l16, rows - 1);
        const int mi = SEVERAL ? r / a.groups : 0, h = hk * a.groups + (SEVERAL ? r % a.groups : r);
        // Q, its channels in the order of K's: steps 2 t and 2 t + 1 take channels 64 t + 16 quad + 0 .. 7 and 8 .. 15
        f16x8 qf[2 * KLOADS];
        {
            const unsigned char* qp = a.q + (int64_t)oseq * a.qs_s + (int64_t)h * a.qs_h + (int64_t)mi * a.qs_m + 32 * quad;
#pragma unroll
            for (int t = 0; t < 2 * KLOADS; t++) qf[t] = *reinterpret_cast<const f16x8*>(qp + 128 * (t / 2) + 16 * (t % 2));
        }
        const int my_last = len - a.M + mi;                                      // last key the row sees
        const int all_see = len - a.M + min(wrow0, rows - 1) / a.groups;  // ... the wave's first row

        const unsigned char* kg = a.k + (int64_t)hk * a.ks_h;
        const unsigned char* vg = a.v + (int64_t)hk * a.vs_h;
        // lanes 0 .. 31: scales of the tile's keys, 32 .. 63: of its values
        const float* sg = lane < 32 ? bs.k + hk * bs.k_h : bs.v + hk * bs.v_h;
        const unsigned ss_p = (unsigned)(lane < 32 ? bs.k_p : bs.v_p), ss_b = (unsigned)(lane < 32 ? bs.k_b : bs.v_b);
        typedef __attribute__((address_space(4))) const int32_t* const_i32_ptr;  // (scalar loads)
        const const_i32_ptr table = (const_i32_ptr)(uintptr_t)(a.table + (int64_t)oseq * a.table_stride);
        auto page_of = [&](int t) { return a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size; };
        auto place_of = [&](int t) { return a.page_shift >= 0 ? t & (a.page_size - 1) : t % a.page_size; };
        auto scale_at = [&](int page, int place) { return sg[(uint64_t)(unsigned)page * ss_p + (uint64_t)(unsigned)bs.of(place) * ss_b]; };

        v4i kf[2][KLOADS], vr[VLOADS];
        float sc;  // the lane's scale
        // The tile's table entries: two in scalar registers, or one per lane, for key key0 + lane % 32.
        int entry[2] = {-1, -1};
        auto load_entries = [&](int key0) {  // (past the end: the last one once more)
            if constexpr (PAGE16) {
#pragma unroll
                for (int u = 0; u < 2; u++) entry[u] = table[page_of(min(key0 + 16 * u, kend - 1))];
            } else {
                entry[0] = a.table[(int64_t)oseq * a.table_stride + page_of(min(key0 + (lane & 31), kend - 1))];
            }
        };
        // K, V and scales of the tile whose entries are here, and which of its keys exist (bit j: key j).  Rows of keys that do not
        // exist read a page that does: finite or not, they are taken out below.
        auto load_tile = [&](int key0) {
            unsigned seen = kend - key0 >= kTileKeys ? ~0u : kend > key0 ? (1u << (kend - key0)) - 1 : 0u;
            if constexpr (PAGE16) {
                const unsigned char *kp[2], *vp[2];
                int pages[2], places[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const bool ok = (unsigned)entry[u] < (unsigned)a.pages;
                    if (!ok) seen &= u ? 0xffffu : 0xffff0000u;
                    const int page = ok ? entry[u] : 0, at = place_of(key0 + 16 * u);
                    kp[u] = kg + row_offset(page, at, a.ks_p, a.ks_n);
                    vp[u] = vg + row_offset(page, at, a.vs_p, a.vs_n);
                    pages[u] = page;
                    places[u] = at;
                }
                const unsigned koff = (unsigned)l16 * (unsigned)a.ks_n + 16 * quad, voff = (unsigned)vr0 * (unsigned)a.vs_n + 16 * vchunk;
                sc = scale_at(quad & 1 ? pages[1] : pages[0], (quad & 1 ? places[1] : places[0]) + l16);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int t = 0; t < KLOADS; t++) kf[u][t] = *reinterpret_cast<const v4i*>(kp[u] + koff + 64 * t);
#pragma unroll
                for (int e = 0; e < VLOADS; e++) {
                    const int r = VSTEP * e;  // (a load's rows lie in one half of the tile)
                    vr[e] = *reinterpret_cast<const v4i*>(vp[r / 16] + (unsigned)(r % 16) * (unsigned)a.vs_n + voff);
                }
            } else {
                const bool ok = (unsigned)entry[0] < (unsigned)a.pages;
                seen &= (unsigned)__builtin_amdgcn_ballot_w64(ok);
                const int page = ok ? entry[0] : 0, at = ok ? place_of(min(key0 + (lane & 31), kend - 1)) : 0;
                const int64_t ko = row_offset(page, at, a.ks_p, a.ks_n), vo = row_offset(page, at, a.vs_p, a.vs_n);
                auto from = [&](int64_t x, int who) {  // the lane that knows the row
                    return ((int64_t)__shfl((int)(x >> 32), who) << 32) | (unsigned)__shfl((int)(unsigned)x, who);
                };
                sc = scale_at(page, at);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const unsigned char* p = kg + from(ko, 16 * u + l16) + 16 * quad;
#pragma unroll
                    for (int t = 0; t < KLOADS; t++) kf[u][t] = *reinterpret_cast<const v4i*>(p + 64 * t);
                }
#pragma unroll
                for (int e = 0; e < VLOADS; e++) vr[e] = *reinterpret_cast<const v4i*>(vg + from(vo, vr0 + VSTEP * e) + 16 * vchunk);
            }
            return seen;
        };

        float m_i = -INFINITY, l_i = 0.0f;
        // Weights are multiplied by w_unit (the same in a row's four lanes); w_top: the largest that this lane has seen, relative to m_i, in that unit.
        float w_unit = 1.0f, w_top = 0.0f;
        v4f o[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) o[ct] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

        int key0 = kbeg + kTileKeys * (wave / row_waves);
        unsigned seen = 0;
        if (key0 < kend) {
            load_entries(key0);
            seen = load_tile(key0);
            load_entries(key0 + kstep);
        }
        __builtin_amdgcn_sched_barrier(0);
        // (after the first tile has been requested)
        float unit = 1.0f;  // of the row's scores: 2^(e - 15)
        if constexpr (std::is_same<QT, __bf16>::value) {
            float top = 0.0f;  // of the finite ones
#pragma unroll
            for (int t = 0; t < 2 * KLOADS; t++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = __builtin_fabsf((float)__builtin_bit_cast(bf16x8, qf[t])[i]);
                    top = fmaxf(top, x < INFINITY ? x : 0.0f);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const int e = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : 15;
            unit = __builtin_amdgcn_ldexpf(1.0f, e - 15);
#pragma unroll
            for (int t = 0; t < 2 * KLOADS; t++) {
                const bf16x8 x = __builtin_bit_cast(bf16x8, qf[t]);
#pragma unroll
                for (int i = 0; i < 8; i++) qf[t][i] = (_Float16)__builtin_amdgcn_ldexpf((float)x[i], 15 - e);
            }
        }
        for (; key0 < kend; key0 += kstep) {
            // ---- S^T = K.Q^T: register i of score tile u is key key0 + 16 u + 4 quad + i of the lane's row
            v4f s[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                s[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < KLOADS; t++) {
                    s[u] = F16::mfma16(to_f16<Code>(v2i{kf[u][t][0], kf[u][t][1]}), qf[2 * t], s[u]);
                    s[u] = F16::mfma16(to_f16<Code>(v2i{kf[u][t][2], kf[u][t][3]}), qf[2 * t + 1], s[u]);
                }
            }
            // ---- V tile and scales -> LDS (the wave's own slice: a wave's LDS instructions run in order, no barrier); rows and
            //      value scales of keys that do not exist as zeros
#pragma unroll
            for (int e = 0; e < VLOADS; e++) {
                const int row = vr0 + VSTEP * e;
                if (seen != ~0u && !((seen >> row) & 1)) vr[e] = v4i{0, 0, 0, 0};
                *reinterpret_cast<v4i*>(vlds + row * D + 16 * (vchunk ^ paged8_v_swizzle<D>(row))) = vr[e];
            }
            slds[lane] = lane < 32 ? sc * a.qk_scale : (seen >> (lane & 31)) & 1 ? sc : 0.0f;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_sched_barrier(0);
            // ---- the registers of K and V are requested anew
            const unsigned tile_seen = seen;
            seen = load_tile(key0 + kstep);
            load_entries(key0 + 2 * kstep);
            __builtin_amdgcn_sched_barrier(0);
            // ---- online softmax
            const bool some_see = SEVERAL && key0 + kTileKeys - 1 > all_see;  // keys that some rows see and others do not
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const v4f ks = *reinterpret_cast<const v4f*>(slds + 16 * u + 4 * quad);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = s[u][i] * ks[i];
                    if (tile_seen != ~0u || some_see) {
                        const int j = 16 * u + 4 * quad + i;
                        x = ((tile_seen >> j) & 1) && (!SEVERAL || key0 + j <= my_last) ? x : -INFINITY;
                    }
                    s[u][i] = x;
                    mx = fmaxf(mx, x);
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m_i, mx);
            const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // (no key seen yet: every P below is exp2(-inf) = 0)
            const bool grown = __builtin_amdgcn_ballot_w64(m_new > m_i) != 0;
            if (grown) {
                const float alpha = __builtin_amdgcn_exp2f((m_i - m_use) * unit);  // 0 for a row without a reference point
                l_i *= alpha;
                w_top *= alpha;
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[ct][i] *= alpha;
                m_i = m_new;
            }
            // Weights; the sum of P is taken before they are rounded
            float psum = 0.0f, top = 0.0f;
            const float m_ref = -m_use * unit;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const v4f vs = *reinterpret_cast<const v4f*>(slds + 32 + 16 * u + 4 * quad);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], unit, m_ref));
                    psum += p;
                    float w = p * vs[i];
                    if (SEVERAL && some_see && key0 + 16 * u + 4 * quad + i > my_last) w = 0.0f;  // (a scale that is not finite, under a hidden key)
                    s[u][i] = w;
                    top = fmaxf(top, __builtin_fabsf(w));
                }
            }
            // Does the unit hold them?  Weights that are too large for it are seen by one lane; that all of a row's are small, by none of its four.
            const float before = w_top;
            w_top = fmaxf(w_top, top * w_unit);
            bool fits = __builtin_amdgcn_ballot_w64(w_top > kUnitTop) == 0;
            if (grown) {
                unsigned long long enough = __builtin_amdgcn_ballot_w64(w_top >= kUnitLow);
                enough |= enough >> 32;
                fits &= ((enough | enough >> 16) & 0xffff) == 0xffff;
            }
            if (!fits) {
                // (weights that are not finite spoil their row in any unit; they have the exponent 0 here)
                const int was = __builtin_amdgcn_frexp_expf(w_unit) - 1;
                int e = max(top > 0.0f ? __builtin_amdgcn_frexp_expf(top) : kUnitLeast, before > 0.0f ? __builtin_amdgcn_frexp_expf(before) - was : kUnitLeast);
                e = max(e, __shfl_xor(e, 16));
                e = max(max(e, __shfl_xor(e, 32)), kUnitLeast);
                const int change = kUnitBits - e - was;
                w_unit = __builtin_amdgcn_ldexpf(1.0f, kUnitBits - e);
                w_top = fminf(fmaxf(__builtin_amdgcn_ldexpf(before, change), top * w_unit), kUnitTop);
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[ct][i] = __builtin_amdgcn_ldexpf(o[ct][i], change);
            }
            f16x8 pf;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) pf[4 * u + i] = (_Float16)(s[u][i] * w_unit);
            l_i += psum;
            // ---- O^T += V^T.P^T
            auto v_fragment = [&](int ct) {  // channels 16 ct ..
                typedef __attribute__((address_space(3))) v2i* lds_v2i_ptr;
                return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i_ptr)(vlds + (vtr ^ (16 * ct))));
            };
            // A NaN among e4m3 codes must not reach the rows that do not see its key (0 times it is NaN): where a tile that some rows
            // see further into than others holds one, the matrix instructions get zeros in its place, and the rows that see it NaN.
            unsigned odd = 0;
            if constexpr (SEVERAL && Code::kHasNan) {
                if (some_see) {
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {
                        const v2i f = v_fragment(ct);
                        odd |= Code::nan_bytes((unsigned)f[0]) | Code::nan_bytes((unsigned)f[1]);
                    }
                }
            }
            if (!(SEVERAL && Code::kHasNan) || __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) == 0, 1)) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++) o[ct] = F16::mfma16(to_f16<Code>(v_fragment(ct)), pf, o[ct]);
            } else if constexpr (SEVERAL && Code::kHasNan) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    v2i f = v_fragment(ct);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const unsigned z = Code::nan_bytes((unsigned)f[i]) >> 7;
                        f[i] &= ~(z * 255);
                    }
                    o[ct] = F16::mfma16(to_f16<Code>(f), pf, o[ct]);
                }
#pragma unroll 1
                for (int j = 0; j < kTileKeys; j++)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) {  // channels 16 ct + 4 quad + i, which the lane's accumulators hold
                        const unsigned word = *reinterpret_cast<const unsigned*>(vlds + j * D + 16 * (ct ^ paged8_v_swizzle<D>(j)) + 4 * quad);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (((word >> (8 * i)) & 0x7f) == 0x7f && key0 + j <= my_last) o[ct][i] = NAN;
                    }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }

        // ---- the waves of the workgroup -> one normalized result and its log-sum-exp
        l_i += __shfl_xor(l_i, 16);
        l_i += __shfl_xor(l_i, 32);
        if (quad == 0) {
            row_m[wave][l16] = m_i;
            row_l[wave][l16] = l_i;
        }
        __syncthreads();
        float m = -INFINITY, l = 0.0f;
        for (int w = row_wave; w < kPagedWaves; w += row_waves) m = fmaxf(m, row_m[w][l16]);
        const float m_use = m == -INFINITY ? 0.0f : m;
        for (int w = row_wave; w < kPagedWaves; w += row_waves) l += row_l[w][l16] * __builtin_amdgcn_exp2f((row_m[w][l16] - m_use) * unit);
        // l = 0: a row that saw no key; its output is 0, its log-sum-exp -inf.  (NaN stays.)
        const float f = l != 0.0f ? __builtin_amdgcn_exp2f((m_i - m_use) * unit) / l : 0.0f;
        const float w_step = 1.0f / w_unit;
        if (wave == row_wave && quad == 0 && wrow0 + l16 < rows) {
            const float lse2 = __builtin_log2f(l) + m_use * unit;
            if (!whole) a.part_lse[(int64_t)slot * a.tile_rows + 16 * row_wave + l16] = lse2;
            else if (a.lse) a.lse[((int64_t)oseq * a.Hq + h) * a.M + mi] = lse2 * 0.693147180559945309f;
        }
        float* slice = reinterpret_cast<float*>(smem);  // (the V tiles have been read, since the barrier above)
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
            *reinterpret_cast<v4f*>(slice + (wave * 16 + l16) * SL_RS + 16 * ct + 4 * quad) = v4f{o[ct][0] * f * w_step, o[ct][1] * f * w_step, o[ct][2] * f * w_step, o[ct][3] * f * w_step};
        __syncthreads();
        const int tile_end = min(16 * row_waves, rows - row0);  // rows that exist
        for (int piece = tid; piece < tile_end * (D / 4); piece += kPagedThreads) {
            const int orow = piece / (D / 4), c = 4 * (piece % (D / 4));
            v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = orow / 16; w < kPagedWaves; w += row_waves) {
                const v4f x = *reinterpret_cast<const v4f*>(slice + (w * 16 + orow % 16) * SL_RS + c);
#pragma unroll
                for (int i = 0; i < 4; i++) sum[i] += x[i];
            }
            const int om = SEVERAL ? (row0 + orow) / a.groups : 0, oh = hk * a.groups + (SEVERAL ? (row0 + orow) % a.groups : row0 + orow);
            if (whole)
                store_rounded(static_cast<QT*>(a.out) + (int64_t)oseq * a.os_s + (int64_t)oh * a.os_h + (int64_t)om * a.os_m + c, sum);
            else
                *reinterpret_cast<v4f*>(a.part_o + ((int64_t)slot * a.tile_rows + orow) * D + c) = sum;
        }
        __syncthreads();  // (the next piece's V tiles go where the results lie)
    }
}

}  // namespace

int64_t paged8_workspace_bytes(const sage_paged8_params& p) { return plan_bytes(plan_paged(p.paged, kPaged8Shares, kPaged8Start), p.paged.head_dim); }

template <int D, typename QT, typename Code>
static int launch_paged8(const PagedArgs& a, const BlockScales& bs, const PagedPlan& plan, hipStream_t stream) {
    const int64_t wgs = plan.shares ? plan.shares : plan.items;
    if (wgs > kMaxThreads / kPagedThreads) return fail(SAGE_E_UNSUPPORTED, "sage_paged8_attn: too many workgroups for one launch");
    const dim3 grid((unsigned)wgs), block(kPagedThreads);
    const bool page16 = a.page_size % 16 == 0;
    if (a.M > 1 && page16) hipLaunchKernelGGL((paged8_attn_kernel<D, QT, Code, true, true>), grid, block, 0, stream, a, bs);
    else if (a.M > 1) hipLaunchKernelGGL((paged8_attn_kernel<D, QT, Code, true, false>), grid, block, 0, stream, a, bs);
    else if (page16) hipLaunchKernelGGL((paged8_attn_kernel<D, QT, Code, false, true>), grid, block, 0, stream, a, bs);
    else hipLaunchKernelGGL((paged8_attn_kernel<D, QT, Code, false, false>), grid, block, 0, stream, a, bs);
    if (int rc = check_launch("paged8_attn_kernel")) return rc;
    return launch_paged_combine<D, QT>(a, plan, stream);
}

template <typename Code>
static int launch_paged8(const sage_paged_params& p, const PagedArgs& a, const BlockScales& bs, const PagedPlan& plan, hipStream_t stream) {
    if (p.head_dim == 128)
        return p.dtype == SAGE_BF16 ? launch_paged8<128, __bf16, Code>(a, bs, plan, stream) : launch_paged8<128, _Float16, Code>(a, bs, plan, stream);
    return p.dtype == SAGE_BF16 ? launch_paged8<64, __bf16, Code>(a, bs, plan, stream) : launch_paged8<64, _Float16, Code>(a, bs, plan, stream);
}

int launch_paged8_attn(const sage_paged8_params& p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    PagedPlan plan = plan_paged(p.paged, kPaged8Shares, kPaged8Start);
    if (!workspace || workspace_bytes < plan_bytes(plan, p.paged.head_dim)) plan.shares = 0;  // (nothing is cut then)
    const PagedArgs a = paged_args(p.paged, plan, workspace, 1);
    const BlockScales bs = block_scales(p.scales, p.paged.page_size);
    return p.scales.codes == SAGE_CODE_INT8 ? launch_paged8<Int8>(p.paged, a, bs, plan, stream) : launch_paged8<E4m3>(p.paged, a, bs, plan, stream);
}

}  // namespace sage
