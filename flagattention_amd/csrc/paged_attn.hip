// Dense attention of the newest tokens of every sequence over a cache of keys and values in pages, for gfx950.
//
// Token t of sequence s lies in page block_table[s][t / page_size] at place t % page_size, for t < seq_lens[s]; the last
// new_tokens of them are the queries' own.  Query m of a sequence sees the keys j <= seq_len - new_tokens + m:
//     o = sum_j 2^(c s_j - m) v_j / l,   l = sum_j 2^(c s_j - m),   s_j = sm_scale q . k_j,   c = log2 e.
//
// Bound by the bytes of K and V: the rows of all query heads that share a K/V head (row r = query r / group, head r % group) are
// multiplied from the same tiles, sixteen by a wave and up to 64 by a workgroup, so that the cache is read from memory once (by two
// waves beyond 16 rows and four beyond 32, each for itself: 8 new tokens of 4 heads a group 72 us where one takes 57).  A workgroup is
// four waves.  They share the rows, sixteen each, and then the keys, and a wave walks over its 32-key tiles without a barrier:
// S^T = K.Q^T and O^T += V^T.P^T on the 16x16 matrix instructions, K rows straight into the operand, V through the wave's slice of
// LDS, from where it is read transposed.  The registers of a tile are requested anew as soon as their contents are used up, and the
// entries of the block table a tile ahead of the rows they lead to.
//
// A workgroup takes an item, the rows of a K/V head of a sequence, where the items fill the chip (plan_paged).  Elsewhere the work
// is one line: sequence after sequence, K/V head after head, in chunks of 128 keys, and every workgroup takes an equal share of it,
// whatever the lengths are, which only the device knows: the end of one item, whole ones, the beginning of another.  Items that are
// cut leave partial results, normalized outputs in fp32 and their base-2 log-sum-exps, for a second kernel.
//
// Measured (contiguous K and V are read at 5.3 TB/s by attn_decode.hip): 128 sequences of 512 to 2048 tokens, 16 heads, D64, fp16
// 111 us = 5.2 TB/s; 32 of up to 8192, H32/8, D128, bf16 57 us = 4.3 TB/s, 5 of them the second kernel; 2 of 50000 to 65536, H32/4
// 57 us = 4.15 TB/s, 6 of them the second kernel; one of 300 tokens 9.5 us: a launch, the first tile, and 1.4 us for every further 128 keys.
#include "serve_common.h"

namespace sage {
namespace {

using namespace attn;

constexpr int kPagedWaves = 4;   // (eight, for one workgroup on a compute unit: 10 to 20 % slower)
constexpr int kPagedThreads = 64 * kPagedWaves;
constexpr int kTileKeys = 32;
constexpr int kChunk = kTileKeys * kPagedWaves;  // keys of a unit of the line
constexpr int kPagedShares = 512;                // two workgroups on each compute unit
constexpr int kCombineThreads = 256;

struct PagedArgs {
    const unsigned char* q;
    const unsigned char* k;
    const unsigned char* v;
    void* out;
    float* lse;  // [seqs, Hq, M] natural log, or null
    const int32_t* table;
    const int32_t* lens;
    int64_t qs_s, qs_h, qs_m, ks_p, ks_h, ks_n, vs_p, vs_h, vs_n;  // bytes
    int64_t os_s, os_h, os_m, table_stride;                        // elements
    int32_t seqs, M, Hq, Hkv, groups, pages, page_size, page_shift;  // page_shift: log2 of page_size, -1: it has none
    int32_t capacity;                                                // keys that a row of the table can lead to
    int32_t row_waves;             // waves that share an item's rows, sixteen each: 1, 2 or 4
    int32_t row_tiles, tile_rows;  // items that the rows of a K/V head make; rows of one
    int32_t shares;                // equal shares of the line; 0: a workgroup per item
    float qk_scale;                // sm_scale * log2(e)
    float* part_o;                 // [2 * shares][tile_rows][D]
    float* part_lse;               // [2 * shares][tile_rows], base 2
};

__device__ __forceinline__ int seq_len(const PagedArgs& a, int s) { return min(max(a.lens[s], 0), a.capacity); }
__device__ __forceinline__ int seq_chunks(const PagedArgs& a, int s) { return max((seq_len(a, s) + kChunk - 1) / kChunk, 1); }

// Chunks of all sequences.
__device__ __forceinline__ int line_total(const PagedArgs& a) {
    int sum = 0;
    for (int s = threadIdx.x & 63; s < a.seqs; s += 64) sum += seq_chunks(a, s);
    return wave_sum(sum) * a.Hkv * a.row_tiles;
}

// V tiles in LDS: 16-byte chunk c of row r lies at chunk c ^ paged_v_swizzle(r), so that the sixteen rows which a transposed read
// touches, 32 bytes each, spread over all banks.
template <int D> __device__ __forceinline__ int paged_v_swizzle(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

// SEVERAL: more than one new token per sequence, whose rows see different keys.  PAGE16: the page size
// is a multiple of 16, so that 16 keys of a tile share a page, whose address is then computed in scalar registers.
template <int D, typename VT, bool SEVERAL, bool PAGE16>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_attn_kernel(PagedArgs a) {
    using PVT = PV<VT>;
    using vec16 = typename PVT::vec;
    constexpr int KSTEPS = D / 32;        // matrix instructions of a 16 x 16 score tile: 64 bytes of a row each
    constexpr int CT = D / 16;            // 16-channel tiles
    constexpr int V_RS = 2 * D;           // bytes per V row in LDS
    constexpr int VCPR = V_RS / 16;       // 16-byte chunks per V row
    constexpr int VLOADS = kTileKeys * VCPR / 64;
    constexpr int VSTEP = 64 / VCPR;      // rows of a V load
    constexpr int V_TILE = kTileKeys * V_RS;
    constexpr int SL_RS = D + 4;          // floats per row of the buffer in which the waves' results meet, sixteen rows at a time
    constexpr int SLICE = kPagedWaves * 16 * SL_RS * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[kPagedWaves * V_TILE > SLICE ? kPagedWaves * V_TILE : SLICE];
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
        if (!find_run(a.seqs, pos, [&](int s) { return seq_chunks(a, s) * per_seq; }, seq, seq_begin)) return;
    }
    const int share_begin = pos;

    const int vr0 = lane / VCPR, vchunk = lane % VCPR;  // V load e of a lane: row vr0 + VSTEP e, this chunk
    unsigned char* vlds = smem + wave * V_TILE;
    // ds_read_b64_tr_b16: in each group of 16 lanes, lane 4 s + c supplies channels 4 c .. of key row s, and lane i receives channel i
    // of the four rows.  Group g reads keys 4 g .. and 16 + 4 g .. of the tile, where the lane's P come from.
    const int vkey = 4 * quad + ((lane >> 2) & 3);
    const int vtr = vkey * V_RS + 16 * (((lane & 3) >> 1) ^ paged_v_swizzle<D>(vkey)) + 8 * (lane & 1);
    static_assert(D == 64 || D == 128, "swizzle periods");

    while (pos < end) {
        // ---- the piece: chunks `first` .. of an item
        const int len = seq_len(a, seq), chunks = seq_chunks(a, seq);
        // (a workgroup per item: all items at once may be more than 31 bits of chunks)
        const int item = a.shares == 0 ? blockIdx.x % per_seq : (pos - seq_begin) / chunks;
        const int first = a.shares == 0 ? 0 : pos - seq_begin - item * chunks;
        const int hk = item / a.row_tiles, row0 = item % a.row_tiles * (16 * row_waves);
        const int n = min(chunks - first, end - pos);
        const bool whole = n == chunks;
        const int slot = 2 * (int)blockIdx.x + (pos != share_begin);
        const int kbeg = first * kChunk, kend = min((first + n) * kChunk, len);
        const int oseq = seq;
        pos += n;
        if (a.shares != 0 && pos - seq_begin == chunks * per_seq) {
            seq_begin = pos;
            seq++;
        }

        // this lane's row; rows past the last one multiply a copy of it
        const int wrow0 = row0 + 16 * row_wave, r = min(wrow0 + l16, rows - 1);
        const int mi = SEVERAL ? r / a.groups : 0, h = hk * a.groups + (SEVERAL ? r % a.groups : r);
        v4i qf[KSTEPS];
        {
            const unsigned char* qp = a.q + (int64_t)oseq * a.qs_s + (int64_t)h * a.qs_h + (int64_t)mi * a.qs_m + 16 * quad;
#pragma unroll
            for (int t = 0; t < KSTEPS; t++) qf[t] = *reinterpret_cast<const v4i*>(qp + 64 * t);
        }
        const int my_last = len - a.M + mi;                                      // last key the row sees
        const int all_see = len - a.M + min(wrow0, rows - 1) / a.groups;  // ... the wave's first row

        const unsigned char* kg = a.k + (int64_t)hk * a.ks_h;
        const unsigned char* vg = a.v + (int64_t)hk * a.vs_h;
        typedef __attribute__((address_space(4))) const int32_t* const_i32_ptr;  // (scalar loads)
        const const_i32_ptr table = (const_i32_ptr)(uintptr_t)(a.table + (int64_t)oseq * a.table_stride);
        auto page_of = [&](int t) { return a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size; };
        auto place_of = [&](int t) { return a.page_shift >= 0 ? t & (a.page_size - 1) : t % a.page_size; };

        v4i kf[2][KSTEPS], vr[VLOADS];
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
        // K and V of the tile whose entries are here, and which of its keys exist (bit j: key j).  Rows of keys that do not
        // exist read a page that does: finite or not, they are taken out below.
        auto load_tile = [&](int key0) {
            unsigned seen = kend - key0 >= kTileKeys ? ~0u : kend > key0 ? (1u << (kend - key0)) - 1 : 0u;
            if constexpr (PAGE16) {
                const unsigned char *kp[2], *vp[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const bool ok = (unsigned)entry[u] < (unsigned)a.pages;
                    if (!ok) seen &= u ? 0xffffu : 0xffff0000u;
                    const int page = ok ? entry[u] : 0, at = place_of(key0 + 16 * u);
                    kp[u] = kg + (int64_t)page * a.ks_p + (int64_t)at * a.ks_n;
                    vp[u] = vg + (int64_t)page * a.vs_p + (int64_t)at * a.vs_n;
                }
                const unsigned koff = (unsigned)l16 * (unsigned)a.ks_n + 16 * quad, voff = (unsigned)vr0 * (unsigned)a.vs_n + 16 * vchunk;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int t = 0; t < KSTEPS; t++) kf[u][t] = *reinterpret_cast<const v4i*>(kp[u] + koff + 64 * t);
#pragma unroll
                for (int e = 0; e < VLOADS; e++) {
                    const int r = VSTEP * e;  // (a load's rows lie in one half of the tile)
                    vr[e] = *reinterpret_cast<const v4i*>(vp[r / 16] + (unsigned)(r % 16) * (unsigned)a.vs_n + voff);
                }
            } else {
                const bool ok = (unsigned)entry[0] < (unsigned)a.pages;
                seen &= (unsigned)__builtin_amdgcn_ballot_w64(ok);
                const int64_t page = ok ? entry[0] : 0, at = ok ? place_of(min(key0 + (lane & 31), kend - 1)) : 0;
                const int64_t ko = page * a.ks_p + at * a.ks_n, vo = page * a.vs_p + at * a.vs_n;
                auto from = [&](int64_t x, int who) {  // the lane that knows the row
                    return ((int64_t)__shfl((int)(x >> 32), who) << 32) | (unsigned)__shfl((int)(unsigned)x, who);
                };
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const unsigned char* p = kg + from(ko, 16 * u + l16) + 16 * quad;
#pragma unroll
                    for (int t = 0; t < KSTEPS; t++) kf[u][t] = *reinterpret_cast<const v4i*>(p + 64 * t);
                }
#pragma unroll
                for (int e = 0; e < VLOADS; e++) vr[e] = *reinterpret_cast<const v4i*>(vg + from(vo, vr0 + VSTEP * e) + 16 * vchunk);
            }
            return seen;
        };

        float m_i = -INFINITY, l_i = 0.0f;
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
        for (; key0 < kend; key0 += kstep) {
            // ---- S^T = K.Q^T: register i of score tile u is key key0 + 16 u + 4 quad + i of the lane's row
            v4f s[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                s[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = 0; t < KSTEPS; t++)
                    s[u] = PVT::mfma16(__builtin_bit_cast(vec16, kf[u][t]), __builtin_bit_cast(vec16, qf[t]), s[u]);
            }
            // ---- V tile -> LDS (the wave's own slice: a wave's LDS instructions run in order, no barrier); rows of keys that do
            //      not exist as zeros
#pragma unroll
            for (int e = 0; e < VLOADS; e++) {
                const int row = vr0 + VSTEP * e;
                if (seen != ~0u && !((seen >> row) & 1)) vr[e] = v4i{0, 0, 0, 0};
                *reinterpret_cast<v4i*>(vlds + row * V_RS + 16 * (vchunk ^ paged_v_swizzle<D>(row))) = vr[e];
            }
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
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = s[u][i] * a.qk_scale;
                    if (tile_seen != ~0u || some_see) {
                        const int j = 16 * u + 4 * quad + i;
                        x = ((tile_seen >> j) & 1) && (!SEVERAL || key0 + j <= my_last) ? x : -INFINITY;
                    }
                    s[u][i] = x;
                    mx = fmaxf(mx, x);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m_i, mx);
            const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // (no key seen yet: every P below is exp2(-inf) = 0)
            if (__builtin_amdgcn_ballot_w64(m_new > m_i) != 0) {
                const float alpha = __builtin_amdgcn_exp2f(m_i - m_use);  // 0 for a row without a reference point
                l_i *= alpha;
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[ct][i] *= alpha;
                m_i = m_new;
            }
            // P is rounded to 16 bits for the matrix instructions (at most 1, half a step of itself off); its sum is taken before that
            vec16 pf;
            float psum = 0.0f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = __builtin_amdgcn_exp2f(s[u][i] - m_use);
                    psum += p;
                    pf[4 * u + i] = (VT)p;
                }
            l_i += psum;
            // ---- O^T += V^T.P^T
            auto v_fragment = [&](int ct) {  // channels 16 ct ..
                const unsigned char* p0 = vlds + (vtr ^ (32 * ct));
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p0);
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p0 + 16 * V_RS));
                return __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            // An infinity or NaN in V must not reach the rows that do not see its key (0 times it is NaN): where a tile that some rows
            // see further into than others holds one, the matrix instructions get zeros in its place, and it is added to the rows
            // that see its key.
            unsigned odd = 0;
            if (SEVERAL && some_see) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    const v4i f = v_fragment(ct);
#pragma unroll
                    for (int i = 0; i < 4; i++) odd |= nonfinite_halves<VT>((unsigned)f[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                asm volatile("" ::: "memory");  // (the fragments are read again below: kept they cost 32 registers)
            }
            if (!SEVERAL || __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) == 0, 1)) {
#pragma unroll
                for (int ct = 0; ct < CT; ct++) o[ct] = PVT::mfma16(__builtin_bit_cast(vec16, v_fragment(ct)), pf, o[ct]);
            } else {
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    o[ct] = PVT::mfma16(__builtin_bit_cast(vec16, finite_only<VT>(v_fragment(ct))), pf, o[ct]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                add_nonfinite<D, VT>(vlds, [](int row) { return paged_v_swizzle<D>(row); }, pf, my_last - key0 + 1, o);
            }
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
        for (int w = row_wave; w < kPagedWaves; w += row_waves) l += row_l[w][l16] * __builtin_amdgcn_exp2f(row_m[w][l16] - m_use);
        // l = 0: a row that saw no key; its output is 0, its log-sum-exp -inf.  (NaN stays.)
        const float f = l != 0.0f ? __builtin_amdgcn_exp2f(m_i - m_use) / l : 0.0f;
        if (wave == row_wave && quad == 0 && wrow0 + l16 < rows) {
            const float lse2 = __builtin_log2f(l) + m_use;
            if (!whole) a.part_lse[(int64_t)slot * a.tile_rows + 16 * row_wave + l16] = lse2;
            else if (a.lse) a.lse[((int64_t)oseq * a.Hq + h) * a.M + mi] = lse2 * 0.693147180559945309f;
        }
        float* slice = reinterpret_cast<float*>(smem);  // (the V tiles have been read, since the barrier above)
#pragma unroll
        for (int ct = 0; ct < CT; ct++)
            *reinterpret_cast<v4f*>(slice + (wave * 16 + l16) * SL_RS + 16 * ct + 4 * quad) = v4f{o[ct][0] * f, o[ct][1] * f, o[ct][2] * f, o[ct][3] * f};
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
                store_rounded(static_cast<VT*>(a.out) + (int64_t)oseq * a.os_s + (int64_t)oh * a.os_h + (int64_t)om * a.os_m + c, sum);
            else
                *reinterpret_cast<v4f*>(a.part_o + ((int64_t)slot * a.tile_rows + orow) * D + c) = sum;
        }
        __syncthreads();  // (the next piece's V tiles go where the results lie)
    }
}

// The parts of the items that were cut: lse = log2 sum_s 2^lse_s, out = sum_s 2^(lse_s - lse) o_s.  A workgroup per item (BY_ITEM) and
// few of its rows, or, where the items outnumber the cuts, per cut between two shares: the first cut inside an item takes care of it
// (per item: 32 sequences x 8 K/V heads 58.2 -> 57.6 us for the whole call, 1000 x 8 450 -> 470).  SG groups of D / 4 threads share
// the parts of a row.
template <int D, typename VT, bool BY_ITEM>
__global__ __launch_bounds__(kCombineThreads) void paged_combine_kernel(PagedArgs a) {
    constexpr int TPR = D / 4, SG = 4, ROWS = kCombineThreads / (TPR * SG);
    constexpr int kBatch = 8;  // loads on their way together
    __shared__ float sm_m[kCombineThreads], sm_den[kCombineThreads];
    __shared__ v4f sm_acc[kCombineThreads];
    const int per_seq = a.Hkv * a.row_tiles;
    int seq, item, begin;  // begin: of the item on the line
    int all = 0, before = 0;  // chunks of the sequences; of those before this workgroup's
    for (int i = threadIdx.x & 63; i < a.seqs; i += 64) {
        const int n = seq_chunks(a, i);
        all += n;
        before += i < (int)blockIdx.x / per_seq ? n : 0;
    }
    const EqualShares line(wave_sum(all) * per_seq, a.shares);
    if (BY_ITEM) {
        seq = blockIdx.x / per_seq;
        item = blockIdx.x % per_seq;
        begin = wave_sum(before) * per_seq + item * seq_chunks(a, seq);
    } else {
        const int pos = line.begin(blockIdx.x + 1);
        if (pos >= line.begin(blockIdx.x + 2)) return;  // (the shares from here on are empty)
        if (!find_run(a.seqs, pos, [&](int s) { return seq_chunks(a, s) * per_seq; }, seq, begin)) return;
        item = (pos - begin) / seq_chunks(a, seq);
        begin += item * seq_chunks(a, seq);
        if (begin == pos || line.owner(begin) != (int)blockIdx.x) return;
    }
    const int chunks = seq_chunks(a, seq);
    const int first = line.owner(begin), last = line.owner(begin + chunks - 1);
    if (first == last) return;  // (whole)
    const int hk = item / a.row_tiles, row0 = item % a.row_tiles * (16 * a.row_waves), rows = a.groups * a.M;
    const int c = 4 * (threadIdx.x % TPR), sg = (threadIdx.x / TPR) % SG;
    const int trow = blockIdx.y * ROWS + threadIdx.x / (TPR * SG);  // row of the tile
    if (row0 + (int)blockIdx.y * ROWS >= rows) return;
    const bool ok = trow < a.tile_rows && row0 + trow < rows;
    const int srow = ok ? trow : 0;
    auto slot = [&](int w) { return (int64_t)(2 * w + (w == first && begin != line.begin(w))) * a.tile_rows + srow; };
    float m = -INFINITY, den = 0.0f;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int w0 = first + sg; w0 <= last; w0 += SG * kBatch) {
        float x[kBatch];
        v4f o[kBatch];
        float top = m;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {  // (past the end: the last part once more)
            const int64_t s = slot(min(w0 + SG * u, last));
            x[u] = a.part_lse[s];
            o[u] = *reinterpret_cast<const v4f*>(a.part_o + s * D + c);
        }
#pragma unroll
        for (int u = 0; u < kBatch; u++) top = x[u] > top || x[u] != x[u] ? x[u] : top;  // (NaN stays)
        if (top == -INFINITY) continue;  // (no key seen so far)
        const float alpha = __builtin_amdgcn_exp2f(m - top);
        den *= alpha;
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] *= alpha;
        m = top;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const float w = w0 + SG * u <= last ? __builtin_amdgcn_exp2f(x[u] - m) : 0.0f;
            den += w;
            // (a part without a key has weight 0 and is all zeros)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = w0 + SG * u <= last ? __builtin_fmaf(w, o[u][i], acc[i]) : acc[i];
        }
    }
    sm_m[threadIdx.x] = m;
    sm_den[threadIdx.x] = den;
    sm_acc[threadIdx.x] = acc;
    __syncthreads();
    if (sg != 0 || !ok) return;
#pragma unroll
    for (int g = 1; g < SG; g++) {
        const float x = sm_m[threadIdx.x + g * TPR];
        m = x > m || x != x ? x : m;
    }
    acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    den = 0.0f;
    if (m != -INFINITY) {
#pragma unroll
        for (int g = 0; g < SG; g++) {
            const float w = __builtin_amdgcn_exp2f(sm_m[threadIdx.x + g * TPR] - m);
            const v4f o = sm_acc[threadIdx.x + g * TPR];
            den = __builtin_fmaf(w, sm_den[threadIdx.x + g * TPR], den);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = __builtin_fmaf(w, o[i], acc[i]);
        }
    }
    const float inv = den != 0.0f ? 1.0f / den : 0.0f;
    const int mi = (row0 + trow) / a.groups, h = hk * a.groups + (row0 + trow) % a.groups;
    store_rounded(static_cast<VT*>(a.out) + (int64_t)seq * a.os_s + (int64_t)h * a.os_h + (int64_t)mi * a.os_m + c,
                  v4f{acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv});
    if (a.lse && c == 0)
        a.lse[((int64_t)seq * a.Hq + h) * a.M + mi] = (__builtin_log2f(den) + (m == -INFINITY ? 0.0f : m)) * 0.693147180559945309f;
}

struct PagedPlan {
    int64_t row_waves, row_tiles, tile_rows, capacity, items, shares;
};

PagedPlan plan_paged(const sage_paged_params& p) {
    PagedPlan plan;
    const int64_t rows = p.heads_q / p.heads_kv * p.new_tokens;
    plan.row_waves = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    plan.row_tiles = (rows + 16 * plan.row_waves - 1) / (16 * plan.row_waves);
    plan.tile_rows = rows < 16 * plan.row_waves ? rows : 16 * plan.row_waves;
    const int64_t most = 0x7fffffffLL - 4 * kChunk;
    plan.capacity = p.table_width > most / p.page_size ? most : p.table_width * p.page_size;
    plan.items = p.seqs * p.heads_kv * plan.row_tiles;
    // Equal shares, or a workgroup per item?  A workgroup needs about 1.4 us for a chunk, and a launch of items lasts as long as its
    // longest one (chunks: what a sequence could hold at most) or as all of them over the chip; shares cost a second launch, and
    // every item in a share a start and an end, about five chunks in all.  Measured, items and shares (bf16, D128): 1 x 32 heads, 700
    // tokens 14.1 and 11.7 us, 8 x 8, 2000 26.6 and 20.2, 32 x 8, up to 8192 99 and 59, 16 x 32, up to 9000 239 and 192; 32 x 8, up to
    // 700 15.7 and 19.5, 128 x 8, up to 500 36.5 and 48, 1000 x 8, up to 1500 378 and 451; D64: 128 x 16, up to 2048 111 and 119.
    const int64_t chunks = (plan.capacity + kChunk - 1) / kChunk;
    plan.shares = plan.items * chunks < kPagedShares ? plan.items * chunks : kPagedShares;
    if (chunks <= 5 + 6 * plan.items / kPagedShares || plan.items > 0x7fffffffLL / chunks) plan.shares = 0;
    return plan;
}

}  // namespace

int64_t paged_workspace_bytes(const sage_paged_params& p) {
    const PagedPlan plan = plan_paged(p);
    return 2 * plan.shares * plan.tile_rows * (p.head_dim + 1) * (int64_t)sizeof(float);
}

template <int D, typename VT>
static int launch_paged(const PagedArgs& a, const PagedPlan& plan, hipStream_t stream) {
    const int64_t wgs = plan.shares ? plan.shares : plan.items;
    if (wgs > kMaxThreads / kPagedThreads) return fail(SAGE_E_UNSUPPORTED, "sage_paged_attn: too many workgroups for one launch");
    const dim3 grid((unsigned)wgs), block(kPagedThreads);
    const bool page16 = a.page_size % 16 == 0;
    if (a.M > 1 && page16) hipLaunchKernelGGL((paged_attn_kernel<D, VT, true, true>), grid, block, 0, stream, a);
    else if (a.M > 1) hipLaunchKernelGGL((paged_attn_kernel<D, VT, true, false>), grid, block, 0, stream, a);
    else if (page16) hipLaunchKernelGGL((paged_attn_kernel<D, VT, false, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_attn_kernel<D, VT, false, false>), grid, block, 0, stream, a);
    if (int rc = check_launch("paged_attn_kernel")) return rc;
    if (a.shares < 2) return SAGE_OK;
    constexpr int rows = kCombineThreads / D;
    const unsigned row_groups = (unsigned)((a.tile_rows + rows - 1) / rows);
    if (plan.items < a.shares)
        hipLaunchKernelGGL((paged_combine_kernel<D, VT, true>), dim3((unsigned)plan.items, row_groups), dim3(kCombineThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_combine_kernel<D, VT, false>), dim3((unsigned)a.shares - 1, row_groups), dim3(kCombineThreads), 0, stream, a);
    return check_launch("paged_combine_kernel");
}

int launch_paged_attn(const sage_paged_params& p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    PagedPlan plan = plan_paged(p);
    if (!workspace || workspace_bytes < paged_workspace_bytes(p)) plan.shares = 0;  // (nothing is cut then)
    PagedArgs a{};
    a.q = (const unsigned char*)p.q.ptr; a.k = (const unsigned char*)p.k_cache.ptr; a.v = (const unsigned char*)p.v_cache.ptr;
    a.out = p.out.ptr; a.lse = p.log_normalizer; a.table = p.block_table; a.lens = p.seq_lens;
    a.qs_s = 2 * p.q.stride_b; a.qs_h = 2 * p.q.stride_h; a.qs_m = 2 * p.q.stride_n;
    a.ks_p = 2 * p.k_cache.stride_b; a.ks_h = 2 * p.k_cache.stride_h; a.ks_n = 2 * p.k_cache.stride_n;
    a.vs_p = 2 * p.v_cache.stride_b; a.vs_h = 2 * p.v_cache.stride_h; a.vs_n = 2 * p.v_cache.stride_n;
    a.os_s = p.out.stride_b; a.os_h = p.out.stride_h; a.os_m = p.out.stride_n; a.table_stride = p.table_stride;
    a.seqs = (int)p.seqs; a.M = (int)p.new_tokens; a.Hq = (int)p.heads_q; a.Hkv = (int)p.heads_kv;
    a.groups = (int)(p.heads_q / p.heads_kv);
    a.pages = (int)p.pages; a.page_size = (int)p.page_size;
    a.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)p.page_size) : -1;
    a.capacity = (int)plan.capacity; a.row_tiles = (int)plan.row_tiles; a.row_waves = (int)plan.row_waves; a.tile_rows = (int)plan.tile_rows;
    a.shares = (int)plan.shares;
    a.qk_scale = p.sm_scale * 1.44269504089f;
    a.part_o = (float*)workspace;
    a.part_lse = a.part_o + 2 * plan.shares * plan.tile_rows * p.head_dim;
    if (p.head_dim == 128) return p.dtype == SAGE_BF16 ? launch_paged<128, __bf16>(a, plan, stream) : launch_paged<128, _Float16>(a, plan, stream);
    return p.dtype == SAGE_BF16 ? launch_paged<64, __bf16>(a, plan, stream) : launch_paged<64, _Float16>(a, plan, stream);
}

}  // namespace sage
