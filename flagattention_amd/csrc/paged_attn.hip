// Dense attention of the newest tokens of every sequence over a cache of keys and values in pages, for gfx950.
//
// Token t of sequence s lies in page block_table[s][t / page_size] at place t % page_size, for t < seq_lens[s]; the last
// new_tokens of them are the queries' own.  Query m of a sequence sees the keys j <= seq_len - new_tokens + m:
//     o = sum_j 2^(c s_j - m) v_j / l,   l = sum_j 2^(c s_j - m),   s_j = sm_scale q . k_j,   c = log2 e.
//
// Bound by the bytes of K and V: the rows of all query heads that share a K/V head (row r = query r / group, head r % group) are
// multiplied from the same tiles, up to 32 rows at a time, so that the cache is read once.  A workgroup is four waves, and a wave
// walks over 32-key tiles of its own without a barrier: S^T = K.Q^T and O^T += V^T.P^T on the 32x32 matrix instructions, K rows
// straight into the operand, V through the wave's slice of LDS, from where it is read transposed.  The entries of the block table
// are fetched a tile ahead of the rows they lead to.
//
// The work is one line: sequence after sequence, K/V head after head, in chunks of 128 keys.  Every workgroup takes an equal
// share of it, whatever the lengths are, which only the device knows: the end of one item (rows of a K/V head of a sequence),
// whole ones, the beginning of another.  Items that are cut leave partial results, normalized outputs in fp32 and their base-2
// log-sum-exps, for a second kernel.
#include "serve_common.h"

namespace sage {
namespace {

using namespace attn;

constexpr int kPagedWaves = 4;
constexpr int kPagedThreads = 64 * kPagedWaves;
constexpr int kTileKeys = 32;
constexpr int kChunk = kTileKeys * kPagedWaves;  // keys of a unit of the line: a tile for every wave
constexpr int kPagedShares = 512;                // two workgroups on each compute unit
constexpr int kRowsPerTile = 32;

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
    int32_t row_tiles, tile_rows;  // tiles of up to 32 rows of an item's queries; rows of one
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

template <int D> __device__ __forceinline__ int paged_v_swizzle(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

// SEVERAL: more than one new token per sequence, whose rows see different keys.
template <int D, typename VT, bool SEVERAL>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_attn_kernel(PagedArgs a) {
    using PVT = PV<VT>;
    using vec16 = typename PVT::vec;
    constexpr int KSTEPS = D / 16;        // matrix instructions of a 32 x 32 score tile: 32 bytes of a row each
    constexpr int DT = D / 32;
    constexpr int V_RS = 2 * D;           // bytes per V row in LDS
    constexpr int VCPR = V_RS / 16;       // 16-byte chunks per V row
    constexpr int VLOADS = kTileKeys * VCPR / 64;
    constexpr int V_TILE = kTileKeys * V_RS;
    constexpr int SL_RS = 32 + 4;         // floats per row of the buffer in which the waves' results meet, 32 channels at a time
    constexpr int SLICE = kPagedWaves * 32 * SL_RS * 4;
    __shared__ __attribute__((aligned(16))) unsigned char smem[kPagedWaves * V_TILE > SLICE ? kPagedWaves * V_TILE : SLICE];
    __shared__ float row_m[kPagedWaves][32], row_l[kPagedWaves][32];

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per_seq = a.Hkv * a.row_tiles;  // items of a sequence
    const int rows = a.groups * a.M;
    int seq, pos, end, seq_begin;  // share of the line; where the sequence begins on it
    if (a.shares == 0) {
        seq = blockIdx.x / per_seq;
        seq_begin = 0;
        const int c = seq_chunks(a, seq);
        pos = blockIdx.x % per_seq * c;
        end = pos + c;
    } else {
        const EqualShares line(line_total(a), a.shares);
        pos = line.begin(blockIdx.x);
        end = line.begin(blockIdx.x + 1);
        if (pos >= end) return;
        if (!find_run(a.seqs, pos, [&](int s) { return seq_chunks(a, s) * per_seq; }, seq, seq_begin)) return;
    }
    const int share_begin = pos;

    const int vr0 = lane / VCPR, vchunk = lane % VCPR;  // V load e of a lane: row vr0 + e * 64 / VCPR, this chunk
    unsigned char* vlds = smem + wave * V_TILE;
    int vtr[DT];  // LDS offsets of the transposed fragment reads (see attn_fast_kernel.h)
    {
        const int s4 = (lane >> 2) & 3, a4 = lane & 3, g1 = (lane >> 4) & 1;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            vtr[dt] = (4 * half + s4) * V_RS + 16 * ((4 * dt + 2 * g1 + (a4 >> 1)) ^ paged_v_swizzle<D>(s4)) + 8 * (a4 & 1);
    }

    while (pos < end) {
        // ---- the piece: chunks `first` .. of an item
        const int len = seq_len(a, seq), chunks = seq_chunks(a, seq);
        const int item = (pos - seq_begin) / chunks, first = pos - seq_begin - item * chunks;
        const int hk = item / a.row_tiles, row0 = item % a.row_tiles * kRowsPerTile;
        const int n = min(chunks - first, end - pos);
        const bool whole = n == chunks;
        const int slot = 2 * (int)blockIdx.x + (pos != share_begin);
        const int kbeg = first * kChunk, kend = min((first + n) * kChunk, len);
        const int oseq = seq;
        pos += n;
        if (pos - seq_begin == chunks * per_seq) {
            seq_begin = pos;
            seq++;
        }

        // this lane's row; rows past the last one multiply a copy of it
        const int r = min(row0 + l32, rows - 1);
        const int mi = r / a.groups, h = hk * a.groups + r % a.groups;
        v4i qf[KSTEPS];
        {
            const unsigned char* qp = a.q + (int64_t)oseq * a.qs_s + (int64_t)h * a.qs_h + (int64_t)mi * a.qs_m + 16 * half;
#pragma unroll
            for (int t = 0; t < KSTEPS; t++) qf[t] = *reinterpret_cast<const v4i*>(qp + 32 * t);
        }
        const int my_last = len - a.M + mi;            // last key the row sees
        const int all_see = len - a.M + row0 / a.groups;  // ... the tile's first row

        const unsigned char* kg = a.k + (int64_t)hk * a.ks_h;
        const unsigned char* vg = a.v + (int64_t)hk * a.vs_h;
        const int32_t* table = a.table + (int64_t)oseq * a.table_stride;
        // Key key0 + l32: its page, or -1 (no such key, or an entry that is no page), and its place in the page.
        auto load_entry = [&](int key0) {
            const int t = key0 + l32;
            const int idx = a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size;
            return t < kend ? table[idx] : -1;
        };
        auto place = [&](int key0) {
            const int t = key0 + l32;
            return a.page_shift >= 0 ? t & (a.page_size - 1) : t % a.page_size;
        };
        v4i kf[KSTEPS], vr[VLOADS];
        // Rows of keys that do not exist read page 0: finite or not, they are taken out below.
        auto load_k = [&](int page, int at) {
            const unsigned char* p = kg + (int64_t)page * a.ks_p + (int64_t)at * a.ks_n + 16 * half;
#pragma unroll
            for (int t = 0; t < KSTEPS; t++) kf[t] = *reinterpret_cast<const v4i*>(p + 32 * t);
        };
        auto load_v = [&](int page, int at) {
            const int64_t mine = (int64_t)page * a.vs_p + (int64_t)at * a.vs_n;
#pragma unroll
            for (int e = 0; e < VLOADS; e++) {
                const int from = vr0 + e * (64 / VCPR);  // the lane that knows the row
                const unsigned lo = __shfl((int)(unsigned)mine, from);
                const int hi = __shfl((int)(mine >> 32), from);
                vr[e] = *reinterpret_cast<const v4i*>(vg + (((int64_t)hi << 32) | lo) + 16 * vchunk);
            }
        };

        float m_i = -INFINITY, l_i = 0.0f;
        v16f o[DT];
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[dt][i] = 0.0f;

        int key0 = kbeg + kTileKeys * wave;
        unsigned seen = 0, seen_next = 0;  // bit j: key j of the tile (of the next one) exists
        int entry = -1;                    // of the next tile
        if (key0 < kend) {
            const int e = load_entry(key0);
            entry = load_entry(key0 + kChunk);
            const bool ok = (unsigned)e < (unsigned)a.pages;
            seen = (unsigned)__builtin_amdgcn_ballot_w64(ok);
            const int page = ok ? e : 0, at = ok ? place(key0) : 0;
            load_k(page, at);
            load_v(page, at);
        }
        for (; key0 < kend; key0 += kChunk) {
            const bool ok = (unsigned)entry < (unsigned)a.pages;  // (behind the last tile: no key, page 0 once more)
            seen_next = (unsigned)__builtin_amdgcn_ballot_w64(ok);
            const int page = ok ? entry : 0, at = ok ? place(key0 + kChunk) : 0;
            entry = load_entry(key0 + 2 * kChunk);
            // ---- S^T = K.Q^T; the K registers are requested anew right behind it
            v16f s;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
            for (int t = 0; t < KSTEPS; t++) s = PVT::mfma(__builtin_bit_cast(vec16, kf[t]), __builtin_bit_cast(vec16, qf[t]), s);
            load_k(page, at);
            __builtin_amdgcn_sched_barrier(0);
            // ---- V tile -> LDS (the wave's own slice: a wave's LDS instructions run in order, no barrier); rows of keys that do
            //      not exist as zeros
#pragma unroll
            for (int e = 0; e < VLOADS; e++) {
                const int row = vr0 + e * (64 / VCPR);
                if (seen != ~0u && !((seen >> row) & 1)) vr[e] = v4i{0, 0, 0, 0};
                *reinterpret_cast<v4i*>(vlds + row * V_RS + 16 * (vchunk ^ paged_v_swizzle<D>(row))) = vr[e];
            }
            load_v(page, at);
            __builtin_amdgcn_sched_barrier(0);
            // ---- online softmax: register i of this lane is key key0 + 8 (i / 4) + 4 half + i % 4 of its row
            const bool some_see = SEVERAL && key0 + kTileKeys - 1 > all_see;  // keys that some rows see and others do not
            const bool hides = seen != ~0u || some_see;
            float x[16];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int j = 8 * (i >> 2) + 4 * half + (i & 3);
                x[i] = s[i] * a.qk_scale;
                if (hides) x[i] = ((seen >> j) & 1) && (!SEVERAL || key0 + j <= my_last) ? x[i] : -INFINITY;
                mx = fmaxf(mx, x[i]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m_i, mx);
            const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // (no key seen yet: every P below is exp2(-inf) = 0)
            if (__builtin_amdgcn_ballot_w64(m_new > m_i) != 0) {
                const float alpha = __builtin_amdgcn_exp2f(m_i - m_use);  // 0 for a row without a reference point
                l_i *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[dt][i] *= alpha;
                m_i = m_new;
            }
            // P is rounded to 16 bits for the matrix instructions (at most 1, so half a step of 1 off); its sum is taken before that
            vec16 pf[2];
            float psum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float p = __builtin_amdgcn_exp2f(x[i] - m_use);
                psum += p;
                pf[i >> 3][i & 7] = (VT)p;
            }
            l_i += psum;
            // ---- O^T += V^T.P^T
            auto v_fragment = [&](int c, int dt) {
                const unsigned char* p0 = vlds + vtr[dt] + 16 * c * V_RS;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p0);
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p0 + 8 * V_RS));
                return __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            // An infinity or NaN in V under a hidden key must not reach the rows that do not see it (0 times it is NaN): where a tile
            // that hides keys holds one, the matrix instructions get zeros in its place, and it is added to the rows that see its key.
            unsigned odd = 0;
            if (SEVERAL && some_see) {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const v4i f = v_fragment(c, dt);
#pragma unroll
                        for (int i = 0; i < 4; i++) odd |= nonfinite_halves<VT>((unsigned)f[i]);
                    }
            }
            if (!SEVERAL || __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) == 0, 1)) {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[dt] = PVT::mfma(__builtin_bit_cast(vec16, v_fragment(c, dt)), pf[c], o[dt]);
            } else {
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
                        o[dt] = PVT::mfma(__builtin_bit_cast(vec16, finite_only<VT>(v_fragment(c, dt))), pf[c], o[dt]);
                add_nonfinite<D, VT>(vlds, [](int row) { return paged_v_swizzle<D>(row); }, pf[0], pf[1], my_last - key0 + 1, o);
            }
            seen = seen_next;
        }

        // ---- the waves of the workgroup -> one normalized result and its log-sum-exp
        const float l_tot = l_i + __shfl_xor(l_i, 32);
        if (half == 0) {
            row_m[wave][l32] = m_i;
            row_l[wave][l32] = l_tot;
        }
        __syncthreads();
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int w = 0; w < kPagedWaves; w++) m = fmaxf(m, row_m[w][l32]);
        const float m_use = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < kPagedWaves; w++) l += row_l[w][l32] * __builtin_amdgcn_exp2f(row_m[w][l32] - m_use);
        // l = 0: a row that saw no key; its output is 0, its log-sum-exp -inf.  (NaN stays.)
        const float f = l != 0.0f ? __builtin_amdgcn_exp2f(m_i - m_use) / l : 0.0f;
        if (wave == 0 && half == 0 && row0 + l32 < rows) {
            const float lse2 = __builtin_log2f(l) + m_use;
            if (!whole) a.part_lse[(int64_t)slot * a.tile_rows + l32] = lse2;
            else if (a.lse) a.lse[((int64_t)oseq * a.Hq + h) * a.M + mi] = lse2 * 0.693147180559945309f;
        }
        float* slice = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            __syncthreads();  // the V tiles / the previous channels have been read
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<v4f*>(slice + (wave * 32 + l32) * SL_RS + 8 * g + 4 * half) =
                    v4f{o[dt][4 * g] * f, o[dt][4 * g + 1] * f, o[dt][4 * g + 2] * f, o[dt][4 * g + 3] * f};
            __syncthreads();
            const int orow = tid / 8, c = 4 * (tid % 8);  // 32 rows of eight groups of four channels
            if (row0 + orow < rows) {
                v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kPagedWaves; w++) {
                    const v4f x = *reinterpret_cast<const v4f*>(slice + (w * 32 + orow) * SL_RS + c);
#pragma unroll
                    for (int i = 0; i < 4; i++) sum[i] += x[i];
                }
                const int om = (row0 + orow) / a.groups, oh = hk * a.groups + (row0 + orow) % a.groups;
                if (whole)
                    store_rounded(static_cast<VT*>(a.out) + (int64_t)oseq * a.os_s + (int64_t)oh * a.os_h + (int64_t)om * a.os_m + 32 * dt + c, sum);
                else
                    *reinterpret_cast<v4f*>(a.part_o + ((int64_t)slot * a.tile_rows + orow) * D + 32 * dt + c) = sum;
            }
        }
        __syncthreads();  // (the next piece's V tiles go where the results lie)
    }
}

// The parts of the items that were cut: lse = log2 sum_s 2^lse_s, out = sum_s 2^(lse_s - lse) o_s.  A workgroup per cut between two
// shares; the first cut inside an item takes care of it.  SG groups of D / 4 threads share the parts of a row.
template <int D, typename VT>
__global__ __launch_bounds__(kPagedThreads) void paged_combine_kernel(PagedArgs a) {
    constexpr int TPR = D / 4, SG = 4, ROWS = kPagedThreads / (TPR * SG);
    constexpr int kBatch = 8;  // loads on their way together
    __shared__ float sm_m[kPagedThreads], sm_den[kPagedThreads];
    __shared__ v4f sm_acc[kPagedThreads];
    const EqualShares line(line_total(a), a.shares);
    const int cut = blockIdx.x + 1, pos = line.begin(cut);
    const int per_seq = a.Hkv * a.row_tiles;
    int seq, seq_begin;
    if (line.begin(cut + 1) <= pos) return;  // (the shares from here on are empty)
    if (!find_run(a.seqs, pos, [&](int s) { return seq_chunks(a, s) * per_seq; }, seq, seq_begin)) return;
    const int chunks = seq_chunks(a, seq), item = (pos - seq_begin) / chunks;
    const int begin = seq_begin + item * chunks;
    const int first = line.owner(begin);
    if (begin == pos || first + 1 != cut) return;
    const int last = line.owner(begin + chunks - 1);
    const int hk = item / a.row_tiles, row0 = item % a.row_tiles * kRowsPerTile, rows = a.groups * a.M;
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
    int64_t row_tiles, tile_rows, capacity, items, shares;
};

PagedPlan plan_paged(const sage_paged_params& p) {
    PagedPlan plan;
    const int64_t rows = p.heads_q / p.heads_kv * p.new_tokens;
    plan.row_tiles = (rows + kRowsPerTile - 1) / kRowsPerTile;
    plan.tile_rows = rows < kRowsPerTile ? rows : kRowsPerTile;
    const int64_t most = 0x7fffffffLL - 4 * kChunk;
    plan.capacity = p.table_width > most / p.page_size ? most : p.table_width * p.page_size;
    plan.items = p.seqs * p.heads_kv * plan.row_tiles;
    // What the sequences could hold at most, in chunks.  Short ones are not cut: a second launch takes as long as four to
    // six chunks more.
    const int64_t chunks = (plan.capacity + kChunk - 1) / kChunk;
    plan.shares = plan.items * chunks < kPagedShares ? plan.items * chunks : kPagedShares;
    if (chunks <= 6 || plan.items > 0x7fffffffLL / chunks) plan.shares = 0;
    return plan;
}

}  // namespace

int64_t paged_workspace_bytes(const sage_paged_params& p) {
    const PagedPlan plan = plan_paged(p);
    return 2 * plan.shares * plan.tile_rows * (p.head_dim + 1) * (int64_t)sizeof(float);
}

template <int D, typename VT>
static int launch_paged(const PagedArgs& a, int64_t wgs, hipStream_t stream) {
    if (a.M > 1) hipLaunchKernelGGL((paged_attn_kernel<D, VT, true>), dim3((unsigned)wgs), dim3(kPagedThreads), 0, stream, a);
    else hipLaunchKernelGGL((paged_attn_kernel<D, VT, false>), dim3((unsigned)wgs), dim3(kPagedThreads), 0, stream, a);
    if (int rc = check_launch("paged_attn_kernel")) return rc;
    if (a.shares < 2) return SAGE_OK;
    constexpr int rows = kPagedThreads / D;
    hipLaunchKernelGGL((paged_combine_kernel<D, VT>), dim3((unsigned)(a.shares - 1), (unsigned)((a.tile_rows + rows - 1) / rows)),
                       dim3(kPagedThreads), 0, stream, a);
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
    a.capacity = (int)plan.capacity; a.row_tiles = (int)plan.row_tiles; a.tile_rows = (int)plan.tile_rows;
    a.shares = (int)plan.shares;
    a.qk_scale = p.sm_scale * 1.44269504089f;
    a.part_o = (float*)workspace;
    a.part_lse = a.part_o + 2 * plan.shares * plan.tile_rows * p.head_dim;
    if (plan.shares == 0 && plan.items > 0x7fffffffLL) return fail(SAGE_E_UNSUPPORTED, "sage_paged_attn: too many workgroups for one launch");
    const int64_t wgs = plan.shares ? plan.shares : plan.items;
    if (p.head_dim == 128) return p.dtype == SAGE_BF16 ? launch_paged<128, __bf16>(a, wgs, stream) : launch_paged<128, _Float16>(a, wgs, stream);
    return p.dtype == SAGE_BF16 ? launch_paged<64, __bf16>(a, wgs, stream) : launch_paged<64, _Float16>(a, wgs, stream);
}

}  // namespace sage
