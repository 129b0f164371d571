// What the kernels that attend over paged caches share (paged_attn.hip: 16-bit caches, paged8_attn.hip: caches of 8-bit codes): their
// arguments, how the keys of all sequences are laid out on a line and shared out, and the kernel that joins the parts.
#pragma once
#include "serve_common.h"

namespace sage {
namespace {

using namespace attn;

constexpr int kPagedWaves = 4;   // (eight, for one workgroup on a compute unit: 10 to 20 % slower)
constexpr int kPagedThreads = 64 * kPagedWaves;
constexpr int kTileKeys = 32;
constexpr int kChunk = kTileKeys * kPagedWaves;  // keys of a unit of the line
constexpr int kPagedWhole = 512;   // items that fill the chip (plan_paged)
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
    int32_t start;                 // units of the line before an item's chunks
    float qk_scale;                // sm_scale * log2(e)
    float* part_o;                 // [2 * shares][tile_rows][D]
    float* part_lse;               // [2 * shares][tile_rows], base 2
};

__device__ __forceinline__ int seq_len(const PagedArgs& a, int s) { return min(max(a.lens[s], 0), a.capacity); }
__device__ __forceinline__ int seq_chunks(const PagedArgs& a, int s) { return max((seq_len(a, s) + kChunk - 1) / kChunk, 1); }
// What an item takes on the line: its chunks, after `start` units for what its beginning and end cost.
__device__ __forceinline__ int seq_units(const PagedArgs& a, int s) { return a.start + seq_chunks(a, s); }

// Units of all sequences.
__device__ __forceinline__ int line_total(const PagedArgs& a) {
    int sum = 0;
    for (int s = threadIdx.x & 63; s < a.seqs; s += 64) sum += seq_units(a, s);
    return wave_sum(sum) * a.Hkv * a.row_tiles;
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
    int all = 0, before = 0;  // units of the sequences; of those before this workgroup's
    for (int i = threadIdx.x & 63; i < a.seqs; i += 64) {
        const int n = seq_units(a, i);
        all += n;
        before += i < (int)blockIdx.x / per_seq ? n : 0;
    }
    const EqualShares line(wave_sum(all) * per_seq, a.shares);
    if (BY_ITEM) {
        seq = blockIdx.x / per_seq;
        item = blockIdx.x % per_seq;
        begin = wave_sum(before) * per_seq + item * seq_units(a, seq);
    } else {
        const int pos = line.begin(blockIdx.x + 1);
        if (pos >= line.begin(blockIdx.x + 2)) return;  // (the shares from here on are empty)
        if (!find_run(a.seqs, pos, [&](int s) { return seq_units(a, s) * per_seq; }, seq, begin)) return;
        item = (pos - begin) / seq_units(a, seq);
        begin += item * seq_units(a, seq);
        if (line.owner(begin + a.start) != (int)blockIdx.x) return;
    }
    const int first = line.owner(begin + a.start), last = line.owner(begin + seq_units(a, seq) - 1);
    if (first == last) return;  // (whole)
    const int hk = item / a.row_tiles, row0 = item % a.row_tiles * (16 * a.row_waves), rows = a.groups * a.M;
    const int c = 4 * (threadIdx.x % TPR), sg = (threadIdx.x / TPR) % SG;
    const int trow = blockIdx.y * ROWS + threadIdx.x / (TPR * SG);  // row of the tile
    if (row0 + (int)blockIdx.y * ROWS >= rows) return;
    const bool ok = trow < a.tile_rows && row0 + trow < rows;
    const int srow = ok ? trow : 0;
    auto slot = [&](int w) { return (int64_t)(2 * w + (w == first && begin > line.begin(w))) * a.tile_rows + srow; };
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
    int64_t row_waves, row_tiles, tile_rows, capacity, items, shares, start;
};

PagedPlan plan_paged(const sage_paged_params& p, int most_shares, int start) {
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
    plan.shares = plan.items * chunks < most_shares ? plan.items * chunks : most_shares;
    if (chunks <= 5 + 6 * plan.items / kPagedWhole || plan.items > 0x7fffffffLL / (chunks + start)) plan.shares = 0;
    plan.start = plan.shares < most_shares ? 0 : start;  // (a share for every chunk: none begins two items)
    return plan;
}

int64_t plan_bytes(const PagedPlan& plan, int64_t head_dim) { return 2 * plan.shares * plan.tile_rows * (head_dim + 1) * (int64_t)sizeof(float); }

// e: bytes of an entry of the caches
PagedArgs paged_args(const sage_paged_params& p, const PagedPlan& plan, void* workspace, int e) {
    PagedArgs a{};
    a.q = (const unsigned char*)p.q.ptr; a.k = (const unsigned char*)p.k_cache.ptr; a.v = (const unsigned char*)p.v_cache.ptr;
    a.out = p.out.ptr; a.lse = p.log_normalizer; a.table = p.block_table; a.lens = p.seq_lens;
    a.qs_s = 2 * p.q.stride_b; a.qs_h = 2 * p.q.stride_h; a.qs_m = 2 * p.q.stride_n;
    a.ks_p = e * p.k_cache.stride_b; a.ks_h = e * p.k_cache.stride_h; a.ks_n = e * p.k_cache.stride_n;
    a.vs_p = e * p.v_cache.stride_b; a.vs_h = e * p.v_cache.stride_h; a.vs_n = e * p.v_cache.stride_n;
    a.os_s = p.out.stride_b; a.os_h = p.out.stride_h; a.os_m = p.out.stride_n; a.table_stride = p.table_stride;
    a.seqs = (int)p.seqs; a.M = (int)p.new_tokens; a.Hq = (int)p.heads_q; a.Hkv = (int)p.heads_kv;
    a.groups = (int)(p.heads_q / p.heads_kv);
    a.pages = (int)p.pages; a.page_size = (int)p.page_size;
    a.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)p.page_size) : -1;
    a.capacity = (int)plan.capacity; a.row_tiles = (int)plan.row_tiles; a.row_waves = (int)plan.row_waves; a.tile_rows = (int)plan.tile_rows;
    a.shares = (int)plan.shares; a.start = (int)plan.start;
    a.qk_scale = p.sm_scale * 1.44269504089f;
    a.part_o = (float*)workspace;
    a.part_lse = a.part_o + 2 * plan.shares * plan.tile_rows * p.head_dim;
    return a;
}

// The second kernel of a launch in shares.
template <int D, typename VT>
int launch_paged_combine(const PagedArgs& a, const PagedPlan& plan, hipStream_t stream) {
    if (a.shares < 2) return SAGE_OK;
    constexpr int rows = kCombineThreads / D;
    const unsigned row_groups = (unsigned)((a.tile_rows + rows - 1) / rows);
    if (plan.items < a.shares)
        hipLaunchKernelGGL((paged_combine_kernel<D, VT, true>), dim3((unsigned)plan.items, row_groups), dim3(kCombineThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((paged_combine_kernel<D, VT, false>), dim3((unsigned)a.shares - 1, row_groups), dim3(kCombineThreads), 0, stream, a);
    return check_launch("paged_combine_kernel");
}

}  // namespace
}  // namespace sage
