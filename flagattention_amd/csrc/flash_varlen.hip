// Dense attention forward over packed sequences for gfx950: the queries, keys and values of all sequences lie one after the other
// in q [total_q, Hq, D], k, v [total_k, Hkv, D], and cu_seqlens say where each sequence begins.
//
//     s_ij = sm_scale q_i . k_j   for keys j <= i + (Lk - Lq) of the sequence (without the causal flag: all of them),
//     o_i  = sum_j 2^(c s_ij - m_i) v_j / l_i,   l_i = sum_j 2^(c s_ij - m_i),   c = log2 e,
//
// one pass over the keys with the running maximum m_i.  Nothing is padded: a workgroup takes 128 rows of one sequence, a row
// being a (query, query head) pair of one K/V head (row r = query r / group, head r % group), so that grouped heads share their
// K and V tiles and the rows of a block lie close to the causal diagonal.  The lengths are read on the device: the grid is
// as large as total_q and the number of sequences allow, and a workgroup finds its sequence by itself (find_run).
//
// S^T = K.Q^T and O^T += V^T.P^T on v_mfma_f32_32x32x16: a lane owns one row, and P goes from the accumulators to the operand
// without leaving its registers.  K and V tiles go straight into LDS for the four waves, two of each resident, one barrier per
// step.  Bound by the matrix cores, with the vector instructions of the softmax in their shadow, in two forms (launch_d):
// * Many blocks: tiles of 32 keys, 168 registers, three workgroups on a compute unit.  They are not tied to each other, so that one's
//   exponentials, barriers, search for a block, first tile and output meet the others' matrix instructions.
// * Few: tiles of 64 keys, two workgroups on a compute unit.  A step makes the scores of the next tile while it takes the exponentials
//   of its own.
// No vector register is spilled (13 to 28 scalar ones, to lanes of vector registers, in the cut forms and the 64-key form at head_dim
// 128): a reload waits for every tile on its way into LDS, since loads return in order (three reloads per step: 4 documents of 512 to
// 8192 tokens, H32/8 D128, 593 -> 811 us).  What is rare is therefore kept out of its registers (careful_row).  Workgroups are handed
// out longest first over all sequences (find_block).
// Measured (bf16, D128, causal; a library product of 8192^3 reaches 1360 to 1380 TFLOP/s here): those documents 577 to 600 us = 1085 to
// 1130 TFLOP/s, one sequence of 16384 tokens with H16/2 960 us = 1145, 48 prompts of 1 to 700 tokens 39 us, 200 of 100 to 200 142 us =
// 4.2 TB/s.
// There a workgroup spends 1.7 us on finding its block, 2.2 on its first tile, 1.3 on every further 64 keys and 1.4 on its output.
#include <math.h>

#include "serve_common.h"
#include "step_lines.h"

namespace sage {
namespace {

using namespace attn;

struct VarlenArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;  // [Hq, total_q] natural log, or null
    const int32_t* cu_q;
    const int32_t* cu_k;
    int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h, os_t, os_h;
    int32_t seqs, total_q, total_k, Hkv, groups, causal;
    float qk_scale;       // sm_scale * log2(e)
    uint32_t inv_groups;  // 2^16 / groups, rounded down, + 1
    // Cut launch: workgroups that share all steps evenly, tokens of a block (a power of two; log2), partial results.
    int32_t shares, tokens_shift;
    float* part_o;    // [2 * shares][4 waves][D / 32][4][64 lanes][4]: normalized outputs in the order of the accumulator registers
    float* part_lse;  // [2 * shares][128], base 2
};

constexpr int kVarWaves = 4;
constexpr int kVarThreads = 64 * kVarWaves;
constexpr int kVarRows = 32 * kVarWaves;
constexpr float kLag = 8.0f;
// From this size of a row's reference point on (in base 2) its rounding to 24 bits, which shifts all exponents of the row alike, can
// take P out of its range: by up to 4 below it.
constexpr float kHuge = 134217728.0f;

// Sequence s of a packed axis.  (Offsets out of order or past the end give no rows that do not exist.)
__device__ __forceinline__ void sequence(const int32_t* cu, int s, int total, int& begin, int& len) {
    begin = min(max(cu[s], 0), total);
    len = min(max(cu[s + 1], begin), total) - begin;
}

constexpr unsigned kOrderless = 256;  // workgroups that have a compute unit each: the order in which they start is of no matter

// The block of 128 rows that workgroup `at` (of a K/V head) takes, and its sequence; false: there is none.
// Up to 64 sequences, a lane each: the blocks that see the most keys first, so that the last workgroups to start are the short
// ones.  With more of them, and where the order is of no matter (3 x 100 to 300 tokens 12.0 -> 11.5 us): sequence after sequence,
// each from its last block on.
__device__ __forceinline__ bool find_block(const VarlenArgs& a, int at, int& q0, int& M, int& k0, int& N, int& block) {
    const int lane = threadIdx.x & 63;
    auto blocks = [&](int m) { return (int)(((int64_t)m * a.groups + kVarRows - 1) / kVarRows); };
    if (a.seqs == 1) {  // (the search for one of several takes 1 us: 77 tokens 7.2 -> 6.4 us, 500 15.4 -> 14.3)
        sequence(a.cu_q, 0, a.total_q, q0, M);
        sequence(a.cu_k, 0, a.total_k, k0, N);
        block = blocks(M) - 1 - at;
        return block >= 0;
    }
    if (a.seqs > 64 || gridDim.x <= kOrderless) {
        auto count = [&](int s) {
            int begin, len;
            sequence(a.cu_q, s, a.total_q, begin, len);
            return blocks(len);
        };
        int seq, first;
        if (!find_run(a.seqs, at, count, seq, first)) return false;
        sequence(a.cu_q, seq, a.total_q, q0, M);
        sequence(a.cu_k, seq, a.total_k, k0, N);
        block = blocks(M) - 1 - (at - first);
        return true;
    }
    int lq0, lm = 0, lk0, ln = 0;
    sequence(a.cu_q, min(lane, a.seqs - 1), a.total_q, lq0, lm);
    sequence(a.cu_k, min(lane, a.seqs - 1), a.total_k, lk0, ln);
    if (lane >= a.seqs) lm = 0;
    const int nb = blocks(lm);
    // blocks below `first_of(l)` visit fewer than l key tiles
    auto first_of = [&](int l) {
        const int before = kVarKeys * (l - 1) - ln;  // keys
        if (!a.causal) return before < 0 ? 0 : nb;
        const int first = min(max(before, -lm), 0) + lm;  // the first query that sees a key of tile l - 1
        return first == lm ? nb : first * a.groups / kVarRows;
    };
    if (at >= wave_sum(nb)) return false;
    int low = 0, high = wave_max(ln) / kVarKeys + 2;  // the largest level l with more than `at` blocks of l tiles and more: low <= l < high
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (wave_sum(nb - first_of(mid)) > at) low = mid;
        else high = mid;
    }
    const int above = first_of(low + 1), mine = above - (low > 0 ? first_of(low) : 0);  // this lane's blocks of the level
    const int rank = at - wave_sum(nb - above);
    const int incl = wave_scan(mine);
    const int seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > rank));
    q0 = __builtin_amdgcn_readlane(lq0, seq);
    M = __builtin_amdgcn_readlane(lm, seq);
    k0 = __builtin_amdgcn_readlane(lk0, seq);
    N = __builtin_amdgcn_readlane(ln, seq);
    block = __builtin_amdgcn_readlane(above - 1 - (rank - (incl - mine)), seq);
    return true;
}

template <int D> __device__ __forceinline__ int var_v_swizzle(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

__device__ __forceinline__ int sequence_steps(const VarlenArgs& a, int s) {
    int begin, m, n;
    sequence(a.cu_q, s, a.total_q, begin, m);
    sequence(a.cu_k, s, a.total_k, begin, n);
    return Steps(m, n, a.tokens_shift, a.causal).total() * a.Hkv;
}

__device__ __forceinline__ int all_steps(const VarlenArgs& a) {
    int sum = 0;
    for (int s = threadIdx.x & 63; s < a.seqs; s += 64) sum += sequence_steps(a, s);
    return wave_sum(sum);
}

// The block that holds step `pos` of the line.
struct BlockAt {
    int q0, M, k0, N;  // its sequence
    int hk, block;
    int begin, tiles;  // its first step on the line; its tiles are the steps from begin + kStart on
    bool found;
    __device__ BlockAt(const VarlenArgs& a, int pos) {
        int seq, first;
        found = find_run(a.seqs, pos, [&](int s) { return sequence_steps(a, s); }, seq, first);
        if (!found) return;
        sequence(a.cu_q, seq, a.total_q, q0, M);
        sequence(a.cu_k, seq, a.total_k, k0, N);
        const Steps line(M, N, a.tokens_shift, a.causal);
        const int per_head = line.total();
        hk = (pos - first) / per_head;
        first += hk * per_head;
        int low = 0, high = line.nb;
        while (high - low > 1) {
            const int mid = (low + high) / 2;
            if (first + line.before(mid) <= pos) low = mid;
            else high = mid;
        }
        block = low;
        begin = first + line.before(low);
        tiles = line.tiles(low);
    }
};

// One row by one wave, from its keys alone: query token qt, head h, the first n keys from k0 on.  A lane is a key for the scores,
// and D / 64 channels for the output.  part_o: where the wave's partial results begin and the row's log-sum-exp goes, for row r of
// the wave, or null.  For rows whose tiles hold infinities or NaN in V and for huge scores: a hundred times and more slower
// than the kernel below, and hardly ever called.
template <int D, typename VT>
__device__ void careful_row(const VarlenArgs& a, int qt, int h, int hk, int k0, int n, float* part_o, float* part_lse, int r) {
    constexpr int CH = D / 64;
    typedef VT vt8 __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63;
    const VT* q = static_cast<const VT*>(a.q) + (int64_t)qt * a.qs_t + (int64_t)h * a.qs_h;
    const VT* k = static_cast<const VT*>(a.k) + (int64_t)k0 * a.ks_t + (int64_t)hk * a.ks_h;
    const VT* v = static_cast<const VT*>(a.v) + (int64_t)k0 * a.vs_t + (int64_t)hk * a.vs_h;
    float m = -INFINITY, l = 0.0f, o[CH] = {};
    for (int n0 = 0; n0 < n; n0 += 64) {
        const int key = min(n0 + lane, n - 1);
        float s = 0.0f;
#pragma unroll 1
        for (int c = 0; c < D; c += 8) {
            const vt8 x = *reinterpret_cast<const vt8*>(q + c), y = *reinterpret_cast<const vt8*>(k + (int64_t)key * a.ks_t + c);
#pragma unroll
            for (int i = 0; i < 8; i++) s = __builtin_fmaf((float)x[i], (float)y[i], s);
        }
        s = n0 + lane < n ? s * a.qk_scale : -INFINITY;
        float top = fmaxf(m, s);
#pragma unroll
        for (int d = 32; d > 0; d /= 2) top = fmaxf(top, __shfl_xor(top, d));
        const float m_use = top == -INFINITY ? 0.0f : top;
        const float alpha = __builtin_amdgcn_exp2f(m - m_use), p = __builtin_amdgcn_exp2f(s - m_use);
        float sum = p;
#pragma unroll
        for (int d = 32; d > 0; d /= 2) sum += __shfl_xor(sum, d);
        l = l * alpha + sum;
#pragma unroll
        for (int i = 0; i < CH; i++) o[i] *= alpha;
        m = top;
        // (an output that is NaN stays so: where all of the row's are, only its statistics can still change)
        bool lost = true;
#pragma unroll
        for (int i = 0; i < CH; i++) lost = lost && o[i] != o[i];
        if (__builtin_amdgcn_ballot_w64(!lost) == 0) {
            if (!part_o && !a.lse) break;
            continue;
        }
#pragma unroll 1
        for (int j = 0; j < min(64, n - n0); j++) {
            const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j));
#pragma unroll
            for (int i = 0; i < CH; i++) o[i] = __builtin_fmaf(pj, (float)v[(int64_t)(n0 + j) * a.vs_t + lane + 64 * i], o[i]);
        }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    if (part_o) {
#pragma unroll
        for (int i = 0; i < CH; i++) {
            const int c = lane + 64 * i;
            part_o[(c / 8) * 256 + (32 * (c / 4 % 2) + r) * 4 + c % 4] = o[i] * inv;
        }
        if (lane == 0) part_lse[r] = __builtin_log2f(l) + (m == -INFINITY ? 0.0f : m);
        return;
    }
#pragma unroll
    for (int i = 0; i < CH; i++) static_cast<VT*>(a.out)[(int64_t)qt * a.os_t + (int64_t)h * a.os_h + lane + 64 * i] = (VT)(o[i] * inv);
    if (a.lse && lane == 0) a.lse[(int64_t)h * a.total_q + qt] = (__builtin_log2f(l) + (m == -INFINITY ? 0.0f : m)) * 0.693147180559945309f;
}

// CUT: a workgroup takes an equal share of the launch's steps instead of a block: the end of one, whole ones, the beginning of another.
// KEYS: of a tile, 64 or 32.
template <int D, typename VT, bool CUT, int KEYS>
__global__ __launch_bounds__(kVarThreads, KEYS == 64 ? 2 : 3) void flash_varlen_kernel(VarlenArgs args) {
    const VarlenArgs& a0 = args;
    using PVT = PV<VT>;
    using vec16 = typename PVT::vec;
    constexpr int KS = D / 16;      // matrix instructions of one 32 x 32 score tile
    constexpr int DT = D / 32;      // 32-channel tiles of the output
    constexpr int RS = 2 * D;       // bytes per K / V row
    constexpr int CPR = RS / 16;    // 16-byte chunks per row
    constexpr int TILE = KEYS * RS;
    constexpr int LOADS = TILE / 1024 / kVarWaves;  // 1 KB loads per wave of a K (of a V) tile
    constexpr int KT = KEYS / 32;
    static_assert(KT == 1 || KT == 2, "one or two halves");
    constexpr int UNIT = kVarKeys / KEYS;  // tiles in a step of the line
    constexpr int O_RS = 2 * D + 16;  // of an output row on its way through LDS
    constexpr int OUT = D == 128 ? 32 * kVarWaves * O_RS : 0;
    __shared__ __attribute__((aligned(16))) unsigned char all_smem[4 * TILE > OUT ? 4 * TILE : OUT];
    auto smem = reinterpret_cast<unsigned char(*)[2][TILE]>(all_smem);  // [K, V][buffer]

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int pos = 0, pos_end = 1, share = 0;  // (CUT) this workgroup's steps
    if constexpr (CUT) {
        // (neighbours on the line, which read the same keys, on one XCD: workgroups go to the eight of them in turn)
        share = blockIdx.x % 8 * (a0.shares / 8) + blockIdx.x / 8;
        const EqualShares line(all_steps(a0), a0.shares);
        pos = line.begin(share);
        pos_end = line.begin(share + 1);
    }
    const int pos_begin = pos;
  while (pos < pos_end) {
    // (CUT: the arguments are read again for each piece, behind an opaque pointer: kept across the pieces they cost scalar registers
    // that the step loop then reloads)
    typedef __attribute__((address_space(4))) const void* const_ptr;
    const_ptr again_args = (const_ptr)__builtin_amdgcn_kernarg_segment_ptr();
    if constexpr (CUT) asm volatile("" : "+s"(again_args));
    const VarlenArgs& a = CUT ? *(const VarlenArgs*)again_args : args;
    int hk = blockIdx.x % a.Hkv, q0, M, k0, N, block;
    int block_rows = kVarRows, first_tile = 0, cut_tiles = 0;
    bool whole = true;
    const int slot = 2 * share + (pos != pos_begin);  // (CUT) of the piece's results, if it is not the whole block
    if constexpr (CUT) {
        const BlockAt at(a, pos);
        if (!at.found) return;
        q0 = at.q0; M = at.M; k0 = at.k0; N = at.N; hk = at.hk; block = at.block;
        block_rows = a.groups << a.tokens_shift;
        first_tile = max(pos - at.begin - kStart, 0);
        const bool later = pos != pos_begin;
        pos = min(at.begin + kStart + at.tiles, pos_end);
        cut_tiles = pos - at.begin - kStart - first_tile;
        if (cut_tiles <= 0) break;  // (no tile of this block: it is the next share's)
        whole = cut_tiles == at.tiles;
        if (later) __syncthreads();  // (the piece before has been read)
    } else {
        pos = pos_end;
        if (!find_block(a, blockIdx.x / a.Hkv, q0, M, k0, N, block)) return;
    }
    // rows of this block; the problem of a piece begins at its first key
    const int row0 = block * block_rows, rows = CUT ? min(row0 + block_rows, M * a.groups) : M * a.groups;
    if constexpr (CUT) {
        k0 += first_tile * kVarKeys;
        N -= first_tile * kVarKeys;
    }
    const int shift = N - M;
    // Row row0 + r is head rem0 + r - groups * j of token tok0 + j, j = tokens_on(r): r < 128, so that products of 16 bits divide it
    // exactly (n inv_groups = 2^16 n / groups + less than n, and n < 256 here) or, for larger groups, a comparison.
    const int tok0 = CUT ? block << a.tokens_shift : row0 / a.groups, rem0 = row0 - tok0 * a.groups;
    auto tokens_on = [&](int r) { return a.groups < kVarRows ? (int)((unsigned)(rem0 + r) * a.inv_groups >> 16) : rem0 + r >= a.groups ? 1 : 0; };
    const int my_row = 32 * wave + l32, last_row = rows - 1 - row0;
    const bool row_ok = my_row <= last_row;
    const int my_on = tokens_on(min(my_row, last_row));
    const int my_m = tok0 + my_on, my_h = hk * a.groups + rem0 + min(my_row, last_row) - my_on * a.groups;

    // Q rows as the B operand: lane (row l32, half) holds elements 16 t + 8 half .. + 7 of its row for step t
    vec16 qf[KS];
    {
        const VT* qp = static_cast<const VT*>(a.q) + (int64_t)(q0 + my_m) * a.qs_t + (int64_t)my_h * a.qs_h + 8 * half;
#pragma unroll
        for (int t = 0; t < KS; t++) qf[t] = *reinterpret_cast<const vec16*>(qp + 16 * t);
    }
    const VT* kbase = static_cast<const VT*>(a.k) + (int64_t)k0 * a.ks_t + (int64_t)hk * a.ks_h;
    const VT* vbase = static_cast<const VT*>(a.v) + (int64_t)k0 * a.vs_t + (int64_t)hk * a.vs_h;

    // keys that any row of the workgroup / of this wave can see, and those that every row of the wave sees
    int n_end = N, wave_end = N, all_see = N;
    if (a.causal) {
        auto sees = [&](int r) { return max(min(N, tok0 + tokens_on(min(r, last_row)) + 1 + shift), 0); };  // keys that row row0 + r sees
        n_end = sees(block_rows - 1);
        wave_end = sees(32 * wave + 31);
        all_see = sees(32 * wave);
    }
    const int my_lim = a.causal ? min(my_m + shift, N - 1) : N - 1;  // last key this lane's row sees
    int ntiles = (n_end + KEYS - 1) / KEYS;
    if (CUT) ntiles = min(ntiles, UNIT * cut_tiles);
    // tiles that this wave multiplies with, and how many of them, the first ones, hide no key
    const int my_tiles = 32 * wave <= last_row ? min((wave_end + KEYS - 1) / KEYS, ntiles) : 0;
    const int clear_tiles = min(all_see / KEYS, my_tiles);

    // Tile t of K and V -> one of the two buffers, straight into LDS (written in assembly, as in attn_fast_kernel.h: the compiler
    // would wait for every outstanding load before each LDS read; m0 holds the LDS address and nothing else here uses it).
    // Chunk c of row r lies at chunk c ^ (r mod chunks) for K and at c ^ var_v_swizzle(r) for V: the load fetches the chunk that
    // belongs where a lane writes, the fragment reads spread over all banks.  Load e of a wave: kRound rows further on, a whole
    // number of swizzle periods.  Rows past the end re-read the last one.
    constexpr int kRound = kVarWaves * 64 / CPR;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)all_smem;
    const int frow = (64 / CPR) * wave + lane / CPR;  // row of load 0
    const unsigned kchunk = 16 * ((lane % CPR) ^ (frow & (CPR - 1))), vchunk = 16 * ((lane % CPR) ^ var_v_swizzle<D>(frow));
    const unsigned koff = (unsigned)frow * (unsigned)(a.ks_t * 2) + kchunk, voff = (unsigned)frow * (unsigned)(a.vs_t * 2) + vchunk;
    auto fetch = [&](auto whole, const VT* base, int64_t stride, unsigned off, unsigned chunk, int t, unsigned dst) {
        const int n0 = KEYS * t;
        const VT* tile = base + (int64_t)n0 * stride;
        const unsigned to = lds0 + dst + 1024 * wave;
        if (decltype(whole)::value || n0 + KEYS <= N) {
#pragma unroll
            for (int e = 0; e < LOADS; e++)
                asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(tile + e * kRound * stride),
                             "s"(to + 1024 * kVarWaves * e) : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < LOADS; e++) {
                const unsigned cut = (unsigned)min(frow + kRound * e, N - 1 - n0) * (unsigned)(stride * 2) + chunk;
                asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(cut), "s"(tile),
                             "s"(to + 1024 * kVarWaves * e) : "memory");
            }
        }
    };
    // whole: tiles that are known to end before the last key
    auto fetch_k = [&](auto whole, int t) { fetch(whole, kbase, a.ks_t, koff, kchunk, t, (unsigned)((t & 1) * TILE)); };
    auto fetch_v = [&](auto whole, int t) { fetch(whole, vbase, a.vs_t, voff, vchunk, t, (unsigned)((2 + (t & 1)) * TILE)); };
    int vtr[DT];  // LDS offsets of the transposed fragment reads (see attn_fast_kernel.h)
    {
        const int s4 = (lane >> 2) & 3, a4 = lane & 3, g1 = (lane >> 4) & 1;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            vtr[dt] = (4 * half + s4) * RS + 16 * ((4 * dt + 2 * g1 + (a4 >> 1)) ^ var_v_swizzle<D>(s4)) + 8 * (a4 & 1);
    }
    const int krow = l32 * RS + 16 * (half ^ (l32 & (CPR - 1)));

    v16f acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[dt][i] = 0.0f;
    float m_i = -INFINITY, l_i = 0.0f;  // running maximum (base-2 units) and this half's part of the row sum

    // scores of tile t, 32 keys each: accumulator i of a lane is key 64 t + 32 kt + 8 (i / 4) + 4 half + i % 4
    auto half_scores = [&](int t, int kt, v16f& s) {
        const unsigned char* ktile = smem[0][t & 1] + 32 * kt * RS;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < KS; c++) s = PVT::mfma(*reinterpret_cast<const vec16*>(ktile + (krow ^ (32 * c))), qf[c], s);
    };
    auto scores = [&](int t, v16f (&s)[KT]) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) half_scores(t, kt, s[kt]);
    };
    auto hide = [&](int t, v16f (&s)[KT]) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            const int last = my_lim - KEYS * t - 32 * kt - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; i++) s[kt][i] = 8 * (i >> 2) + (i & 3) <= last ? s[kt][i] : -INFINITY;
        }
    };
    auto largest = [&](const v16f (&s)[KT]) {
        float x = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) x = fmaxf(x, s[kt][i]);
        return x * a.qk_scale;
    };
    // The reference point of a row moves up to its maximum where that is more than 2^kLag above it: P up to 2^kLag serve as well as P up
    // to 1, their rounding is relative, and most steps then multiply no accumulator (5 % of the documents' time).  A row's point depends on its own scores alone.
    auto raise = [&](float top) {
        if (__builtin_amdgcn_ballot_w64(top > m_i + kLag) != 0) {
            top = fmaxf(top, __shfl_xor(top, 32));
            const float m_new = top > m_i + kLag ? top : m_i;
            // (a row that has seen no key yet keeps m = -inf: every p below is then 0)
            const float alpha = m_i == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_i - m_new);
            l_i *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[dt][i] *= alpha;
            m_i = m_new;
        }
    };
    // P is rounded to 16 bits for the matrix instructions (half a step of itself off); its sum is taken before that
    auto half_weights = [&](const v16f& s, vec16& lo, vec16& hi) {
        const float m_use = m_i == -INFINITY ? 0.0f : m_i;
        float psum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.qk_scale, -m_use));  // hidden keys: exp2(-inf) = 0
            psum += p;
            if (i < 8) lo[i & 7] = (VT)p;
            else hi[i & 7] = (VT)p;
        }
        l_i += psum;
    };
    auto weights = [&](const v16f (&s)[KT], vec16 (&pf)[2 * KT]) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) half_weights(s[kt], pf[2 * kt], pf[2 * kt + 1]);
    };
    auto v_fragment = [&](int t, int c, int dt) {  // keys 16 c .. of the tile
        const unsigned char* p0 = smem[1][t & 1] + vtr[dt] + 16 * c * RS;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p0);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p0 + 8 * RS));
        return __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto add_slice = [&](int t, int c, const vec16& p) {
#pragma unroll
        for (int dt = 0; dt < DT; dt++) acc[dt] = PVT::mfma(__builtin_bit_cast(vec16, v_fragment(t, c, dt)), p, acc[dt]);
    };
    auto add = [&](int t, const vec16 (&pf)[2 * KT]) {
#pragma unroll
        for (int c = 0; c < 2 * KT; c++) add_slice(t, c, pf[c]);
    };
    // ---- K of tile t + 1 and V of tile t are in LDS, or on their way, when step t begins; the step fetches K of t + 2 and V of t + 1
    if (ntiles > 0) {
        fetch_k(IC<0>{}, 0);
        fetch_v(IC<0>{}, 0);
        if (ntiles > 1) fetch_k(IC<0>{}, 1);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __builtin_amdgcn_s_barrier();
    // (Q is here by now: inside the loop the compiler's waits for it would also wait for the tiles on their way)
#pragma unroll
    for (int t = 0; t < KS; t++) {
        v4i bits = __builtin_bit_cast(v4i, qf[t]);
        asm volatile("" : "+v"(bits));
        qf[t] = __builtin_bit_cast(vec16, bits);
    }
    auto next = [&](auto whole, int t) {
        // vmcnt(0): what this step needs has landed, for all waves past the barrier; what it overwrites has been read
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __builtin_amdgcn_s_barrier();
        if (decltype(whole)::value || t + 2 < ntiles) fetch_k(whole, t + 2);
        if (decltype(whole)::value || t + 1 < ntiles) fetch_v(whole, t + 1);
    };
    v16f sa[KT];
    if (my_tiles > 0) {
        scores(0, sa);
        if (clear_tiles < 1) hide(0, sa);
        raise(largest(sa));
    }
    int t = 0;
    if constexpr (KT == 2) {
        v16f sb[KT];
        // A step that hides no key, nor does the next: the scores of the next tile are made while this one's exponentials are.
        auto clear_step = [&](int t, v16f (&cur)[KT], v16f (&nxt)[KT]) {
            vec16 pf[2 * KT];
            // (in two parts, so that no more than three of the four 32-key score tiles are in registers at a time: without the barrier one
            // sequence of 2000 tokens takes 4 % longer)
            half_scores(t + 1, 0, nxt[0]);
            half_weights(cur[0], pf[0], pf[1]);
            __builtin_amdgcn_sched_barrier(0);
            half_weights(cur[1], pf[2], pf[3]);
            half_scores(t + 1, 1, nxt[1]);
            add_slice(t, 0, pf[0]);
            add_slice(t, 1, pf[1]);
            add_slice(t, 2, pf[2]);
            add_slice(t, 3, pf[3]);
            raise(largest(nxt));
        };
        for (; t + 3 < clear_tiles; t += 2) {
            next(IC<1>{}, t);
            clear_step(t, sa, sb);
            next(IC<1>{}, t + 1);
            clear_step(t + 1, sb, sa);
        }
    }
    if constexpr (KT == 1) {
        // (the matrix instructions one after the other, so that the maximum of the next scores is taken while V is added)
        auto short_step = [&](int t) {
            vec16 pf[2];
            half_weights(sa[0], pf[0], pf[1]);
            half_scores(t + 1, 0, sa[0]);
            add_slice(t, 0, pf[0]);
            add_slice(t, 1, pf[1]);
            raise(largest(sa));
        };
        for (; t + 3 < clear_tiles; t += 2) {
            next(IC<1>{}, t);
            short_step(t);
            next(IC<1>{}, t + 1);
            short_step(t + 1);
        }
    }
    for (; t < ntiles; t++) {
        next(IC<0>{}, t);
        if (t >= my_tiles) continue;
        vec16 pf[2 * KT];
        weights(sa, pf);
        add(t, pf);
        if (t + 1 < my_tiles) {
            scores(t + 1, sa);
            if (t + 1 >= clear_tiles) hide(t + 1, sa);
            raise(largest(sa));
        }
    }
    __syncthreads();  // (all waves are done with the tiles; nothing is on its way into LDS)

    // accumulator i of tile dt: channel 32 dt + 8 (i / 4) + 4 half + i % 4
    float* part_o = whole ? nullptr : a.part_o + ((int64_t)slot * kVarWaves + wave) * (32 * D);
    float* part_lse = whole ? nullptr : a.part_lse + (int64_t)slot * kVarRows + 32 * wave;
    // An infinity or NaN in V under a hidden key must not reach the rows that do not see it (0 times it is NaN): where an output is not
    // finite and a tile that hides keys holds one, the wave's rows are computed again, key by key.  (Looking at those tiles inside the
    // loop: 48 prompts of 1 to 700 tokens, H32/8 D128, 43.5 us instead of 42.1.)
    // So they are where a reference point is huge, or was: infinite P leave a NaN sum then, though neither Q nor K holds one.
    auto any_odd = [&](const VT* base, int64_t stride, int first, int end) {
        // (the lane anew in tiles of 32 keys: kept through the steps it is spilled)
        const int me = KEYS == 32 ? __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)) : lane;
        unsigned odd = 0;
#pragma unroll 1
        for (int n = first + me / CPR; n < end; n += 64 / CPR) {
            const v4i f = *reinterpret_cast<const v4i*>(base + (int64_t)n * stride + 8 * (me % CPR));
#pragma unroll
            for (int w = 0; w < 4; w++) odd |= nonfinite_halves<VT>((unsigned)f[w]);
        }
        return __builtin_amdgcn_ballot_w64(odd != 0) != 0;
    };
    const bool huge = __builtin_amdgcn_ballot_w64(__builtin_fabsf(m_i) >= kHuge && __builtin_fabsf(m_i) < INFINITY) != 0;
    if (clear_tiles < my_tiles || huge || __builtin_amdgcn_ballot_w64(l_i != l_i) != 0) {
        float zero[2] = {0.0f, 0.0f};
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int i = 0; i < 16; i++) zero[i & 1] = __builtin_fmaf(acc[dt][i], 0.0f, zero[i & 1]);
        if (__builtin_expect(huge || __builtin_amdgcn_ballot_w64(zero[0] + zero[1] != 0.0f) != 0, 0)) {
            unsigned odd_q = 0;
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
                for (int w = 0; w < 4; w++) odd_q |= nonfinite_halves<VT>((unsigned)__builtin_bit_cast(v4i, qf[t])[w]);
            odd_q |= __shfl_xor((int)odd_q, 32);
            const int end = min(KEYS * my_tiles, N);
            if (huge || any_odd(vbase, a.vs_t, KEYS * clear_tiles, end) ||
                (__builtin_amdgcn_ballot_w64(l_i != l_i && odd_q == 0) != 0 && !any_odd(kbase, a.ks_t, 0, end))) {
                for (int r = 32 * wave; r < 32 * wave + 32 && r <= last_row; r++) {
                    const int on = tokens_on(r), m = tok0 + on, n = a.causal ? min(m + shift, N - 1) + 1 : N;
                    careful_row<D, VT>(a, q0 + m, hk * a.groups + rem0 + r - on * a.groups, hk, k0, CUT ? min(n, KEYS * ntiles) : n, part_o, part_lse, r - 32 * wave);
                }
                continue;
            }
        }
    }
    const float l_tot = l_i + __shfl_xor(l_i, 32);
    // l = 0: a row that saw no key: zero row.  (NaN stays.)
    const float inv = l_tot != 0.0f ? 1.0f / l_tot : 0.0f;
    const float lse2 = __builtin_log2f(l_tot) + (m_i == -INFINITY ? 0.0f : m_i);
    if (CUT && !whole) {
        if (row_ok) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *reinterpret_cast<v4f*>(part_o + ((4 * dt + g) * 64 + lane) * 4) =
                        v4f{acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv};
            if (half == 0) part_lse[l32] = lse2;
        }
    } else if (D == 64) {
        if (row_ok) {
            VT* op = static_cast<VT*>(a.out) + (int64_t)(q0 + my_m) * a.os_t + (int64_t)my_h * a.os_h + 4 * half;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    store_rounded(op + 32 * dt + 8 * g, v4f{acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv});
            if (a.lse && half == 0) a.lse[(int64_t)my_h * a.total_q + q0 + my_m] = lse2 * 0.693147180559945309f;
        }
    } else {
        // rows of 256 bytes through LDS, so that sixteen lanes store a whole one (48 prompts of 1 to 700 tokens, H32/8: 11 % less time;
        // at head_dim 64 the stores of 8 bytes from the registers are as fast, 19.6 and 20.6 us with H16)
        unsigned char* mine = all_smem + wave * 32 * O_RS;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                store_rounded(reinterpret_cast<VT*>(mine + l32 * O_RS) + 32 * dt + 8 * g + 4 * half,
                              v4f{acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv});
        if (a.lse && half == 0 && row_ok) a.lse[(int64_t)my_h * a.total_q + q0 + my_m] = lse2 * 0.693147180559945309f;
#pragma unroll
        for (int e = 0; e < 32 * CPR / 64; e++) {
            const int r = (64 / CPR) * e + lane / CPR, on = tokens_on(32 * wave + r);
            const v4i x = *reinterpret_cast<const v4i*>(mine + r * O_RS + 16 * (lane % CPR));
            if (32 * wave + r <= last_row)
                *reinterpret_cast<v4i*>(static_cast<VT*>(a.out) + (int64_t)(q0 + tok0 + on) * a.os_t +
                                        (int64_t)(hk * a.groups + rem0 + 32 * wave + r - on * a.groups) * a.os_h + 8 * (lane % CPR)) = x;
        }
    }
  }
}

// The blocks of a cut launch that lie in more than one share: lse = log2 sum_s 2^lse_s, out = sum_s 2^(lse_s - lse) o_s.  A workgroup per
// cut between two shares and wave of a block; the first cut inside a block takes care of it.  A wave adds 32 channels of 32 rows
// in the order of the registers that left them.
template <int D, typename VT>
__global__ __launch_bounds__(2 * D) void varlen_combine_kernel(VarlenArgs a) {
    const EqualShares line(all_steps(a), a.shares);
    const int cut = blockIdx.x + 1, pos = line.begin(cut), wave = blockIdx.y;
    if (line.begin(cut + 1) <= pos) return;  // (the shares from here on are empty)
    const BlockAt at(a, pos);
    if (!at.found) return;
    const int first = line.owner(at.begin + kStart);
    if (pos <= at.begin + kStart || first + 1 != cut) return;
    const int last = line.owner(at.begin + kStart + at.tiles - 1);
    const int block_rows = a.groups << a.tokens_shift;
    const int row0 = at.block * block_rows + 32 * wave, rows = min((at.block + 1) * block_rows, at.M * a.groups);
    if (row0 >= rows) return;
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5, dt = threadIdx.x >> 6;
    auto slot = [&](int w) { return (int64_t)(2 * w + (w == first && at.begin > line.begin(w))); };
    v4f acc[4];
#pragma unroll
    for (int g = 0; g < 4; g++) acc[g] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, den = 0.0f;
    constexpr int kBatch = 4;  // parts on their way together
    for (int w0 = first; w0 <= last; w0 += kBatch) {
        float x[kBatch];
        v4f o[kBatch][4];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {  // (past the end: the last part once more)
            const int64_t s = slot(min(w0 + u, last));
            x[u] = a.part_lse[s * kVarRows + 32 * wave + l32];
#pragma unroll
            for (int g = 0; g < 4; g++)
                o[u][g] = *reinterpret_cast<const v4f*>(a.part_o + ((s * kVarWaves + wave) * (D / 8) + 4 * dt + g) * 256 + lane * 4);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < kBatch; u++) top = x[u] > top || x[u] != x[u] ? x[u] : top;  // (NaN stays)
        const float use = top == -INFINITY ? 0.0f : top;  // (no key seen so far: weights of 0)
        const float alpha = __builtin_amdgcn_exp2f(m - use);
        den *= alpha;
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[g][i] *= alpha;
        m = top;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            if (w0 + u > last) break;
            const float w = __builtin_amdgcn_exp2f(x[u] - use);
            den += w;
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[g][i] = __builtin_fmaf(w, o[u][g][i], acc[g][i]);
        }
    }
    const int row = row0 + l32;
    if (row >= rows) return;
    const float inv = den != 0.0f ? 1.0f / den : 0.0f;
    const int my_m = row / a.groups, my_h = at.hk * a.groups + row % a.groups;
    VT* op = static_cast<VT*>(a.out) + (int64_t)(at.q0 + my_m) * a.os_t + (int64_t)my_h * a.os_h + 32 * dt + 4 * half;
#pragma unroll
    for (int g = 0; g < 4; g++) store_rounded(op + 8 * g, v4f{acc[g][0] * inv, acc[g][1] * inv, acc[g][2] * inv, acc[g][3] * inv});
    if (a.lse && dt == 0 && half == 0)
        a.lse[(int64_t)my_h * a.total_q + at.q0 + my_m] = (__builtin_log2f(den) + (m == -INFINITY ? 0.0f : m)) * 0.693147180559945309f;
}

constexpr int kVarShares = 512;  // two workgroups on each compute unit

// Does a cut launch pay?  By its time against that of whole blocks, in steps of the kernel, for sequences of the mean lengths (the
// real ones are the device's): whole blocks take the longest one, or an even share where there are more than fit the chip; a cut
// launch takes an even share with the blocks' starts, one more start and about 15 steps for the partial results and the second
// launch.  Measured, whole and cut: H32/8 D128, 512 queries against 16512 keys 286 and 156 us, 3 x 100 to 400 against up to 8000
// 146 and 79, 8 x 64 to 256 against up to 4000 86 and 77; 2000 causal 49 and 63, 2048 against 32000 951 and 1021; H16 D64, 6 x 129
// to 512 against up to 7000 85 and 58, 2 x 3000 causal 51 and 68.
bool cut_pays(const sage_varlen_params& p) {
    const double blocks = (double)p.total_q * (p.heads_q / p.heads_kv) / kVarRows + 0.5 * p.seqs, load = blocks * p.heads_kv / kVarShares;
    const double longest = (double)p.total_k / p.seqs / kVarKeys;
    const double mean = p.causal ? longest - 0.5 * fmin((double)p.total_q / p.seqs / kVarKeys, longest) : longest;
    const double whole = kStart + (load > 1.0 ? load * mean : longest), cut = load * (kStart + mean) + kStart + 15.0;
    return 1.1 * cut < whole;
}

struct VarlenPlan { int64_t blocks; int shares, tokens_shift; };

// Whole blocks, or (with_workspace) a cut launch.  The lengths are the device's: what the host knows are the totals.
VarlenPlan plan_varlen(const sage_varlen_params& p, bool with_workspace) {
    const int64_t groups = p.heads_q / p.heads_kv;
    VarlenPlan plan{p.total_q * groups / kVarRows + p.seqs, 0, 0};  // at most: a ragged last block for every sequence
    if (!with_workspace || groups > kVarRows) return plan;
    while (2 * groups << plan.tokens_shift <= kVarRows) plan.tokens_shift++;
    const int64_t blocks = (p.total_q >> plan.tokens_shift) + p.seqs, tiles = p.total_k / kVarKeys + 1;
    if (blocks * p.heads_kv > 0x7fffffffLL / (tiles + kStart)) return plan;
    if (cut_pays(p)) plan.shares = kVarShares;
    return plan;
}

// Tiles of 32 keys where blocks are many, of 64 where they are few: a workgroup by itself is slower with the former, but three of them
// share a compute unit instead of two.  Measured, 64 and 32 (H32/8 D128, causal): 1 x 500 tokens 15.4 and 17.0 us, 1 x 3000 80 and 88,
// 24 x 1 to 700 (860 workgroups) 24.4 and 26.0, 1 x 3500 (880) 107 and 109; 1 x 4000 (1010) 138 and 131, 32 x 1 to 700 (1150) 31.7 and 27.4,
// 16 x 100 to 2000 139 and 125, 200 x 100 to 200 166 and 142, the documents 626 and 589; H16 D64: 1 x 700 12.3 and 13.0,
// 2 x 3000 (780) 52.7 and 53.6, 4 x 4096 176 and 170, 48 x 1 to 700 20.4 and 18.6.
constexpr int64_t kManyBlocks = 1000;

template <int D, typename VT>
int launch_d(const VarlenArgs& a, int64_t blocks, hipStream_t stream) {
    if (a.shares) {
        hipLaunchKernelGGL((flash_varlen_kernel<D, VT, true, 64>), dim3((unsigned)a.shares), dim3(kVarThreads), 0, stream, a);
        if (int rc = check_launch("flash_varlen_kernel")) return rc;
        hipLaunchKernelGGL((varlen_combine_kernel<D, VT>), dim3((unsigned)a.shares - 1, kVarWaves), dim3(2 * D), 0, stream, a);
        return check_launch("varlen_combine_kernel");
    }
    if (blocks * a.Hkv > kMaxThreads / kVarThreads) return fail(SAGE_E_UNSUPPORTED, "sage_flash_varlen_fwd: too many workgroups for one launch");
    if (blocks * a.Hkv > kManyBlocks)
        hipLaunchKernelGGL((flash_varlen_kernel<D, VT, false, 32>), dim3((unsigned)(blocks * a.Hkv)), dim3(kVarThreads), 0, stream, a);
    else
        hipLaunchKernelGGL((flash_varlen_kernel<D, VT, false, 64>), dim3((unsigned)(blocks * a.Hkv)), dim3(kVarThreads), 0, stream, a);
    return check_launch("flash_varlen_kernel");
}

}  // namespace

int64_t varlen_workspace_bytes(const sage_varlen_params& p) {
    return 2LL * plan_varlen(p, true).shares * kVarRows * (p.head_dim + 1) * (int64_t)sizeof(float);
}

int launch_flash_varlen(const sage_varlen_params& p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    const VarlenPlan plan = plan_varlen(p, workspace != nullptr && workspace_bytes >= varlen_workspace_bytes(p));
    VarlenArgs a{};
    a.q = p.q.ptr; a.k = p.k.ptr; a.v = p.v.ptr; a.out = p.out.ptr; a.lse = p.log_normalizer;
    a.cu_q = p.cu_seqlens_q; a.cu_k = p.cu_seqlens_k;
    a.qs_t = p.q.stride_n; a.qs_h = p.q.stride_h; a.ks_t = p.k.stride_n; a.ks_h = p.k.stride_h;
    a.vs_t = p.v.stride_n; a.vs_h = p.v.stride_h; a.os_t = p.out.stride_n; a.os_h = p.out.stride_h;
    a.seqs = (int)p.seqs; a.total_q = (int)p.total_q; a.total_k = (int)p.total_k;
    a.Hkv = (int)p.heads_kv; a.groups = (int)(p.heads_q / p.heads_kv); a.causal = p.causal ? 1 : 0;
    a.qk_scale = p.sm_scale * 1.44269504089f;
    a.inv_groups = (1u << 16) / a.groups + 1;
    a.shares = plan.shares; a.tokens_shift = plan.tokens_shift;
    a.part_o = (float*)workspace;
    a.part_lse = a.part_o + 2LL * plan.shares * kVarRows * p.head_dim;
    if (p.head_dim == 128) return p.dtype == SAGE_BF16 ? launch_d<128, __bf16>(a, plan.blocks, stream) : launch_d<128, _Float16>(a, plan.blocks, stream);
    return p.dtype == SAGE_BF16 ? launch_d<64, __bf16>(a, plan.blocks, stream) : launch_d<64, _Float16>(a, plan.blocks, stream);
}

}  // namespace sage
