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
// without leaving its registers.  Bound by the matrix cores, with the vector instructions of the softmax in their shadow:
// * K and V tiles of 64 keys go straight into LDS for the four waves, two of each resident, one barrier per step.  Two workgroups
//   share a compute unit and are not tied to each other, so one's exponentials meet the other's matrix instructions.
// * A step makes the scores of the next tile while it takes the exponentials of its own.
// * Nothing of the step loop is spilled: a reload waits for every tile on its way into LDS, since loads return in order (three
//   reloads per step: 4 documents of 512 to 8192 tokens, H32/8 D128, 593 -> 811 us).  What is rare is therefore kept out of its
//   registers (careful_row).
// * Workgroups are handed out longest first over all sequences (find_block).
// Measured (bf16, D128, causal): those documents 593 us = 1100 TFLOP/s, one sequence of 16384 tokens with H16/2 952 us = 1155 TFLOP/s (a
// library product of 8192^3 reaches 1356 here); 48 prompts of 1 to 700 tokens 48 us.  Tiles of 32 keys, each multiplied, weighed and
// added in turn: 811, 1272 and 54 us.  Eight waves per workgroup: 2 % more for long sequences, 28 % less for short ones.
#include "serve_common.h"

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
    float qk_scale;  // sm_scale * log2(e)
};

constexpr int kVarWaves = 4;
constexpr int kVarThreads = 64 * kVarWaves;
constexpr int kVarRows = 32 * kVarWaves;
constexpr int kVarKeys = 64;  // keys per tile
constexpr float kLag = 8.0f;

// Sequence s of a packed axis.  (Offsets out of order or past the end give no rows that do not exist.)
__device__ __forceinline__ void sequence(const int32_t* cu, int s, int total, int& begin, int& len) {
    begin = min(max(cu[s], 0), total);
    len = min(max(cu[s + 1], begin), total) - begin;
}

// The block of 128 rows that workgroup `at` (of a K/V head) takes, and its sequence; false: there is none.
// Up to 64 sequences, a lane each: the blocks that see the most keys first, so that the last workgroups to start are the short
// ones.  With more of them: sequence after sequence, each from its last block on.
__device__ __forceinline__ bool find_block(const VarlenArgs& a, int at, int& q0, int& M, int& k0, int& N, int& block) {
    const int lane = threadIdx.x & 63;
    auto blocks = [&](int m) { return (int)(((int64_t)m * a.groups + kVarRows - 1) / kVarRows); };
    if (a.seqs > 64) {
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
    const int nb = blocks(lm), rows = lm * a.groups;
    // blocks below `first_of(l)` visit fewer than l key tiles
    auto first_of = [&](int l) {
        if (!a.causal) return kVarKeys * (l - 1) < ln ? 0 : nb;
        const int64_t x = ((int64_t)kVarKeys * (l - 1) - (ln - lm)) * a.groups;  // the first row that sees a key of tile l - 1
        return x >= rows ? nb : x <= 0 ? 0 : (int)(x / kVarRows);
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

// One row by one wave, from its keys alone: query token qt, head h, the first n keys from k0 on.  A lane is a key for the scores,
// and D / 64 channels for the output.  For rows whose tiles hold infinities or NaN in V: a thousand times slower than a tile's share
// of the kernel below, and hardly ever called.
template <int D, typename VT>
__device__ void careful_row(const VarlenArgs& a, int qt, int h, int hk, int k0, int n) {
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
#pragma unroll 1
        for (int j = 0; j < min(64, n - n0); j++) {
            const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j));
#pragma unroll
            for (int i = 0; i < CH; i++) o[i] = __builtin_fmaf(pj, (float)v[(int64_t)(n0 + j) * a.vs_t + lane + 64 * i], o[i]);
        }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < CH; i++) static_cast<VT*>(a.out)[(int64_t)qt * a.os_t + (int64_t)h * a.os_h + lane + 64 * i] = (VT)(o[i] * inv);
    if (a.lse && lane == 0) a.lse[(int64_t)h * a.total_q + qt] = (__builtin_log2f(l) + (m == -INFINITY ? 0.0f : m)) * 0.693147180559945309f;
}

template <int D, typename VT>
__global__ __launch_bounds__(kVarThreads, 2) void flash_varlen_kernel(VarlenArgs a) {
    using PVT = PV<VT>;
    using vec16 = typename PVT::vec;
    constexpr int KS = D / 16;      // matrix instructions of one 32 x 32 score tile
    constexpr int DT = D / 32;      // 32-channel tiles of the output
    constexpr int RS = 2 * D;       // bytes per K / V row
    constexpr int CPR = RS / 16;    // 16-byte chunks per row
    constexpr int TILE = kVarKeys * RS;
    constexpr int LOADS = TILE / 1024 / kVarWaves;  // 1 KB loads per wave of a K (of a V) tile
    constexpr int KT = kVarKeys / 32;
    static_assert(KT == 2, "halves of a tile");
    __shared__ __attribute__((aligned(16))) unsigned char smem[2][2][TILE];  // [K, V][buffer]

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % a.Hkv;
    int q0, M, k0, N, block;
    if (!find_block(a, blockIdx.x / a.Hkv, q0, M, k0, N, block)) return;
    const int rows = M * a.groups, row0 = block * kVarRows;
    const int shift = N - M;
    const int row = row0 + 32 * wave + l32;
    const bool row_ok = row < rows;
    const int my_m = min(row, rows - 1) / a.groups, my_h = hk * a.groups + min(row, rows - 1) % a.groups;

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
        n_end = max(min(N, (min(row0 + kVarRows, rows) - 1) / a.groups + 1 + shift), 0);
        wave_end = max(min(N, (min(row0 + 32 * wave + 32, rows) - 1) / a.groups + 1 + shift), 0);
        all_see = max(min(N, min(row0 + 32 * wave, rows - 1) / a.groups + 1 + shift), 0);
    }
    const int my_lim = a.causal ? min(my_m + shift, N - 1) : N - 1;  // last key this lane's row sees
    const int ntiles = (n_end + kVarKeys - 1) / kVarKeys;
    const int my_tiles = row0 + 32 * wave < rows ? (wave_end + kVarKeys - 1) / kVarKeys : 0;  // that this wave multiplies with
    const int clear_tiles = all_see / kVarKeys;                                               // the first ones hide no key

    // Tile t of K and V -> one of the two buffers, straight into LDS (written in assembly, as in attn_fast_kernel.h: the compiler
    // would wait for every outstanding load before each LDS read; m0 holds the LDS address and nothing else here uses it).
    // Chunk c of row r lies at chunk c ^ (r mod chunks) for K and at c ^ var_v_swizzle(r) for V: the load fetches the chunk that
    // belongs where a lane writes, the fragment reads spread over all banks.  Load e of a wave: kRound rows further on, a whole
    // number of swizzle periods.  Rows past the end re-read the last one.
    constexpr int kRound = kVarWaves * 64 / CPR;
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)&smem[0][0][0];
    const int frow = (64 / CPR) * wave + lane / CPR;  // row of load 0
    const unsigned kchunk = 16 * ((lane % CPR) ^ (frow & (CPR - 1))), vchunk = 16 * ((lane % CPR) ^ var_v_swizzle<D>(frow));
    const unsigned koff = (unsigned)frow * (unsigned)(a.ks_t * 2) + kchunk, voff = (unsigned)frow * (unsigned)(a.vs_t * 2) + vchunk;
    auto fetch = [&](auto whole, const VT* base, int64_t stride, unsigned off, unsigned chunk, int t, unsigned dst) {
        const int n0 = kVarKeys * t;
        const VT* tile = base + (int64_t)n0 * stride;
        const unsigned to = lds0 + dst + 1024 * wave;
        if (decltype(whole)::value || n0 + kVarKeys <= N) {
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
            const int last = my_lim - kVarKeys * t - 32 * kt - 4 * half;
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
            top = fmaxf(top, __shfl_xor(top, 32));  // (two lanes share a row)
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
    // An infinity or NaN in V under a hidden key must not reach the rows that do not see it (0 times it is NaN): where a tile that
    // hides keys holds one, the wave's rows are computed again at the end, key by key.
    bool again = false;
    auto look = [&](int t) {
        unsigned odd = 0;
#pragma unroll
        for (int c = 0; c < 2 * KT; c++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const v4i f = v_fragment(t, c, dt);
#pragma unroll
                for (int i = 0; i < 4; i++) odd |= nonfinite_halves<VT>((unsigned)f[i]);
                if (dt % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // (two fragments at a time: registers)
            }
        again |= __builtin_amdgcn_ballot_w64(odd != 0) != 0;
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
    v16f sa[KT], sb[KT];
    if (my_tiles > 0) {
        scores(0, sa);
        if (clear_tiles < 1) hide(0, sa);
        raise(largest(sa));
    }
    // A step that hides no key, nor does the next: the scores of the next tile are made while this one's exponentials are.
    auto clear_step = [&](int t, v16f (&cur)[KT], v16f (&nxt)[KT]) {
        vec16 pf[2 * KT];
        // (in three parts, so that no more than three of the four 32-key score tiles are in registers at a time)
        half_scores(t + 1, 0, nxt[0]);
        half_weights(cur[0], pf[0], pf[1]);
        __builtin_amdgcn_sched_barrier(0);
        half_scores(t + 1, 1, nxt[1]);
        half_weights(cur[1], pf[2], pf[3]);
        add_slice(t, 0, pf[0]);
        add_slice(t, 1, pf[1]);
        __builtin_amdgcn_sched_barrier(0);
        add_slice(t, 2, pf[2]);
        add_slice(t, 3, pf[3]);
        raise(largest(nxt));
    };
    int t = 0;
    for (; t + 3 < clear_tiles; t += 2) {
        next(IC<1>{}, t);
        clear_step(t, sa, sb);
        next(IC<1>{}, t + 1);
        clear_step(t + 1, sb, sa);
    }
    for (; t < ntiles; t++) {
        next(IC<0>{}, t);
        if (t >= my_tiles) continue;
        vec16 pf[2 * KT];
        weights(sa, pf);
        if (t >= clear_tiles) look(t);
        add(t, pf);
        if (t + 1 < my_tiles) {
            scores(t + 1, sa);
            if (t + 1 >= clear_tiles) hide(t + 1, sa);
            raise(largest(sa));
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // nothing of this workgroup is on its way into LDS when it ends

    if (__builtin_expect(again, 0)) {
        for (int r = row0 + 32 * wave; r < min(row0 + 32 * wave + 32, rows); r++) {
            const int m = r / a.groups;
            careful_row<D, VT>(a, q0 + m, hk * a.groups + r % a.groups, hk, k0, a.causal ? min(m + shift, N - 1) + 1 : N);
        }
        return;
    }
    const float l_tot = l_i + __shfl_xor(l_i, 32);
    // l = 0: a row that saw no key: zero row.  (NaN stays.)
    const float inv = l_tot != 0.0f ? 1.0f / l_tot : 0.0f;
    if (!row_ok) return;
    // accumulator i of tile dt: channel 32 dt + 8 (i / 4) + 4 half + i % 4
    VT* op = static_cast<VT*>(a.out) + (int64_t)(q0 + my_m) * a.os_t + (int64_t)my_h * a.os_h + 4 * half;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            store_rounded(op + 32 * dt + 8 * g, v4f{acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv});
    if (a.lse && half == 0) {
        a.lse[(int64_t)my_h * a.total_q + q0 + my_m] = (__builtin_log2f(l_tot) + (m_i == -INFINITY ? 0.0f : m_i)) * 0.693147180559945309f;
    }
}

template <int D, typename VT>
int launch_d(const VarlenArgs& a, hipStream_t stream) {
    const int64_t blocks = ((int64_t)a.total_q * a.groups) / kVarRows + a.seqs;  // at most: a ragged last block for every sequence
    if (blocks * a.Hkv > 0x7fffffffLL) return fail(SAGE_E_UNSUPPORTED, "sage_flash_varlen_fwd: too many workgroups for one launch");
    hipLaunchKernelGGL((flash_varlen_kernel<D, VT>), dim3((unsigned)(blocks * a.Hkv)), dim3(kVarThreads), 0, stream, a);
    return check_launch("flash_varlen_kernel");
}

}  // namespace

int launch_flash_varlen(const sage_varlen_params& p, hipStream_t stream) {
    VarlenArgs a{};
    a.q = p.q.ptr; a.k = p.k.ptr; a.v = p.v.ptr; a.out = p.out.ptr; a.lse = p.log_normalizer;
    a.cu_q = p.cu_seqlens_q; a.cu_k = p.cu_seqlens_k;
    a.qs_t = p.q.stride_n; a.qs_h = p.q.stride_h; a.ks_t = p.k.stride_n; a.ks_h = p.k.stride_h;
    a.vs_t = p.v.stride_n; a.vs_h = p.v.stride_h; a.os_t = p.out.stride_n; a.os_h = p.out.stride_h;
    a.seqs = (int)p.seqs; a.total_q = (int)p.total_q; a.total_k = (int)p.total_k;
    a.Hkv = (int)p.heads_kv; a.groups = (int)(p.heads_q / p.heads_kv); a.causal = p.causal ? 1 : 0;
    a.qk_scale = p.sm_scale * 1.44269504089f;
    if (p.head_dim == 128) return p.dtype == SAGE_BF16 ? launch_d<128, __bf16>(a, stream) : launch_d<128, _Float16>(a, stream);
    return p.dtype == SAGE_BF16 ? launch_d<64, __bf16>(a, stream) : launch_d<64, _Float16>(a, stream);
}

}  // namespace sage
