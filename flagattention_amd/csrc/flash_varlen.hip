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
// without leaving its registers.  Tiles of 32 keys go straight into LDS for the four waves, one tile ahead, one barrier each.
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
constexpr int kVarKeys = 32;  // keys per tile

// Sequence s of a packed axis.  (Offsets out of order or past the end give no rows that do not exist.)
__device__ __forceinline__ void sequence(const int32_t* cu, int s, int total, int& begin, int& len) {
    begin = min(max(cu[s], 0), total);
    len = min(max(cu[s + 1], begin), total) - begin;
}

template <int D> __device__ __forceinline__ int var_v_swizzle(int row) { return D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

template <int D, typename VT>
__global__ __launch_bounds__(kVarThreads, D == 128 ? 2 : 3) void flash_varlen_kernel(VarlenArgs a) {
    using PVT = PV<VT>;
    using vec16 = typename PVT::vec;
    constexpr int KS = D / 16;      // matrix instructions of one 32 x 32 score tile
    constexpr int DT = D / 32;      // 32-channel tiles of the output
    constexpr int RS = 2 * D;       // bytes per K / V row
    constexpr int CPR = RS / 16;    // 16-byte chunks per row
    constexpr int TILE = kVarKeys * RS;
    constexpr int LOADS = TILE / 1024 / kVarWaves;  // 1 KB loads per wave of a K (of a V) tile
    __shared__ __attribute__((aligned(16))) unsigned char smem[2][2][TILE];  // [buffer][K, V]

    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % a.Hkv, block = blockIdx.x / a.Hkv;
    auto blocks = [&](int s) {
        int begin, len;
        sequence(a.cu_q, s, a.total_q, begin, len);
        return (int)(((int64_t)len * a.groups + kVarRows - 1) / kVarRows);
    };
    int seq, first_block;
    if (!find_run(a.seqs, block, blocks, seq, first_block)) return;
    int q0, M, k0, N;
    sequence(a.cu_q, seq, a.total_q, q0, M);
    sequence(a.cu_k, seq, a.total_k, k0, N);
    const int rows = M * a.groups;
    const int row0 = (blocks(seq) - 1 - (block - first_block)) * kVarRows;  // (the last queries, which see the most keys, first)
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
    // (waited for here: inside the loop the compiler's waits for them would also wait for the tile on its way)
#pragma unroll
    for (int t = 0; t < KS; t++) {
        v4i bits = __builtin_bit_cast(v4i, qf[t]);
        asm volatile("" : "+v"(bits));
        qf[t] = __builtin_bit_cast(vec16, bits);
    }
    const VT* kbase = static_cast<const VT*>(a.k) + (int64_t)k0 * a.ks_t + (int64_t)hk * a.ks_h;
    const VT* vbase = static_cast<const VT*>(a.v) + (int64_t)k0 * a.vs_t + (int64_t)hk * a.vs_h;

    // keys that any row of the workgroup / of this wave can see
    int n_end = N, wave_end = N;
    if (a.causal) {
        n_end = max(min(N, (min(row0 + kVarRows, rows) - 1) / a.groups + 1 + shift), 0);
        wave_end = (min(row0 + 32 * wave + 32, rows) - 1) / a.groups + 1 + shift;
    }
    const int my_lim = a.causal ? min(my_m + shift, N - 1) : N - 1;  // last key this lane's row sees
    const int first_lim = a.causal ? min(min(row0 + 32 * wave, rows - 1) / a.groups + shift, N - 1) : N - 1;  // ... the wave's first row
    const int ntiles = (n_end + kVarKeys - 1) / kVarKeys;

    // Tile t of K and V -> one of the two buffers, straight into LDS (written in assembly, as in attn_fast_kernel.h: the compiler
    // would wait for every outstanding load before each LDS read; m0 holds the LDS address and nothing else here uses it).
    // Chunk c of row r lies at chunk c ^ (r mod chunks) for K and at c ^ var_v_swizzle(r) for V: the load fetches the chunk that
    // belongs where a lane writes, the fragment reads spread over all banks.  Rows past the end re-read the last one.
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)&smem[0][0][0];
    unsigned koff[LOADS], voff[LOADS];
    auto set_offsets = [&](int last) {  // last: the tile's last row
#pragma unroll
        for (int e = 0; e < LOADS; e++) {
            const int r = (64 / CPR) * (LOADS * wave + e) + lane / CPR;
            koff[e] = (unsigned)min(r, last) * (unsigned)(a.ks_t * 2) + 16 * ((lane % CPR) ^ (r & (CPR - 1)));
            voff[e] = (unsigned)min(r, last) * (unsigned)(a.vs_t * 2) + 16 * ((lane % CPR) ^ var_v_swizzle<D>(r));
        }
    };
    set_offsets(kVarKeys - 1);
    auto fetch = [&](int t, int buf) {
        const int n0 = kVarKeys * t;
        if (n0 + kVarKeys > N) set_offsets(N - 1 - n0);  // (the last tile)
        const VT* kt = kbase + (int64_t)n0 * a.ks_t;
        const VT* vt = vbase + (int64_t)n0 * a.vs_t;
        const unsigned dst = lds0 + (unsigned)(buf * 2 * TILE + 1024 * LOADS * wave);
#pragma unroll
        for (int e = 0; e < LOADS; e++) {
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(koff[e]), "s"(kt), "s"(dst + 1024 * e) : "memory");
            asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff[e]), "s"(vt), "s"(dst + TILE + 1024 * e) : "memory");
        }
    };
    int vtr[DT];  // LDS offsets of the transposed fragment reads (see attn_fast_kernel.h)
    {
        const int s4 = (lane >> 2) & 3, a4 = lane & 3, g1 = (lane >> 4) & 1;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
            vtr[dt] = (4 * half + s4) * RS + 16 * ((4 * dt + 2 * g1 + (a4 >> 1)) ^ var_v_swizzle<D>(s4)) + 8 * (a4 & 1);
    }

    v16f acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[dt][i] = 0.0f;
    float m_i = -INFINITY, l_i = 0.0f;  // running maximum (base-2 units) and this half's part of the row sum

    if (ntiles > 0) fetch(0, 0);
    for (int t = 0; t < ntiles; t++) {
        // vmcnt(0): this tile has landed, for all waves past the barrier; the one before has been read
        __builtin_amdgcn_s_waitcnt(0x0F70);
        __builtin_amdgcn_s_barrier();
        if (t + 1 < ntiles) fetch(t + 1, (t + 1) & 1);
        const int n0 = kVarKeys * t;
        if (n0 >= wave_end) continue;  // (no row of this wave sees a key of the tile)
        const unsigned char* ktile = smem[t & 1][0];
        const unsigned char* vtile = smem[t & 1][1];

        v16f s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
        int krow = l32 * RS + 16 * (half ^ (l32 & (CPR - 1)));
        asm volatile("" : "+v"(krow));  // (the addresses of the fragments, krow ^ 32 c, are not kept from tile to tile)
#pragma unroll
        for (int c = 0; c < KS; c++) s = PVT::mfma(*reinterpret_cast<const vec16*>(ktile + (krow ^ (32 * c))), qf[c], s);

        // accumulator i of this lane: key n0 + 8 (i / 4) + 4 half + i % 4
        const bool hides = n0 + kVarKeys - 1 > first_lim;
        if (hides) {
            const int last = my_lim - n0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = 8 * (i >> 2) + (i & 3) <= last ? s[i] : -INFINITY;
        }
        float tile_max = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) tile_max = fmaxf(tile_max, s[i]);
        tile_max *= a.qk_scale;
        // (a tile that raises no row of the wave needs no exchange between the two lanes of a row)
        if (__builtin_amdgcn_ballot_w64(tile_max > m_i) != 0) {
            const float m_new = fmaxf(m_i, fmaxf(tile_max, __shfl_xor(tile_max, 32)));
            // (a row that has seen no key yet keeps m = -inf: every p below is then 0)
            const float alpha = m_i == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_i - m_new);
            l_i *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[dt][i] *= alpha;
            m_i = m_new;
        }
        const float m_use = m_i == -INFINITY ? 0.0f : m_i;
        // P is rounded to 16 bits for the matrix instructions (at most 1, so half a step of 1 off); its sum is taken before that
        vec16 pf[2];
        float p[16], psum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.qk_scale, -m_use));  // hidden keys: exp2(-inf) = 0
            psum += p[i];
            pf[i >> 3][i & 7] = (VT)p[i];
        }
        l_i += psum;
        auto v_fragment = [&](int c, int dt) {
            const unsigned char* p0 = vtile + vtr[dt] + 16 * c * RS;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)p0);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p0 + 8 * RS));
            return __builtin_bit_cast(v4i, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // An infinity or NaN in V under a hidden key must not reach the rows that do not see it (0 times it is NaN): where a tile
        // that hides keys holds one, the matrix instructions get zeros in its place, and it is added to the rows that see its key.
        unsigned odd = 0;
        if (hides) {
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const v4i f = v_fragment(c, dt);
#pragma unroll
                    for (int i = 0; i < 4; i++) odd |= nonfinite_halves<VT>((unsigned)f[i]);
                }
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) == 0, 1)) {
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++) acc[dt] = PVT::mfma(__builtin_bit_cast(vec16, v_fragment(c, dt)), pf[c], acc[dt]);
        } else {
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
                    acc[dt] = PVT::mfma(__builtin_bit_cast(vec16, finite_only<VT>(v_fragment(c, dt))), pf[c], acc[dt]);
            add_nonfinite<D, VT>(vtile, [](int row) { return var_v_swizzle<D>(row); }, p, my_lim - n0 + 1, acc);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // nothing of this workgroup is on its way into LDS when it ends

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
