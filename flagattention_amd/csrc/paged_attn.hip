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
#include "paged_common.h"

namespace sage {
namespace {

constexpr int kPagedShares = 512;  // two workgroups on each compute unit

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

}  // namespace

int64_t paged_workspace_bytes(const sage_paged_params& p) { return plan_bytes(plan_paged(p, kPagedShares, 0), p.head_dim); }

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
    return launch_paged_combine<D, VT>(a, plan, stream);
}

int launch_paged_attn(const sage_paged_params& p, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    PagedPlan plan = plan_paged(p, kPagedShares, 0);
    if (!workspace || workspace_bytes < plan_bytes(plan, p.head_dim)) plan.shares = 0;  // (nothing is cut then)
    const PagedArgs a = paged_args(p, plan, workspace, 2);
    if (p.head_dim == 128) return p.dtype == SAGE_BF16 ? launch_paged<128, __bf16>(a, plan, stream) : launch_paged<128, _Float16>(a, plan, stream);
    return p.dtype == SAGE_BF16 ? launch_paged<64, __bf16>(a, plan, stream) : launch_paged<64, _Float16>(a, plan, stream);
}

}  // namespace sage
