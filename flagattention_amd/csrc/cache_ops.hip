// The movements of a paged key-value cache for gfx950: rows of new tokens into their slots, and whole pages to other pages.  Bound by
// bytes: 16 of them per lane and load, K and V in the same launch.  Slots and pages that do not exist move nothing.
// Measured (read and written bytes; a copy of 4 GiB reaches 4.78 TB/s): 16384 tokens of 8 heads, D128, bf16 25 to 27 us = 4.9 to 5.3
// TB/s, 700 pages of 8 layers 142 us = 5.2 TB/s; a step of 28 tokens 2.8 us of GPU time, 12 pages 2.9: a launch.
#include "common.h"

namespace sage {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t index_at(const void* list, int wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(list)[i] : (int64_t) static_cast<const int32_t*>(list)[i];
}

struct AppendArgs {
    const unsigned char* src[2];  // k, v
    unsigned char* dst[2];        // caches
    int64_t ss_t[2], ss_h[2], ds_p[2], ds_h[2], ds_n[2];  // bytes
    const void* slots;
    int64_t pieces, slot_limit;  // 16-byte pieces of k (of v); slots of the cache
    int32_t wide, page_size, heads, row_pieces;
};

// A thread moves a 16-byte piece of a row of k and the same one of v.
__global__ __launch_bounds__(kThreads) void cache_append_kernel(AppendArgs a) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= a.pieces) return;
    const int per_token = a.heads * a.row_pieces;
    const int64_t t = i / per_token;
    const int r = (int)(i - t * per_token), h = r / a.row_pieces, c = r - h * a.row_pieces;
    const int64_t slot = index_at(a.slots, a.wide, t);
    if (slot < 0 || slot >= a.slot_limit) return;
    const int64_t page = slot / a.page_size, at = slot - page * a.page_size;
#pragma unroll
    for (int x = 0; x < 2; x++)
        *reinterpret_cast<v4i*>(a.dst[x] + page * a.ds_p[x] + h * a.ds_h[x] + at * a.ds_n[x] + 16 * c) =
            *reinterpret_cast<const v4i*>(a.src[x] + t * a.ss_t[x] + h * a.ss_h[x] + 16 * c);
}

struct CopyArgs {
    unsigned char* cache[2];
    int64_t stride_l[2], stride_p[2];  // bytes: layer, page
    const void* src;
    const void* dst;
    int64_t pages;
    int32_t src_wide, dst_wide, page_pieces, count;
};

constexpr int kCopyPieces = 4;  // per thread, on their way together

// blockIdx: part of a page, pair, layer * 2 + cache
__global__ __launch_bounds__(kThreads) void cache_copy_kernel(CopyArgs a) {
    const int which = blockIdx.z & 1;
    const int64_t layer = blockIdx.z >> 1;
    const int first = blockIdx.x * (kThreads * kCopyPieces) + threadIdx.x;
    for (int i = blockIdx.y; i < a.count; i += gridDim.y) {
        const int64_t from = index_at(a.src, a.src_wide, i), to = index_at(a.dst, a.dst_wide, i);
        if (from < 0 || from >= a.pages || to < 0 || to >= a.pages) continue;
        unsigned char* base = a.cache[which] + layer * a.stride_l[which];
        const v4i* s = reinterpret_cast<const v4i*>(base + from * a.stride_p[which]);
        v4i* d = reinterpret_cast<v4i*>(base + to * a.stride_p[which]);
        v4i x[kCopyPieces];
#pragma unroll
        for (int e = 0; e < kCopyPieces; e++)
            if (first + e * kThreads < a.page_pieces) x[e] = s[first + e * kThreads];
#pragma unroll
        for (int e = 0; e < kCopyPieces; e++)
            if (first + e * kThreads < a.page_pieces) d[first + e * kThreads] = x[e];
    }
}

}  // namespace

int launch_cache_append(const sage_append_params& p, hipStream_t stream) {
    AppendArgs a{};
    const sage_tensor* src[2] = {&p.k, &p.v};
    const sage_tensor* dst[2] = {&p.k_cache, &p.v_cache};
    const int64_t e = dtype_bytes(p.dtype);
    for (int x = 0; x < 2; x++) {
        a.src[x] = (const unsigned char*)src[x]->ptr; a.ss_t[x] = e * src[x]->stride_n; a.ss_h[x] = e * src[x]->stride_h;
        a.dst[x] = (unsigned char*)dst[x]->ptr; a.ds_p[x] = e * dst[x]->stride_b; a.ds_h[x] = e * dst[x]->stride_h; a.ds_n[x] = e * dst[x]->stride_n;
    }
    a.slots = p.slots; a.wide = p.slots_int64 ? 1 : 0;
    a.slot_limit = p.pages * p.page_size;
    a.page_size = (int)p.page_size; a.heads = (int)p.heads_kv; a.row_pieces = (int)(p.head_dim * e / 16);
    a.pieces = p.tokens * a.heads * a.row_pieces;
    const int64_t wgs = (a.pieces + kThreads - 1) / kThreads;
    if (wgs > kMaxThreads / kThreads) return fail(SAGE_E_UNSUPPORTED, "sage_cache_append: too many rows for one launch");
    hipLaunchKernelGGL(cache_append_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, stream, a);
    return check_launch("cache_append_kernel");
}

int launch_cache_copy(const sage_copy_params& p, hipStream_t stream) {
    CopyArgs a{};
    a.cache[0] = (unsigned char*)p.k_cache; a.cache[1] = (unsigned char*)p.v_cache;
    a.stride_l[0] = p.k_stride_layer; a.stride_l[1] = p.v_stride_layer;
    a.stride_p[0] = p.k_stride_page; a.stride_p[1] = p.v_stride_page;
    a.src = p.src; a.dst = p.dst; a.src_wide = p.src_int64 ? 1 : 0; a.dst_wide = p.dst_int64 ? 1 : 0;
    a.pages = p.pages; a.page_pieces = (int)(p.page_bytes / 16); a.count = (int)p.count;
    const int parts = (a.page_pieces + kThreads * kCopyPieces - 1) / (kThreads * kCopyPieces);
    const unsigned pairs = (unsigned)(p.count < 65535 ? p.count : 65535);
    hipLaunchKernelGGL(cache_copy_kernel, dim3((unsigned)parts, pairs, (unsigned)(2 * p.layers)), dim3(kThreads), 0, stream, a);
    return check_launch("cache_copy_kernel");
}

}  // namespace sage
