// How the steps of a launch are laid out on a line and shared out: arithmetic of the kernels for packed sequences and paged caches,
// which the host compiler takes too.
#pragma once
#ifndef __HIP__
#include <algorithm>
#define __host__
#define __device__
using std::max;
using std::min;
#endif

namespace sage {
namespace attn {

// A line of steps in equal shares: share w has `base` of them, one more for w < rest.
struct EqualShares {
    int total, base, rest;
    __host__ __device__ EqualShares(int total_, int shares) : total(total_), base(total_ / shares), rest(total_ % shares) {}
    __host__ __device__ int begin(int w) const { return w * base + (w < rest ? w : rest); }
    // The share that holds step pos.  (One outside the line belongs to its first or last share: sequences whose offsets overlap can
    // have more steps than 31 bits count, and lie on the line anywhere; what is read for them has to exist all the same.)
    __host__ __device__ int owner(int pos) const {
        pos = max(min(pos, total - 1), 0);
        const int longer = rest * (base + 1);
        return pos < longer ? pos / (base + 1) : rest + (pos - longer) / base;
    }
};

constexpr int kVarKeys = 64;  // keys per tile of flash_varlen_kernel

// The steps of a cut launch as one line: sequence after sequence, K/V head after head, block after block of 2^tokens_shift
// queries each.  A block is kStart steps for what its start and end cost, and a step for each key tile (one for a block that
// sees no key).
constexpr int kStart = 4;
struct Steps {
    int M, N, nb, shift, causal;  // queries, keys and blocks of the sequence, tokens_shift
    __host__ __device__ Steps(int m, int n, int tokens_shift, int causal_)
        : M(m), N(n), nb((m + (1 << tokens_shift) - 1) >> tokens_shift), shift(tokens_shift), causal(causal_) {}
    __host__ __device__ int end(int j) const { return causal ? min((j + 1) << shift, M) + N - M : N; }  // keys that block j sees (0 or less: none)
    __host__ __device__ int tiles(int j) const { return max((end(j) + kVarKeys - 1) / kVarKeys, 1); }
    // 1 + 2 + .. + n modulo 2^32: the odd one of n and n + 1 times half of the even one
    __host__ __device__ static unsigned triangle(unsigned n) { return (n | 1) * ((n + 1) / 2); }
    // tiles of the first j < nb blocks: the first `ones` of them one each, block i of the others ceil(((i + 1) 2^shift + N - M) / 64).
    // (Sums from the sequence's first tile on pass 32 bits where a block sees 3 million keys; modulo 2^32 their differences, which do
    // not, are exact.)
    __host__ __device__ int tiles_before(int j) const {
        if (!causal) return j * max((N + kVarKeys - 1) / kVarKeys, 1);
        const int d = N - M;
        const int ones = d > kVarKeys ? 0 : min((kVarKeys - d) >> shift, j);
        const int over = j - ones;
        if (over == 0) return ones;
        static_assert(kVarKeys == 64, "2^6 keys");
        if (shift > 6) return (int)(ones + ((triangle(j) - triangle(ones)) << (shift - 6)) + (unsigned)over * (unsigned)((d + kVarKeys - 1) >> 6));
        const int q = 6 - shift, c = -(-d >> shift);  // 2^q blocks a tile; d / 2^shift rounded up
        auto sum = [&](int n) {  // of ceil(k / 2^q) for k = 1 .. n
            const unsigned m = (unsigned)n >> q, r = (unsigned)n & ((1u << q) - 1);
            return (triangle(m) << q) + r * (m + 1);
        };
        return (int)(ones + (sum(j + c) - sum(ones + c)));
    }
    __host__ __device__ int before(int j) const { return tiles_before(j) + kStart * j; }  // steps of the first j < nb blocks
    __host__ __device__ int total() const { return nb == 0 ? 0 : before(nb - 1) + tiles(nb - 1) + kStart; }
};

}  // namespace attn
}  // namespace sage
