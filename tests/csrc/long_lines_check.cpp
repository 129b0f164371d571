// The lines of steps (step_lines.h) of sequences with up to 2^30 keys against counting in 64 bits.  Lines of 2^31 steps and more
// are none: a launch is not cut then.
#include <cstdint>
#include <cstdio>
#include <random>

#include "../../flagattention_amd/csrc/step_lines.h"

using namespace sage::attn;

static long g_lines = 0;

static bool check(int m, int n, int shift, int causal) {
    const int nb = (int)((m + (1LL << shift) - 1) >> shift);
    auto tiles = [&](int64_t j) {
        const int64_t last = std::min((j + 1) << shift, (int64_t)m), seen = causal ? last + n - m : n;
        return seen <= 0 ? 1 : (seen + 63) / 64;
    };
    int64_t sum = 0;
    for (int j = 0; j < nb; j++) sum += tiles(j) + kStart;
    if (sum >= 1LL << 31) return true;
    g_lines++;
    const Steps s(m, n, shift, causal);
    if (s.nb != nb || s.total() != sum) return printf("total of M %d N %d shift %d causal %d: %d, not %lld\n", m, n, shift, causal, s.total(), (long long)sum), false;
    sum = 0;
    for (int j = 0; j < nb; j++) {
        if (s.tiles(j) != tiles(j) || s.before(j) != sum) return printf("block %d of M %d N %d shift %d causal %d\n", j, m, n, shift, causal), false;
        sum += tiles(j) + kStart;
    }
    return true;
}

int main() {
    std::mt19937 rng(1);
    auto between = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo)); };
    for (int causal = 0; causal < 2; causal++)
        for (int shift = 0; shift <= 7; shift++) {
            for (int n = 2965000; n < 2971000; n += 97)  // m (m + 1) passes 2^31 where a block sees 46341 tiles
                if (!check(512, n, shift, causal)) return 1;
            for (int i = 0; i < 600; i++) {
                const int top = i % 3 == 0 ? 1 << 30 : i % 3 == 1 ? 1 << 26 : 1 << 22;
                if (!check(between(0, 1500), between(1 << 21, top), shift, causal)) return 1;
            }
            for (int m : {1, 63, 64, 65, 128, 1000})
                for (int n : {(1 << 30) - 1, (1 << 30) - 64, (1 << 30) - 65, 1 << 29, 46341 * 64, 46341 * 64 - 1, 65536 * 64, 65536 * 64 + 1})
                    if (!check(m, n, shift, causal)) return 1;
            for (int m : {70000, 300001})  // more queries than keys
                for (int n : {0, 1, 5000, 69000})
                    if (!check(m, n, shift, causal)) return 1;
        }
    printf("ok %ld\n", g_lines);
    return 0;
}
