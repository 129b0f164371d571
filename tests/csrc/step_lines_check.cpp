// The lines of steps (step_lines.h) against counting: every block's tiles and its place on the line, every share and its owner.
#include <cstdio>

#include "../../flagattention_amd/csrc/step_lines.h"

using namespace sage::attn;

int main() {
    long blocks = 0;
    for (int causal = 0; causal < 2; causal++)
        for (int shift = 0; shift <= 7; shift++)
            for (int m = 0; m <= 400; m += 1 + m / 40)
                for (int n = 0; n <= 700; n += 1 + n / 30) {
                    const Steps s(m, n, shift, causal);
                    int sum = 0;
                    for (int j = 0; j < s.nb; j++, blocks++) {
                        const int last = min((j + 1) << shift, m) - 1, seen = causal ? last + 1 + n - m : n;
                        const int tiles = seen <= 0 ? 1 : (seen + 63) / 64;
                        if (s.tiles(j) != tiles || s.before(j) != sum) return printf("block %d of M %d N %d shift %d causal %d\n", j, m, n, shift, causal), 1;
                        sum += tiles + kStart;
                    }
                    if (s.total() != sum) return printf("total of M %d N %d shift %d causal %d\n", m, n, shift, causal), 1;
                }
    for (int shares : {1, 2, 7, 512})
        for (int total = 0; total < 3000; total += 1 + total / 50) {
            const EqualShares line(total, shares);
            if (line.begin(0) != 0 || line.begin(shares) != total) return printf("ends of %d in %d\n", total, shares), 1;
            for (int w = 0; w < shares; w++)
                for (int pos = line.begin(w); pos < line.begin(w + 1); pos++)
                    if (line.owner(pos) != w) return printf("owner of %d of %d in %d\n", pos, total, shares), 1;
        }
    printf("ok %ld\n", blocks);
    return 0;
}
