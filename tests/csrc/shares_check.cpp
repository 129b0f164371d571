// Steps that do not lie on a line (step_lines.h) belong to its first or last share that holds any.
#include <cstdio>

#include "../../flagattention_amd/csrc/step_lines.h"

using namespace sage::attn;

int main() {
    for (int shares : {1, 2, 512})
        for (int total : {1, 2, 5, 511, 512, 513, 70000, 0x7ffffffe}) {
            const EqualShares line(total, shares);
            const int last = line.owner(total - 1);
            if (last >= shares || line.begin(last) > total - 1 || line.owner(0) != 0) return printf("ends of %d in %d\n", total, shares), 1;
            for (int past : {1, 2, 3, 600, 1 << 20, 0x7fffffff})
                if (line.owner(-past) != 0 || (past <= 0x7fffffff - total && line.owner(total - 1 + past) != last))
                    return printf("%d outside of %d in %d\n", past, total, shares), 1;
        }
    printf("ok\n");
    return 0;
}
