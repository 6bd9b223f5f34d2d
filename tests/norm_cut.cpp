// How rows of tsn_gate_add_norm are launched (gate_norm_cut, no GPU): one launch a line of stdin,
//   rows mod_rows waves chunks
// one answer a line of stdout: rows in turn, workgroups, threads of one
#include <hip/hip_runtime.h>

#include <cstdio>

#include "kernels.h"

int main() {
    unsigned rows, mod_rows, waves, chunks;
    while (scanf("%u %u %u %u", &rows, &mod_rows, &waves, &chunks) == 4) {
        const tsn::GateNormCut c = tsn::gate_norm_cut(rows, mod_rows, waves, chunks);
        printf("%u %u %u\n", c.per, c.grid, c.block);
    }
    return 0;
}
