// Reads "rows groups row_tiles chunks sms" per line and writes the pass size that is chosen, its estimate and the least estimate.
#include <cstdio>

#include "mxfp4_passes.h"

int main() {
    int rows, groups, tiles, chunks, sms;
    while (std::scanf("%d %d %d %d %d", &rows, &groups, &tiles, &chunks, &sms) == 5) {
        const int chosen = sb::choose_cap(rows, groups, tiles, chunks, sms);
        double least = 1e300;
        for (int cap = sb::MT_BOX; cap <= sb::MT_MAX_N; cap += sb::MT_BOX) {
            least = std::min(least, sb::pass_estimate(rows, groups, tiles, chunks, sms, cap));
            if (cap >= rows) break;
        }
        std::printf("%d %.17g %.17g\n", chosen, sb::pass_estimate(rows, groups, tiles, chunks, sms, chosen), least);
    }
}
