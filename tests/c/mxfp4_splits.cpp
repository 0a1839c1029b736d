// Reads "units chunks half sms" per line and writes the blocks of a cluster that are chosen.
#include <cstdio>

#include "mxfp4_passes.h"

int main() {
    long long units;
    int chunks, half, sms;
    while (std::scanf("%lld %d %d %d", &units, &chunks, &half, &sms) == 4) std::printf("%d\n", sb::choose_split(units, chunks, half, sms));
}
