// Sizes of the MXFP4 products' tiles and passes, and how many rows a pass gets.  Plain C++, for the host's tests too.
#pragma once
#include <algorithm>
#include <cmath>

#ifdef __CUDACC__
#define SB_BOTH __host__ __device__ __forceinline__
#else
#define SB_BOTH inline
#endif

namespace sb {

constexpr int MX_TILE_ROWS = 128, MX_TILE_COLS = 256;
constexpr int MX_CODE_BYTES = MX_TILE_ROWS * MX_TILE_COLS / 2;
constexpr int MX_TILE_BYTES = MX_CODE_BYTES + MX_TILE_ROWS * MX_TILE_COLS / 32;

constexpr int MT_CHUNK = 128;            // packed bytes of a K chunk
constexpr int MT_BOX = 32;               // rows of an activation copy
constexpr int MT_MAX_N = 224;            // two accumulators of 224 columns and 64 columns of scales fill TMEM
constexpr int MT_MAX_SPLIT = 8;
constexpr int MT_SMALL_N = 96;           // two of 96 columns and the scales half of it: two blocks per SM

// Passes of a group of n rows: as few as the cap allows, of equal size up to the multiple of 16.
SB_BOTH int pass_rows(int n, int cap) {
    const int passes = (n + cap - 1) / cap;
    return passes ? ((n + passes - 1) / passes + 15) & ~15 : cap;
}

// Microseconds of all passes of `groups` groups of `rows` rows by passes of up to `cap`, without what every call costs, by what was
// measured: a chunk takes a block 0.3, or 0.4 with a second one beside it, a column of results 0.022, and all SMs together load 11 TB/s
// from L2.  A round of units that does not fill the chip counts half as a whole one and half as the share of the SMs that it keeps busy
// (8 experts of 256 x 3648, gate | up, 6456 rows: 19.7 us by passes of 192 and 15.9 by 224; estimates 11.3 and 11.5, by whole rounds
// 12.9 and 13.7).  Over 140 sizes the choice below takes 2.8 % less than without its limit, 6.6 % more at worst; by whole rounds 23 % more.
inline double pass_estimate(int rows, int groups, int row_tiles, int chunks, int sms, int cap) {
    const bool large = cap > MT_SMALL_N, pairs = large && row_tiles > 1;
    const double passes = (double)groups * ((rows + cap - 1) / cap), units = passes * (pairs ? (row_tiles + 1) / 2 : row_tiles);
    const int n = pass_rows(rows, cap);
    const bool two = !large && units > sms;
    const double share = units / (pairs ? sms / 2 : two ? 2 * sms : sms), rounds = (std::ceil(share) + std::max(share, 1.0)) / 2;
    const double loop = chunks * (two ? 0.4 : 0.3), store = 0.022 * n;
    const double loads = passes * row_tiles * chunks * (MX_TILE_BYTES + (large ? n / 2 : n) * MT_CHUNK) / 11e6;
    return std::max(rounds * std::max(loop, store) + std::min(loop, store), loads);
}

// Most rows of a pass, for `groups` groups that are expected to have `rows` rows (of expert groups a quarter and 8 above the average:
// a longer one takes a pass more, which reads its weights again, from L2).  Longer passes load less in all; shorter ones keep more
// SMs busy, write their results sooner, and up to 96 rows two blocks share an SM.  Fewer passes are taken for up to a tenth more than
// the size before them, which is within what the estimate leaves out (37 rows of 2112 x 2816: estimates 4.0 and 4.4, measured 7.1 us in
// two passes, 6.4 in one), and never for more than 15 % above the least estimate: without that limit the tenths add up (2134 rows of
// 465 x 4864: estimates 7.1 / 7.8 / 8.5 / 9.2 / 9.9 / 10.6 for 64 to 224 rows, measured 10.2 / 11.2 / 11.8 / 12.1 / 13.2 / 14.3).
inline int choose_cap(int rows, int groups, int row_tiles, int chunks, int sms) {
    const int last = std::min(MT_MAX_N, (rows + MT_BOX - 1) / MT_BOX * MT_BOX);
    double least = 0;
    for (int cap = MT_BOX; cap <= last; cap += MT_BOX) {
        const double t = pass_estimate(rows, groups, row_tiles, chunks, sms, cap);
        if (cap == MT_BOX || t < least) least = t;
    }
    int best = 0;
    double taken = 0, fewest = 0;
    for (int cap = MT_BOX; cap <= last; cap += MT_BOX) {
        const double passes = (double)groups * ((rows + cap - 1) / cap), t = pass_estimate(rows, groups, row_tiles, chunks, sms, cap);
        if (t <= 1.15 * least && (!best || (passes < fewest && t < 1.1 * taken))) {
            best = cap;
            taken = t;
            fewest = passes;
        }
    }
    return best;
}

// Blocks of a cluster that share a unit's chunks (1, 2, 4 or 8), where there are few units.  Two blocks fit on an SM where the share is
// at most `half` chunks; 0: never.
// Joining the parts costs about as much as four to six chunks of one block (0.33 us each); by 1 / 2 / 4 / 8 blocks one row of 2304 x 4096
// takes 7.4 / 6.6 / 6.4 / 6.5 us, of 1920 x 16384 18.4 / 12.2 / 9.2 / 8.6 (32 units of 16 chunks are the exception: 7.5 / 6.8 / 7.2).
// Units that wait for a place cost more than they save.  Blocks that fill an SM each find one for 74 clusters of two, 33 of four and 15
// of eight among 148 SMs: 16 units of 64 chunks take 9.4 us by four and 13.4 by eight, 34 of them 13.6 by two and 18.8 by four; 130
// blocks are within both smaller forms.  Two to an SM, 160 blocks still gain nothing and lose nothing (40 units of 16 chunks: 7.1 by
// two, 7.3 by four), 256 of eight lose (36 units: 12.1).
inline int choose_split(long long units, int chunks, int half, int sms) {
    int best = 1, cost = chunks;
    for (int split = 2; split <= MT_MAX_SPLIT; split *= 2) {
        const int share = (chunks + split - 1) / split;
        const int places = share <= half ? sms + sms / 12 : split == 8 ? sms * 13 / 16 : sms - sms / 8;
        if (units * split <= places && share + 4 + split / 4 < cost) {
            best = split;
            cost = share + 4 + split / 4;
        }
    }
    return best;
}

}  // namespace sb
