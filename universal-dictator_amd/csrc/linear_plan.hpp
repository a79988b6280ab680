// Which kernel an int8 product takes, by its sizes (plain C++).
#pragma once
#include <stdint.h>

namespace ud {

// Kernels for a few rows, 16 at most: workgroups of 16 channels whose waves share out k, 4 or 8 of them, with blocks of 64 u of k.
// For some rows: the waves share out k too, through LDS tiles of their own.
// For many: tiles of rows and channels through two or four LDS tiles, by four waves (eight where it says so).
enum LinearKernel {
    FEW_16x16,          // 4 waves, blocks of 1,024 of k
    FEW_16x16_DEEP,     // 8 waves
    FEW_16x16_SHORT,    // 4 waves, blocks of 512
    SPLIT_16x16,        // 8 waves
    SPLIT_16x32,        // 4
    SPLIT_32x32,        // 4
    SPLIT_64x32,        // 4
    PANEL_64x64,        // 4 LDS tiles
    PANEL_64x128,       // 4
    PANEL_128x64,       // 4
    PANEL_128x128,      // 4: one workgroup a CU
    PANEL_128x128_TWO,  // 2: two workgroups a CU
    PANEL_256x192,      // 2
    PANEL_256x256,      // 2, eight waves
    LINEAR_KERNELS
};

constexpr int64_t tiles_of(int64_t M, int64_t N, int64_t tm, int64_t tn) { return ((M + tm - 1) / tm) * ((N + tn - 1) / tn); }

// Up to four rows the weights' way from memory is the time (one row of 4,096 -> 32,000 23.2 us, 16 x 32 split 26.2), in all of k at one
// time where it fits: in blocks of 1,024 24.0, of 512 31.8, but of 2,048 -> 32,001 14.1 and 12.9, with 8 waves of 12,288 -> 4,096 10.9, with 4
// 11.8.  Tiles of 16 x 16 that are between one and two rounds of the chip leave half of it idle, 16 x 32 that are one round do not: one row of
// 4,096 -> 6,144 7.7 and 6.8.
//
// Some rows: the smallest tiles that are one round of the chip (us, weights from HBM): 16 rows of 4,096 -> 4,096 16 x 16 5.7, 16 x 32 6.5; 32 rows
// 16 x 32 6.6, 32 x 32 7.6; 64 rows 32 x 32 7.5, 64 x 32 9.9; 128 rows 32 x 32 11.1, 64 x 32 9.7, 64 x 64 by four waves 12.2.  While they are
// one or two tiles of rows, more rounds cost less than larger tiles: 16 rows of 4,096 -> 32,000 16 x 32 26.9, 32 rows 32 x 32 30.2,
// 64 x 128 by four waves 31.8 and 33.2; of 2,048 -> 32,001, whose tiles are short, 14.6, 16.8 and 14.5, 15.0.
//
// Otherwise the tile with the least time on the CU that has the most of them: for each 128 of k of each tile, and beside that for each time
// that the CU is filled with as many as its LDS holds of them (us, fitted to 425 sizes with 33 to 8,192 rows: with 2 us between launches
// they lie within 7 to 15 % of the measured times at the median; the choice costs 0.4 % over the best tile on average, 3 % at the 95th
// percentile, 28 % at most, for 2,048 rows of 1,024 -> 2,048: 128 x 128 14.4, two a CU 11.3; after it 16 %, for 1,466 of 944 -> 11,826).
// us predicted and measured: 563 rows of 4,096 -> 6,144 128 x 128 21 and 24, two a CU 24 and 33, 64 x 64 41 and 33;
// 1,695 of 5,072 -> 2,914 two a CU 44 and 47, one 48 and 58, 64 x 64 62 and 66; 2,469 of 12,288 -> 4,096 256 x 192 117 and 128, 256 x 256 133 and
// 145; 8,192 of 4,096 -> 6,144 256 x 256 151 and 185.
inline LinearKernel linear_kernel(int64_t M, int64_t N, int64_t K) {
    const int64_t small = tiles_of(M, N, 16, 16), wide = tiles_of(M, N, 16, 32);
    if (M <= 4 && (small <= 256 || wide > 256)) return K >= 8192 ? FEW_16x16_DEEP : K > 2048 ? FEW_16x16 : FEW_16x16_SHORT;
    if (small <= 256) return SPLIT_16x16;
    if (wide <= 256 || M <= 16) return SPLIT_16x32;
    if (tiles_of(M, N, 32, 32) <= 256 || (M <= 32 && K > 2048)) return SPLIT_32x32;
    if (tiles_of(M, N, 64, 32) <= 256) return SPLIT_64x32;
    struct Shape { LinearKernel kernel; int tm, tn, held; double step, once; };
    const Shape shapes[] = {{PANEL_64x64, 64, 64, 2, 0.27, 2.03},       {PANEL_64x128, 64, 128, 1, 0.44, 2.55},
                            {PANEL_128x64, 128, 64, 1, 0.37, 2.65},     {PANEL_128x128, 128, 128, 1, 0.42, 6.02},
                            {PANEL_128x128_TWO, 128, 128, 2, 0.42, 8.25},{PANEL_256x192, 256, 192, 1, 1.10, 8.90},
                            {PANEL_256x256, 256, 256, 1, 1.27, 9.14}};
    const int64_t steps = (K + 127) / 128;
    LinearKernel best = PANEL_256x256;
    double least = 1e300;
    for (const Shape& s : shapes) {
        const int64_t tiles = (tiles_of(M, N, s.tm, s.tn) + 255) / 256;    // on one CU
        const double cost = (double)((tiles + s.held - 1) / s.held) * s.once + (double)(tiles * steps) * s.step;
        if (cost < least) { least = cost; best = s.kernel; }
    }
    return best;
}

}  // namespace ud
