// Which kernel an int8 product takes, by its sizes (plain C++).
#pragma once
#include <stdint.h>

namespace ud {

// Kernels for few rows: workgroups of 16 rows and 16 (or 32) channels whose waves share out k, 4 or 8 of them, with blocks of 64 u of k.
// Kernels for many: tiles of rows and channels through two or four LDS tiles, by four waves (eight where it says so).
enum LinearKernel {
    FEW_16x16,          // 4 waves, blocks of 1,024 of k
    FEW_16x16_DEEP,     // 8 waves
    FEW_16x16_SHORT,     // 4 waves, blocks of 512
    FEW_16x32,          // 4 waves, blocks of 512
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

// Few rows while their workgroups are one round of the chip, or the rows so few that reading them again for every 16 channels costs
// nothing: the weights' way from memory is the time then, and small tiles spread it over all CUs.  us, 16 x 16 / 16 x 32 / 64 x 64 (weights
// from HBM): 16 rows of 4,096 -> 4,096 6.1 / 7.9 / 9.6, 24 rows 8.9 / 7.8 / 9.8, 48 rows 13 / 12 / 9.8; one row of 4,096 -> 6,144 7.6 / 8.4 / 11.4;
// 13 rows of 2,048 -> 32,001 18.2 / 17.0 / 15.0 (64 x 128: 14.1).  All of k at one time where it fits: one row of 4,096 -> 32,000 in blocks of
// 1,024 24.0, of 512 31.8, but of 2,048 -> 32,001 14.1 and 12.9, with 8 waves of 12,288 -> 4,096 10.9, with 4 11.8.
//
// Otherwise the tile whose rounds over the 256 CUs cost least, from what one tile took per 128 of k and beside them (us, all CUs at
// work).  us predicted and measured: 563 rows of 4,096 -> 6,144 128 x 128 20 and 21.3, 64 x 64 36 and 30.4, 256 x 256 60 and 49; 2,469 of
// 12,288 -> 4,096 256 x 192 142 and 129, 128 x 128 165 and 164, 256 x 256 169 and 145; 8,192 of 4,096 -> 6,144 256 x 256 181 and 181,
// 256 x 192 206 and 200.
inline LinearKernel linear_kernel(int64_t M, int64_t N, int64_t K) {
    const int64_t few = tiles_of(M, N, 16, 16);
    if (M <= 4 || few <= 256) return K >= 8192 ? FEW_16x16_DEEP : K > 2048 ? FEW_16x16 : FEW_16x16_SHORT;
    if (tiles_of(M, N, 16, 32) <= 256) return FEW_16x32;
    struct Shape { LinearKernel kernel; int tm, tn; double step, once; };
    const Shape shapes[] = {{PANEL_64x64, 64, 64, 0.23, 1.5},   {PANEL_64x128, 64, 128, 0.31, 2},  {PANEL_128x64, 128, 64, 0.29, 2},
                            {PANEL_128x128, 128, 128, 0.54, 3}, {PANEL_256x192, 256, 192, 1.42, 6}, {PANEL_256x256, 256, 256, 1.70, 6}};
    const int64_t steps = (K + 127) / 128;
    LinearKernel best = PANEL_256x256;
    double least = 1e300;
    for (const Shape& s : shapes) {
        const int64_t tiles = tiles_of(M, N, s.tm, s.tn);
        const double cost = (double)((tiles + 255) / 256) * ((double)steps * s.step + s.once);
        if (cost < least) { least = cost; best = s.kernel == PANEL_128x128 && tiles > 256 ? PANEL_128x128_TWO : s.kernel; }
    }
    return best;
}

}  // namespace ud
