// Which kernel a grouped product takes, from the mean rows of an expert (the counts
// themselves are on the device).
//
// Measured on MI355X (us, int8 / e4m3; tiled weights out of HBM, experts' shares uneven as a
// router's are, one run on one card; runs differ by 2% to 4%):
//   experts of n x k, SwiGLU  rows         stream       band 64      band 128         tiles
//   32 of  2816 x 2048, yes      8    34.2 / 32.7   35.8 / 35.6   40.0 / 39.7   49.6 / 47.6
//                               16    42.6 / 41.6   36.4 / 36.7   40.7 / 40.3   53.0 / 48.0
//                               48    86.1 / 85.7   41.3 / 42.3   42.3 / 40.9   57.9 / 50.9
//                              100                  49.1 / 48.3   50.0 / 49.9   60.3 / 61.7
//                              200                  73.0 / 68.8   71.9 / 65.5   85.4 / 66.2
//                              300                  96.8 / 92.1   90.2 / 83.1    106 / 89.5
//                              400                    121 / 115     120 / 111    112 / 94.3
//                              600                    168 / 158     153 / 144     139 / 120
//                              800                    215 / 206     192 / 190     196 / 173
//                             2048                    551 / 525     473 / 463     409 / 360
//    8 of 14336 x 5376, yes      8    84.9 / 96.4     106 / 111     112 / 117     111 / 115
//                               16      152 / 130     114 / 114     118 / 117     119 / 115
//                               48      341 / 327     120 / 118     123 / 128     123 / 127
//                              100                    162 / 155     150 / 150     150 / 149
//                              200                    220 / 224     192 / 192     221 / 217
//                              300                    289 / 288     253 / 249     288 / 269
//                              400                    357 / 365     301 / 300     298 / 275
//                              600                    500 / 498     404 / 412     427 / 385
//                              800                    661 / 656     524 / 535     518 / 463
//                             2048                  1628 / 1610   1317 / 1290   1148 / 1033
//   64 of  2048 x 1408, no       8    34.8 / 36.6   36.0 / 36.9   41.6 / 40.4   42.8 / 43.5
//                               16    49.0 / 47.6   37.6 / 37.0   41.2 / 41.5   44.1 / 44.1
//                               48    95.2 / 95.8   41.6 / 42.2   48.0 / 49.7   50.2 / 53.6
//                              100                  56.2 / 53.8   54.1 / 55.6   72.7 / 72.0
//                              200                  79.0 / 77.9   78.7 / 77.4   84.7 / 81.8
//                              300                    107 / 107    99.4 / 104     104 / 108
//                              400                    137 / 134     128 / 125     128 / 122
//                              600                    194 / 189     180 / 175     162 / 145
//                              800                    254 / 247     228 / 222     213 / 192
//                             2048                    632 / 618     541 / 526     469 / 452
//   16 of  4096 x 2048, no       8    24.6 / 25.8   29.1 / 29.4   29.9 / 30.1   31.9 / 32.1
//                               16    31.7 / 31.9   29.3 / 29.5   30.1 / 32.3   32.8 / 32.9
//                               48    65.7 / 64.4   33.2 / 33.4   30.9 / 31.5   34.3 / 33.7
//                              100                  40.5 / 40.5   39.9 / 39.7   40.6 / 40.5
//                              200                  57.5 / 56.4   48.5 / 55.1   70.7 / 66.1
//                              300                  73.7 / 72.6   66.3 / 64.4   70.8 / 66.1
//                              400                  89.7 / 86.8   83.0 / 83.3    102 / 94.3
//                              600                    123 / 119     115 / 114    105 / 95.6
//                              800                    158 / 154     140 / 138     137 / 123
//                             2048                    405 / 391     355 / 343     314 / 277
// The borders lie where most of these cross: at 8 rows the streams lead, at 16 the 64-row bands;
// between 48 and 100 either band does, by up to 18%; tiles lead from 400 rows of e4m3 (16 of
// 4096 x 2048 from 600) and from 600 of int8 (8 of 14336 x 5376 from 800; 2816 x 2048 loses 2%
// there).
#include "h3q_kernels.hpp"

namespace h3q {

namespace {

enum GroupedKernel : int { kGroupedStream = 1, kGroupedBand64 = 4, kGroupedBand128 = 8, kGroupedTile = 256 };

GroupedKernel grouped_kernel(int kind, const GroupedArgs& a) {
    const int64_t mean = a.rows / a.experts;
    if (mean <= 10) return kGroupedStream;
    if (mean <= 64) return kGroupedBand64;
    // Wide products (see GroupedMfma) exist for the kernels that stream weights.
    if (mean <= (kind == kOpE4M3 ? 384 : 512) || !grouped_tile_supported(a) || (kind == kOpE4M3 && a.wide))
        return kGroupedBand128;
    return kGroupedTile;
}

}  // namespace

bool grouped_mm_fits(int kind, const GroupedArgs& a) {
    const GroupedKernel kernel = grouped_kernel(kind, a);
    if (kernel == kGroupedTile) return true;
    // A grid of n workgroups of 256 threads takes n * 256 < 2^32.
    return (kernel == kGroupedStream ? grouped_stream_grid(a) : grouped_band_grid(a, kernel)) < (int64_t(1) << 24);
}

hipError_t launch_grouped_mm(int kind, const GroupedArgs& a, hipStream_t st) {
    const GroupedKernel kernel = grouped_kernel(kind, a);
    if (kernel == kGroupedStream) return launch_grouped_stream(kind, a, st);
    if (kernel == kGroupedTile) return launch_grouped_tile(kind, a, st);
    return launch_grouped_band(kind, a, kernel, st);
}

}  // namespace h3q
