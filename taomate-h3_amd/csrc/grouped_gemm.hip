// Which kernel a grouped product takes, from the mean rows of an expert (the counts
// themselves are on the device).
//
// Measured on MI355X (us; int8, tiled weights out of HBM, experts' shares uneven as a
// router's are; e4m3 within a few percent of it up to 200 rows):
//   experts of n x k, SwiGLU       rows   stream  band 32  band 64  band 128  tiles
//   32 of  2816 x 2048, yes          4     28.5     33.2     38.8     42.8     50.2
//                                   12     34.9     38.9     40.7     44.3     50.3
//                                   18     44.4     40.3     41.2     44.4
//                                   40     59.9     58.5     43.9     46.9     50.7
//                                  100      114     98.9     69.0     53.6     75.5
//                                  400      372      185      156      130      113
//                                 1024                                 276      251
//   8 of  14336 x 5376, yes          4     89.5      108      110      114      115
//                                   18      163      116      115      116
//                                   40      157      129      119      124      124
//                                  160      513      325      203      178      167
//                                  400     1191      694      419      318      310
//                                 2048                                1312     1209
//   16 of 4096 x 2048, no           12     28.3     30.9     30.1     32.1     31.5
//                                  160      130     57.4     52.5     46.6     73.4
//                                  700                                 121      134
//                                 2048                                 353      309
#include "h3q_kernels.hpp"

namespace h3q {

namespace {

enum GroupedKernel : int { kGroupedStream = 1, kGroupedTile = 256 };  // else: 16-row blocks of a band

int grouped_kernel(int kind, const GroupedArgs& a) {
    const int64_t mean = a.rows / a.experts;
    if (mean <= 12) return kGroupedStream;
    if (mean <= 20) return 2;
    if (mean <= 48) return 4;
    // Wide products (see GroupedMfma) exist for the kernels that stream weights.
    if (mean <= 384 || !grouped_tile_supported(a) || (kind == kOpE4M3 && a.wide)) return 8;
    return kGroupedTile;
}

}  // namespace

bool grouped_mm_fits(int kind, const GroupedArgs& a) {
    const int kernel = grouped_kernel(kind, a);
    if (kernel == kGroupedTile) return true;
    // A grid of n workgroups of 256 threads takes n * 256 < 2^32.
    return (kernel == kGroupedStream ? grouped_stream_grid(a) : grouped_band_grid(a, kernel)) < (int64_t(1) << 24);
}

hipError_t launch_grouped_mm(int kind, const GroupedArgs& a, hipStream_t st) {
    const int kernel = grouped_kernel(kind, a);
    if (kernel == kGroupedStream) return launch_grouped_stream(kind, a, st);
    if (kernel == kGroupedTile) return launch_grouped_tile(kind, a, st);
    return launch_grouped_band(kind, a, kernel, st);
}

}  // namespace h3q
