// Which kernel a grouped product takes, from the mean rows of an expert (the counts
// themselves are on the device).
//
// Measured on MI355X (us; int8, tiled weights out of HBM, experts' shares uneven as a
// router's are; e4m3 the same within a few percent, its tiles 5% to 10% faster):
//   experts of n x k, SwiGLU       rows   stream  band 64  band 128  tiles
//   32 of  2816 x 2048, yes          8     31.7     36.2              50.2
//                                   16     42.6     36.3     41.2     51.2
//                                   48     84.0     42.6     41.4     51.7
//                                  100      147     48.6     51.1     72.5
//                                  400      516      117      112      112
//                                  800     1011      209      192      207
//   8 of  14336 x 5376, yes          8     92.7      111               117
//                                   16      131      115      118      118
//                                   48      330      120      126      127
//                                  200     1307      231      185      236
//                                  800     5195      662      544      526
//                                 2048                       1290     1170
//   16 of 4096 x 2048, no            8     24.5     29.3              30.9
//                                   48     64.2     33.3     30.9     34.5
//                                  200      219     55.6     56.5     73.2
//                                  800      833      153      138      135
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
