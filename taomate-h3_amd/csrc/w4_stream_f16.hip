// The instances of w4_stream.hpp for binary16 activations.
#include "w4_stream.hpp"

namespace h3q {

hipError_t launch_w4_stream_f16(const W4Args& a, hipStream_t st) {
    return a.zeros ? launch_w4_stream_groups<true, true>(a, st) : launch_w4_stream_groups<true, false>(a, st);
}

}  // namespace h3q
