// The instances of w4_stream.hpp for bf16 activations, and the choice between the types.
#include "w4_stream.hpp"

namespace h3q {

hipError_t launch_w4_stream_f16(const W4Args& a, hipStream_t st);  // w4_stream_f16.hip

hipError_t launch_w4_stream(const W4Args& a, hipStream_t st) {
    if (a.f16) return launch_w4_stream_f16(a, st);
    return a.zeros ? launch_w4_stream_groups<false, true>(a, st) : launch_w4_stream_groups<false, false>(a, st);
}

}  // namespace h3q
