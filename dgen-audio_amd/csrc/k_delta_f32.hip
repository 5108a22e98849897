// Gated delta rule in fp32: k_delta.h's kernels.
#include "k_delta.h"

namespace dgen {

void delta_enqueue_f32(const dgen_hip_delta& a, bool backward, hipStream_t st) { delta_width<float>(a, backward, st); }

}  // namespace dgen
