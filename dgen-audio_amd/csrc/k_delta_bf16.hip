// Gated delta rule in bf16: k_delta.h's kernels.
#include "k_delta.h"

namespace dgen {

void delta_enqueue_bf16(const dgen_hip_delta& a, bool backward, hipStream_t st) { delta_width<bf16>(a, backward, st); }

}  // namespace dgen
