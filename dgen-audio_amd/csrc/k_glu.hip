#include "seq.h"
namespace dgen {
int64_t mlp_workspace(const dgen_hip_mlp&, bool) { return 0; }
int mlp_run(const dgen_hip_mlp&, bool, hipStream_t, bool) { return fail(DGEN_HIP_E_INVALID, "not yet"); }
}
