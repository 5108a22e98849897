// C entries of the sequence operators (dgen_hip.h, "sequence operators on
// device tensors").
#include "seq.h"

using namespace dgen;

// One operator's entries: descriptor test, device, launch; and its scratch,
// for a descriptor that is complete but for the workspace.
#define DGEN_SEQ_ENTRY(name, type, run, backward)                                                   \
  extern "C" int dgen_hip_##name(int device, const type* d, void* stream) {                         \
    if (!d) return fail(DGEN_HIP_E_INVALID, #name ": null descriptor");                             \
    if (int rc = run(*d, backward, nullptr, true)) return rc;                                       \
    DeviceScope on(device);                                                                         \
    if (!on.ok()) return fail(DGEN_HIP_E_DEVICE, #name ": device %d", device);                      \
    return run(*d, backward, static_cast<hipStream_t>(stream), false);                              \
  }
#define DGEN_SEQ_WORKSPACE(name, type, run, need)                                                   \
  extern "C" int dgen_hip_##name##_workspace(int device, const type* d, int backward, uint64_t* bytes) { \
    if (!d || !bytes) return fail(DGEN_HIP_E_INVALID, #name "_workspace: null argument");           \
    if (d->struct_size != sizeof(*d)) return fail(DGEN_HIP_E_INVALID, #name "_workspace: struct_size"); \
    type t = *d;                                                                                    \
    t.workspace = reinterpret_cast<void*>(256);                                                     \
    t.workspace_bytes = ~0ull;                                                                      \
    if (int rc = run(t, backward != 0, nullptr, true)) return rc;                                   \
    *bytes = (uint64_t)need(*d, backward != 0);                                                     \
    return 0;                                                                                       \
  }
#define DGEN_SEQ(name, type, run, need)          \
  DGEN_SEQ_ENTRY(name, type, run, false)         \
  DGEN_SEQ_ENTRY(name##_backward, type, run, true) \
  DGEN_SEQ_WORKSPACE(name, type, run, need)

DGEN_SEQ(rms_norm, dgen_hip_norm, norm_run, norm_workspace)
DGEN_SEQ(causal_conv, dgen_hip_conv, conv_run, conv_workspace)
DGEN_SEQ(selective_scan, dgen_hip_scan, scan_run, scan_workspace)
DGEN_SEQ(gated_mlp, dgen_hip_mlp, mlp_run, mlp_workspace)
