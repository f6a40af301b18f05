// rt_internal.h -- runtime helpers shared by libvearo_hip.so's translation
// units. Hidden: not part of the C ABI.
#pragma once
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/vearo_hip.h"

struct VhErrRecord;

namespace vh_rt {
#define VH_RT_HIDDEN __attribute__((visibility("hidden")))
// Records msg as this thread's vh_last_error() text and returns code.
VH_RT_HIDDEN int fail(int code, const std::string& msg);
// VH_OK once vh_init has run, else VH_ERR_NOT_INIT.
VH_RT_HIDDEN int require_init();
// The stream a `void* stream` argument names (NULL: the runtime's own).
VH_RT_HIDDEN hipStream_t stream_of(void* s);
// An unbatched dense product (no addend, or a bias over the output columns;
// accumulation allowed) through hipBLASLt; *taken is false when it does not
// take the layout or has no algorithm, and the caller runs its own kernel.
// akc / bkc: A / B have their unit stride along k.
VH_RT_HIDDEN int blaslt_gemm(const vh_gemm_desc* d, bool akc, bool bkc, void* stream, bool* taken);
// Releases hipBLASLt's handle, workspace and cached plans (vh_shutdown).
VH_RT_HIDDEN void blaslt_shutdown();
// Takes the current device's address of the device-resident scratch
// (noalloc.hip) once per device; vh_init calls it with `device` current.
VH_RT_HIDDEN int noalloc_setup(int device);
// That address (VH_NOALLOC_SCRATCH_BYTES bytes), or NULL before setup.
VH_RT_HIDDEN void* noalloc_scratch(int device);
// Launches a kernel of either code object with its argument struct (as the template in
// runtime.cpp, which says what grids it refuses).
VH_RT_HIDDEN int launch_args(const std::string& name, int64_t gx, int64_t gy, int64_t gz, unsigned block, hipStream_t s,
                             void* args);
// The device error record.
VH_RT_HIDDEN VhErrRecord* error_record();
// Compute units of the device.
VH_RT_HIDDEN int cu_count();
// VH_OK if a layout is not null, has a rank in [0, 8] and no negative dim or stride.
VH_RT_HIDDEN int check_layout(const vh_layout* l, const char* what);

// Scratch of one call: the caller's buffer, or a block of the arena that goes back
// when the call's launches are queued.
struct VH_RT_HIDDEN CallScratch {
  void* p = nullptr;
  hipStream_t s = nullptr;
  bool owned = false;
  ~CallScratch();
  // Refuses NULL on a stream under capture: a captured graph would go on using the
  // block after it has gone back.
  int get(hipStream_t stream, void* user, size_t user_bytes, size_t need);
};
}  // namespace vh_rt
