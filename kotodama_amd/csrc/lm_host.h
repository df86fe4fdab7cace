// What the host sources of the language-model operators share (lm_capi.cpp,
// serving_capi.cpp): errors, types, alignment and launches.
#ifndef KOTODAMA_AMD_LM_HOST_H
#define KOTODAMA_AMD_LM_HOST_H

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "attnres.h"
#include "attnres_internal.h"

namespace {

constexpr int kServingSlots = 100;  // the kernel slots from here on are serving_capi.cpp's

inline int fail(int code, const char* fmt, ...) {
  char buf[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return attnres_internal_fail(code, buf);
}

inline bool valid_dtype(int d) { return d == ATTNRES_DTYPE_F32 || d == ATTNRES_DTYPE_BF16; }
inline bool valid_index(int d) { return d == ATTNRES_INDEX_I32 || d == ATTNRES_INDEX_I64; }
inline int esize(int d) { return d == ATTNRES_DTYPE_BF16 ? 2 : 4; }
inline bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

template <typename Params>
int launch(int slot, int part, const char* name, unsigned gx, unsigned gy, unsigned block, unsigned lds, Params& P,
           void* stream) {
  if ((uint64_t)gx * block > UINT32_MAX)  // a launch's threads along one axis
    return fail(ATTNRES_ERR_UNSUPPORTED, "%s: too many rows for one call", name);
  hipFunction_t f = nullptr;
  int cus = 0;
  int rc = attnres_internal_kernel(slot, part, name, &f, &cus);
  if (rc != ATTNRES_OK) return rc;
  size_t sz = sizeof(Params);
  void* cfg[] = {HIP_LAUNCH_PARAM_BUFFER_POINTER, &P, HIP_LAUNCH_PARAM_BUFFER_SIZE, &sz, HIP_LAUNCH_PARAM_END};
  hipError_t e = hipModuleLaunchKernel(f, gx, gy, 1, block, 1, 1, lds, (hipStream_t)stream, nullptr, cfg);
  if (e != hipSuccess) return fail(ATTNRES_ERR_HIP, "hipModuleLaunchKernel(%s) failed: %s", name, hipGetErrorString(e));
  return ATTNRES_OK;
}

}  // namespace

#endif  // KOTODAMA_AMD_LM_HOST_H
