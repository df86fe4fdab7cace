/* What the host sources of libattnres_hip.so share; none of it is exported. */
#ifndef KOTODAMA_AMD_ATTNRES_INTERNAL_H
#define KOTODAMA_AMD_ATTNRES_INTERNAL_H

#include <hip/hip_runtime.h>

#define ATTNRES_INTERNAL_SLOTS 128 /* kernels of lm_capi.cpp and serving_capi.cpp */
#define ATTNRES_HIDDEN __attribute__((visibility("hidden")))

#ifdef __cplusplus
extern "C" {
#endif

/* Sets attnres_last_error() and returns `code`. */
ATTNRES_HIDDEN int attnres_internal_fail(int code, const char* msg);

/* Kernel `name` of code-object part `part` on the current device, kept in slot
 * `slot` (one name per slot), and the device's CU count. */
ATTNRES_HIDDEN int attnres_internal_kernel(int slot, int part, const char* name, hipFunction_t* f, int* num_cus);

/* The current device's CU count. */
ATTNRES_HIDDEN int attnres_internal_num_cus(int* num_cus);

#ifdef __cplusplus
}
#endif

#endif /* KOTODAMA_AMD_ATTNRES_INTERNAL_H */
