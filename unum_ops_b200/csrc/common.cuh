// Shared helpers for the unum_ops_b200 kernels: error reporting across the
// C ABI and small device utilities.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>
#include <cstdarg>
#include <cstdio>

#include "../../include/unum_ops_b200.h"

namespace unum {

// Thread-local message of the last failing entry point (read by unum_last_error).
void set_error(const char *fmt, ...);
void clear_error();

#define UNUM_CHECK_ARG(cond, ...)              \
    do {                                       \
        if (!(cond)) {                         \
            ::unum::set_error(__VA_ARGS__);    \
            return UNUM_ERR_INVALID;           \
        }                                      \
    } while (0)

#define UNUM_CHECK_CUDA(expr)                                                          \
    do {                                                                               \
        cudaError_t e_ = (expr);                                                       \
        if (e_ != cudaSuccess) {                                                       \
            ::unum::set_error("%s failed: %s", #expr, cudaGetErrorString(e_));         \
            return UNUM_ERR_CUDA;                                                      \
        }                                                                              \
    } while (0)

// Check the launch that was just enqueued.
inline int check_launch(const char *what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_error("%s launch failed: %s", what, cudaGetErrorString(e));
        return UNUM_ERR_CUDA;
    }
    return UNUM_OK;
}

inline int sm_count() {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n > 0 ? n : 148;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Programmatic dependent launch: a kernel launched with this attribute may start while the one before it in the stream
// still runs, so that its launch is not waited for.  Such a kernel begins with wait_for_previous_kernel in every thread,
// before it reads or writes anything and before any block ends: it returns when everything before has completed and is
// visible, and from then on lets the kernel behind it start in the same way.  Nothing that the kernel before may write is
// read through the read-only path (__ldg, const __restrict__): that is for memory which does not change while a kernel runs,
// and this one runs before those writes end; its lines are not made visible by the wait, and the compiler may move such a
// load ahead of it.
inline cudaLaunchAttribute behind_previous_kernel() {
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    return a;
}

#ifdef __CUDACC__
__device__ __forceinline__ void wait_for_previous_kernel() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
#endif

}  // namespace unum
