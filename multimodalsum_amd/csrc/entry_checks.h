// Argument checks and launch shapes that C entries share.
#pragma once
#include <hip/hip_runtime.h>

namespace {
// one of these required pointers is missing: the kernel would read or write address 0
template <typename... P> inline bool any_null(P... p) { return ((p == nullptr) || ...); }
// An axis of a launch holds fewer than 2^32 threads (beyond, the count wraps without an error and workgroups are missing): n workgroups of up to
// 1,024 threads on two axes.  Those with block_index() >= n, less than a row of them, have to leave at once.
inline dim3 grid_of(long n) {
    const long wide = n < 1 << 21 ? n : 1 << 21;
    return dim3((unsigned)wide, (unsigned)((n + wide - 1) / wide));
}
__device__ __forceinline__ long block_index() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }
}  // namespace
