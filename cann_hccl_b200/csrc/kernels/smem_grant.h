// Dynamic shared memory beyond what a kernel may have unasked (48 KB with what it has of its own).  The limit belongs to the function on a
// device, not to a call: two threads that each set their own call's size would take it from each other before their launches.  So it is
// set once for a kernel and device, to the most that any call asks for.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include <mutex>
#include "common/log.h"

namespace hcclb {

inline HcclResult grant_smem(const void *fn, size_t most, const char *what)
{
    struct Kernel { const void *fn; uint64_t devices; };  // devices: a bit for each that has the grant
    static std::mutex mu;
    static Kernel known[128];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return HCCL_E_RUNTIME;
    std::lock_guard<std::mutex> lk(mu);
    Kernel *k = known;
    while (k < known + 128 && k->fn && k->fn != fn) ++k;  // beyond the table a kernel is granted the same anew, which changes nothing
    if (k < known + 128 && k->fn == fn && (k->devices >> dev & 1)) return HCCL_SUCCESS;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    CHK_RET_LOG(e != cudaSuccess, HCCL_E_RUNTIME, "%s set-up failed: %s", what, cudaGetErrorString(e));
    if (k < known + 128) { k->fn = fn; k->devices |= 1ull << dev; }
    return HCCL_SUCCESS;
}

}  // namespace hcclb
