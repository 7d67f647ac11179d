// Host-side helpers shared by the translation units of the library: the one driver entry point it uses,
// device facts asked of the runtime once, per-kernel shared-memory opt-in.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>
#include <unordered_map>

#include "../../include/qssm.h"

namespace qssm {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = []() -> EncodeTiledFn {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// Driver-API calls (tensor map encoding) need the primary context current on the calling thread;
// a thread that has only inherited a device ordinal (e.g. an autograd worker) may not have one yet.
inline void ensure_context() {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaSetDevice(dev);
}

inline int dtype_size(int dt) { return dt == QSSM_F32 ? 4 : (dt == QSSM_F16 || dt == QSSM_BF16) ? 2 : 0; }

constexpr int MAX_DEVICES = 64;

inline int current_device() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return 0;
    return dev;
}

// SM count of the current device (looked up once per device ordinal).
inline int sm_count() {
    static int cached[MAX_DEVICES];
    const int dev = current_device();
    int n = __atomic_load_n(&cached[dev], __ATOMIC_RELAXED);
    if (n <= 0) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
        n = v;
        __atomic_store_n(&cached[dev], n, __ATOMIC_RELAXED);
    }
    return n;
}

// Per kernel instantiation and device: the largest dynamic shared-memory size the function has been
// opted into, and how many of its CTAs fit on an SM at a given size.  Both are asked of the runtime
// once, not on every launch.
struct KernelCache {
    std::mutex mu;
    std::unordered_map<unsigned long long, int> smem_set;   // (kernel, device) -> bytes
    std::unordered_map<unsigned long long, int> per_sm;     // (kernel, device, smem, threads) -> CTAs per SM
};
inline KernelCache& kernel_cache() {
    static KernelCache c;
    return c;
}
inline unsigned long long kernel_key(const void* fn, int dev) {
    return (unsigned long long)reinterpret_cast<uintptr_t>(fn) * 64ull + (unsigned long long)dev;
}

template <typename K> int ensure_smem(K kernel, int smem_bytes) {
    KernelCache& kc = kernel_cache();
    const unsigned long long key = kernel_key(reinterpret_cast<const void*>(kernel), current_device());
    std::lock_guard<std::mutex> lock(kc.mu);
    auto it = kc.smem_set.find(key);
    if (it != kc.smem_set.end() && it->second >= smem_bytes) return 0;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
    if (e != cudaSuccess) return (int)e;
    kc.smem_set[key] = smem_bytes;
    return 0;
}

}  // namespace qssm
