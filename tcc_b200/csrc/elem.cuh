// elem.cuh -- element types (fp32, fp16, bf16) and 16-byte packs shared by the
// embedding, group norm and clipping kernels.  All arithmetic is fp32 or wider;
// a value is rounded to its storage type once, when it is stored.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace tcc {

// Lets a kernel use `bytes` of dynamic shared memory, once per device.
template <typename Kernel>
void allow_smem(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    TCC_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return;
    TCC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) done.fetch_or(bit, std::memory_order_release);
}

inline bool valid_type(int t) { return t == TCC_F32 || t == TCC_F16 || t == TCC_BF16; }
inline uint32_t type_bytes(int t) { return t == TCC_F32 ? 4u : 2u; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One element of an array whose type is known at run time (parameters that a
// thread reads once).
__device__ __forceinline__ float load_typed(const void* p, int type, uint64_t i) {
    if (type == TCC_F32) return static_cast<const float*>(p)[i];
    if (type == TCC_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_typed(void* p, int type, uint64_t i, float v) {
    if (type == TCC_F32) static_cast<float*>(p)[i] = v;
    else if (type == TCC_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// V elements moved as one aligned load or store (V * sizeof(T) <= 16).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

template <int BYTES>
struct RawOf;
template <> struct RawOf<2> { using type = unsigned short; };
template <> struct RawOf<4> { using type = unsigned int; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };

template <typename T, int V>
union PackBits {
    typename RawOf<sizeof(T) * V>::type raw;
    Pack<T, V> pack;
    __device__ PackBits() {}
};

// Plain, read-only and streaming (evict-first) accesses to one pack.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    PackBits<T, V> b;
    b.raw = *reinterpret_cast<const decltype(b.raw)*>(p);
    return b.pack;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack_nc(const T* p) {
    PackBits<T, V> b;
    b.raw = __ldg(reinterpret_cast<const decltype(b.raw)*>(p));
    return b.pack;
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack_cs(const T* p) {
    PackBits<T, V> b;
    b.raw = __ldcs(reinterpret_cast<const decltype(b.raw)*>(p));
    return b.pack;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    PackBits<T, V> b;
    b.pack = v;
    *reinterpret_cast<decltype(b.raw)*>(p) = b.raw;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack_cs(T* p, const Pack<T, V>& v) {
    PackBits<T, V> b;
    b.pack = v;
    __stcs(reinterpret_cast<decltype(b.raw)*>(p), b.raw);
}

// Asynchronous copies global -> shared of one pack (4 bytes at least); a
// thread waits for its own.
template <typename T, int V>
__device__ __forceinline__ void copy_pack_async(Pack<T, V>* smem, const T* global) {
    constexpr int bytes = sizeof(T) * V;
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(smem);
    if constexpr (bytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(global) : "memory");
    else if constexpr (bytes >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(global), "n"(bytes) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most LEFT of the thread's groups of copies are under way
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Kernels of one call that follow each other: launch_after lets the next one's
// CTAs take their places once the previous kernel's have all begun, and
// after_previous, first in each such kernel, holds them until that kernel is
// through and what it wrote can be seen.  What it wrote is read by plain loads
// (no __restrict__, no __ldg), which the compiler moves past no such wait.
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
void launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    TCC_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
}

// The widest V (of 8, 4, 2, 1; V * bytes <= 16) that divides every count in
// `counts` and keeps every pointer aligned to V elements of its own size.
struct VecRule {
    uint64_t bits = 8;  // or-ed element counts; starts at the widest V
    uint32_t max_bytes = 2;
    void count(uint64_t n) { bits |= n; }
    void pointer(const void* p, uint32_t bytes) {
        bits |= reinterpret_cast<uintptr_t>(p) / bytes;
        if (bytes > max_bytes) max_bytes = bytes;
    }
    int width() const {
        int v = 8;
        while ((uint64_t)v * max_bytes > 16 || (bits & (uint64_t)(v - 1))) v >>= 1;
        return v;
    }
};

}  // namespace tcc
