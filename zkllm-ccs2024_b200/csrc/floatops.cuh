// Types, vectors and argument checks shared by the float operators of a layer (rope.cu, block_norm.cu, glu.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cstddef>

#include "common.cuh"

namespace zkb {

typedef __nv_bfloat16 bf16;

// ---- values: all arithmetic is in 32 bits, a result is rounded once, to nearest even, when it is stored ------------------
template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<bf16>(bf16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive values; V * sizeof(T) is 16 for the wide paths, V is 1 for the path without alignment.
template <class T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };
template <class T> constexpr int kWide = 16 / (int)sizeof(T);

template <class T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&out)[V]) {
    const Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32<T>(x.v[i]);
}
template <class T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
    Vec<T, V> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<Vec<T, V>*>(p) = x;
}

inline size_t type_size(int dtype) { return dtype == ZKB_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == ZKB_F32 || dtype == ZKB_F16 || dtype == ZKB_BF16; }
inline bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// A pointer argument of the float operators: where it is given it has to be a whole element's address and memory that the
// current device reaches, so that a host array or another device's tensor ends in an error and not in a fault.
int check_device(const void* p, size_t align, const char* who, const char* what);

// A kernel that was launched beside its predecessor waits for that one's end and results; a kernel lets its successor be launched.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launch of a kernel that may start beside its predecessor on the stream: every thread of it that touches global memory, in
// whichever way, does so after grid_wait().
template <class... P, class... A>
int launch_beside(const char* name, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, const A&... args) {
    cudaLaunchAttribute beside;
    beside.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    beside.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c = {};
    c.gridDim = grid, c.blockDim = block, c.dynamicSmemBytes = smem, c.stream = s, c.attrs = &beside;
    c.numAttrs = g_profile_on ? 0 : 1;   // timed alone: the events around it would not order it
    if (g_profile_on) profile_begin(name, s);
    ZKB_CUDA(cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...));
    if (g_profile_on) profile_end(s);
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return ZKB_OK;
}

}  // namespace zkb
