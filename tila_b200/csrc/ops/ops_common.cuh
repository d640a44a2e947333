// Shared by the hand-written operators: element types, status reporting and
// launch attributes.
#pragma once

#include "../../../include/tila_b200.h"
#include "../tile/tila_tile.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>

namespace tila_ops {

using tila::i32;
using tila::i64;
using tila::u32;
using tila::u64;

// Device error of the operators, beside tila::ErrorCode: an index read from
// device memory (a slot, a page) points outside its pool.
constexpr u32 kErrIndex = 5;

constexpr int kSms = 148;

inline int fail(int status, char *log, size_t cap, const char *fmt, ...) {
  if (log != nullptr && cap != 0) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(log, cap, fmt, ap);
    va_end(ap);
  }
  return status;
}

inline int launch_status(cudaError_t e, const char *what, char *log, size_t cap) {
  if (e == cudaSuccess) return TILA_OK;
  cudaGetLastError();  // the error is returned here, not left for the next call
  int code = (e == cudaErrorInvalidValue || e == cudaErrorLaunchOutOfResources)
                 ? TILA_ERR_RESOURCES : TILA_ERR_DRIVER;
  return fail(code, log, cap, "%s: %s", what, cudaGetErrorString(e));
}

// Launches `kernel`; `after_previous`: it may start while the previous kernel of
// the stream still runs (programmatic dependent launch).  Kernels launched so end
// or begin with tila::grid_dep_wait(), which returns when that kernel is done.
template <typename... P, typename... A>
cudaError_t launch_kernel(void (*kernel)(P...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t stream,
                          bool after_previous, const A &...args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = after_previous ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Lets `kernel` have `bytes` of dynamic shared memory, once for each device.
template <auto kernel> cudaError_t allow_shared_memory(int bytes) {
  static std::atomic<u64> allowed{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const u64 bit = device < 64 ? u64{1} << device : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// Two neighbouring elements as two floats, and back (each rounded to nearest).
template <typename T> __device__ __forceinline__ float2 unpack_pair(u32 w);
template <> __device__ __forceinline__ float2 unpack_pair<__half>(u32 w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <> __device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(u32 w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ u32 pack_pair(float lo, float hi);
template <> __device__ __forceinline__ u32 pack_pair<__half>(float lo, float hi) { return tila::pack_f16x2(lo, hi); }
template <> __device__ __forceinline__ u32 pack_pair<__nv_bfloat16>(float lo, float hi) {
  u32 r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// V elements moved by one access.
template <typename T, int V> struct __align__(sizeof(T) * V) Vec { T e[V]; };

}  // namespace tila_ops
