// What the hand-written CUDA entry points share: the error channel, launches that overlap the
// kernel before them, and the descriptions of a paged cache as the kernels see it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/ptxgen_b200.h"

// Records `msg` as the calling thread's last error (launcher.cpp) and returns `code`.
int pg_detail_fail(int code, const char *msg);

namespace pg {

inline int runtime_fail(cudaError_t e, const char *what) {
  char buf[512];
  snprintf(buf, sizeof buf, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
  return pg_detail_fail(PG_ERR_RUNTIME, buf);
}

__attribute__((format(printf, 1, 2))) inline int argument_fail(const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return pg_detail_fail(PG_ERR_ARGUMENT, buf);
}

// Arguments take the kernel's own types on the way.
template <class... P, class... A>
cudaError_t launch_kernel(const cudaLaunchConfig_t &cfg, void (*kernel)(P...), A... args) {
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Launches with programmatic stream serialization: the kernel's blocks may become resident
// while the kernel ahead of it on the stream drains, which hides a launch's set-up. Every kernel
// launched this way calls cudaGridDependencySynchronize() before its first access to memory, in
// every thread and on every path, so it still sees all that came before it and a kernel behind
// it cannot run ahead of what this one waits for.
// `Kernel` always has the same `smem`, so the opt-in above the default 48 KiB is made once a device.
template <auto Kernel, class... A>
int launch(const char *name, dim3 grid, int block, int smem, cudaStream_t stream, A... args) {
  cudaError_t e;
  if (smem > 32 * 1024) {  // with a kernel's static shared memory more than the default
    static std::atomic<uint64_t> done{0};
    int device = 0;
    if ((e = cudaGetDevice(&device)) != cudaSuccess) return runtime_fail(e, name);
    const uint64_t bit = 1ull << (device & 63);
    if (device > 63 || !(done.load(std::memory_order_relaxed) & bit)) {
      e = cudaFuncSetAttribute(reinterpret_cast<const void *>(Kernel),
                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return runtime_fail(e, name);
      done.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = launch_kernel(cfg, Kernel, args...);
  return e == cudaSuccess ? PG_OK : runtime_fail(e, name);
}

inline int sm_count(int *out) {
  static std::atomic<int> known[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && device < 64 && (*out = known[device].load(std::memory_order_relaxed)))
    return PG_OK;
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return runtime_fail(e, "cudaDeviceGetAttribute");
  if (device < 64) known[device].store(*out, std::memory_order_relaxed);
  return PG_OK;
}

__device__ __forceinline__ void wait_for_earlier_kernels() {
#if defined(__CUDA_ARCH__)
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
#endif
}

// The largest of three; NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two 32-bit numbers that one instruction multiplies and adds.
struct Two {
  uint64_t v;
  Two() = default;
  __device__ Two(uint64_t x) : v(x) {}
  __device__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ void get(float &x, float &y) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
  }
};
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two add(Two a, Two b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a.v), "l"(b.v));
  return r;
}

__device__ __forceinline__ uint4 load16(const void *p) {
  return *reinterpret_cast<const uint4 *>(p);
}

}  // namespace pg
