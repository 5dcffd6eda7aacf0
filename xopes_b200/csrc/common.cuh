// Shared helpers for the xopes_b200 kernels (sm_100a only).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/xopes_b200.h"

namespace la {

template <typename T> struct Cvt;
template <> struct Cvt<float> {
  static __device__ __forceinline__ float to_f(float x) { return x; }
  static __device__ __forceinline__ float from_f(float x) { return x; }
};
template <> struct Cvt<__nv_bfloat16> {
  static __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Cvt<__half> {
  static __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
};

static inline size_t dtype_size(int dtype) { return dtype == LA_F32 ? 4 : 2; }

// Text of the last CUDA error this library met on the calling thread (la_debug_last_cuda_error).
char *last_cuda_error_buf();
static inline void note_cuda_error(cudaError_t e, const char *where) {
  snprintf(last_cuda_error_buf(), 256, "%s: %s", where, cudaGetErrorString(e));
}

// Launch-error check that never synchronises: reports configuration errors only.
static inline int launch_status() {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) note_cuda_error(e, "kernel launch");
  return e == cudaSuccess ? LA_OK : LA_ERR_CUDA;
}

// Launch of a kernel that may start while the kernel before it on the stream still runs: it calls after_previous() in every
// thread before it touches global memory (a kernel that ends without would let the one after it start too early), and
// lets_next_start() at its beginning.  What that saves is the next kernel's launch and setup, about 1 us a kernel (10.4 to 9.6 us for a token through 4096 x 4096).
// cluster > 0: size of the clusters of a kernel without a fixed one.
template <typename... K, typename... A>
static inline int launch_early(void (*kernel)(K...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, int cluster,
                               A &&...args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(args)...);
  if (e == cudaSuccess) return LA_OK;
  cudaGetLastError();
  note_cuda_error(e, "kernel launch");
  return LA_ERR_CUDA;
}
#ifdef __CUDACC__
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void lets_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

// While one of these lives, calls that a stream capture forbids on its thread (making a pool, a stream or an
// event) are allowed: for what the library makes once, on first need, which may be in a capture.
struct CaptureRelaxed {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  CaptureRelaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~CaptureRelaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// Address (on the current device) of the watchdog word that la_device_status() reads.
// Defined in api.cu; kernels that can time out receive it as a parameter.
int *status_word_ptr();
// The same for kernels that do without the word where it cannot be had: looking it up for the first time on a device
// would end a stream capture, so there the word stays null.  False on a CUDA error.
bool status_word_for(cudaStream_t st, int **word);

}  // namespace la
