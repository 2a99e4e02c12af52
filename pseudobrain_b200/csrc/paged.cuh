// The paged key-value cache: addressing shared by its kernels, and their launchers (called
// by the C ABI after validation).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "../../include/pbk.h"

namespace pbk {

namespace paged {

// A ring of `stages` buffers, each with a barrier whose phase ends when a unit's copy has landed:
// unit u lies in stage u % stages and ends its (u / stages)-th phase, so this is the parity to wait
// for. A reader that gives up at unit i waits for the units i .. ring_issued(i, ...) - 1 before the
// buffers are left: those that were issued (a unit is issued when the one `stages` before it has
// been read) and not read.
struct RingWait {
  int stage;
  uint32_t parity;
};
__host__ __device__ inline RingWait ring_wait(int64_t u, int stages) {
  return {(int)(u % stages), (uint32_t)(u / stages & 1)};
}
__host__ __device__ inline int64_t ring_issued(int64_t i, int stages, int64_t count) {
  return i + stages < count ? i + stages : count;
}

}  // namespace paged

#ifdef __CUDACC__
namespace paged {

// Entries of sequence b that the table can hold (lengths outside [0, capacity] are clamped).
__device__ __forceinline__ int clamp_length(int n, int width, int page) {
  const int64_t cap = (int64_t)width * page;
  return n < 0 ? 0 : (n > cap ? (int)cap : n);
}

// Pool page of entry j of table row `row`, -1 when the id lies outside the pool.
__device__ __forceinline__ int page_of(const int32_t* row, int j, int log_page, int pages) {
  const int id = row[j >> log_page];
  return (unsigned)id < (unsigned)pages ? id : -1;
}

// The cache's kernels are launched so that each may start while the one before it in the stream
// ends (programmatic dependent launch): every kernel lets its successor start at once and waits
// for its predecessor's writes before it touches memory. A serving step is a chain of short
// kernels, and this hides most of each launch.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace paged

template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, dim3 block, int smem, cudaStream_t st, int cluster,
                         Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = (size_t)smem, cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}
#endif

// SMs of the current device (looked up once per device).
inline int paged_sm_count() {
  static std::atomic<int> cached[64] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if ((n = cached[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
  cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

// An attribute of a kernel, set once per device (bit dev of `done`).
inline cudaError_t paged_allow(const void* kernel, cudaFuncAttribute what, int value, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, what, value);
  if (e == cudaSuccess && dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  return e;
}
inline cudaError_t paged_allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  return paged_allow(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes, done);
}

inline int paged_log2(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}

cudaError_t launch_paged_append(const pbk_paged_cache& c, const pbk_paged_batch& b, const void* k, const void* v,
                                int64_t stride_t, int64_t stride_h, int tokens, const int32_t* cu_seqlens,
                                cudaStream_t st);
size_t paged_attend_workspace(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_attend_desc& d);
cudaError_t launch_paged_attend(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_attend_desc& d,
                                void* ws, cudaStream_t st);
size_t paged_observe_workspace(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_observe_desc& d);
cudaError_t launch_paged_observe(const pbk_paged_cache& c, const pbk_paged_batch& b, const pbk_paged_observe_desc& d,
                                 void* ws, cudaStream_t st);
cudaError_t launch_paged_select(const pbk_paged_cache& c, const pbk_paged_batch& b, int budget, int recent, int sinks,
                                int32_t* src, int32_t* dst, int32_t* count, int moves, cudaStream_t st);
cudaError_t launch_paged_move(const pbk_paged_cache& c, const pbk_paged_batch& b, const int32_t* src,
                              const int32_t* dst, const int32_t* count, int moves, cudaStream_t st);

}  // namespace pbk
