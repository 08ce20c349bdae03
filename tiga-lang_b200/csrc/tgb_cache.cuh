// Shared by the kernels over a paged key/value cache: place lookup with bounds,
// device-side checks, and programmatic dependent launch.
#pragma once

#include "tgb_common.cuh"

namespace tgb {

__device__ __forceinline__ void cache_fault(const tgb_paged_cache &c, int code) {
  *reinterpret_cast<volatile int32_t *>(c.fault) = code;
}

__device__ __forceinline__ int cache_capacity(const tgb_paged_cache &c) { return c.pages_per_sequence * c.page_size; }

// places that sequence b holds, inside [0, capacity]
__device__ __forceinline__ int cache_length(const tgb_paged_cache &c, int b) {
  const int length = c.lengths[b], capacity = cache_capacity(c);
  if ((unsigned)length > (unsigned)capacity) {
    cache_fault(c, TGB_CACHE_BAD_LENGTH);
    return length < 0 ? 0 : capacity;
  }
  return length;
}

// row of place t (inside the capacity) of sequence b, or -1 where its page does not exist
__device__ __forceinline__ int64_t cache_row(const tgb_paged_cache &c, int b, int t) {
  const int at = t / c.page_size;
  const int page = c.page_table[(int64_t)b * c.pages_per_sequence + at];
  if ((unsigned long long)(long long)page >= (unsigned long long)c.num_pages) {
    cache_fault(c, TGB_CACHE_BAD_PAGE);
    return -1;
  }
  return (int64_t)page * c.page_size + (t - at * c.page_size);
}

// A kernel launched by launch_dependent may start while the one before it still runs; it reads nothing
// that one writes before wait_for_previous().
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                             Args... args) {
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, args...);
}

// Shared memory beyond 48 KB has to be asked for once per kernel and device. `asked` is one word per kernel, a bit
// per device; two threads that both find the bit clear ask twice, which is harmless.
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t> &asked) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  int device;
  cudaError_t status = cudaGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (status != cudaSuccess || (device < 64 && (asked.load(std::memory_order_relaxed) & bit))) return status;
  status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (status == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return status;
}

int32_t check_cache(const tgb_paged_cache *cache);

}  // namespace tgb
