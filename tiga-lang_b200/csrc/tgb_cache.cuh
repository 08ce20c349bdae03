// Shared by the kernels over query / key heads and over a paged key/value cache:
// dependent launches, place lookup with bounds, device-side checks.
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

// Every kernel over heads and caches is launched by launch_dependent and begins with wait_for_previous: it is set up
// while the one before it runs and touches no memory until that one has ended (and, as it began the same way,
// everything before it). One token per sequence appended and the cache evicted in place: 16.4 -> 12.9 us. Letting the
// next kernel's blocks take their places before that (griddepcontrol.launch_dependents) was slower everywhere, and
// by 40 % for attention, whose blocks then share SMs with waiting ones of the next call.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Args>
cudaError_t launch_clusters(void (*kernel)(Args...), int cluster, dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                            Args... args) {
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = cluster, attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  config.attrs = attribute;
  config.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t status = cudaLaunchKernelEx(&config, kernel, args...);
  if (status == cudaSuccess) g_launches.fetch_add(1);
  return status;
}
template <typename T> struct Same { using type = T; };
template <typename... Args>
cudaError_t launch_dependent(void (*kernel)(Args...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                             typename Same<Args>::type... args) {
  return launch_clusters(kernel, 1, grid, block, shared, stream, args...);
}

// Shared memory beyond 48 KB has to be asked for once per kernel and device: the most that any call of the kernel
// needs, because the limit holds for all threads' launches and one set for a small call would fail another thread's
// large one. `asked` is one word per kernel, a bit per device; two threads that both find the bit clear ask for the same.
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
