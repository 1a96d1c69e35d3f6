// The paged key / value cache as the kernels see it, and launches that overlap the end of the one before.
#pragma once
#include "common.cuh"

#include <algorithm>
#include <atomic>
#include <utility>

namespace fa4b {

// Strides and row sizes in bytes.
struct KvView {
  uint8_t* k;
  uint8_t* v;
  int64_t k_layer, k_page, v_layer, v_page;
  int layers, pages, heads, page_tokens, page_shift, row_bytes, block_bytes;  // block: the dense [heads, tokens, D] of a page
  int32_t* table;
  int64_t table_stride;
  int max_seqs, width;
  int32_t* lens;
  int32_t* refs;
  int32_t* work;
};

// `work` in 32-bit words: findings of the page calls, findings of the attention over the cache, then what one call keeps
constexpr int kKvStatus = 0, kKvAttnStatus = 4, kKvHead = 8, kKvStatusWords = 8;

// checks a cache's description and turns it into what the kernels take
int kv_view(const fa4b_kv_cache* c, KvView* out);

inline bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

// A launch that may begin while the kernel before it on the stream still runs: every kernel launched this way runs
// pdl_wait() before it touches memory (which returns once the kernel before has ended and its writes are visible), so only
// the launch itself overlaps.  pdl_trigger() lets the next such launch come up early.  Pointer parameters of such a kernel are not
// __restrict__: loads through them might move above the wait.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_overlapped(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(std::forward<A>(args))...);
}

// A launch may have 48 KB of shared memory without more ado, of which static variables and the system take their part; more than this
// much dynamic memory is asked for.
constexpr size_t kSmemUnasked = 40 * 1024;

// More dynamic shared memory than that is allowed once per kernel and device; one `done` for each kernel.
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  FA4B_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return FA4B_OK;
  FA4B_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  FA4B_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));  // CTAs of two launches share an SM
  done.fetch_or(bit, std::memory_order_release);
  return FA4B_OK;
}

}  // namespace fa4b
