// Paged key / value cache: what its kernels share - argument checks on the host, addresses on the device.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "internal.h"

namespace b200q {

constexpr int KV_MAX_SEQUENCES = 1024;      // one CTA scans the sequences, one thread each
constexpr int KV_MAX_PAGES = 1 << 20;       // its bitmap of free pages fits in shared memory
constexpr int KV_MAX_HEAD_DIM = 256;

int kv_check_pool(const char* who, const b200q_kv_pool* pool);
int kv_check_cache(const char* who, const b200q_kv_cache* cache);
// 32-bit arguments whose addresses the device takes as they are (null: not given)
int kv_check_words(const char* who, std::initializer_list<const void*> words);

// Makes the device that holds `p` current for the life of the object (the launch goes to that device whichever one the
// caller has current); rc is not B200Q_OK when `p` is no device memory.
class OnDeviceOf {
 public:
  OnDeviceOf(const char* who, const void* p);
  ~OnDeviceOf();
  OnDeviceOf(const OnDeviceOf&) = delete;
  OnDeviceOf& operator=(const OnDeviceOf&) = delete;
  int rc = B200Q_OK;
  int device = 0;

 private:
  int before_ = -1;
};

// SMs of a device; negative when it cannot be asked.
int sm_count(int device);

#ifdef __CUDACC__
// Launches a kernel that may become resident while its predecessor on the stream drains: every thread of it executes griddep_wait
// before it reads or writes anything outside the block, and it lets its own successor come early too.
template <typename... Formal, typename... Actual>
int launch_dependent(void (*kernel)(Formal...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Actual&&... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<Formal>(args)...));
  return B200Q_OK;
}
// Pages that sequence `s` holds, within its row of the table.
__device__ __forceinline__ int kv_held(const b200q_kv_pool& pool, int s) {
  const int n = pool.held[s];
  return n < 0 ? 0 : n < pool.table_width ? n : pool.table_width;
}
// Page of position `pos` of sequence `s`, or -1 where it holds none of the pool.
__device__ __forceinline__ int kv_page(const b200q_kv_pool& pool, int s, int pos) {
  const int j = (int)((unsigned)pos / (unsigned)pool.page_size);
  if (pos < 0 || j >= pool.table_width) return -1;
  const int p = pool.table[s * pool.table_stride + j];   // (read beside held, not after it)
  return j < kv_held(pool, s) && (unsigned)p < (unsigned)pool.pages ? p : -1;
}
// Element offset of (page, slot of pos) in one layer's keys or values, head 0; -1 where there is no page.
__device__ __forceinline__ int64_t kv_entry(const b200q_kv_cache& c, const b200q_kv_pool& pool, int s, int pos) {
  const int p = kv_page(pool, s, pos);
  if (p < 0) return -1;
  return p * c.page_stride + (int64_t)((unsigned)pos % (unsigned)pool.page_size) * c.slot_stride;
}
__device__ __forceinline__ int kv_length(const b200q_kv_pool& pool, int s) {
  const int n = pool.length[s], most = pool.table_width * pool.page_size;
  return n < 0 ? 0 : n < most ? n : most;
}
#endif

}  // namespace b200q
