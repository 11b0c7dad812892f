// The pages of a key / value cache: reserving, freeing, forking (with the copy of ragged pages) and compacting.
//
// All state lives on the device: a decoding loop needs no copy to the host and can be captured.  A page is free when its
// reference count is zero, and pages are handed out lowest number first, so the outcome does not depend on the order in
// which threads run: counts change by integer atomics only, and every page's new place is computed from scans.
//
// What bounds them: the bookkeeping kernels are one CTA and latency (a scan of the counts with all its loads in flight); the copies are HBM.
#include "kv_cache.h"
#include "ptx_sm100.cuh"

namespace b200q {

// ---------------------------------------------------------------------------------------------- host checks
int kv_check_pool(const char* who, const b200q_kv_pool* pool) {
  if (!pool) return set_error(B200Q_ERR_INVALID, "%s: null pool", who);
  const b200q_kv_pool& p = *pool;
  if (!p.table || !p.length || !p.held || !p.refcount) return set_error(B200Q_ERR_INVALID, "%s: null pointer in the pool", who);
  if (((uintptr_t)p.table | (uintptr_t)p.length | (uintptr_t)p.held | (uintptr_t)p.refcount | (uintptr_t)p.scratch) & 3)
    return set_error(B200Q_ERR_INVALID, "%s: a pointer in the pool is not 4-byte aligned", who);
  if (p.sequences < 0 || p.table_width < 1 || p.pages < 1 || p.page_size < 1 || p.table_stride < p.table_width)
    return set_error(B200Q_ERR_INVALID, "%s: bad shape of the pool", who);
  if (p.sequences > KV_MAX_SEQUENCES || p.pages > KV_MAX_PAGES || (int64_t)p.table_width * p.page_size > 0x7fffffffLL)
    return set_error(B200Q_ERR_UNSUPPORTED, "%s: at most %d sequences, %d pages and 2^31 - 1 positions in a row of the table", who,
                     KV_MAX_SEQUENCES, KV_MAX_PAGES);
  return B200Q_OK;
}

int kv_check_cache(const char* who, const b200q_kv_cache* cache) {
  if (!cache) return set_error(B200Q_ERR_INVALID, "%s: null cache", who);
  const b200q_kv_cache& c = *cache;
  if (!c.k || !c.v) return set_error(B200Q_ERR_INVALID, "%s: null pointer in the cache", who);
  if (((uintptr_t)c.k | (uintptr_t)c.v) & 15) return set_error(B200Q_ERR_INVALID, "%s: keys and values must be 16-byte aligned", who);
  if (c.dtype != B200Q_DT_BF16 && c.dtype != B200Q_DT_F16) return set_error(B200Q_ERR_UNSUPPORTED, "%s: the cache must be bf16 or f16", who);
  if (c.layers < 1 || c.heads < 1 || c.head_dim < 1) return set_error(B200Q_ERR_INVALID, "%s: bad shape of the cache", who);
  if (c.head_dim % 8 || c.head_dim > KV_MAX_HEAD_DIM)
    return set_error(B200Q_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8, at most %d", who, KV_MAX_HEAD_DIM);
  if (c.heads > 65535 || c.layers > 65535) return set_error(B200Q_ERR_UNSUPPORTED, "%s: at most 65535 heads and layers", who);
  if ((c.layer_stride | c.page_stride | c.slot_stride | c.head_stride) & 7)
    return set_error(B200Q_ERR_INVALID, "%s: the cache's strides must be multiples of 8 elements", who);
  if (c.layer_stride < 0 || c.page_stride < 1 || c.slot_stride < 1 || c.head_stride < 1 || c.page_stride >= 1LL << 38 ||
      c.slot_stride >= 1LL << 38 || c.head_stride >= 1LL << 38)
    return set_error(B200Q_ERR_INVALID, "%s: the cache's strides must be positive (and below 2^38 elements)", who);
  return B200Q_OK;
}

OnDeviceOf::OnDeviceOf(const char* who, const void* p) {
  cudaPointerAttributes a{};
  cudaError_t e = cudaPointerGetAttributes(&a, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    rc = cuda_error(e, "cudaPointerGetAttributes", __FILE__, __LINE__);
    return;
  }
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) {
    rc = set_error(B200Q_ERR_INVALID, "%s: the pointers must be device memory", who);
    return;
  }
  int now = 0;
  if ((e = cudaGetDevice(&now)) != cudaSuccess) {
    rc = cuda_error(e, "cudaGetDevice", __FILE__, __LINE__);
    return;
  }
  device = a.type == cudaMemoryTypeManaged ? now : a.device;
  if (device != now) {
    if ((e = cudaSetDevice(device)) != cudaSuccess) rc = cuda_error(e, "cudaSetDevice", __FILE__, __LINE__);
    else before_ = now;
  }
}
OnDeviceOf::~OnDeviceOf() {
  if (before_ >= 0) cudaSetDevice(before_);
}

int sm_count(int device) {
  int n = 0;
  cudaError_t e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  return e == cudaSuccess ? n : cuda_error(e, "cudaDeviceGetAttribute", __FILE__, __LINE__);
}

namespace {

constexpr int PLAN_THREADS = 1024;

// Inclusive sum over the block's threads, one value each; every thread also gets the total.  buf: 33 words of shared memory.
__device__ __forceinline__ long long block_scan(long long v, long long* buf, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();   // buf may still be read from the scan before
  if (lane == 31) buf[warp] = v;
  __syncthreads();
  if (warp == 0) {
    long long w = lane < (int)(blockDim.x >> 5) ? buf[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    buf[lane] = w;
  }
  __syncthreads();
  *total = buf[31];
  return v + (warp ? buf[warp - 1] : 0);
}

// The `need` lowest free pages, in order: give(rank, page) is called once for every rank below `need`, by some thread.  Nothing is
// called and false returned when there are fewer.  All threads of a block of PLAN_THREADS call it; bitmap: a word for 32 pages.
//
// Free pages become bits (a lane looks at four counts, eight lanes' nibbles make a word), 32768 pages a step so that all loads of a
// step are in flight, and the steps end once enough are found; ranks are the sums of the bits before, by a scan over the threads'
// runs of words.
template <typename Give>
__device__ bool lowest_free(const int32_t* refcount, int pages, long long need, uint32_t* bitmap, long long* buf, Give give) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = PLAN_THREADS / 32;
  const bool wide = (reinterpret_cast<uintptr_t>(refcount) & 15) == 0;
  constexpr int PER_WARP = 1024;                   // pages of a step that a warp looks at, 128 at a time
  int seen = 0;                                    // pages whose bits are set up (a multiple of 128 but for the last)
  long long found = 0;
  while (seen < pages && found < need) {
    const int first = seen + warp * PER_WARP;
    int4 c[PER_WARP / 128];
#pragma unroll
    for (int i = 0; i < PER_WARP / 128; ++i) {
      const int p = first + i * 128 + lane * 4;
      c[i] = make_int4(1, 1, 1, 1);
      if (wide && p + 4 <= pages) {
        c[i] = *reinterpret_cast<const int4*>(refcount + p);
      } else {
        if (p < pages) c[i].x = refcount[p];
        if (p + 1 < pages) c[i].y = refcount[p + 1];
        if (p + 2 < pages) c[i].z = refcount[p + 2];
        if (p + 3 < pages) c[i].w = refcount[p + 3];
      }
    }
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER_WARP / 128; ++i) {
      uint32_t w = (uint32_t)(c[i].x == 0) | (uint32_t)(c[i].y == 0) << 1 | (uint32_t)(c[i].z == 0) << 2 | (uint32_t)(c[i].w == 0) << 3;
      w <<= 4 * (lane & 7);
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      const int at = first + i * 128 + (lane >> 3) * 32;
      if ((lane & 7) == 0 && at < pages) {
        bitmap[at >> 5] = w;
        mine += __popc(w);
      }
    }
    long long total;
    block_scan(mine, buf, &total);
    found += total;
    seen = seen + warps * PER_WARP < pages ? seen + warps * PER_WARP : pages;
  }
  if (found < need) return false;
  const int words = (seen + 31) >> 5, each = (words + PLAN_THREADS - 1) / PLAN_THREADS;
  const int w0 = threadIdx.x * each;
  int mine = 0;
  for (int i = 0; i < each; ++i)
    if (w0 + i < words) mine += __popc(bitmap[w0 + i]);
  long long total;
  long long rank = block_scan(mine, buf, &total) - mine;
  // a warp goes through its lanes' words together, a bit a lane: neighbouring ranks are handed out by neighbouring lanes
  for (int i = 0; i < each; ++i) {
    const uint32_t w = w0 + i < words ? bitmap[w0 + i] : 0u;
    uint32_t some = __ballot_sync(0xffffffffu, w != 0u && rank < need);
    while (some) {
      const int src = __ffs(some) - 1;
      some &= some - 1;
      const uint32_t bits = __shfl_sync(0xffffffffu, w, src);
      const long long base = __shfl_sync(0xffffffffu, rank, src);
      const int word = __shfl_sync(0xffffffffu, w0, src) + i;
      const long long r = base + __popc(bits & ((1u << lane) - 1u));
      if ((bits >> lane & 1u) && r < need) give(r, word * 32 + lane);
    }
    rank += __popc(w);
  }
  return true;
}

// The first of n ascending sums that is above `rank`.
__device__ __forceinline__ int owner(const long long* sums, int n, long long rank) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > rank) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) reserve_kernel(b200q_kv_pool pool, const int32_t* __restrict__ extra, int32_t* status) {
  extern __shared__ uint32_t bitmap[];
  __shared__ long long buf[33], sums[KV_MAX_SEQUENCES];
  __shared__ int base[KV_MAX_SEQUENCES];
  const int s = threadIdx.x;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  long long need = 0;
  int held = 0, narrow = 0;
  if (s < pool.sequences && extra[s] >= 0) {
    const int n = pool.length[s];
    held = pool.held[s];
    held = held < 0 ? 0 : held < pool.table_width ? held : pool.table_width;
    const long long want = ((long long)(n < 0 ? 0 : n) + extra[s] + pool.page_size - 1) / pool.page_size;
    need = want > held ? want - held : 0;
    narrow = want > pool.table_width;
  }
  long long total;
  const long long upto = block_scan(need, buf, &total);
  sums[s] = upto;
  base[s] = held - (int)(upto - need);   // column of rank r: base + r
  if (__syncthreads_or(narrow)) {
    if (s == 0 && status) *status = 2;
    return;
  }
  if (total == 0) return;
  const bool ok = lowest_free(pool.refcount, pool.pages, total, bitmap, buf, [&](long long r, int page) {
    const int t = owner(sums, pool.sequences, r);
    pool.table[t * pool.table_stride + base[t] + (int)r] = page;
    pool.refcount[page] = 1;
  });
  if (!ok) {
    if (s == 0 && status) *status = 1;
    return;
  }
  if (need) pool.held[s] = held + (int)need;
}

__global__ void __launch_bounds__(128) free_kernel(b200q_kv_pool pool, const int32_t* __restrict__ which) {
  const int s = blockIdx.x;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if (which[s] == 0) return;
  int n = pool.held[s];
  n = n < pool.table_width ? n : pool.table_width;
  int32_t* row = pool.table + s * pool.table_stride;
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int p = row[j];
    if ((unsigned)p < (unsigned)pool.pages) atomicSub(pool.refcount + p, 1);
    row[j] = -1;
  }
  __syncthreads();   // every thread has read held
  if (threadIdx.x == 0) pool.held[s] = pool.length[s] = 0;
}

// ---- fork.  What the second kernel reads from scratch: words 0 = may go on, 1 = ragged children; then for every sequence the
// length and the pages before the call, the child's own page (-1: none), the page that it is a copy of (read here: the
// parent's row may be a child's too) and the list of ragged children.
struct ForkScratch {
  int32_t *go, *ragged, *length, *held, *page, *source, *list;
};
constexpr int64_t scratch_words(int64_t n) { return 2 + 5 * n; }
__device__ __forceinline__ ForkScratch fork_scratch(int32_t* w, int n) {
  return {w, w + 1, w + 2, w + 2 + n, w + 2 + 2 * n, w + 2 + 3 * n, w + 2 + 4 * n};
}

__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(b200q_kv_pool pool, const int32_t* __restrict__ parent, int32_t* status) {
  extern __shared__ uint32_t bitmap[];
  __shared__ long long buf[33];
  __shared__ int list[KV_MAX_SEQUENCES], lengths[KV_MAX_SEQUENCES];
  const int s = threadIdx.x, n = pool.sequences;
  const ForkScratch f = fork_scratch(pool.scratch, n);
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if (s < n) lengths[s] = kv_length(pool, s);
  __syncthreads();
  const int p = s < n ? parent[s] : -1;
  const bool child = p >= 0 && p < n && p != s;
  const int count = child ? lengths[p] : 0, ragged = count % pool.page_size != 0;
  long long total;
  const long long rank = block_scan(ragged, buf, &total) - ragged;
  if (ragged) list[rank] = s;
  if (s < n) {
    f.length[s] = lengths[s];
    f.held[s] = pool.held[s];
    f.page[s] = -1;
    f.source[s] = ragged ? kv_page(pool, p, count) : -1;
  }
  if (s == 0) {
    *f.ragged = (int)total;
    *f.go = 1;
  }
  __syncthreads();
  if (s < total) f.list[s] = list[s];
  const bool ok = total == 0 || lowest_free(pool.refcount, pool.pages, total, bitmap, buf, [&](long long r, int page) { f.page[list[r]] = page; });
  if (!ok) {
    if (s == 0) {
      *f.go = 0;
      if (status) *status = 1;
    }
    return;
  }
  if (child) {
    pool.length[s] = count;
    pool.held[s] = (count + pool.page_size - 1) / pool.page_size;
  }
}

constexpr int FORK_THREADS = 256;
constexpr int FORK_TILE = 8192;   // table entries of a tile: at least 8 columns of 1024 sequences

// Blocks below `table_blocks` take the tables, a run of columns each: all sequences' entries of these columns are read before the
// first is written, so children may be parents.  The other blocks copy ragged pages, a (child, layer, keys or values) at a time.
__global__ void __launch_bounds__(FORK_THREADS)
fork_kernel(b200q_kv_cache cache, b200q_kv_pool pool, const int32_t* __restrict__ parent, int table_blocks, int columns) {
  __shared__ int32_t old[FORK_TILE];
  const int n = pool.sequences;
  const ForkScratch f = fork_scratch(pool.scratch, n);
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if (*f.go == 0) return;
  if ((int)blockIdx.x < table_blocks) {
    for (int c0 = blockIdx.x * columns; c0 < pool.table_width; c0 += table_blocks * columns) {
      for (int i = threadIdx.x; i < n * columns; i += FORK_THREADS) {
        const int s = i / columns, c = c0 + i % columns;
        old[i] = c < pool.table_width ? pool.table[s * pool.table_stride + c] : -1;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < n * columns; i += FORK_THREADS) {
        const int s = i / columns, c = c0 + i % columns, p = parent[s];
        if (p < 0 || p >= n || p == s || c >= pool.table_width) continue;
        const int full = f.length[p] / pool.page_size;
        int entry = -1;
        if (c < full) {
          entry = old[p * columns + i % columns];
          if ((unsigned)entry < (unsigned)pool.pages) atomicAdd(pool.refcount + entry, 1);
        } else if (c == full && f.page[s] >= 0) {
          entry = f.page[s];
          atomicAdd(pool.refcount + entry, 1);
        }
        if (c < f.held[s] && (unsigned)old[i] < (unsigned)pool.pages) atomicSub(pool.refcount + old[i], 1);
        pool.table[s * pool.table_stride + c] = entry;
      }
      __syncthreads();
    }
    return;
  }
  // the order of a page's elements that is nearer to the one in memory: slots outside heads, or heads outside slots
  const int chunks = cache.head_dim / 8, ragged = *f.ragged, parts = 2 * cache.layers;
  const bool slots_outside = cache.slot_stride >= cache.head_stride;
  for (int item = blockIdx.x - table_blocks; item < ragged * parts; item += gridDim.x - table_blocks) {
    const int s = f.list[item / parts], part = item % parts, from = f.source[s], to = f.page[s];
    if (from < 0) continue;
    const int slots = f.length[parent[s]] % pool.page_size;
    uint16_t* base = static_cast<uint16_t*>(part & 1 ? cache.v : cache.k) + (part >> 1) * cache.layer_stride;
    const int inner = slots_outside ? cache.heads : slots;
    for (int i = threadIdx.x; i < slots * cache.heads * chunks; i += FORK_THREADS) {
      const int d = i % chunks, row = i / chunks, a = row / inner, b = row % inner;
      const int64_t at = (slots_outside ? a * cache.slot_stride + b * cache.head_stride : b * cache.slot_stride + a * cache.head_stride) + d * 8;
      *reinterpret_cast<uint4*>(base + to * cache.page_stride + at) = *reinterpret_cast<const uint4*>(base + from * cache.page_stride + at);
    }
  }
}

// ---- compact.  A block takes a (sequence, layer, keys or values); a thread takes 16 bytes of a head and walks along the path.
// Entry i is moved to place i <= path[i], and no later source lies at or before place i (the path ascends), so loads may run ahead of
// stores but not the other way: eight loads, then their stores.
constexpr int COMPACT_THREADS = 128, PATH_MOST = 1024, COMPACT_AHEAD = 8;

__global__ void __launch_bounds__(COMPACT_THREADS)
compact_kernel(b200q_kv_cache cache, b200q_kv_pool pool, const int32_t* __restrict__ path, int64_t path_stride, int path_width,
               const int32_t* __restrict__ path_length, int32_t* __restrict__ length_out) {
  __shared__ int64_t from[PATH_MOST], to[PATH_MOST];
  __shared__ int good;
  const int parts = 2 * cache.layers, chunks = cache.head_dim / 8;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  for (int item = blockIdx.x; item < pool.sequences * parts; item += gridDim.x) {
    const int s = item / parts, part = item % parts, length = kv_length(pool, s);
    int n = path_length[s];
    n = n < 0 ? 0 : n < path_width ? n : path_width;
    if (threadIdx.x == 0) good = n;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += COMPACT_THREADS) {
      const int32_t* row = path + s * path_stride;
      const int node = row[i], before = i ? row[i - 1] : -1;
      const bool in = node > before && node >= i && (int64_t)length + node <= 0x7fffffffLL;
      from[i] = in ? kv_entry(cache, pool, s, length + node) : -1;
      to[i] = in ? kv_entry(cache, pool, s, length + i) : -1;
      if (from[i] < 0 || to[i] < 0) atomicMin(&good, i);
    }
    __syncthreads();
    n = good;
    if (part == 0 && threadIdx.x == 0) length_out[s] = length + n;
    uint16_t* base = static_cast<uint16_t*>(part & 1 ? cache.v : cache.k) + (part >> 1) * cache.layer_stride;
    for (int c = threadIdx.x; c < cache.heads * chunks; c += COMPACT_THREADS) {
      uint16_t* p = base + (c / chunks) * cache.head_stride + (c % chunks) * 8;
      for (int i0 = 0; i0 < n; i0 += COMPACT_AHEAD) {
        uint4 v[COMPACT_AHEAD];
#pragma unroll
        for (int j = 0; j < COMPACT_AHEAD; ++j)
          if (i0 + j < n && from[i0 + j] != to[i0 + j]) v[j] = *reinterpret_cast<const uint4*>(p + from[i0 + j]);
#pragma unroll
        for (int j = 0; j < COMPACT_AHEAD; ++j)
          if (i0 + j < n && from[i0 + j] != to[i0 + j]) *reinterpret_cast<uint4*>(p + to[i0 + j]) = v[j];
      }
    }
    __syncthreads();   // from, to and good are the next item's
  }
}

// The new lengths take the place of the old ones once no block needs those.
__global__ void __launch_bounds__(KV_MAX_SEQUENCES) lengths_kernel(const int32_t* __restrict__ from, int32_t* __restrict__ to, int n) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if ((int)threadIdx.x < n) to[threadIdx.x] = from[threadIdx.x];
}

int check_scratch(const char* who, const b200q_kv_pool* pool) {
  if (!pool->scratch || pool->scratch_words < scratch_words(pool->sequences))
    return set_error(B200Q_ERR_INVALID, "%s: the pool's scratch holds fewer than b200q_kv_scratch_words(sequences) words", who);
  return B200Q_OK;
}

// Raises a kernel's shared-memory limit to what a bitmap of this pool's pages takes.
int bitmap_bytes(const void* kernel, int pages, size_t* bytes) {
  *bytes = ((size_t)pages + 31) / 32 * 4;
  if (*bytes > 32 * 1024) CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KV_MAX_PAGES / 8));
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int64_t b200q_kv_scratch_words(int32_t sequences) { return scratch_words(sequences > 0 ? sequences : 0); }

int b200q_kv_reserve_dev(const b200q_kv_pool* pool, const int32_t* extra, int32_t* status, void* stream) {
  B200Q_TRY(kv_check_pool("kv_reserve", pool));
  if (!extra) return set_error(B200Q_ERR_INVALID, "kv_reserve: null extra");
  if (pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("kv_reserve", pool->table);
  B200Q_TRY(dev.rc);
  size_t bytes;
  B200Q_TRY(bitmap_bytes((const void*)reserve_kernel, pool->pages, &bytes));
  return launch_dependent(reserve_kernel, dim3(1), dim3(PLAN_THREADS), bytes, static_cast<cudaStream_t>(stream), *pool, extra, status);
}

int b200q_kv_free_dev(const b200q_kv_pool* pool, const int32_t* which, void* stream) {
  B200Q_TRY(kv_check_pool("kv_free", pool));
  if (!which) return set_error(B200Q_ERR_INVALID, "kv_free: null which");
  if (pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("kv_free", pool->table);
  B200Q_TRY(dev.rc);
  return launch_dependent(free_kernel, dim3(pool->sequences), dim3(128), 0, static_cast<cudaStream_t>(stream), *pool, which);
}

int b200q_kv_fork_dev(const b200q_kv_cache* cache, const b200q_kv_pool* pool, const int32_t* parent, int32_t* status, void* stream) {
  B200Q_TRY(kv_check_pool("kv_fork", pool));
  B200Q_TRY(kv_check_cache("kv_fork", cache));
  B200Q_TRY(check_scratch("kv_fork", pool));
  if (!parent) return set_error(B200Q_ERR_INVALID, "kv_fork: null parent");
  if ((int64_t)pool->page_size * cache->heads * (cache->head_dim / 8) > 0x7fffffffLL)
    return set_error(B200Q_ERR_UNSUPPORTED, "kv_fork: a page of one layer has more than 2^31 - 1 pieces of 16 bytes");
  if (pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("kv_fork", pool->table);
  B200Q_TRY(dev.rc);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  size_t bytes;
  B200Q_TRY(bitmap_bytes((const void*)fork_plan_kernel, pool->pages, &bytes));
  B200Q_TRY(launch_dependent(fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), bytes, s, *pool, parent, status));
  // 32 columns a tile where they fit, at least 8
  int columns = FORK_TILE / pool->sequences;
  columns = columns > 32 ? 32 : columns;
  const int tiles = ceil_div(pool->table_width, columns), table_blocks = tiles < sms ? tiles : sms;
  const int64_t copies = (int64_t)pool->sequences * 2 * cache->layers;
  const int copy_blocks = (int)(copies < 4 * sms ? copies : 4 * sms);
  return launch_dependent(fork_kernel, dim3(table_blocks + copy_blocks), dim3(FORK_THREADS), 0, s, *cache, *pool, parent, table_blocks, columns);
}

int b200q_kv_compact_dev(const b200q_kv_cache* cache, const b200q_kv_pool* pool, const int32_t* path, int64_t path_stride,
                         int32_t path_width, const int32_t* path_length, int32_t* length_out, void* stream) {
  B200Q_TRY(kv_check_pool("kv_compact", pool));
  B200Q_TRY(kv_check_cache("kv_compact", cache));
  if (!path || !path_length || !length_out) return set_error(B200Q_ERR_INVALID, "kv_compact: null argument");
  if (path_width < 0 || path_stride < path_width) return set_error(B200Q_ERR_INVALID, "kv_compact: bad shape of the paths");
  if (path_width > PATH_MOST) return set_error(B200Q_ERR_UNSUPPORTED, "kv_compact: a path has at most %d nodes", PATH_MOST);
  const bool in_place = length_out == pool->length;
  if (in_place) B200Q_TRY(check_scratch("kv_compact", pool));
  if (pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("kv_compact", pool->table);
  B200Q_TRY(dev.rc);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // (a block with nothing to move is gone in a microsecond: the grid only has to keep the memory busy)
  const int64_t items = (int64_t)pool->sequences * 2 * cache->layers;
  B200Q_TRY(launch_dependent(compact_kernel, dim3((unsigned)(items < 65536 ? items : 65536)), dim3(COMPACT_THREADS), 0, s, *cache, *pool, path,
                             path_stride, path_width, path_length, in_place ? pool->scratch : length_out));
  if (in_place) B200Q_TRY(launch_dependent(lengths_kernel, dim3(1), dim3(KV_MAX_SEQUENCES), 0, s, pool->scratch, pool->length, pool->sequences));
  return B200Q_OK;
}

}  // extern "C"
