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

int kv_check_words(const char* who, std::initializer_list<const void*> words) {
  for (const void* p : words)
    if ((uintptr_t)p & 3) return set_error(B200Q_ERR_INVALID, "%s: an array of 32-bit numbers is not 4-byte aligned", who);
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

// The planning kernels are one block, compiled for two an SM (32 registers): it fits beside what the kernel before it still runs, and
// starts while that drains (at 60 registers the fork of 16 beams took 4 us more).
constexpr int PLAN_THREADS = 1024;

// Inclusive sum over the block's threads, one value each; every thread also gets the total.  buf: 32 of shared memory.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* buf, T* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  __syncthreads();   // buf may still be read from the scan before
  if (lane == 31) buf[warp] = v;
  __syncthreads();
  if (warp == 0) {
    T w = buf[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const T o = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += o;
    }
    buf[lane] = w;
  }
  __syncthreads();
  *total = buf[31];
  return v + (warp ? buf[warp - 1] : 0);
}

// Four pages' bits where sixteen bytes cannot be read at once.
__device__ __noinline__ uint32_t free_one_by_one(const int32_t* refcount, int at, int pages) {
  uint32_t w = 0;
#pragma unroll 1
  for (int e = 0; e < 4 && at + e < pages; ++e) w |= (uint32_t)(refcount[at + e] == 0) << e;
  return w;
}

// The `need` lowest free pages, in order: give(first, rank, page, mine) is called by whole warps, `mine` once for every rank below `need`;
// `first` is the rank of the warp's first free page.  Nothing is called and false returned when there are fewer.  All threads of a block of
// PLAN_THREADS call it; bitmap: a word for 32 pages.
//
// Free pages become bits (a lane looks at four counts, eight lanes' nibbles make a word), 16384 pages a step so that all loads of a
// step are in flight, and the steps end once enough are found.  Then, 1024 words a step, ranks are the sums of the bits before (a scan),
// and the words are dealt out to the warps one by one, a bit a lane: free pages stand together, and a warp that had a run of them to
// itself took 17 us for 5000.
template <typename Give>
__device__ bool lowest_free(const int32_t* refcount, int pages, long long need, uint32_t* bitmap, int* ranks, int* buf, Give give) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = PLAN_THREADS / 32;
  const bool wide = (reinterpret_cast<uintptr_t>(refcount) & 15) == 0;
  constexpr int PER_WARP = 512;                    // pages of a step that a warp looks at, 128 at a time
  int seen = 0, found = 0;                         // pages whose bits are set up; how many of them are free
  if (threadIdx.x == 0) ranks[0] = 0;
  __syncthreads();
  while (seen < pages && found < need) {
    const int first = seen + warp * PER_WARP + lane * 4;
    int4 c[PER_WARP / 128];
#pragma unroll
    for (int i = 0; i < PER_WARP / 128; ++i)
      c[i] = wide && first + i * 128 + 4 <= pages ? *reinterpret_cast<const int4*>(refcount + first + i * 128) : make_int4(1, 1, 1, 1);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER_WARP / 128; ++i) {
      const int at = first + i * 128;
      uint32_t w = (uint32_t)(c[i].x == 0) | (uint32_t)(c[i].y == 0) << 1 | (uint32_t)(c[i].z == 0) << 2 | (uint32_t)(c[i].w == 0) << 3;
      if (at < pages && !(wide && at + 4 <= pages)) w = free_one_by_one(refcount, at, pages);
      w <<= 4 * (lane & 7);
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      if ((lane & 7) == 0 && at < pages) {
        bitmap[at >> 5] = w;
        mine += __popc(w);
      }
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0 && mine) atomicAdd(&ranks[0], mine);
    __syncthreads();
    found = ranks[0];
    __syncthreads();   // (before the next step adds to it)
    seen = seen + warps * PER_WARP < pages ? seen + warps * PER_WARP : pages;
  }
  if (found < need) return false;
  const int words = (seen + 31) >> 5;
  long long before = 0;
  for (int w0 = 0; w0 < words && before < need; w0 += PLAN_THREADS) {
    const int mine = w0 + (int)threadIdx.x < words ? __popc(bitmap[w0 + threadIdx.x]) : 0;
    int total;
    const int upto = block_scan(mine, buf, &total);
    ranks[threadIdx.x] = upto - mine;
    __syncthreads();
#pragma unroll 1
    for (int k = warp; k < PLAN_THREADS && w0 + k < words && before + ranks[k] < need; k += warps) {
      const uint32_t bits = bitmap[w0 + k];
      const long long first = before + ranks[k], r = first + __popc(bits & ((1u << lane) - 1u));
      give(first, r, (w0 + k) * 32 + lane, (bits >> lane & 1u) && r < need);
    }
    before += total;
  }
  return true;
}

// The first of PLAN_THREADS ascending sums that is above `rank`, found by a warp: which 32 of them, then which of those.
__device__ __forceinline__ int owner(const long long* sums, long long rank) {
  const int lane = threadIdx.x & 31;
  const int group = __popc(__ballot_sync(0xffffffffu, sums[lane * 32 + 31] <= rank));
  return group * 32 + __popc(__ballot_sync(0xffffffffu, sums[(group & 31) * 32 + lane] <= rank));
}

__global__ void __launch_bounds__(PLAN_THREADS, 2) reserve_kernel(b200q_kv_pool pool, const int32_t* __restrict__ extra, int32_t* status) {
  extern __shared__ uint32_t bitmap[];
  __shared__ long long wide_buf[32], sums[KV_MAX_SEQUENCES];
  __shared__ int base[KV_MAX_SEQUENCES], ranks[PLAN_THREADS], buf[32];
  const int s = threadIdx.x;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  long long need = 0;
  int held = 0, narrow = 0;
  if (s < pool.sequences && extra[s] >= 0) {
    const int n = pool.length[s];
    held = kv_held(pool, s);
    const long long want = ((long long)(n < 0 ? 0 : n) + extra[s] + pool.page_size - 1) / pool.page_size;
    need = want > held ? want - held : 0;
    narrow = want > pool.table_width;
  }
  long long total;
  const long long upto = block_scan(need, wide_buf, &total);
  sums[s] = upto;
  base[s] = held - (int)(upto - need);   // column of rank r: base + r
  if (__syncthreads_or(narrow)) {
    if (s == 0 && status) *status = 2;
    return;
  }
  if (total == 0) return;
  const bool ok = lowest_free(pool.refcount, pool.pages, total, bitmap, ranks, buf, [&](long long first, long long r, int page, bool mine) {
    int t = owner(sums, first);
    if (!mine) return;
    while (sums[t] <= r) ++t;
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
  const int n = kv_held(pool, s);
  int32_t* row = pool.table + s * pool.table_stride;
  for (unsigned j = threadIdx.x; j < (unsigned)n; j += blockDim.x) {   // (n may be 2^31 - 1)
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

__global__ void __launch_bounds__(PLAN_THREADS, 2) fork_plan_kernel(b200q_kv_pool pool, const int32_t* __restrict__ parent, int32_t* status) {
  extern __shared__ uint32_t bitmap[];
  __shared__ int buf[32], list[KV_MAX_SEQUENCES], lengths[KV_MAX_SEQUENCES], ranks[PLAN_THREADS];
  const int s = threadIdx.x, n = pool.sequences;
  const ForkScratch f = fork_scratch(pool.scratch, n);
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  // (positions without pages are not passed on)
  if (s < n) lengths[s] = (int)min((int64_t)kv_length(pool, s), (int64_t)kv_held(pool, s) * pool.page_size);
  __syncthreads();
  const int p = s < n ? parent[s] : -1;
  const bool child = p >= 0 && p < n && p != s;
  // a ragged last page that is none of the pool's is passed on as it is: positions without a page
  const int count = child ? lengths[p] : 0, source = count % pool.page_size ? kv_page(pool, p, count) : -1, ragged = source >= 0;
  int total;
  const int rank = block_scan(ragged, buf, &total) - ragged;
  if (ragged) list[rank] = s;
  if (s < n) {
    f.length[s] = lengths[s];
    f.held[s] = pool.held[s];
    f.page[s] = -1;
    f.source[s] = source;
  }
  if (s == 0) {
    *f.ragged = total;
    *f.go = 1;
  }
  __syncthreads();
  if (s < total) f.list[s] = list[s];
  const bool ok = total == 0 || lowest_free(pool.refcount, pool.pages, total, bitmap, ranks, buf, [&](long long, long long r, int page, bool mine) {
    if (mine) f.page[list[r]] = page;
  });
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

constexpr int FORK_THREADS = 256, FORK_AT_ONCE = 4, FORK_PER_SM = 4;
constexpr int FORK_TILE = 2048;   // table entries of a tile: at least 2 columns of 1024 sequences

// Blocks below `table_blocks` take the tables, a run of columns each: all sequences' entries of these columns are read before the
// first is written, so children may be parents.  The other blocks copy ragged pages, a (child, layer, keys or values) at a time.
__global__ void __launch_bounds__(FORK_THREADS, FORK_PER_SM)
fork_kernel(b200q_kv_cache cache, b200q_kv_pool pool, const int32_t* __restrict__ parent, int table_blocks, int columns) {
  __shared__ int32_t old[FORK_TILE];
  const int n = pool.sequences;
  const ForkScratch f = fork_scratch(pool.scratch, n);
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if (*f.go == 0) return;
  if ((int)blockIdx.x < table_blocks) {
    // (64 bits: a row of the table may have 2^31 - 1 entries)
    for (int64_t c0 = (int64_t)blockIdx.x * columns; c0 < pool.table_width; c0 += table_blocks * columns) {
      for (int i = threadIdx.x; i < n * columns; i += FORK_THREADS) {
        const int s = i / columns;
        const int64_t c = c0 + i % columns;
        old[i] = c < pool.table_width ? pool.table[s * pool.table_stride + c] : -1;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < n * columns; i += FORK_THREADS) {
        const int s = i / columns, p = parent[s];
        const int64_t c = c0 + i % columns;
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
    const int slots = f.length[parent[s]] % pool.page_size;
    uint16_t* base = static_cast<uint16_t*>(part & 1 ? cache.v : cache.k) + (part >> 1) * cache.layer_stride;
    const int inner = slots_outside ? cache.heads : slots, count = slots * cache.heads * chunks;
    const uint16_t* src = base + from * cache.page_stride;
    uint16_t* dst = base + to * cache.page_stride;
    for (int i0 = threadIdx.x; i0 < count; i0 += FORK_AT_ONCE * FORK_THREADS) {
      uint4 v[FORK_AT_ONCE];
      int64_t at[FORK_AT_ONCE];
#pragma unroll
      for (int j = 0; j < FORK_AT_ONCE; ++j) {
        const int i = i0 + j * FORK_THREADS, row = i / chunks, x = row / inner, y = row - x * inner;
        at[j] = (slots_outside ? x * cache.slot_stride + y * cache.head_stride : y * cache.slot_stride + x * cache.head_stride) + (i - row * chunks) * 8;
        if (i < count) v[j] = *reinterpret_cast<const uint4*>(src + at[j]);
      }
#pragma unroll
      for (int j = 0; j < FORK_AT_ONCE; ++j)
        if (i0 + j * FORK_THREADS < count) *reinterpret_cast<uint4*>(dst + at[j]) = v[j];
    }
  }
}

// ---- compact.  A block takes some (layer, keys or values) of a sequence, whose places it looks up once; a thread takes 16 bytes of a head
// and walks along the path.
// Entry i is moved to place i <= path[i], and no later source lies at or before place i (the path ascends), so loads may run ahead of
// stores but not the other way: eight loads, then their stores.
constexpr int COMPACT_THREADS = 128, PATH_MOST = 1024, COMPACT_AHEAD = 8;

__global__ void __launch_bounds__(COMPACT_THREADS)
compact_kernel(b200q_kv_cache cache, b200q_kv_pool pool, const int32_t* __restrict__ path, int64_t path_stride, int path_width,
               const int32_t* __restrict__ path_length, int32_t* __restrict__ length_out, int parts_each) {
  __shared__ int64_t from[PATH_MOST], to[PATH_MOST];
  __shared__ int good;
  const int parts = 2 * cache.layers, chunks = cache.head_dim / 8;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int blocks_each = (parts + parts_each - 1) / parts_each, s = blockIdx.x / blocks_each, part0 = blockIdx.x % blocks_each * parts_each;
  const int length = pool.length[s];
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
  if (part0 == 0 && threadIdx.x == 0) length_out[s] = length + n;
  for (int part = part0; part < part0 + parts_each && part < parts; ++part) {
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

// Shared memory of a bitmap of this pool's pages, within the kernel's raised limit.
int bitmap_bytes(const void* kernel, int pages, size_t* bytes) {
  *bytes = ((size_t)pages + 31) / 32 * 4;
  CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, KV_MAX_PAGES / 8));
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
  B200Q_TRY(kv_check_words("kv_reserve", {extra, status}));
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
  B200Q_TRY(kv_check_words("kv_free", {which}));
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
  B200Q_TRY(kv_check_words("kv_fork", {parent, status}));
  if ((int64_t)pool->page_size * cache->heads * (cache->head_dim / 8) > 1 << 30)
    return set_error(B200Q_ERR_UNSUPPORTED, "kv_fork: a page of one layer has more than 2^30 pieces of 16 bytes");
  if (pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("kv_fork", pool->table);
  B200Q_TRY(dev.rc);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  size_t bytes;
  B200Q_TRY(bitmap_bytes((const void*)fork_plan_kernel, pool->pages, &bytes));
  B200Q_TRY(launch_dependent(fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), bytes, s, *pool, parent, status));
  // 32 columns a tile where they fit, at least 2
  int columns = FORK_TILE / pool->sequences;
  columns = columns > 32 ? 32 : columns;
  const int64_t tiles = ((int64_t)pool->table_width + columns - 1) / columns;
  const int table_blocks = (int)(tiles < sms ? tiles : sms);
  const int64_t copies = (int64_t)pool->sequences * 2 * cache->layers;
  const int copy_blocks = (int)(copies < FORK_PER_SM * sms ? copies : FORK_PER_SM * sms);
  return launch_dependent(fork_kernel, dim3(table_blocks + copy_blocks), dim3(FORK_THREADS), 0, s, *cache, *pool, parent, table_blocks, columns);
}

int b200q_kv_compact_dev(const b200q_kv_cache* cache, const b200q_kv_pool* pool, const int32_t* path, int64_t path_stride,
                         int32_t path_width, const int32_t* path_length, int32_t* length_out, void* stream) {
  B200Q_TRY(kv_check_pool("kv_compact", pool));
  B200Q_TRY(kv_check_cache("kv_compact", cache));
  if (!path || !path_length || !length_out) return set_error(B200Q_ERR_INVALID, "kv_compact: null argument");
  B200Q_TRY(kv_check_words("kv_compact", {path, path_length, length_out}));
  if (path_width < 0 || path_stride < path_width) return set_error(B200Q_ERR_INVALID, "kv_compact: bad shape of the paths");
  if (path_width > PATH_MOST) return set_error(B200Q_ERR_UNSUPPORTED, "kv_compact: a path has at most %d nodes", PATH_MOST);
  const bool in_place = length_out == pool->length;
  if (in_place) B200Q_TRY(check_scratch("kv_compact", pool));
  if (pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("kv_compact", pool->table);
  B200Q_TRY(dev.rc);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  // Parts of a block: as few as keep the grid within 16 blocks an SM.  (Nine are resident at once, by 50 registers a thread; 13 by the 16 KB of
  // places.  64 paths in 32 layers, 61 MB: 15.0 us, 15.2 with nine, 18.0 with five, 15.7 with a part a block: the short second wave of 16 costs no
  // more than longer blocks in one.)
  const int parts = 2 * cache->layers;
  const int64_t items = (int64_t)pool->sequences * parts;
  const int parts_each = (int)((items + 16 * sms - 1) / (16 * sms)), each = parts_each < parts ? parts_each : parts;
  B200Q_TRY(launch_dependent(compact_kernel, dim3((unsigned)(pool->sequences * ((parts + each - 1) / each))), dim3(COMPACT_THREADS), 0, s, *cache, *pool,
                             path, path_stride, path_width, path_length, in_place ? pool->scratch : length_out, each));
  if (in_place) B200Q_TRY(launch_dependent(lengths_kernel, dim3(1), dim3(KV_MAX_SEQUENCES), 0, s, pool->scratch, pool->length, pool->sequences));
  return B200Q_OK;
}

}  // extern "C"
