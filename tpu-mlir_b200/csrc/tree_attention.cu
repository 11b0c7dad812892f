// Attention of drafted trees (chains, single tokens) over a paged key / value cache.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i k_j - max_j),  j over the committed positions of the row's sequence and
//   the drafted nodes that its mask names.
//
// One pass over keys and values with a running maximum and sum.  The heads that share a cache head are stacked: its rows are
// (node, head of the group), 16, 32 or 64 of them in a tile, so that a key is read once for all of them.  Work is counted in units of
// 64 positions of one (sequence, cache head, row tile); the units of the whole batch stand in one line and every block takes an
// equal run of them, so uneven contexts do not wait for each other and one long context fills the GPU.  Lengths stay on the
// device: each block adds up the batch's units for itself.  An item that a run's end cuts leaves fp32 partial sums in the workspace
// (at most two a block), which a second kernel joins, in the order of the positions.
//
// Loads run ahead of the products across items: a ring of stages of 64 keys and values, filled with 16-byte cp.async through
// the page table, whose entries are looked up one unit earlier.  Shared memory is swizzled by 16-byte pieces (piece ^ row % 8),
// so that ldmatrix meets no bank twice.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "kv_cache.h"
#include "ptx_sm100.cuh"

namespace b200q {
namespace {

constexpr int UNIT = 64;   // positions of a unit

struct AttnArgs {
  b200q_kv_cache cache;
  b200q_kv_pool pool;
  b200q_tree_attention io;
  int group;          // query heads of a cache head
  float scale_log2;   // scale * log2(e)
  int min_units;      // units that a block takes at least, if there are any
  float* partial;     // [blocks][2][rows of a tile][dim + 2]: sums, maximum (log2 domain), total
  struct SplitItem* items;   // [blocks]
};

// The item that starts in a block's run and ends in a later one's.
struct SplitItem {
  int parts;       // blocks that hold a part of it; 0: none
  int first_row;   // of its sequence
  int row0, rows;  // its tile's first (node, head of the group) and how many the sequence has
  int head;        // cache head
};

struct Sequence {
  int first_row, nodes, length, total;   // total: committed positions and nodes
};
__device__ __forceinline__ Sequence load_sequence(const AttnArgs& a, int s) {
  Sequence q;
  const int64_t b = a.io.row_start[s], e = a.io.row_start[s + 1];
  const int64_t end = e < a.io.rows ? e : a.io.rows;
  q.first_row = (int)b;
  q.nodes = b >= 0 && end > b ? (int)(end - b) : 0;
  q.length = kv_length(a.pool, s);
  const int64_t most = (int64_t)a.pool.table_width * a.pool.page_size, all = (int64_t)q.length + q.nodes;
  q.total = (int)(all < most ? all : most);
  return q;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;   // 0: the 16 bytes become zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool F16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// a 16-bit number that is infinite or NaN
template <bool F16>
__device__ __forceinline__ bool not_finite(uint32_t bits) {
  constexpr uint32_t E = F16 ? 0x7c00u : 0x7f80u;
  return (bits & E) == E;
}
template <bool F16>
__device__ __forceinline__ float from_bits(uint32_t bits) {
  return F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16);
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// Which of the 64 positions from `p0` on node `node` sees: all committed ones, and the nodes that its mask names (a chain: up to
// itself).  mask: the row's words.
__device__ __forceinline__ uint64_t sees(const AttnArgs& a, const uint32_t* mask, int node, int length, int p0) {
  const int base = p0 - length;   // node at the first position, negative: committed
  if (base <= -64) return ~0ull;
  if (!a.io.mask) return low_bits(node - base + 1);
  const int from = base > 0 ? base : 0;
  const int64_t w = from >> 5;
  const int sh = from & 31;
  const uint64_t w0 = w < a.io.mask_stride ? mask[w] : 0u, w1 = w + 1 < a.io.mask_stride ? mask[w + 1] : 0u,
                 w2 = w + 2 < a.io.mask_stride ? mask[w + 2] : 0u;
  uint64_t bits = (w0 | w1 << 32) >> sh;
  if (sh) bits |= w2 << (64 - sh);
  return base >= 0 ? bits : low_bits(-base) | bits << -base;
}

template <int DIM, int WR, int WC>
struct Shape {
  static constexpr int ROWS = 16 * WR, THREADS = 32 * WR * WC, STAGES = DIM > 128 ? 2 : 3, COLS = UNIT / WC;
  static constexpr int TILE = UNIT * DIM * 2;                         // bytes of a stage's keys, and of its values
  static constexpr int MERGE = WC > 1 ? ROWS * 64 * 4 + 2 * WC * ROWS * 4 : 0;
  static constexpr int FIXED = STAGES * 2 * TILE + MERGE;
  static size_t bytes(int sequences) { return FIXED + (size_t)sequences * (sizeof(long long) + sizeof(Sequence)); }
};

// DIM: head size that the registers and the tiles are laid out for (head_dim <= DIM; pieces past it stay zero).
// WR x WC warps: WR take 16 rows each, WC share a unit's positions.
template <bool F16, int DIM, int WR, int WC>
__global__ void __launch_bounds__(32 * WR * WC) tree_attention_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shape<DIM, WR, WC>;
  constexpr int STAGES = S::STAGES, THREADS = S::THREADS, NT = S::COLS / 8, PIECES = DIM / 8, SLOTS = STAGES + 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t offset[SLOTS][UNIT];        // element offset of a unit's rows in keys and values, -1: none
  __shared__ uint32_t there[SLOTS][2];           // which rows have one
  __shared__ long long scan_buf[33];
  __shared__ uint32_t bad[2];                    // rows of the unit whose values hold infinities or NaN
  float* merge = reinterpret_cast<float*>(smem + STAGES * 2 * S::TILE);
  float* merge_ml = merge + S::ROWS * 64;
  long long* sums = reinterpret_cast<long long*>(smem + S::FIXED);
  Sequence* seqs = reinterpret_cast<Sequence*>(sums + a.pool.sequences);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wr = warp / WC, wc = warp % WC;
  const int n = a.pool.sequences, dim = a.cache.head_dim, heads = a.cache.heads, group = a.group;
  ptx::griddep_launch_dependents();

  // ---- the batch's units, sequence by sequence
  const int each = (n + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int i = 0; i < each; ++i) {
    const int s = tid * each + i;
    if (s >= n) break;
    const Sequence q = load_sequence(a, s);
    const long long tiles = ((long long)q.nodes * group + S::ROWS - 1) / S::ROWS;
    mine += heads * tiles * ((q.total + UNIT - 1) / UNIT);
    seqs[s] = q;
    sums[s] = mine;
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) scan_buf[warp] = upto;
  if (tid < 2) bad[tid] = 0;
  // pieces past head_dim are never loaded: zero once
  for (int i = tid; i < STAGES * 2 * UNIT * PIECES; i += THREADS)
    if (i % PIECES >= dim / 8) {
      const int row = i / PIECES % UNIT, piece = i % PIECES;
      *reinterpret_cast<uint4*>(smem + (i / (PIECES * UNIT)) * S::TILE + row * DIM * 2 + ((piece ^ (row & 7)) * 16)) = make_uint4(0, 0, 0, 0);
    }
  __syncthreads();
  long long before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WR * WC; ++w) {
    if (w < warp) before += scan_buf[w];
    total += scan_buf[w];
  }
  for (int i = 0; i < each; ++i)
    if (tid * each + i < n) sums[tid * each + i] += before;
  __syncthreads();

  long long run = (total + gridDim.x - 1) / gridDim.x;
  if (run < a.min_units) run = a.min_units;
  const long long u0 = (long long)blockIdx.x * run, u1 = u0 + run < total ? u0 + run : total;
  if (tid == 0) a.items[blockIdx.x].parts = 0;
  if (u0 >= u1) return;

  // ---- where the loads are: unit `u` of the line
  struct Place {
    int s, head, tile, unit, tiles, units;   // row tile, unit of the item; how many there are
    int total, length, nodes, first_row;
  };
  auto enter = [&](Place& p, int s) {
    const Sequence q = seqs[s];
    p.s = s;
    p.tiles = (q.nodes * group + S::ROWS - 1) / S::ROWS;
    p.units = (q.total + UNIT - 1) / UNIT;
    p.total = q.total;
    p.length = q.length;
    p.nodes = q.nodes;
    p.first_row = q.first_row;
  };
  auto next_item = [&](Place& p) {   // row tiles of a head next to each other: they read the same keys
    p.unit = 0;
    if (++p.tile < p.tiles) return;
    p.tile = 0;
    if (++p.head < heads) return;
    p.head = 0;
    int s = p.s + 1;
    while (s < n && seqs[s].nodes == 0) ++s;
    if (s < n) enter(p, s);
  };
  Place load;
  {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] > u0) hi = mid;
      else lo = mid + 1;
    }
    enter(load, lo);
    const long long local = u0 - (lo ? sums[lo - 1] : 0), item = local / load.units;
    load.unit = (int)(local - item * load.units);
    load.head = (int)(item / load.tiles);
    load.tile = (int)(item - (long long)load.head * load.tiles);
  }
  Place at = load;
  const int count = (int)(u1 - u0);

  // the offset of row `tid` of the unit that `load` stands at, which then goes one further
  auto look_up = [&]() -> int64_t {
    int64_t off = -1;
    if (tid < UNIT) {
      const int pos = load.unit * UNIT + tid;
      if (pos < load.total) {
        off = kv_entry(a.cache, a.pool, load.s, pos);
        if (off >= 0) off += load.head * a.cache.head_stride;
      }
    }
    if (++load.unit == load.units) next_item(load);
    return off;
  };
  auto note = [&](int slot, int64_t off) {
    if (tid < UNIT) {
      offset[slot][tid] = off;
      const uint32_t m = __ballot_sync(0xffffffffu, off >= 0);
      if (lane == 0) there[slot][warp] = m;
    }
  };
  const uint16_t* kp = static_cast<const uint16_t*>(a.cache.k) + a.io.layer * a.cache.layer_stride;
  const uint16_t* vp = static_cast<const uint16_t*>(a.cache.v) + a.io.layer * a.cache.layer_stride;
  const uint32_t smem_base = ptx::smem_u32(smem);
  auto fetch = [&](int stage, int slot) {
    const int piece = tid % PIECES;
    if (piece < dim / 8) {
#pragma unroll
      for (int i = 0; i < UNIT * PIECES / THREADS; ++i) {
        const int row = tid / PIECES + i * (THREADS / PIECES);
        const int64_t off = offset[slot][row];
        const int64_t at16 = (off >= 0 ? off : 0) + piece * 8;
        const uint32_t dst = smem_base + stage * 2 * S::TILE + row * DIM * 2 + ((piece ^ (row & 7)) * 16);
        cp_async16(dst, kp + at16, off >= 0);
        cp_async16(dst + S::TILE, vp + at16, off >= 0);
      }
    }
  };

#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (i < count) note(i, look_up());
  __syncthreads();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < count) fetch(i, i);
    cp_async_commit();
  }

  // ---- registers: queries (A fragments), sums, running maximum (log2 domain) and total of rows lane / 4 and lane / 4 + 8
  uint32_t q[DIM / 16][4];
  float o[DIM / 8][4], m[2], l[2];
  const uint32_t* mask[2];
  int node[2];
  int started = at.unit;   // unit of the item that this block's part starts with
  int stage = 0, slot = 0;

  for (int i = 0; i < count; ++i) {
    if (i == 0 || at.unit == 0) {
      // a new item (or this block's part of one)
      started = at.unit;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = at.tile * S::ROWS + wr * 16 + lane / 4 + 8 * h;
        const bool real = r < at.nodes * group;
        const int t = r / group, row = at.first_row + (real ? t : 0);
        node[h] = t;
        mask[h] = a.io.mask ? a.io.mask + (int64_t)row * a.io.mask_stride : nullptr;
        m[h] = -INFINITY;
        l[h] = 0.f;
        const uint16_t* src = static_cast<const uint16_t*>(a.io.q) + (int64_t)row * a.io.q_row_stride + (at.head * group + r % group) * a.io.q_head_stride;
#pragma unroll
        for (int k = 0; k < DIM / 16; ++k) {
          const int d = k * 16 + (lane & 3) * 2;
          q[k][h] = real && d < dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          q[k][h + 2] = real && d + 8 < dim ? *reinterpret_cast<const uint32_t*>(src + d + 8) : 0u;
        }
      }
#pragma unroll
      for (int k = 0; k < DIM / 8; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][e] = 0.f;
    }

    cp_async_wait<STAGES - 2>();
    __syncthreads();   // unit i is here, and every warp is done with unit i - 1
    if (i + STAGES - 1 < count) fetch((stage + STAGES - 1) % STAGES, (slot + STAGES - 1) % SLOTS);
    cp_async_commit();
    int64_t ahead = -1;
    if (i + STAGES < count) ahead = look_up();

    // ---- scores of 16 rows x COLS positions
    const uint32_t ks = smem_base + stage * 2 * S::TILE, vs = ks + S::TILE;
    float sc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[t][e] = 0.f;
#pragma unroll
    for (int k = 0; k < DIM / 16; ++k) {
      if (k * 16 < dim) {
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
          uint32_t b[4];
          const int row = wc * S::COLS + t * 8 + (lane >> 4) * 8 + (lane & 7), piece = k * 2 + ((lane >> 3) & 1);
          ldmatrix4(b, ks + row * DIM * 2 + ((piece ^ (row & 7)) * 16));
          mma16816<F16>(sc[t], q[k], b[0], b[1]);
          mma16816<F16>(sc[t + 1], q[k], b[2], b[3]);
        }
      }
    }

    // ---- what is not seen
    const int p0 = at.unit * UNIT;
    const uint64_t in_pool = (uint64_t)there[slot][1] << 32 | there[slot][0];
    const bool drafted = p0 + UNIT > at.length;
    uint64_t see[2] = {~0ull, ~0ull};
    bool fix = false;
    if (drafted || in_pool != ~0ull) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        see[h] = in_pool & sees(a, mask[h], node[h], at.length, p0);
        const uint64_t mine64 = see[h] >> (wc * S::COLS + (lane & 3) * 2);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!(mine64 >> (t * 8 + e) & 1)) sc[t][2 * h + e] = -INFINITY;
      }
      if (drafted) {
        // Values of drafted nodes meet weights of zero in rows that do not see them: infinite or NaN ones are taken out of the
        // tile (and added below where they are seen), or they would make those rows NaN.
        int found = 0;
        for (int c = tid; c < UNIT * PIECES; c += THREADS) {
          const int row = c / PIECES, piece = c % PIECES;
          uint32_t* w = reinterpret_cast<uint32_t*>(smem + (vs - smem_base) + row * DIM * 2 + ((piece ^ (row & 7)) * 16));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = w[j];
            const bool lo = not_finite<F16>(x & 0xffffu), hi = not_finite<F16>(x >> 16);
            if (lo || hi) {
              found = 1;
              w[j] = (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
              atomicOr(&bad[row >> 5], 1u << (row & 31));
            }
          }
        }
        fix = __syncthreads_or(found);
      }
    }

    // ---- running maximum and sum
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; ++t) top = fmaxf(top, fmaxf(sc[t][2 * h], sc[t][2 * h + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float now = fmaxf(m[h], top * a.scale_log2), base = now == -INFINITY ? 0.f : now;
      alpha[h] = exp2_approx(m[h] - base);
      m[h] = now;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_approx(fmaf(sc[t][2 * h + e], a.scale_log2, -base));
          sc[t][2 * h + e] = p;
          sum += p;
        }
      l[h] = l[h] * alpha[h] + sum;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int k = 0; k < DIM / 8; ++k) {
        o[k][0] *= alpha[0];
        o[k][1] *= alpha[0];
        o[k][2] *= alpha[1];
        o[k][3] *= alpha[1];
      }
    }

    // ---- weights (rounded to the 16-bit type: the tensor cores take no wider pair; the rounding is unbiased and averages out
    // over positions) times values
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      const uint32_t p[4] = {pack_pair<F16>(sc[2 * j][0], sc[2 * j][1]), pack_pair<F16>(sc[2 * j][2], sc[2 * j][3]),
                             pack_pair<F16>(sc[2 * j + 1][0], sc[2 * j + 1][1]), pack_pair<F16>(sc[2 * j + 1][2], sc[2 * j + 1][3])};
#pragma unroll
      for (int k = 0; k < DIM / 16; ++k) {
        if (k * 16 < dim) {
          uint32_t b[4];
          const int row = wc * S::COLS + j * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), piece = k * 2 + (lane >> 4);
          ldmatrix4_t(b, vs + row * DIM * 2 + ((piece ^ (row & 7)) * 16));
          mma16816<F16>(o[2 * k], p, b[0], b[1]);
          mma16816<F16>(o[2 * k + 1], p, b[2], b[3]);
        }
      }
    }
    if (fix) {
      for (int c = 0; c < S::COLS; ++c) {
        const int row = wc * S::COLS + c;
        if (!(bad[row >> 5] >> (row & 31) & 1)) continue;
        float w[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (t * 8 + (lane & 3) * 2 + e == c) {
              w[0] = sc[t][e];
              w[1] = sc[t][2 + e];
            }
        const int from = (lane & ~3) | ((c & 7) >> 1);
        w[0] = __shfl_sync(0xffffffffu, w[0], from);
        w[1] = __shfl_sync(0xffffffffu, w[1], from);
        const int64_t off = offset[slot][row];
        if (off < 0) continue;
#pragma unroll
        for (int k = 0; k < DIM / 8; ++k) {
          const int d = k * 8 + (lane & 3) * 2;
          const uint32_t x = d < dim ? *reinterpret_cast<const uint32_t*>(vp + off + d) : 0u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t v = e ? x >> 16 : x & 0xffffu;
            if (not_finite<F16>(v)) {
              if (see[0] >> row & 1) o[k][e] += w[0] * from_bits<F16>(v);
              if (see[1] >> row & 1) o[k][2 + e] += w[1] * from_bits<F16>(v);
            }
          }
        }
      }
      __syncthreads();
      if (tid < 2) bad[tid] = 0;
    }
    if (i + STAGES < count) note((slot + STAGES) % SLOTS, ahead);
    stage = (stage + 1) % STAGES;
    slot = (slot + 1) % SLOTS;

    // ---- the end of the item, or of this block's part
    if (++at.unit == at.units || i + 1 == count) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      }
      if (WC > 1) {
        // the warps that shared the positions: a common maximum, then their sums one after the other, 64 columns at a time
        __syncthreads();   // (the buffer may still be read for the item before)
        if ((lane & 3) == 0)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = wr * 16 + lane / 4 + 8 * h;
            merge_ml[wc * S::ROWS + r] = m[h];
            merge_ml[(WC + wc) * S::ROWS + r] = l[h];
          }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = wr * 16 + lane / 4 + 8 * h;
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int w = 0; w < WC; ++w) top = fmaxf(top, merge_ml[w * S::ROWS + r]);
          const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int w = 0; w < WC; ++w) sum += merge_ml[(WC + w) * S::ROWS + r] * exp2_approx(merge_ml[w * S::ROWS + r] - base);
          const float f = exp2_approx(m[h] - base);
#pragma unroll
          for (int k = 0; k < DIM / 8; ++k) {
            o[k][2 * h] *= f;
            o[k][2 * h + 1] *= f;
          }
          m[h] = top;
          l[h] = sum;
        }
#pragma unroll
        for (int c = 0; c < DIM / 64; ++c) {
          float4* buf = reinterpret_cast<float4*>(merge) + wr * 8 * 32;
#pragma unroll
          for (int w = 0; w < WC; ++w) {
            if (wc == w) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                float(&x)[4] = o[c * 8 + k];
                if (w > 0) {
                  const float4 y = buf[k * 32 + lane];
                  x[0] += y.x;
                  x[1] += y.y;
                  x[2] += y.z;
                  x[3] += y.w;
                }
                if (w < WC - 1) buf[k * 32 + lane] = make_float4(x[0], x[1], x[2], x[3]);
              }
            }
            __syncthreads();
          }
        }
      }
      const bool whole = started == 0 && at.unit == at.units;
      if (wc == WC - 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int rt = wr * 16 + lane / 4 + 8 * h, r = at.tile * S::ROWS + rt;
          if (r >= at.nodes * group) continue;
          if (whole) {
            const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
            uint16_t* dst = static_cast<uint16_t*>(a.io.out) + (int64_t)(at.first_row + r / group) * a.io.out_row_stride +
                            (at.head * group + r % group) * a.io.out_head_stride;
#pragma unroll
            for (int k = 0; k < DIM / 8; ++k) {
              const int d = k * 8 + (lane & 3) * 2;
              if (d < dim) *reinterpret_cast<uint32_t*>(dst + d) = pack_pair<F16>(o[k][2 * h] * inv, o[k][2 * h + 1] * inv);
            }
          } else {
            float* dst = a.partial + ((int64_t)(blockIdx.x * 2 + (started == 0)) * S::ROWS + rt) * (DIM + 2);
#pragma unroll
            for (int k = 0; k < DIM / 8; ++k) *reinterpret_cast<float2*>(dst + k * 8 + (lane & 3) * 2) = make_float2(o[k][2 * h], o[k][2 * h + 1]);
            if ((lane & 3) == 0) *reinterpret_cast<float2*>(dst + DIM) = make_float2(m[h], l[h]);
          }
        }
      }
      if (tid == 0 && started == 0 && !whole) {
        // the item's first unit is unit u1 - at.unit of the line
        const long long last = u1 - at.unit + at.units - 1;
        a.items[blockIdx.x] = SplitItem{(int)(last / run) - (int)blockIdx.x + 1, at.first_row, at.tile * S::ROWS, at.nodes * group, at.head};
      }
      if (at.unit == at.units) next_item(at);
    }
  }
}

// Joins the parts of the items that were cut: block x looks after the item that starts in block x's run, a warp takes a row.
template <bool F16, int DIM>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ AttnArgs a, int tile_rows) {
  constexpr int PER = DIM / 32;
  ptx::griddep_wait();
  ptx::griddep_launch_dependents();
  const SplitItem it = a.items[blockIdx.x];
  const int rt = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, r = it.row0 + rt, dim = a.cache.head_dim;
  if (it.parts == 0 || r >= it.rows) return;
  // part 0 lies in its block's second place, the others in their blocks' first
  auto part = [&](int i) { return a.partial + ((int64_t)((blockIdx.x + i) * 2 + (i == 0)) * tile_rows + rt) * (DIM + 2); };
  float top = -INFINITY;
  for (int i = lane; i < it.parts; i += 32) top = fmaxf(top, part(i)[DIM]);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float base = top == -INFINITY ? 0.f : top;
  float acc[PER], sum = 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < it.parts; ++i) {
    const float* p = part(i);
    const float2 ml = *reinterpret_cast<const float2*>(p + DIM);
    const float w = exp2_approx(ml.x - base);
    sum += w * ml.y;
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
      const float2 x = *reinterpret_cast<const float2*>(p + e * 32 + lane * 2);
      acc[e] += w * x.x;
      acc[e + 1] += w * x.y;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* dst = static_cast<uint16_t*>(a.io.out) + (int64_t)(it.first_row + r / a.group) * a.io.out_row_stride +
                  (it.head * a.group + r % a.group) * a.io.out_head_stride;
#pragma unroll
  for (int e = 0; e < PER; e += 2) {
    const int d = e * 32 + lane * 2;
    if (d < dim) *reinterpret_cast<uint32_t*>(dst + d) = pack_pair<F16>(acc[e] * inv, acc[e + 1] * inv);
  }
}

constexpr int BLOCKS_PER_SM = 2, MAX_TILE_ROWS = 64;

// Layout of the workspace for `blocks` blocks.
int64_t workspace_bytes(int blocks, int dim) {
  const int64_t items = ((int64_t)blocks * sizeof(SplitItem) + 255) / 256 * 256;
  return items + (int64_t)blocks * 2 * MAX_TILE_ROWS * (dim + 2) * 4;
}
int padded_dim(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

template <bool F16, int DIM, int WR, int WC>
int launch(const AttnArgs& a, int sms, cudaStream_t s) {
  using S = Shape<DIM, WR, WC>;
  auto kernel = tree_attention_kernel<F16, DIM, WR, WC>;
  const size_t smem = S::bytes(a.pool.sequences);
  CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::bytes(KV_MAX_SEQUENCES)));
  const int blocks = sms * (DIM > 128 ? 1 : BLOCKS_PER_SM);
  kernel<<<blocks, S::THREADS, smem, s>>>(a);
  CUDA_TRY(cudaGetLastError());
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = launch_config(dim3(blocks, S::ROWS / 4), dim3(128), 0, s, &attr, true);
  CUDA_TRY(cudaLaunchKernelEx(&cfg, join_kernel<F16, DIM>, a, (int)S::ROWS));
  return B200Q_OK;
}

// Rows of a tile by the batch's average of (node, head of the group) a cache head, which the host knows.
template <bool F16, int DIM>
int launch_rows(const AttnArgs& a, int sms, cudaStream_t s) {
  const int64_t rows = (a.io.rows + a.pool.sequences - 1) / a.pool.sequences * a.group;
  if (rows <= 16) return launch<F16, DIM, 1, 4>(a, sms, s);
  if constexpr (DIM <= 128)
    if (rows > 32) return launch<F16, DIM, 4, 1>(a, sms, s);
  return launch<F16, DIM, 2, 2>(a, sms, s);
}

template <bool F16>
int launch_dim(const AttnArgs& a, int sms, cudaStream_t s) {
  switch (padded_dim(a.cache.head_dim)) {
    case 64: return launch_rows<F16, 64>(a, sms, s);
    case 128: return launch_rows<F16, 128>(a, sms, s);
    default: return launch_rows<F16, 256>(a, sms, s);
  }
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_tree_attention_workspace(const b200q_kv_cache* cache, int32_t q_heads, int64_t* bytes) {
  B200Q_TRY(kv_check_cache("tree_attention_workspace", cache));
  if (!bytes || q_heads < 1 || q_heads % cache->heads) return set_error(B200Q_ERR_INVALID, "tree_attention_workspace: bad argument");
  OnDeviceOf dev("tree_attention_workspace", cache->k);
  B200Q_TRY(dev.rc);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  *bytes = workspace_bytes(sms * BLOCKS_PER_SM, padded_dim(cache->head_dim));
  return B200Q_OK;
}

int b200q_tree_attention_dev(const b200q_kv_cache* cache, const b200q_kv_pool* pool, const b200q_tree_attention* args, void* stream) {
  B200Q_TRY(kv_check_cache("tree_attention", cache));
  B200Q_TRY(kv_check_pool("tree_attention", pool));
  if (!args) return set_error(B200Q_ERR_INVALID, "tree_attention: null args");
  const b200q_tree_attention& io = *args;
  if (!io.q || !io.out || !io.row_start || !io.workspace) return set_error(B200Q_ERR_INVALID, "tree_attention: null argument");
  if (io.rows < 0 || io.rows > 0x7fffffffLL || io.q_heads < 1 || io.q_heads % cache->heads)
    return set_error(B200Q_ERR_INVALID, "tree_attention: rows must fit 31 bits and q_heads be a multiple of the cache's heads");
  if (io.rows * (io.q_heads / cache->heads) > 0x7fffffffLL) return set_error(B200Q_ERR_UNSUPPORTED, "tree_attention: too many rows");
  if (io.layer < 0 || io.layer >= cache->layers) return set_error(B200Q_ERR_INVALID, "tree_attention: no layer %d in the cache", io.layer);
  if (!(io.scale > 0.f) || !isfinite(io.scale)) return set_error(B200Q_ERR_INVALID, "tree_attention: scale must be positive");
  if (((uintptr_t)io.q | (uintptr_t)io.out | (uintptr_t)io.workspace) & 15)
    return set_error(B200Q_ERR_INVALID, "tree_attention: q, out and workspace must be 16-byte aligned");
  if (((uintptr_t)io.row_start | (uintptr_t)io.mask) & 3)
    return set_error(B200Q_ERR_INVALID, "tree_attention: row_start and mask must be 4-byte aligned");
  if ((io.q_row_stride | io.q_head_stride | io.out_row_stride | io.out_head_stride) & 7)
    return set_error(B200Q_ERR_INVALID, "tree_attention: strides of q and out must be multiples of 8 elements");
  if (io.mask && io.mask_stride < 0) return set_error(B200Q_ERR_INVALID, "tree_attention: negative mask_stride");
  if (io.rows == 0 || pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("tree_attention", pool->table);
  B200Q_TRY(dev.rc);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  const int blocks = sms * BLOCKS_PER_SM;
  if (io.workspace_bytes < workspace_bytes(blocks, padded_dim(cache->head_dim)))
    return set_error(B200Q_ERR_INVALID, "tree_attention: the workspace is smaller than b200q_tree_attention_workspace says");
  AttnArgs a{};
  a.cache = *cache;
  a.pool = *pool;
  a.io = io;
  a.group = io.q_heads / cache->heads;
  a.scale_log2 = io.scale * 1.4426950408889634f;
  a.min_units = 2;
  a.items = static_cast<SplitItem*>(io.workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(io.workspace) + ((int64_t)blocks * sizeof(SplitItem) + 255) / 256 * 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == B200Q_DT_F16 ? launch_dim<true>(a, sms, s) : launch_dim<false>(a, sms, s);
}

}  // extern "C"
