// Attention of drafted trees (chains, single tokens) over a paged key / value cache.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i k_j - max_j),  j over the committed positions of the row's sequence and
//   the drafted nodes that its mask names.
//
// One pass over keys and values with a running maximum and sum.  The heads that share a cache head are stacked: its rows are
// (node, head of the group), 16 or 32 of them in a tile, so that a key is read once for all of them.  Work is counted in units of
// 64 positions of one (sequence, cache head, row tile); the units of the whole batch stand in one line and every block takes an
// equal run of them, so uneven contexts do not wait for each other and one long context fills the GPU.  Lengths stay on the
// device: each block adds up the batch's units for itself.  An item that a run's end cuts leaves fp32 partial sums in the workspace
// (at most two a block), which a second kernel joins, in the order of the positions.
//
// One warp of a block only loads, with TMA boxes of as many rows as both a page and a unit are made of: a lane looks a box's page
// up and issues its copy, ahead of the products and across items, into a ring of stages of 64 keys and values; four warps
// compute.  Shared memory holds 64 elements a row, swizzled by 16-byte pieces (piece ^ row % 8), so that ldmatrix meets no bank
// twice.  (Loading with 16-byte cp.async instead, one or two warps a block, took 640 instructions a warp and unit and held the
// computing warps up: 108 us where this takes %%%.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "igemm.h"
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
  int box;            // rows of a TMA box
  int min_run;        // the shortest run of the line that a block takes, if there is so much
  unsigned long long wait_ns;   // no wait inside the kernel lasts longer
  int expect_extra;             // test aid: bytes that a stage waits for and that never come (0 in normal use)
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

// a box of a page's rows: x byte of the head, y slot, z head, w page; what lies outside becomes zeros
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
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
// itself).
__device__ __forceinline__ uint64_t sees(const AttnArgs& a, int row, int node, int length, int p0) {
  const int base = p0 - length;   // node at the first position, negative: committed
  if (base <= -64) return ~0ull;
  if (!a.io.mask) return low_bits(node - base + 1);
  const uint32_t* mask = a.io.mask + (int64_t)row * a.io.mask_stride;
  const int from = base > 0 ? base : 0;
  const int64_t w = from >> 5;
  const int sh = from & 31;
  const uint64_t w0 = w < a.io.mask_stride ? mask[w] : 0u, w1 = w + 1 < a.io.mask_stride ? mask[w + 1] : 0u,
                 w2 = w + 2 < a.io.mask_stride ? mask[w + 2] : 0u;
  uint64_t bits = (w0 | w1 << 32) >> sh;
  if (sh) bits |= w2 << (64 - sh);
  return base >= 0 ? bits : low_bits(-base) | bits << -base;
}

// ---- the line of units: which unit stands at a position of it
struct Line {
  const Sequence* seqs;
  int sequences, heads, group, tile_rows;
};
// An item (sequence, cache head, row tile) takes ITEM_COST positions of the line and one for each unit: what a block spends on an
// item besides its units (queries, the sums' way out) counts when runs are made equal.
constexpr int ITEM_COST = 1;
struct Place {
  long long pos;                     // in the line
  int s, head, tile, unit;           // row tile of the sequence, unit of the item
  int tiles, units, total, length, nodes, first_row;
  __device__ __forceinline__ void enter(const Line& line, int seq) {
    const Sequence q = line.seqs[seq];
    s = seq;
    tiles = (int)(((long long)q.nodes * line.group + line.tile_rows - 1) / line.tile_rows);
    units = (q.total + UNIT - 1) / UNIT;
    total = q.total;
    length = q.length;
    nodes = q.nodes;
    first_row = q.first_row;
  }
  // the unit at `pos` or the first one after it; sums: the line's length up to and with each sequence
  __device__ __forceinline__ void find(const Line& line, const long long* sums, long long at) {
    int lo = 0, hi = line.sequences - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] > at) hi = mid;
      else lo = mid + 1;
    }
    enter(line, lo);
    const long long local = at - (lo ? sums[lo - 1] : 0), item = local / (units + ITEM_COST);
    const int in = (int)(local - item * (units + ITEM_COST)) - ITEM_COST;
    head = (int)(item / tiles);
    tile = (int)(item - (long long)head * tiles);
    unit = in > 0 ? in : 0;
    pos = at + (in < 0 ? -in : 0);
  }
  // row tiles of a head stand next to each other: they read the same keys
  __device__ __forceinline__ void next(const Line& line) {
    ++pos;
    if (++unit < units) return;
    unit = 0;
    pos += ITEM_COST;
    if (++tile < tiles) return;
    tile = 0;
    if (++head < line.heads) return;
    head = 0;
    int q = s + 1;
    while (q < line.sequences && line.seqs[q].nodes == 0) ++q;
    if (q < line.sequences) enter(line, q);
  }
};

// Fills seqs and sums (the line's length up to and with each sequence) for all threads of the block; returns the line's length.
template <int THREADS>
__device__ __forceinline__ long long lay_out(const AttnArgs& a, int tile_rows, Sequence* seqs, long long* sums, long long* buf) {
  const int n = a.pool.sequences, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (n + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int i = 0; i < each; ++i) {
    const int s = tid * each + i;
    if (s >= n) break;
    const Sequence q = load_sequence(a, s);
    const long long tiles = ((long long)q.nodes * a.group + tile_rows - 1) / tile_rows;
    mine += a.cache.heads * tiles * ((q.total + UNIT - 1) / UNIT + ITEM_COST);
    seqs[s] = q;
    sums[s] = mine;
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) buf[warp] = upto;
  __syncthreads();
  long long before = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += buf[w];
    total += buf[w];
  }
  for (int i = 0; i < each; ++i)
    if (tid * each + i < n) sums[tid * each + i] += before;
  __syncthreads();
  return total;
}

// ---- loading.  Layout of a tile: [64 elements of the head][row][128 bytes], 16-byte pieces swizzled by the row.
__device__ __forceinline__ uint32_t tile_at(int row, int piece) {
  return (piece >> 3) * (UNIT * 128) + row * 128 + (((piece & 7) ^ (row & 7)) * 16);
}
// The loading warp's life: every unit of the block's run into the ring.  A box is `box` rows (the greatest common divisor of a page's
// and a unit's, so no box is cut by either) of 64 elements.  there[stage]: rows that are positions of the sequence in a page of the pool
// (the others are zeros, or whatever a page holds past the sequence's end).
template <int DIM, int STAGES, typename Wait>
__device__ __forceinline__ void load_units(const AttnArgs& a, const CUtensorMap* km, const CUtensorMap* vm, const Line& line, Place at, long long end,
                                           uint8_t* ring, uint64_t* full_bar, uint64_t* empty_bar, uint64_t* there, Wait wait) {
  constexpr int TILE = UNIT * DIM * 2, PARTS = 2 * (DIM / 64);
  const int lane = threadIdx.x & 31, box = a.box, boxes = UNIT / box, page_size = a.pool.page_size;
  int stage = 0;
  uint32_t phase = 1, sent = 0;   // the first pass over the ring finds it empty
  // the place of box `lane` (and lane + 32) of the unit that `at` stands at: page (-1: none) and slot of its first row
  int page[2], slot[2], rows;
  auto look_up = [&]() {
    rows = at.total - at.unit * UNIT;   // may be more than a unit's
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int b = lane + 32 * j, pos = at.unit * UNIT + b * box;
      page[j] = -1;
      slot[j] = 0;
      if (b < boxes && pos < at.total) {
        page[j] = kv_page(a.pool, at.s, pos);
        slot[j] = (int)((unsigned)pos % (unsigned)page_size);
      }
    }
  };
  look_up();
  while (at.pos < end) {
    const int head = at.head, pg0 = page[0], pg1 = page[1], sl0 = slot[0], sl1 = slot[1], here = rows;
    at.next(line);
    if (at.pos < end) look_up();   // the next unit's entries are on their way while this one's boxes go out
    if (!wait(&empty_bar[stage], phase, 1)) break;
    ++sent;
    uint64_t in = 0;
    if (pg0 >= 0) in |= low_bits(box) << (lane * box);
    if (pg1 >= 0) in |= low_bits(box) << ((lane + 32) * box);
    in = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(in >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)in);
    const uint32_t bar = ptx::smem_u32(&full_bar[stage]), dst = ptx::smem_u32(ring) + stage * 2 * TILE;
    if (lane == 0) {
      there[stage] = in & low_bits(here);
      ptx::mbar_arrive_expect_tx(bar, 2 * TILE + a.expect_extra);
    }
    __syncwarp();
    // a copy a lane: box, then keys or values and which 64 elements
    for (int i = lane; i - lane < boxes * PARTS; i += 32) {
      const int b = i / PARTS, part = i % PARTS;
      const int p0 = __shfl_sync(0xffffffffu, pg0, b & 31), p1 = __shfl_sync(0xffffffffu, pg1, b & 31);
      const int s0 = __shfl_sync(0xffffffffu, sl0, b & 31), s1 = __shfl_sync(0xffffffffu, sl1, b & 31);
      if (b < boxes) {
        const int pg = b < 32 ? p0 : p1, sl = b < 32 ? s0 : s1, x = part >> 1;
        tma_load_4d(dst + (part & 1) * TILE + x * (UNIT * 128) + b * box * 128, part & 1 ? vm : km, bar, x * 128, sl, head, pg < 0 ? a.pool.pages : pg);
      }
    }
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (at.pos < end) {
    // given up: what is still on its way lands before the block is gone
    int flag = 0;
    for (uint32_t i = 0; i < STAGES; ++i)
      if (i < sent) ptx::mbar_wait_bounded(ptx::smem_u32(&full_bar[i]), ((sent - i - 1) / STAGES) & 1, &flag, 1, a.wait_ns);
  }
}

constexpr int COMPUTERS = 128, BLOCK = COMPUTERS + 32;

__device__ __forceinline__ void computers_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool computers_or(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, 1, 128, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(r)
      : "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

template <int DIM, int WR, int WC>
struct Shape {
  static constexpr int ROWS = 16 * WR, STAGES = DIM > 128 ? 2 : 3, COLS = UNIT / WC;
  static constexpr int TILE = UNIT * DIM * 2;                         // bytes of a stage's keys, and of its values
  static constexpr int MERGE = WC > 1 ? ROWS * 64 * 4 + 2 * WC * ROWS * 4 : 0;
  static constexpr int FIXED = STAGES * 2 * TILE + MERGE;
  static size_t bytes(int sequences) { return 1024 + FIXED + (size_t)sequences * (sizeof(long long) + sizeof(Sequence)); }
};

// DIM: head size that the registers and the tiles are laid out for (head_dim <= DIM; pieces past it stay zero).
// WR x WC computing warps: WR take 16 rows each, WC share a unit's positions.
template <bool F16, int DIM, int WR, int WC>
__global__ void __launch_bounds__(BLOCK, DIM > 128 ? 1 : 2)
tree_attention_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm, const __grid_constant__ AttnArgs a) {
  using S = Shape<DIM, WR, WC>;
  static_assert(WR * WC * 32 == COMPUTERS, "");
  constexpr int STAGES = S::STAGES, NT = S::COLS / 8, PIECES = DIM / 8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-ptx::smem_u32(smem_raw) & 1023);   // the swizzle goes by the address
  __shared__ uint64_t there[STAGES];             // which rows of a unit are positions with a page
  __shared__ long long scan_buf[BLOCK / 32];
  __shared__ uint32_t bad[2];                    // rows of the unit whose values hold infinities or NaN
  __shared__ alignas(8) uint64_t full_bar[STAGES], empty_bar[STAGES];
  __shared__ int abort_flag;
  float* merge = reinterpret_cast<float*>(smem + STAGES * 2 * S::TILE);
  float* merge_ml = merge + S::ROWS * 64;
  long long* sums = reinterpret_cast<long long*>(smem + S::FIXED);
  Sequence* seqs = reinterpret_cast<Sequence*>(sums + a.pool.sequences);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int dim = a.cache.head_dim, group = a.group;
  ptx::griddep_launch_dependents();

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full_bar[i]), 1);
      ptx::mbar_init(ptx::smem_u32(&empty_bar[i]), COMPUTERS / 32);
    }
    ptx::fence_barrier_init();
    abort_flag = 0;
    bad[0] = bad[1] = 0;
  }
  const long long total = lay_out<BLOCK>(a, S::ROWS, seqs, sums, scan_buf);
  const Line line{seqs, a.pool.sequences, a.cache.heads, group, S::ROWS};

  long long run = (total + gridDim.x - 1) / gridDim.x;
  if (run < a.min_run) run = a.min_run;
  const long long u0 = (long long)blockIdx.x * run, u1 = u0 + run < total ? u0 + run : total;
  if (tid == 0) a.items[blockIdx.x].parts = 0;
  if (u0 >= u1) return;
  Place at;
  at.find(line, sums, u0);
  const uint16_t* vp = static_cast<const uint16_t*>(a.cache.v) + a.io.layer * a.cache.layer_stride;
  const uint32_t smem_base = ptx::smem_u32(smem);
  // A wait that runs out (it cannot, short of a fault) ends all waiting: the roles go on without, so that no barrier is left short,
  // and the status says so.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
    if (!dead) dead = !ptx::mbar_wait_bounded(ptx::smem_u32(bar), parity, &abort_flag, where, a.wait_ns);
    return !dead;
  };

  if (warp >= COMPUTERS / 32) {
    // ---------------------------------------------------------------- loading
    load_units<DIM, STAGES>(a, &km, &vm, line, at, u1, smem, full_bar, empty_bar, there, wait);
    if (dead && lane == 0 && a.io.status) atomicMax(a.io.status, abort_flag);
    return;
  }

  // ------------------------------------------------------------------ computing
  const int wr = warp / WC, wc = warp % WC;
  // queries (A fragments), sums, running maximum (log2 domain) and total of rows lane / 4 and lane / 4 + 8
  uint32_t q[DIM / 16][4];
  float o[DIM / 8][4], m[2], l[2];
  int node[2];
  int started = 0;   // unit of the item that this block's part starts with
  bool fresh = true;
  int stage = 0;
  uint32_t phase = 0;

  while (at.pos < u1) {
    if (fresh) {
      // a new item (or this block's part of one)
      fresh = false;
      started = at.unit;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = at.tile * S::ROWS + wr * 16 + lane / 4 + 8 * h;
        const bool real = r < at.nodes * group;
        const int t = r / group, row = at.first_row + (real ? t : 0);
        node[h] = t;
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
    wait(&full_bar[stage], phase, 2);

    // ---- scores of 16 rows x COLS positions
    // (pieces 2k and 2k + 1 of a row: the swizzle makes the step from k to k + 1 an exclusive or of 32 bytes)
    const uint32_t ks = smem_base + stage * 2 * S::TILE, vs = ks + S::TILE;
    const uint32_t k_lane = ks + tile_at(wc * S::COLS + (lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
    const uint32_t v_lane = vs + tile_at(wc * S::COLS + ((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
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
          ldmatrix4(b, ((k_lane + t * 8 * 128) ^ ((k & 3) * 32)) + (k >> 2) * (UNIT * 128));
          mma16816<F16>(sc[t], q[k], b[0], b[1]);
          mma16816<F16>(sc[t + 1], q[k], b[2], b[3]);
        }
      }
    }

    // ---- what is not seen
    const int p0 = at.unit * UNIT;
    const uint64_t in_pool = there[stage];
    const bool drafted = p0 + UNIT > at.length;
    uint64_t see[2] = {~0ull, ~0ull};
    bool fix = false;
    if (drafted || in_pool != ~0ull) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        see[h] = in_pool & sees(a, at.first_row + (node[h] < at.nodes ? node[h] : 0), node[h], at.length, p0);
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
        bool found = false;
        for (int c = tid; c < UNIT * PIECES; c += COMPUTERS) {
          const int row = c / PIECES;
          uint32_t* w = reinterpret_cast<uint32_t*>(smem + (vs - smem_base) + tile_at(row, c % PIECES));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = w[j];
            const bool lo = not_finite<F16>(x & 0xffffu), hi = not_finite<F16>(x >> 16);
            if (lo || hi) {
              found = true;
              w[j] = (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
              atomicOr(&bad[row >> 5], 1u << (row & 31));
            }
          }
        }
        fix = computers_or(found);
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
          ldmatrix4_t(b, ((v_lane + j * 16 * 128) ^ ((k & 3) * 32)) + (k >> 2) * (UNIT * 128));
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
        const int64_t entry = kv_entry(a.cache, a.pool, at.s, p0 + row);
        if (entry < 0) continue;
        const uint16_t* value = vp + entry + at.head * a.cache.head_stride;
#pragma unroll
        for (int k = 0; k < DIM / 8; ++k) {
          const int d = k * 8 + (lane & 3) * 2;
          const uint32_t x = d < dim ? *reinterpret_cast<const uint32_t*>(value + d) : 0u;
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
      computers_sync();
      if (tid < 2) bad[tid] = 0;   // (before anyone looks for the next unit's: that ends in a barrier, and starts with one wait more)
      computers_sync();
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&empty_bar[stage]));
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }

    // ---- the end of the item, or of this block's part
    const bool done = at.unit + 1 == at.units;
    const long long first = at.pos - at.unit;   // where the item's units start in the line
    if (done || at.pos + 1 == u1) {
      fresh = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      }
      if (WC > 1) {
        // the warps that shared the positions: a common maximum, then their sums one after the other, 64 columns at a time
        computers_sync();   // (the buffer may still be read for the item before)
        if ((lane & 3) == 0)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = wr * 16 + lane / 4 + 8 * h;
            merge_ml[wc * S::ROWS + r] = m[h];
            merge_ml[(WC + wc) * S::ROWS + r] = l[h];
          }
        computers_sync();
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
            computers_sync();
          }
        }
      }
      const bool whole = started == 0 && done;
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
      if (tid == 0 && started == 0 && !whole)
        a.items[blockIdx.x] = SplitItem{(int)((first + at.units - 1) / run) - (int)blockIdx.x + 1, at.first_row, at.tile * S::ROWS, at.nodes * group, at.head};
    }
    at.next(line);
  }
  if (dead && lane == 0 && a.io.status) atomicMax(a.io.status, abort_flag);
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

// Keys or values of the layer as a TMA tensor [page][head][slot][bytes], boxes of `box` slots x 128 bytes.
int make_map(CUtensorMap* map, const AttnArgs& a, const void* base) {
  const uint64_t dims[4] = {(uint64_t)a.cache.head_dim * 2, (uint64_t)a.pool.page_size, (uint64_t)a.cache.heads, (uint64_t)a.pool.pages};
  const uint64_t strides[3] = {(uint64_t)a.cache.slot_stride * 2, (uint64_t)a.cache.head_stride * 2, (uint64_t)a.cache.page_stride * 2};
  const uint32_t box[4] = {128, (uint32_t)a.box, 1, 1};
  return make_tmap_u8(map, static_cast<const uint16_t*>(base) + a.io.layer * a.cache.layer_stride, 4, dims, strides, box);
}

template <bool F16, int DIM, int WR, int WC>
int launch(const AttnArgs& a, int sms, cudaStream_t s) {
  using S = Shape<DIM, WR, WC>;
  auto kernel = tree_attention_kernel<F16, DIM, WR, WC>;
  const size_t smem = S::bytes(a.pool.sequences);
  CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::bytes(KV_MAX_SEQUENCES)));
  const int blocks = sms * (DIM > 128 ? 1 : BLOCKS_PER_SM);
  CUtensorMap km, vm;
  B200Q_TRY(make_map(&km, a, a.cache.k));
  B200Q_TRY(make_map(&vm, a, a.cache.v));
  kernel<<<blocks, BLOCK, smem, s>>>(km, vm, a);
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
  a.box = UNIT;
  while (pool->page_size % a.box) a.box /= 2;   // the greatest power of two that divides a page, up to a unit
  igemm_wait_test(&a.expect_extra, &a.wait_ns);
  a.min_run = 2 + ITEM_COST;
  a.items = static_cast<SplitItem*>(io.workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(io.workspace) + ((int64_t)blocks * sizeof(SplitItem) + 255) / 256 * 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == B200Q_DT_F16 ? launch_dim<true>(a, sms, s) : launch_dim<false>(a, sms, s);
}

}  // extern "C"
