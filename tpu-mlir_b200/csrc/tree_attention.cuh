// What the two kernels of the attention over the paged cache share: the line of units and its runs, masks, the loading warp.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv_cache.h"
#include "ptx_sm100.cuh"

namespace b200q {
namespace attn {

constexpr int UNIT = 64;   // positions of a unit

struct AttnArgs {
  b200q_kv_cache cache;
  b200q_kv_pool pool;
  b200q_tree_attention io;
  int group;          // query heads of a cache head
  float scale_log2;   // scale * log2(e)
  int box;            // rows of a TMA box
  unsigned long long wait_ns;   // no wait inside the kernel lasts longer
  int expect_extra;             // test aid: bytes that a stage waits for and that never come (0 in normal use)
  // partial sums: [block][2][dim / 4 + 1][rows of a tile][4]; the last four of a row are its maximum (log2 domain) and its total.
  // (Four columns of all rows next to each other: the writers' threads are rows.)
  float* partial;
  struct SplitItem* items;   // [blocks]
};

// floats of a part, and where four columns of a row stand in it
constexpr __host__ __device__ int64_t part_size(int tile_rows, int dim) { return (int64_t)tile_rows * (dim + 4); }
__device__ __forceinline__ int part_at(int tile_rows, int row, int four) { return (four * tile_rows + row) * 4; }

// The item that starts in a block's run and ends in a later one's.
struct SplitItem {
  int parts;       // blocks that hold a part of it; 0: none
  int first_row;   // of its sequence
  int row0, rows;  // its tile's first (node, head of the group) and how many the sequence has
  int head;        // cache head
};

struct Sequence {
  int first_row, nodes, length, total;   // total: committed positions and nodes, as far as pages are held
};
// (rows without a single page still have a unit, in which they see nothing)
__device__ __forceinline__ int units_of(int total) { return total > 0 ? (int)(((unsigned)total + UNIT - 1) / UNIT) : 1; }
__device__ __forceinline__ Sequence load_sequence(const AttnArgs& a, int s) {
  Sequence q;
  const int64_t b = a.io.row_start[s], e = a.io.row_start[s + 1];
  const int64_t end = e < a.io.rows ? e : a.io.rows;
  q.first_row = (int)b;
  q.nodes = b >= 0 && end > b ? (int)(end - b) : 0;
  q.length = kv_length(a.pool, s);
  const int64_t held = (int64_t)kv_held(a.pool, s) * a.pool.page_size, all = (int64_t)q.length + q.nodes;
  q.total = (int)(all < held ? all : held);
  return q;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  const int n = there ? 16 : 0;   // 0: the 16 bytes become zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// A box of a page's rows: x byte of the head, y slot, z head, w page; what lies outside becomes zeros.  Called by a whole warp with
// the same arguments, issued by one elected thread (a copy from a branch, or one a lane, took 100 clocks each).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "{\n\t"
      ".reg .pred one;\n\t"
      "elect.sync _|one, 0xffffffff;\n\t"
      "@one cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n\t"
      "}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
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
// Weights are 2^lift times what the formula says (sums alike, so the quotient is the formula's): the smallest half precision number is
// 2^-24, and a long context's many weights below half of that beside one large weight would all be rounded to nothing.  They are at most
// 1, or 2^8 where sums are rescaled late, so 2^7 stays below 65504.  bfloat16 reaches 2^-133.
template <bool F16>
__device__ __forceinline__ constexpr float lift() {
  return F16 ? 7.f : 0.f;
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
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
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
// GROWS: for long chains (prompts).  Nodes of a chain do not see later ones, so its row tiles end at their own last node, rounded up to
// what makes the line's sums a formula: the units of the committed positions, then `grow` for every tile, up to the sequence's end.
// (A prompt of 4096 nodes, 32 heads on 8, 164 us instead of 493, eight of 1000 138 instead of 290.  Short items would lose 1 us of 10 to the
// formula, so only calls of long chains have it.)
template <bool GROWS>
struct Line {
  const Sequence* seqs;
  int sequences, heads, group, tile_rows, cost;
  __device__ __forceinline__ int grow() const { return ((tile_rows + group - 1) / group + UNIT - 1) / UNIT; }
  __device__ __forceinline__ int tile_units(int all, int length, int tile) const {
    if (!GROWS) return all;
    const int n = (int)(((unsigned)length + UNIT - 1) / UNIT) + (tile + 1) * grow();
    return n < all ? n : all;
  }
  // positions of a head's first `tiles` row tiles; all: units of the sequence
  __device__ __forceinline__ long long before_tile(int all, int length, int tiles) const {
    if (!GROWS) return (long long)tiles * (all + cost);
    const int base = (int)(((unsigned)length + UNIT - 1) / UNIT), room = all > base ? (all - base) / grow() : 0;
    const long long growing = room < tiles ? room : tiles;   // tiles that end at their last node
    return (long long)tiles * cost + growing * base + growing * (growing + 1) / 2 * grow() + (tiles - growing) * all;
  }
};
// An item (sequence, cache head, row tile) takes line.cost positions and one for each unit: what a block spends on an item besides
// its units (queries, the first scores, the sums' way out) counts when runs are made equal.
template <bool GROWS>
struct Place {
  using Line = attn::Line<GROWS>;
  long long pos;                     // in the line
  int s, head, tile, unit;           // row tile of the sequence, unit of the item
  int tiles, units, total, length, nodes, first_row;
  __device__ __forceinline__ void enter(const Line& line, int seq) {
    const Sequence q = line.seqs[seq];
    s = seq;
    tiles = (int)(((long long)q.nodes * line.group + line.tile_rows - 1) / line.tile_rows);
    units = units_of(q.total);
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
    const long long local = at - (lo ? sums[lo - 1] : 0);
    // (a 64-bit division takes hundreds of clocks)
    if (GROWS) {
      const long long all = line.before_tile(units, length, tiles);
      head = (int)(local <= 0x7fffffff && all <= 0x7fffffff ? (unsigned)local / (unsigned)all : local / all);
      const long long rest = local - head * all;
      int above = tiles;   // before_tile(tile) <= rest < before_tile(above)
      tile = 0;
      while (above - tile > 1) {
        const int mid = (int)(((unsigned)tile + (unsigned)above) / 2);
        if (line.before_tile(units, length, mid) <= rest) tile = mid;
        else above = mid;
      }
      const int in = (int)(rest - line.before_tile(units, length, tile)) - line.cost;
      units = line.tile_units(units, length, tile);
      unit = in > 0 ? in : 0;
      pos = at + (in < 0 ? -in : 0);
      return;
    }
    const int stretch = units + line.cost;   // of an item
    const long long item = local <= 0x7fffffff ? (unsigned)local / (unsigned)stretch : local / stretch;
    const int in = (int)(local - item * stretch) - line.cost;
    head = (int)(item <= 0x7fffffff ? (unsigned)item / (unsigned)tiles : item / tiles);
    tile = (int)(item - (long long)head * tiles);
    unit = in > 0 ? in : 0;
    pos = at + (in < 0 ? -in : 0);
  }
  __device__ __forceinline__ void next(const Line& line) { skip(line, 1); }
  // past `count` units of the item, no more than it has left.  Row tiles of a head stand next to each other: they read the same keys
  __device__ __forceinline__ void skip(const Line& line, int count) {
    pos += count;
    if ((unit += count) < units) return;
    unit = 0;
    pos += line.cost;
    if (++tile < tiles) {
      if (GROWS) units = line.tile_units(units_of(total), length, tile);
      return;
    }
    tile = 0;
    if (++head < line.heads) {
      if (GROWS) units = line.tile_units(units_of(total), length, 0);
      return;
    }
    head = 0;
    int q = s + 1;
    while (q < line.sequences && line.seqs[q].nodes == 0) ++q;
    if (q < line.sequences) enter(line, q);
    if (GROWS) units = line.tile_units(units, length, 0);
  }
  // The first position that some row of the item may not see: what lies before needs no mask.
  __device__ __forceinline__ int unseen(const Line& line) const {
    if (!GROWS) return min(length, total);
    const int64_t n = length + (int64_t)((unsigned)(tile * line.tile_rows) / (unsigned)line.group) + 1;
    return (int)(n < total ? n : total);
  }
};

// Fills seqs and sums (the line's length up to and with each sequence) for all threads of the block; returns the line's length.
template <int THREADS, bool GROWS>
__device__ __forceinline__ long long lay_out(const AttnArgs& a, int tile_rows, int cost, Sequence* seqs, long long* sums, long long* buf) {
  const int n = a.pool.sequences, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (n + THREADS - 1) / THREADS;
  long long mine = 0;
  for (int i = 0; i < each; ++i) {
    const int s = tid * each + i;
    if (s >= n) break;
    const Sequence q = load_sequence(a, s);
    const long long tiles = ((long long)q.nodes * a.group + tile_rows - 1) / tile_rows;
    if (GROWS) mine += a.cache.heads * Line<true>{nullptr, n, a.cache.heads, a.group, tile_rows, cost}.before_tile(units_of(q.total), q.length, (int)tiles);
    else mine += a.cache.heads * tiles * (units_of(q.total) + cost);
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

// Positions of a block's run.  Short ones too: a short batch's units one after the other in a few blocks take longer than the join of many
// parts (measured together: one token at 430 positions 9.8 us with a unit a block, 11.2 with four; seven at 1000 14.9 and 17.4).
__device__ __forceinline__ long long run_of(long long total) {
  // (a 64-bit division takes hundreds of clocks)
  const long long all = total + gridDim.x - 1;
  return all <= 0x7fffffff ? (unsigned)all / gridDim.x : all / gridDim.x;
}

// ---- loading.  Layout of a tile: [64 elements of the head][row][128 bytes], 16-byte pieces swizzled by the row.
__device__ __forceinline__ uint32_t tile_at(int row, int piece) {
  return (piece >> 3) * (UNIT * 128) + row * 128 + (((piece & 7) ^ (row & 7)) * 16);
}
// Takes infinite and NaN numbers out of the rows from `from` on of a tile of values, `count` threads of which this is number `me`; marks
// their rows in `bad` (a word for 32) and says whether there were any.
template <bool F16, int PIECES>
__device__ __forceinline__ bool clean_values(uint8_t* tile, int from, int me, int count, uint32_t* bad) {
  constexpr uint32_t E = F16 ? 0x7c007c00u : 0x7f807f80u;
  bool found = false;
#pragma unroll 4
  for (int c = from * PIECES + me; c < UNIT * PIECES; c += count) {
    uint4* at = reinterpret_cast<uint4*>(tile + tile_at(c / PIECES, c % PIECES));
    uint4 x = *at;
    const uint4 m = make_uint4(__vcmpeq2(x.x & E, E), __vcmpeq2(x.y & E, E), __vcmpeq2(x.z & E, E), __vcmpeq2(x.w & E, E));
    if (m.x | m.y | m.z | m.w) {
      found = true;
      *at = make_uint4(x.x & ~m.x, x.y & ~m.y, x.z & ~m.z, x.w & ~m.w);
      atomicOr(&bad[c / PIECES >> 5], 1u << (c / PIECES & 31));
    }
  }
  return found;
}
constexpr int LOADERS = 2;   // warps: one for keys, one for values
template <int STAGES>
struct Ring {
  static constexpr int NOTES = 16;   // units whose `there` is kept: more than any role is behind the loads
  uint64_t full[STAGES], empty[STAGES];
  // which rows of a unit are positions of the sequence in a page of the pool (the others are zeros, or whatever a page holds past the
  // sequence's end)
  uint64_t there[NOTES];
  static_assert(STAGES + 4 < NOTES, "");
  __device__ __forceinline__ void init(int readers) {
    for (int i = 0; i < STAGES; ++i) {
      ptx::mbar_init(ptx::smem_u32(&full[i]), LOADERS);
      ptx::mbar_init(ptx::smem_u32(&empty[i]), readers);
    }
  }
};
// a place in a ring, and the parity of the phase that is waited for there
template <int N>
struct Slot {
  int i = 0;
  uint32_t phase;
  __device__ __forceinline__ explicit Slot(uint32_t p) : phase(p) {}
  __device__ __forceinline__ void next() {
    if (++i == N) {
      i = 0;
      phase ^= 1;
    }
  }
};

// A warp's wait for a barrier; false once any wait of the block has run out (dead: this warp's memory of that).  The first look costs 40
// clocks when the phase is over; going through the bounded loop for it, 100 to 170.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, bool& dead, int* abort_flag, int where, unsigned long long ns) {
  const uint32_t b = ptx::smem_u32(bar);
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(b, parity))) return !dead;
  const bool here = !dead && ptx::mbar_wait_bounded_fast<20>(b, parity, abort_flag, where, ns);
  dead = !__all_sync(0xffffffffu, here);
  return !dead;
}

// A loading warp's life: the keys (which 0) or the values (1) of every unit of the block's run into the ring.  A box is `box` rows (the
// greatest common divisor of a page's and a unit's, so no box is cut by either) of 64 elements.  A lane looks up one box: 32 lanes
// serve the next 32 * box / 64 units at once, a group ahead of their copies, or the table's latency (700 clocks) would be paid for
// every unit.  (With boxes of one row a unit has 64: a lane looks up two.)  Issuing a copy takes 95 clocks, which is why there are two
// such warps: sixteen copies, what a unit of pages of 16 slots takes, are 1530.
template <int DIM, int STAGES, bool GROWS, typename Wait>
__device__ __forceinline__ void load_units(const AttnArgs& a, const CUtensorMap* map, const Line<GROWS>& line, Place<GROWS> at, long long end,
                                           uint32_t stages, Ring<STAGES>& ring, int which, Wait wait) {
  constexpr int TILE = UNIT * DIM * 2, PARTS = DIM / 64;
  const int lane = threadIdx.x & 31, box = a.box, boxes = UNIT / box, page_size = a.pool.page_size;
  const int group = boxes < 32 ? 32 / boxes : 1, box0 = lane % boxes;   // units of a group; this lane's box of its unit
  Slot<STAGES> at_stage(1);     // the first pass over the ring finds it empty
  uint32_t sent = 0;
  // what a lane knows of its unit: the table's entry for its box (as it stands there, so that nothing waits for it; -1: none) and slot of
  // the box's first row, cache head, rows up to the sequence's end (RUN_OVER: no unit)
  constexpr int RUN_OVER = -0x7fffffff;
  struct Found {
    int page[2], slot[2], head, rows;
  };
  // `at` goes from the run's start to this lane's unit, then a group at a time
  auto advance = [&](int count) {
    while (count > 0 && at.pos < end) {
      const int step = count < at.units - at.unit ? count : at.units - at.unit;
      at.skip(line, step);
      count -= step;
    }
  };
  auto look_up = [&]() {
    Found f;
    f.rows = at.pos < end ? at.total - at.unit * UNIT : RUN_OVER;
    f.head = at.head;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int b = box0 + 32 * j, pos = at.unit * UNIT + b * box;
      f.page[j] = -1;
      f.slot[j] = 0;
      if (b < boxes && b * box < f.rows) {
        // (total is within the pages that are held, and those within the table)
        f.page[j] = a.pool.table[at.s * a.pool.table_stride + (unsigned)pos / (unsigned)page_size];
        f.slot[j] = (int)((unsigned)pos % (unsigned)page_size);
      }
    }
    return f;
  };
  bool more = true;
  advance(lane / boxes);   // (0 for 32 boxes and more)
  Found next = look_up();
  while (more) {
    const Found now = next;
    advance(group);
    next = look_up();   // the next group's entries are on their way while this one's boxes go out
    for (int g = 0; g < group; ++g) {
      const int first = boxes < 32 ? g * boxes : 0;   // the lane that knows the unit's first box
      const int here = __shfl_sync(0xffffffffu, now.rows, first), head = __shfl_sync(0xffffffffu, now.head, first);
      if (here == RUN_OVER) {
        more = false;
        break;
      }
      uint64_t in = 0;
      if (which == 0) {
        const bool mine = boxes >= 32 || lane / boxes == g;
        if (mine && (unsigned)now.page[0] < (unsigned)a.pool.pages) in |= low_bits(box) << (box0 * box);
        if (mine && (unsigned)now.page[1] < (unsigned)a.pool.pages) in |= low_bits(box) << ((box0 + 32) * box);
        in = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(in >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)in);
      }
      if (!wait(&ring.empty[at_stage.i], at_stage.phase, 1)) {
        more = false;
        break;
      }
      const uint32_t bar = ptx::smem_u32(&ring.full[at_stage.i]), dst = stages + (at_stage.i * 2 + which) * TILE;
      if (lane == 0) {
        if (which == 0) ring.there[sent % ring.NOTES] = in & low_bits(here);
        ptx::mbar_arrive_expect_tx(bar, TILE + a.expect_extra);
      }
      __syncwarp();
#pragma unroll 4
      for (int b = 0; b < boxes; ++b) {
        const int pg = __shfl_sync(0xffffffffu, b < 32 ? now.page[0] : now.page[1], (first + b) & 31);
        const int sl = __shfl_sync(0xffffffffu, b < 32 ? now.slot[0] : now.slot[1], (first + b) & 31);
#pragma unroll
        for (int x = 0; x < PARTS; ++x)
          tma_load_4d(dst + x * (UNIT * 128) + b * box * 128, map, bar, x * 128, sl, head, (unsigned)pg < (unsigned)a.pool.pages ? pg : a.pool.pages);
      }
      ++sent;
      at_stage.next();
    }
  }
  // what is still on its way (when a wait ran out somewhere) lands before the block is gone
  int flag = 0;
  for (uint32_t i = 0; i < STAGES; ++i)
    if (i < sent) ptx::mbar_wait_bounded(ptx::smem_u32(&ring.full[i]), ((sent - i - 1) / STAGES) & 1, &flag, 1, a.wait_ns);
  __syncwarp();
}

// Launchers: the kernel on mma.sync (tree_attention.cu) and the one on tcgen05 (tree_attention_umma.cu), each followed by the join.
int make_map(CUtensorMap* map, const AttnArgs& a, const void* base);
int launch_join(const AttnArgs& a, int blocks, int tile_rows, int dim, cudaStream_t s);
constexpr int UMMA_ROWS = 128;
// pair: two row tiles at a time; grows: a pair of a chain ends at its own last node
int launch_umma(const AttnArgs& a, bool pair, bool grows, int sms, cudaStream_t s);

}  // namespace attn
}  // namespace b200q
