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
// Two warps of a block only load, one keys and one values, with TMA boxes of as many rows as both a page and a unit are made of, ahead of
// the products and across items, into a ring of stages of 64 keys and values; four warps compute.  Shared memory holds 64 elements
// a row, swizzled by 16-byte pieces (piece ^ row % 8), so that ldmatrix meets no bank twice.  (Loading with 16-byte cp.async took 640
// instructions a warp and unit: 108 us for 48 sequences of one token, 450 MB, that take 81 this way: 5.55 TB/s, 0.85 of the measured rate.)
//
// What bounds it: DRAM; 10 us of a launch, the batch's lengths, the first unit's way through table and memory, and the join are fixed.  At head size
// 128 two blocks an SM fit up to 480 sequences (24 bytes of shared memory each); beyond, one does, and the grid of two an SM runs in two waves: one
// token at 500 positions 5.2 TB/s for 470 sequences, 3.75 for 500, 4.0 for 1024.
#include <math.h>

#include "igemm.h"
#include "tree_attention.cuh"

namespace b200q {
using namespace attn;
namespace {

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
// What an item costs, in units (48 sequences of one token: 91 / 84.5 / 81.6 / 81.6 us at 1 / 2 / 3 / 4).
constexpr int ITEM_COST = 3;
constexpr int COMPUTERS = 128, BLOCK = COMPUTERS + 32 * LOADERS;

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
  __shared__ long long scan_buf[BLOCK / 32];
  __shared__ uint32_t bad[2];                    // rows of the unit whose values hold infinities or NaN
  __shared__ Ring<STAGES> ring;
  __shared__ int abort_flag;
  float* merge = reinterpret_cast<float*>(smem + STAGES * 2 * S::TILE);
  float* merge_ml = merge + S::ROWS * 64;
  long long* sums = reinterpret_cast<long long*>(smem + S::FIXED);
  Sequence* seqs = reinterpret_cast<Sequence*>(sums + a.pool.sequences);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int dim = a.cache.head_dim, group = a.group;
  ptx::griddep_launch_dependents();

  if (tid == 0) {
    ring.init(COMPUTERS / 32);
    ptx::fence_barrier_init();
    abort_flag = 0;
    bad[0] = bad[1] = 0;
    ptx::prefetch_tensormap(&km);
    ptx::prefetch_tensormap(&vm);
  }
  ptx::griddep_wait();
  const long long total = lay_out<BLOCK, false>(a, S::ROWS, ITEM_COST, seqs, sums, scan_buf);
  const Line<false> line{seqs, a.pool.sequences, a.cache.heads, group, S::ROWS, ITEM_COST};

  const long long run = run_of(total);
  const long long u0 = (long long)blockIdx.x * run, u1 = u0 + run < total ? u0 + run : total;
  if (tid == 0) a.items[blockIdx.x].parts = 0;
  if (u0 >= u1) return;
  Place<false> at;
  at.find(line, sums, u0);
  const uint16_t* vp = static_cast<const uint16_t*>(a.cache.v) + a.io.layer * a.cache.layer_stride;
  const uint32_t smem_base = ptx::smem_u32(smem);
  // A wait that runs out (it cannot, short of a fault) ends all waiting: the roles go on without (or stop, where they would load), so
  // that no barrier is left short, and the status says so.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int where) { return warp_wait(bar, parity, dead, &abort_flag, where, a.wait_ns); };

  if (warp >= COMPUTERS / 32) {
    // ---------------------------------------------------------------- loading
    if (warp == COMPUTERS / 32) load_units<DIM>(a, &km, line, at, u1, smem_base, ring, 0, wait);
    else load_units<DIM>(a, &vm, line, at, u1, smem_base, ring, 1, wait);
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
  uint32_t count = 0;
  Slot<STAGES> slot(0);

  while (at.pos < u1) {
    if (fresh) {
      // a new item (or this block's part of one)
      fresh = false;
      started = at.unit;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = at.tile * S::ROWS + wr * 16 + lane / 4 + 8 * h;
        const bool real = r < at.nodes * group;
        const int t = (unsigned)r / (unsigned)group, row = at.first_row + (real ? t : 0);
        node[h] = t;
        if (a.io.mask && a.io.mask_stride && (lane & 3) == 0) prefetch(a.io.mask + (int64_t)row * a.io.mask_stride);
        m[h] = -INFINITY;
        l[h] = 0.f;
        const uint16_t* src = static_cast<const uint16_t*>(a.io.q) + (int64_t)row * a.io.q_row_stride + (at.head * group + r - t * group) * a.io.q_head_stride;
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
    wait(&ring.full[slot.i], slot.phase, 3);

    // ---- scores of 16 rows x COLS positions
    // (pieces 2k and 2k + 1 of a row: the swizzle makes the step from k to k + 1 an exclusive or of 32 bytes)
    const uint32_t ks = smem_base + slot.i * 2 * S::TILE, vs = ks + S::TILE;
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
    const uint64_t in_pool = ring.there[count++ % ring.NOTES];
    const int unseen = min(at.length, at.total);
    const bool drafted = p0 > unseen - UNIT;   // or past the sequence's end: what lies there is anybody's
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
        // The stage's next values come by TMA, which does not wait for ordinary stores by itself: the fence puts these before them.
        const bool found = clean_values<F16, PIECES>(smem + (vs - smem_base), unseen > p0 ? unseen - p0 : 0, tid, COMPUTERS, bad);
        if (found) ptx::fence_proxy_async_smem();
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
      const float now = fmaxf(m[h], top * a.scale_log2), base = now == -INFINITY ? 0.f : now, lifted = base - lift<F16>();
      alpha[h] = exp2_approx(m[h] - base);
      m[h] = now;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp2_approx(fmaf(sc[t][2 * h + e], a.scale_log2, -lifted));
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
    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&ring.empty[slot.i]));
    slot.next();

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
            uint16_t* dst = static_cast<uint16_t*>(a.io.out) + (int64_t)(at.first_row + node[h]) * a.io.out_row_stride +
                            (at.head * group + r - node[h] * group) * a.io.out_head_stride;
#pragma unroll
            for (int k = 0; k < DIM / 8; ++k) {
              const int d = k * 8 + (lane & 3) * 2;
              if (d < dim) *reinterpret_cast<uint32_t*>(dst + d) = pack_pair<F16>(o[k][2 * h] * inv, o[k][2 * h + 1] * inv);
            }
          } else {
            float* dst = a.partial + (blockIdx.x * 2 + (started == 0)) * part_size(S::ROWS, DIM);
#pragma unroll
            for (int k = 0; k < DIM / 8; ++k)
              *reinterpret_cast<float2*>(dst + part_at(S::ROWS, rt, k * 2 + (lane & 3) / 2) + (lane & 1) * 2) = make_float2(o[k][2 * h], o[k][2 * h + 1]);
            if ((lane & 3) == 0) *reinterpret_cast<float2*>(dst + part_at(S::ROWS, rt, DIM / 4)) = make_float2(m[h], l[h]);
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

// Joins the parts of the items that were cut: block x looks after the item that starts in block x's run.  A warp takes eight rows, four
// lanes of each: four columns a lane; or, with more than JOIN_MANY parts (one long context over the whole GPU), one four-column piece
// whose parts the lanes share.  Parts are taken four at a time, their loads in flight together, with a running maximum.
constexpr int JOIN_THREADS = 256, JOIN_MANY = 8, JOIN_AT_ONCE = 4;
template <bool F16>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ AttnArgs a, int tile_rows, int dim_padded) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const SplitItem it = a.items[blockIdx.x];
  if (it.parts == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = a.cache.head_dim;
  const bool many = it.parts > JOIN_MANY;
  const int rows = it.rows - it.row0 < tile_rows ? it.rows - it.row0 : tile_rows;
  const int wide = (dim + 3) / 4, pieces = many ? wide : (wide + 3) / 4, works = (rows + 7) / 8 * pieces;   // of a warp
  const int share = many ? 4 : 1, mine = many ? lane >> 3 : 0;
  for (int w = blockIdx.y * (JOIN_THREADS / 32) + warp; w < works; w += gridDim.y * (JOIN_THREADS / 32)) {
    const int rt = w / pieces * 8 + (lane & 7), four = many ? w % pieces : w % pieces * 4 + (lane >> 3);
    const bool there = rt < rows && four < wide;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    for (int i0 = mine; i0 < it.parts; i0 += share * JOIN_AT_ONCE) {
      float2 ml[JOIN_AT_ONCE];
      float4 x[JOIN_AT_ONCE];
#pragma unroll
      for (int u = 0; u < JOIN_AT_ONCE; ++u) {
        const int i = i0 + u * share;
        // part 0 lies in its block's second place, the others in their blocks' first
        const float* p = a.partial + ((blockIdx.x + i) * 2 + (i == 0)) * part_size(tile_rows, dim_padded);
        ml[u] = make_float2(-INFINITY, 0.f);
        x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there && i < it.parts) {
          ml[u] = *reinterpret_cast<const float2*>(p + part_at(tile_rows, rt, dim_padded / 4));
          x[u] = *reinterpret_cast<const float4*>(p + part_at(tile_rows, rt, four));
        }
      }
      float now = top;
#pragma unroll
      for (int u = 0; u < JOIN_AT_ONCE; ++u) now = fmaxf(now, ml[u].x);
      const float base = now == -INFINITY ? 0.f : now, alpha = exp2_approx(top - base);
      top = now;
      sum *= alpha;
      acc = make_float4(acc.x * alpha, acc.y * alpha, acc.z * alpha, acc.w * alpha);
#pragma unroll
      for (int u = 0; u < JOIN_AT_ONCE; ++u) {
        const float f = exp2_approx(ml[u].x - base);
        sum += f * ml[u].y;
        acc.x += f * x[u].x;
        acc.y += f * x[u].y;
        acc.z += f * x[u].z;
        acc.w += f * x[u].w;
      }
    }
    if (many) {
      // the lanes that shared a row's parts: a common maximum, then the sums in a fixed order
      float now = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 16));
      const float f = exp2_approx(top - (now == -INFINITY ? 0.f : now));
      sum *= f;
      acc = make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f);
#pragma unroll
      for (int d = 8; d <= 16; d += 8) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        acc.x += __shfl_xor_sync(0xffffffffu, acc.x, d);
        acc.y += __shfl_xor_sync(0xffffffffu, acc.y, d);
        acc.z += __shfl_xor_sync(0xffffffffu, acc.z, d);
        acc.w += __shfl_xor_sync(0xffffffffu, acc.w, d);
      }
    }
    if (!there || mine) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int r = it.row0 + rt;
    uint16_t* dst = static_cast<uint16_t*>(a.io.out) + (int64_t)(it.first_row + r / a.group) * a.io.out_row_stride +
                    (it.head * a.group + r % a.group) * a.io.out_head_stride + four * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_pair<F16>(acc.x * inv, acc.y * inv), pack_pair<F16>(acc.z * inv, acc.w * inv));
  }
}

constexpr int BLOCKS_PER_SM = 2;

// Layout of the workspace for `blocks` blocks: what was cut, then the partial sums.
int64_t workspace_bytes(int blocks, int dim) {
  const int64_t items = ((int64_t)blocks * sizeof(SplitItem) + 255) / 256 * 256;
  const int rows = dim > 128 ? 32 : UMMA_ROWS;   // (two tiles a block of half as many blocks are the same)
  return items + blocks * 2 * part_size(rows, dim) * 4;
}
int padded_dim(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }

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
  B200Q_TRY(launch_dependent(kernel, dim3(blocks), dim3(BLOCK), smem, s, km, vm, a));
  return launch_join(a, blocks, S::ROWS, DIM, s);
}

// Rows of a tile by the average of (node, head of the group) a sequence of the call, which is what the host knows: rows / sequences * group.
// Both sides of each rule, us, bf16, 32 heads on 8 of 128 unless said otherwise, contexts spread evenly over the range:
//   up to 16 rows, 16-row tiles on mma.sync: 4 rows x 48 sequences of 200..8000 132.9 (32-row tiles 148.5, tcgen05 tiles 162.1), 4 rows x one of
//     430 10.3 (10.7, 12.5), 16 rows x 16 of 700..5000 43.6 (44.5, 46.8), 8 rows x 64 of 20..600 30.8 (34.9, 44.5);
//   up to 32 rows, 32-row tiles: 32 rows x 64 of 20..600 40.9 (16-row tiles 59.6, tcgen05 49.7), 20 rows x one of 131,000 at dim 64 71.9 (96.6,
//     72.0), though 24 and 32 rows x 16 of 700..5000 49.5 and 49.9 (58.7 and 60.2; 47.3 and 47.7); from 48 rows on a 64-row tile of the same kernel was
//     slower than tcgen05, and at dim 128 it spilled (96 rows x 16 sequences: 163 us), so there is none;
//   more rows: tcgen05, 128 rows a tile, two streams of units a block (49 rows x one of 120,000 at dim 64 68.6, 32-row tiles 108.8; 96 rows x 16 52.3,
//     110.1).  Above 128 rows the two streams take two row tiles and share each unit's keys and values: 160 rows x 8 of 700..8000 50.2 (two
//     streams of one tile: 63.0), 512 rows 99.1 (129.0); below, one tile would idle: 96 rows 52.3 shared out by units against 58.9, 128 rows x 8 45.5
//     against 49.3.
// Chains of more than two row tiles on average (prompts) take the form in which tiles end at their own last node (a prompt of 4096 nodes
// 164 us, without 493; in short calls its formula costs 1 us of 10).
// Sequences without rows, or of another kind, count in the average: 8 trees of 64 nodes at 12,500..16,000 positions take 130 us in a pool of 8 and 588 in one of
// 64, a prompt of 4096 171 and 503, and 7425 in one of 1024.  A call over the run of sequences that has the rows is without that (130, 171).
// Heads of more than 128 keep the 32-row tile: two streams' scores and sums do not fit tensor memory beside one another, and there is no form of
// one stream, whose 256 columns of sums and twice 64 of scores would fit.  That is far from the floor where there are many rows: at 256, 8 trees of 64
// nodes at 8000 positions take 2135 us (floor 81), a prompt of 2000 3141 (39), 48 tokens at 4000 278 (240).
template <bool F16, int DIM>
int launch_rows(const AttnArgs& a, int sms, cudaStream_t s) {
  const int64_t rows = (a.io.rows + a.pool.sequences - 1) / a.pool.sequences * a.group;
  if (rows <= 16) return launch<F16, DIM, 1, 4>(a, sms, s);
  if (rows <= 32 || DIM > 128) return launch<F16, DIM, 2, 2>(a, sms, s);
  return launch_umma(a, rows > UMMA_ROWS, !a.io.mask && rows > 2 * UMMA_ROWS, sms, s);
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

namespace attn {
// Keys or values of the layer as a TMA tensor [page][head][slot][bytes], boxes of `box` slots x 128 bytes.
int make_map(CUtensorMap* map, const AttnArgs& a, const void* base) {
  const uint64_t dims[4] = {(uint64_t)a.cache.head_dim * 2, (uint64_t)a.pool.page_size, (uint64_t)a.cache.heads, (uint64_t)a.pool.pages};
  const uint64_t strides[3] = {(uint64_t)a.cache.slot_stride * 2, (uint64_t)a.cache.head_stride * 2, (uint64_t)a.cache.page_stride * 2};
  const uint32_t box[4] = {128, (uint32_t)a.box, 1, 1};
  return make_tmap_u8(map, static_cast<const uint16_t*>(base) + a.io.layer * a.cache.layer_stride, 4, dims, strides, box);
}

int launch_join(const AttnArgs& a, int blocks, int tile_rows, int dim, cudaStream_t s) {
  // What the host knows: how many rows a tile has at most, and about how many items there are.  Few items are cut into many parts each,
  // and get a block for every eight warps' work; many get half of that each, and keep the launch small.
  const int64_t most = a.io.rows * a.group, rows = most < tile_rows ? most : tile_rows, items = a.cache.heads * (a.pool.sequences + most / tile_rows);
  const bool few = items * JOIN_MANY < blocks;
  const int64_t warps = (rows + 7) / 8 * (dim / (few ? 4 : 16)), per_block = JOIN_THREADS / 32 * (few ? 1 : 2);
  const dim3 grid(blocks, (unsigned)((warps + per_block - 1) / per_block)), block(JOIN_THREADS);
  return a.cache.dtype == B200Q_DT_F16 ? launch_dependent(join_kernel<true>, grid, block, 0, s, a, tile_rows, dim)
                                       : launch_dependent(join_kernel<false>, grid, block, 0, s, a, tile_rows, dim);
}
}  // namespace attn
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
  // (a tile's rows are counted in 32 bits, past the last row too)
  if (io.rows * (io.q_heads / cache->heads) > 0x7fffffffLL - 2 * UMMA_ROWS) return set_error(B200Q_ERR_UNSUPPORTED, "tree_attention: too many rows");
  if (io.layer < 0 || io.layer >= cache->layers) return set_error(B200Q_ERR_INVALID, "tree_attention: no layer %d in the cache", io.layer);
  if (!(io.scale > 0.f) || !isfinite(io.scale)) return set_error(B200Q_ERR_INVALID, "tree_attention: scale must be positive");
  if (((uintptr_t)io.q | (uintptr_t)io.out | (uintptr_t)io.workspace) & 15)
    return set_error(B200Q_ERR_INVALID, "tree_attention: q, out and workspace must be 16-byte aligned");
  B200Q_TRY(kv_check_words("tree_attention", {io.row_start, io.mask, io.status}));
  if ((io.q_row_stride | io.q_head_stride | io.out_row_stride | io.out_head_stride) & 7)
    return set_error(B200Q_ERR_INVALID, "tree_attention: strides of q and out must be multiples of 8 elements");
  if (io.q == io.out && (io.q_row_stride != io.out_row_stride || io.q_head_stride != io.out_head_stride))
    return set_error(B200Q_ERR_INVALID, "tree_attention: in place, the strides of q and out must be the same");
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
  a.items = static_cast<SplitItem*>(io.workspace);
  a.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(io.workspace) + ((int64_t)blocks * sizeof(SplitItem) + 255) / 256 * 256);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == B200Q_DT_F16 ? launch_dim<true>(a, sms, s) : launch_dim<false>(a, sms, s);
}

}  // extern "C"
