// Attention over the paged cache for many rows a cache head (trees, wide groups), on tcgen05: row tiles of 128.
//
// The line of units, its runs, the loads and the join are those of tree_attention.cu.  Per unit of 64 positions
//   S = Q K^T     128 x 64, both operands in shared memory, the queries loaded once an item
//   P = 2^(S - m) a thread owns a row: 64 scores from tensor memory, the running maximum and sum without a shuffle, the weights back
//                 into tensor memory over the scores that they came from, rounded to the 16-bit type
//   O += P V      128 x dim, P from tensor memory, V as it lies (positions x head: the operand is MN-major)
// Scores have two buffers, so that a unit's S is made while the one before is exponentiated; two blocks an SM fill each other's
// gaps.  O is rescaled in tensor memory only when a row's maximum has grown by more than 2^8 since its weights were last based on it:
// weights up to 2^8 are as exact as those up to 1, and the division by the sum takes the base out again.
//
// What bounds it: DRAM up to one row tile a cache head; beyond, shared memory (768 of 128-byte reads and writes a unit and tile) and
// the exponentials (512 of its clocks) share the SM's time.
#include <math.h>

#include "igemm.h"
#include "tree_attention.cuh"

namespace b200q {
using namespace attn;
namespace {

constexpr int ROWS = UMMA_ROWS, BLOCK = ROWS + 64;   // four warps of rows, one loading, one issuing products
constexpr int RING = 2;
constexpr float SLACK = 8.f;                         // log2 of how far weights may exceed 1

// B operand that is contiguous along N: blocks of 64 elements (128-byte swizzle) `lead` bytes apart, groups of 8 rows of K 1024 apart
__device__ __forceinline__ uint64_t make_smem_desc_mnmajor(uint32_t addr, uint32_t lead) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)((lead >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t IDESC_B_MN = 1u << 16;

// One unit of O += P V: A in tensor memory (8 columns a step of 16 positions), B 2048 bytes a step.
__device__ __forceinline__ void umma_pv(uint32_t d_tmem, uint32_t p_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b32 at, bl;\n\t"
      ".reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t"
      "setp.eq.b32 p, %4, %4;\n\t"
      "add.u32 at, %1, 8;\n\t"
      "add.u32 bl, %2, 128;\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [at], db, %4, p;\n\t"
      "add.u32 at, %1, 16;\n\t"
      "add.u32 bl, %2, 256;\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [at], db, %4, p;\n\t"
      "add.u32 at, %1, 24;\n\t"
      "add.u32 bl, %2, 384;\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [at], db, %4, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(p_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Wait for this thread's loads; the registers are operands, so that no use of them comes before the wait.
__device__ __forceinline__ void tmem_ld_wait_8(uint32_t (&x)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_32(uint32_t (&x)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]),
                 "+r"(x[8]), "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]),
                 "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]), "+r"(x[21]), "+r"(x[22]), "+r"(x[23]),
                 "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]), "+r"(x[30]), "+r"(x[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait_64(uint32_t (&x)[32], uint32_t (&y)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]),
                 "+r"(x[8]), "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]),
                 "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]), "+r"(x[20]), "+r"(x[21]), "+r"(x[22]), "+r"(x[23]),
                 "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]), "+r"(x[30]), "+r"(x[31]),
                 "+r"(y[0]), "+r"(y[1]), "+r"(y[2]), "+r"(y[3]), "+r"(y[4]), "+r"(y[5]), "+r"(y[6]), "+r"(y[7]),
                   "+r"(y[8]), "+r"(y[9]), "+r"(y[10]), "+r"(y[11]), "+r"(y[12]), "+r"(y[13]), "+r"(y[14]), "+r"(y[15]),
                   "+r"(y[16]), "+r"(y[17]), "+r"(y[18]), "+r"(y[19]), "+r"(y[20]), "+r"(y[21]), "+r"(y[22]), "+r"(y[23]),
                   "+r"(y[24]), "+r"(y[25]), "+r"(y[26]), "+r"(y[27]), "+r"(y[28]), "+r"(y[29]), "+r"(y[30]), "+r"(y[31])
               :
               : "memory");
}
__device__ __forceinline__ void rows_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool rows_or(bool x) {
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

template <int DIM>
struct Shape {
  static constexpr int TILE = UNIT * DIM * 2, QUERIES = ROWS * DIM * 2, FIXED = QUERIES + 2 * RING * TILE;
  static constexpr uint32_t COLUMNS = 256, S0 = 0, O = 128;   // tensor memory: scores 2 x 64, sums up to 128
  static size_t bytes(int sequences) { return 1024 + FIXED + (size_t)sequences * (sizeof(long long) + sizeof(Sequence)); }
};

template <bool F16, int DIM>
__global__ void __launch_bounds__(BLOCK, 2)
tree_attention_umma_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm, const __grid_constant__ AttnArgs a) {
  using S = Shape<DIM>;
  constexpr int PIECES = DIM / 8, HALVES = DIM / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-ptx::smem_u32(smem_raw) & 1023);   // the swizzle goes by the address
  __shared__ Rings<RING, RING> rings;
  // queries in place; a unit's scores made, its weights in place, its products done
  __shared__ uint64_t q_full, s_full[2], p_full, o_done, drained;
  __shared__ long long scan_buf[BLOCK / 32];
  __shared__ uint32_t bad[2], tmem_slot;
  __shared__ int abort_flag;
  long long* sums = reinterpret_cast<long long*>(smem + S::FIXED);
  Sequence* seqs = reinterpret_cast<Sequence*>(sums + a.pool.sequences);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int dim = a.cache.head_dim, group = a.group;
  const uint32_t q_tile = ptx::smem_u32(smem), k_ring = q_tile + S::QUERIES, v_ring = k_ring + RING * S::TILE;

  if (tid == 0) {
    rings.init(1);
    ptx::mbar_init(ptx::smem_u32(&q_full), ROWS);
    ptx::mbar_init(ptx::smem_u32(&s_full[0]), 1);
    ptx::mbar_init(ptx::smem_u32(&s_full[1]), 1);
    ptx::mbar_init(ptx::smem_u32(&p_full), ROWS);
    ptx::mbar_init(ptx::smem_u32(&o_done), 1);
    ptx::mbar_init(ptx::smem_u32(&drained), 1);
    ptx::fence_barrier_init();
    abort_flag = 0;
    bad[0] = bad[1] = 0;
    ptx::prefetch_tensormap(&km);
    ptx::prefetch_tensormap(&vm);
  }
  ptx::griddep_wait();
  const long long total = lay_out<BLOCK>(a, ROWS, seqs, sums, scan_buf);
  const Line line{seqs, a.pool.sequences, a.cache.heads, group, ROWS};
  long long run = (total + gridDim.x - 1) / gridDim.x;
  if (run < a.min_run) run = a.min_run;
  const long long u0 = (long long)blockIdx.x * run, u1 = u0 + run < total ? u0 + run : total;
  if (tid == 0) a.items[blockIdx.x].parts = 0;
  if (u0 >= u1) return;
  // Tensor memory before the successor may come: a successor that takes all of it while this block still waits for its share would
  // wait for this block's end.
  if (warp == ROWS / 32 + 1) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), S::COLUMNS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  ptx::griddep_launch_dependents();
  const uint32_t tmem = tmem_slot;

  Place at;
  at.find(line, sums, u0);
  // A wait that runs out ends all waiting: the roles go on without (or stop, where they would load or multiply), and the status says
  // so.  A warp agrees on it; `wait1` is for the one thread that issues products.
  bool dead = false;
  auto wait1 = [&](uint64_t* bar, uint32_t parity, int where) {
    if (!dead) dead = !ptx::mbar_wait_bounded_fast<20>(ptx::smem_u32(bar), parity, &abort_flag, where, a.wait_ns);
    return !dead;
  };
  auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
    const bool here = !dead && ptx::mbar_wait_bounded_fast<20>(ptx::smem_u32(bar), parity, &abort_flag, where, a.wait_ns);
    dead = !__all_sync(0xffffffffu, here);
    return !dead;
  };

  if (warp == ROWS / 32) {
    load_units<DIM>(a, &km, &vm, line, at, u1, k_ring, v_ring, rings, wait);
  } else if (warp == ROWS / 32 + 1) {
    // ---------------------------------------------------------------- products, issued by one thread
    if (lane == 0) {
      constexpr uint32_t FORMAT = F16 ? 0 : 1;
      constexpr uint32_t idesc_s = ptx::make_idesc(1, FORMAT, FORMAT, ROWS, UNIT);
      constexpr uint32_t idesc_o = ptx::make_idesc(1, FORMAT, FORMAT, ROWS, DIM) | IDESC_B_MN;
      const uint64_t q_desc = ptx::make_smem_desc_kmajor(q_tile, 1024, 2);
      Slot<RING> ks(0), vs(0);
      uint32_t n = 0, q_phase = 0;   // units whose scores were asked for
      auto scores = [&](bool new_item) {
        if (new_item) {
          if (!wait1(&q_full, q_phase, 5)) return;
          q_phase ^= 1;
        }
        // The buffer held the weights of unit n - 2: its products have to be done.  (Unit n - 1's are not issued yet, except at a
        // new item, where theirs are waited for: the barrier may have gone past the phase of n - 2 by then.)
        const uint32_t back = new_item ? 1 : 2;
        if (n >= back && !wait1(&o_done, (n - back) & 1, 6)) return;
        if (!wait1(&rings.k_full[ks.i], ks.phase, 3)) return;
        ptx::tc_fence_after_sync();
        const uint64_t k_desc = ptx::make_smem_desc_kmajor(k_ring + ks.i * S::TILE, 1024, 2);
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          ptx::umma_kblock_f16(tmem + S::S0 + (n & 1) * UNIT, (uint32_t)q_desc + h * (ROWS * 128 >> 4), (uint32_t)k_desc + h * (UNIT * 128 >> 4),
                               (uint32_t)(q_desc >> 32), (uint32_t)(k_desc >> 32), idesc_s, h > 0);
        ptx::umma_commit(ptx::smem_u32(&rings.k_empty[ks.i]));
        ptx::umma_commit(ptx::smem_u32(&s_full[n & 1]));
        ks.next();
        ++n;
      };
      uint32_t i = 0;
      bool first = true;   // of the item, or of this block's part
      scores(true);
      while (at.pos < u1 && !dead) {
        const bool last = at.unit + 1 == at.units;
        at.next(line);
        const bool more = at.pos < u1;
        if (more && !last) scores(false);
        if (dead || !wait1(&p_full, i & 1, 7) || !wait1(&rings.v_full[vs.i], vs.phase, 4)) break;
        ptx::tc_fence_after_sync();
        const uint64_t v_desc = make_smem_desc_mnmajor(v_ring + vs.i * S::TILE, UNIT * 128);
        umma_pv(tmem + S::O, tmem + S::S0 + (i & 1) * UNIT, (uint32_t)v_desc, (uint32_t)(v_desc >> 32), idesc_o, !first);
        ptx::umma_commit(ptx::smem_u32(&rings.v_empty[vs.i]));
        ptx::umma_commit(ptx::smem_u32(&o_done));
        vs.next();
        ++i;
        first = last;
        if (more && last) scores(true);
      }
      if (dead) {
        // products that are still running end before tensor memory is given back
        int flag = 0;
        ptx::umma_commit(ptx::smem_u32(&drained));
        ptx::mbar_wait_bounded_fast<20>(ptx::smem_u32(&drained), 0, &flag, 1, a.wait_ns);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- a row a thread
    const uint16_t* vp = static_cast<const uint16_t*>(a.cache.v) + a.io.layer * a.cache.layer_stride;
    const uint32_t mine = tmem + ((uint32_t)warp << 21);   // this warp's 32 lanes
    float m = -INFINITY, l = 0.f;
    int started = 0, node = 0;
    bool fresh = true, real = false;
    Slot<RING> vs(0);
    for (uint32_t i = 0; at.pos < u1; ++i) {
      if (fresh) {
        // a new item (or this block's part of one).  All products with the old queries are done: their last unit's scores were read
        started = at.unit;
        const int r0 = at.tile * ROWS, rows = at.nodes * group;
        for (int c = tid; c < ROWS * PIECES; c += ROWS) {
          const int row = c / PIECES, piece = c % PIECES, r = r0 + row;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (r < rows && piece * 8 < dim)
            x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.io.q) + (int64_t)(at.first_row + r / group) * a.io.q_row_stride +
                                                (at.head * group + r % group) * a.io.q_head_stride + piece * 8);
          *reinterpret_cast<uint4*>(smem + (piece >> 3) * (ROWS * 128) + row * 128 + (((piece & 7) ^ (row & 7)) * 16)) = x;
        }
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(ptx::smem_u32(&q_full));
        real = r0 + tid < rows;
        node = (r0 + tid) / group;
        m = -INFINITY;
        l = 0.f;
      }
      // ---- scores
      wait(&s_full[i & 1], (i >> 1) & 1, 8);
      ptx::tc_fence_after_sync();
      const uint32_t s_tmem = mine + S::S0 + (i & 1) * UNIT;
      uint32_t s_lo[32], s_hi[32];
      ptx::tmem_ld_32x32b_x32(s_tmem, s_lo);
      ptx::tmem_ld_32x32b_x32(s_tmem + 32, s_hi);
      tmem_ld_wait_64(s_lo, s_hi);
      float s[UNIT];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        s[j] = __uint_as_float(s_lo[j]);
        s[j + 32] = __uint_as_float(s_hi[j]);
      }
      // ---- what is not seen
      const int p0 = at.unit * UNIT;
      const uint64_t in_pool = rings.there[i % rings.NOTES];
      const bool drafted = p0 + UNIT > at.length;
      uint64_t see = ~0ull;
      bool fix = false;
      if (drafted || in_pool != ~0ull) {
        see = in_pool & sees(a, at.first_row + (real ? node : 0), node, at.length, p0);
#pragma unroll
        for (int j = 0; j < UNIT; ++j)
          if (!(see >> j & 1)) s[j] = -INFINITY;
        if (drafted) {
          // infinite and NaN values of drafted nodes leave the tile: rows that do not see them would become NaN (tree_attention.cu)
          wait(&rings.v_full[vs.i], vs.phase, 9);
          bool found = false;
          for (int c = tid; c < UNIT * PIECES; c += ROWS) {
            const int row = c / PIECES;
            uint32_t* w = reinterpret_cast<uint32_t*>(smem + (v_ring - q_tile) + vs.i * S::TILE + tile_at(row, c % PIECES));
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
          if (found) ptx::fence_proxy_async_smem();
          fix = rows_or(found);
        }
      }
      // ---- running maximum
      float top = s[0];
#pragma unroll
      for (int j = 1; j < UNIT; ++j) top = fmaxf(top, s[j]);
      top *= a.scale_log2;
      const bool grown = top > m + SLACK;   // (-inf: any score)
      if (__any_sync(0xffffffffu, grown)) {
        const float now = grown ? top : m;
        const float alpha = grown ? exp2_approx(m - now) : 1.f;
        m = now;
        l *= alpha;
        if (!fresh) {
          wait(&o_done, (i - 1) & 1, 10);
          ptx::tc_fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < DIM; c += 16) {
            uint32_t x[16];
            ptx::tmem_ld_32x32b_x16(mine + S::O + c, x);
            ptx::tmem_ld_wait_16(x);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
            ptx::tmem_st_32x32b_x16(mine + S::O + c, x);
          }
          ptx::tmem_st_wait();
        }
      }
      // ---- weights (rounded to the 16-bit type: what the tensor cores take; the rounding is unbiased and averages out over positions)
      const float base = m == -INFINITY ? 0.f : m;
      uint32_t p[2][16];   // two weights a word
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int j = 0; j < UNIT; j += 2) {
        const float x = exp2_approx(fmaf(s[j], a.scale_log2, -base)), y = exp2_approx(fmaf(s[j + 1], a.scale_log2, -base));
        sum0 += x;
        sum1 += y;
        p[j / 32][j / 2 % 16] = pack_pair<F16>(x, y);
      }
      l += sum0 + sum1;
      ptx::tmem_st_32x32b_x16(s_tmem, p[0]);
      ptx::tmem_st_32x32b_x16(s_tmem + 16, p[1]);
      ptx::tmem_st_wait();
      ptx::tc_fence_before_sync();
      ptx::mbar_arrive(ptx::smem_u32(&p_full));
      if (fix) {
        wait(&o_done, i & 1, 11);
        ptx::tc_fence_after_sync();
        for (int row = 0; row < UNIT; ++row) {
          if (!(bad[row >> 5] >> (row & 31) & 1)) continue;
          uint32_t pair = 0;
#pragma unroll
          for (int j = 0; j < UNIT / 2; ++j)
            if (j == row >> 1) pair = p[j / 16][j % 16];
          const float w = from_bits<F16>(row & 1 ? pair >> 16 : pair & 0xffffu);
          const int64_t entry = kv_entry(a.cache, a.pool, at.s, p0 + row);
          if (entry < 0) continue;
          const uint16_t* value = vp + entry + at.head * a.cache.head_stride;
#pragma unroll 1
          for (int c = 0; c < dim; c += 8) {
            uint32_t x[8];
            __syncwarp();
            ptx::tmem_ld_32x32b_x8(mine + S::O + c, x);
            tmem_ld_wait_8(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t v = value[c + e];
              if (not_finite<F16>(v) && (see >> row & 1)) x[e] = __float_as_uint(__uint_as_float(x[e]) + w * from_bits<F16>(v));
            }
            __syncwarp();
            ptx::tmem_st_32x32b_x8(mine + S::O + c, x);
          }
          ptx::tmem_st_wait();
        }
        ptx::tc_fence_before_sync();
        rows_sync();
        if (tid < 2) bad[tid] = 0;
        rows_sync();
      }
      vs.next();
      fresh = false;

      // ---- the end of the item, or of this block's part
      const bool done = at.unit + 1 == at.units;
      const long long first = at.pos - at.unit;
      if (done || at.pos + 1 == u1) {
        fresh = true;
        wait(&o_done, i & 1, 12);
        ptx::tc_fence_after_sync();
        const bool whole = started == 0 && done;
        const int r = at.tile * ROWS + tid;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* dst = static_cast<uint16_t*>(a.io.out) + (int64_t)(at.first_row + (real ? r / group : 0)) * a.io.out_row_stride +
                        (at.head * group + r % group) * a.io.out_head_stride;
        float* part = a.partial + ((int64_t)(blockIdx.x * 2 + (started == 0)) * ROWS + tid) * (DIM + 4);
#pragma unroll
        for (int c = 0; c < DIM; c += 32) {
          uint32_t x[32];
          float o[32];
          __syncwarp();   // (loads from tensor memory are the whole warp's)
          ptx::tmem_ld_32x32b_x32(mine + S::O + c, x);
          tmem_ld_wait_32(x);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(x[e]);
          if (!real) {
          } else if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (c + e < dim)
                *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(pack_pair<F16>(o[e] * inv, o[e + 1] * inv), pack_pair<F16>(o[e + 2] * inv, o[e + 3] * inv),
                                                                    pack_pair<F16>(o[e + 4] * inv, o[e + 5] * inv), pack_pair<F16>(o[e + 6] * inv, o[e + 7] * inv));
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(part + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
        if (real && !whole) *reinterpret_cast<float2*>(part + DIM) = make_float2(m, l);
        ptx::tc_fence_before_sync();
        if (tid == 0 && started == 0 && !whole)
          a.items[blockIdx.x] = SplitItem{(int)((first + at.units - 1) / run) - (int)blockIdx.x + 1, at.first_row, at.tile * ROWS, at.nodes * group, at.head};
      }
      at.next(line);
    }
  }
  if (dead && lane == 0 && a.io.status) atomicMax(a.io.status, abort_flag);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  if (warp == ROWS / 32 + 1) ptx::tmem_dealloc(tmem, S::COLUMNS);
}

template <bool F16, int DIM>
int launch(const AttnArgs& a, int sms, cudaStream_t s) {
  using S = Shape<DIM>;
  auto kernel = tree_attention_umma_kernel<F16, DIM>;
  CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::bytes(KV_MAX_SEQUENCES)));
  CUtensorMap km, vm;
  B200Q_TRY(make_map(&km, a, a.cache.k));
  B200Q_TRY(make_map(&vm, a, a.cache.v));
  const int blocks = 2 * sms;
  B200Q_TRY(launch_dependent(kernel, dim3(blocks), dim3(BLOCK), S::bytes(a.pool.sequences), s, km, vm, a));
  return launch_join(a, blocks, ROWS, DIM, s);
}

}  // namespace

namespace attn {
int launch_umma(const AttnArgs& a, int sms, cudaStream_t s) {
  const bool f16 = a.cache.dtype == B200Q_DT_F16;
  if (a.cache.head_dim <= 64) return f16 ? launch<true, 64>(a, sms, s) : launch<false, 64>(a, sms, s);
  return f16 ? launch<true, 128>(a, sms, s) : launch<false, 128>(a, sms, s);
}
}  // namespace attn
}  // namespace b200q
