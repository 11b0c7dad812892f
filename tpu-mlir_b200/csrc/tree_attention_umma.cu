// Attention over the paged cache for many rows a cache head (trees, wide groups), on tcgen05.
//
// The line of units, its runs, the loads and the join are those of tree_attention.cu.  Per unit of 64 positions and 128 rows
//   S = Q K^T     128 x 64, both operands in shared memory, the queries loaded once an item
//   P = 2^(S - m) a thread owns a row: 64 scores from tensor memory, the running maximum and sum without a shuffle, the weights back
//                 into tensor memory over the scores that they came from, rounded to the 16-bit type
//   O += P V      128 x dim, P from tensor memory, V as it lies (positions x head: the operand is MN-major)
// A block (one an SM: the rings of keys and values have to be deep, four to eight units, or their latency sets the pace: with two
// stages and two blocks an SM 8 trees of 49 to 64 nodes over 9800 to 16,000 positions took 204 us where this took 115 in short runs) keeps two streams of this
// going, each with four warps, two buffers of scores and sums of its own.  With more than 128 rows a cache head the streams are two row
// tiles that share every unit of keys and values (PAIR); with fewer they take the units of one row tile in turn, and are merged at the
// item's end.
// O is rescaled in tensor memory only when a row's maximum has grown by more than 2^8 since its weights were last based on it:
// weights up to 2^8 are as exact as those up to 1, and the division by the sum takes the base out again.
//
// What bounds it: DRAM up to 128 rows a cache head (a unit every 0.65 us an SM, 7.3 TB/s with what L2 holds, and 10 us of start and join; an
// item more costs a block 5 us); beyond, exponentials, products and issue slots, 55, 55 and 46 % busy, wait for one another: 8 trees
// of 49 to 64 nodes, up to 256 rows, 428 MB and 95 GFLOP in 135 us under steady load (707 TFLOP/s; the power cap's clocks) and 116 in short runs.
#include <math.h>

#include "igemm.h"
#include "tree_attention.cuh"

namespace b200q {
using namespace attn;
namespace {

constexpr int ROWS = UMMA_ROWS, COMPUTERS = 2 * ROWS, MAKERS = COMPUTERS / 32 + LOADERS;   // two streams of rows, loading warps,
constexpr int BLOCK = 32 * (MAKERS + 2);                                                      // a warp a stream that issues products
// What an item costs, in units (16 trees of 24 nodes 52.1 / 50.4 / 49.0 / 48.1 us at 2 / 4 / 6 / 8, 50.5 at 16; queries, the first scores, the
// sums' way out).
constexpr int ITEM_COST = 8;
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

// The products are issued by a whole warp in step, of which one thread is elected for each instruction: addresses then live in uniform
// registers.  Issued from a branch that one thread takes, an instruction took 70 clocks whatever its size, more than its work.
// 64 elements of the head of S = Q K^T: four steps of 16, 32 bytes further each.
__device__ __forceinline__ void umma_qk(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, one;\n\t"
      ".reg .b32 al, bl;\n\t"
      ".reg .b64 da, db;\n\t"
      "elect.sync _|one, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "setp.eq.b32 p, %5, %5;\n\t"
      "add.u32 al, %1, 2;\n\t"
      "add.u32 bl, %3, 2;\n\t"
      "mov.b64 da, {al, %2};\n\t"
      "mov.b64 db, {bl, %4};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "add.u32 al, %1, 4;\n\t"
      "add.u32 bl, %3, 4;\n\t"
      "mov.b64 da, {al, %2};\n\t"
      "mov.b64 db, {bl, %4};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "add.u32 al, %1, 6;\n\t"
      "add.u32 bl, %3, 6;\n\t"
      "mov.b64 da, {al, %2};\n\t"
      "mov.b64 db, {bl, %4};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One unit of O += P V: A in tensor memory (8 columns a step of 16 positions), B 2048 bytes a step.
__device__ __forceinline__ void umma_pv(uint32_t d_tmem, uint32_t p_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p, one;\n\t"
      ".reg .b32 at, bl;\n\t"
      ".reg .b64 db;\n\t"
      "elect.sync _|one, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t"
      "setp.eq.b32 p, %4, %4;\n\t"
      "add.u32 at, %1, 8;\n\t"
      "add.u32 bl, %2, 128;\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [at], db, %4, p;\n\t"
      "add.u32 at, %1, 16;\n\t"
      "add.u32 bl, %2, 256;\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [at], db, %4, p;\n\t"
      "add.u32 at, %1, 24;\n\t"
      "add.u32 bl, %2, 384;\n\t"
      "mov.b64 db, {bl, %3};\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], [at], db, %4, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "r"(p_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The elected thread (the same one every time) signals `bar` when its products so far are done.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t"
      ".reg .pred one;\n\t"
      "elect.sync _|one, 0xffffffff;\n\t"
      "@one tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "}\n" ::"r"(ptx::smem_u32(bar))
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
// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t bits2(float2 v) { return (uint64_t)__float_as_uint(v.y) << 32 | __float_as_uint(v.x); }
__device__ __forceinline__ float2 float2_of(uint64_t b) { return make_float2(__uint_as_float((uint32_t)b), __uint_as_float((uint32_t)(b >> 32))); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return float2_of(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
  return float2_of(d);
}
// Barriers 1 and 2 are a stream's, 3 is for both, 4 and 5 pass the turn to the first and to the second stream.
template <int THREADS>
__device__ __forceinline__ void rows_sync(int id) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void rows_arrive(int id) {
  asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ bool rows_or(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.b32 q, %3, 0;\n\t"
      "barrier.cta.red.or.pred p, %1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(r)
      : "r"(id), "n"(THREADS), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

template <int DIM, bool PAIR>
struct Shape {
  static constexpr int TILES = PAIR ? 2 : 1, RING = DIM > 64 ? (PAIR ? 4 : 5) : 8;
  static constexpr int TILE = UNIT * DIM * 2, QUERIES = ROWS * DIM * 2, FIXED = TILES * QUERIES + 2 * RING * TILE;
  // tensor memory, a stream: scores 2 x 64, sums up to 128 columns
  static constexpr uint32_t COLUMNS = 512, STREAM = 256, O = 128;
  static size_t bytes(int sequences) { return 1024 + FIXED + (size_t)sequences * (sizeof(long long) + sizeof(Sequence)); }
};

template <bool F16, int DIM, bool PAIR, bool GROWS>
__global__ void __launch_bounds__(BLOCK, 1)
tree_attention_umma_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm, const __grid_constant__ AttnArgs a) {
  using S = Shape<DIM, PAIR>;
  constexpr int PIECES = DIM / 8, HALVES = DIM / 64, RING = S::RING, TILE_ROWS = S::TILES * ROWS;
  constexpr int SHARERS = PAIR ? COMPUTERS : ROWS;   // threads that a unit of values concerns
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-ptx::smem_u32(smem_raw) & 1023);   // the swizzle goes by the address
  __shared__ Ring<RING> ring;
  // Of a stream: queries in place; a unit's scores made, its weights in place, its products done.  The last three alternate between two
  // barriers, step by step: a barrier tells two phases apart, and the roles can be two steps away from each other (a step's scores are
  // asked for when the products two steps before are done).
  __shared__ uint64_t q_full[2], s_full[2][2], p_full[2][2], o_done[2][2], drained[2];
  __shared__ long long scan_buf[BLOCK / 32];
  __shared__ float2 other_ml[2][ROWS];               // not PAIR: what the streams tell each other at an item's end
  __shared__ uint32_t bad[2][2], tmem_slot;          // rows of a stream's unit whose values hold infinities or NaN (PAIR: the first)
  __shared__ int abort_flag;
  long long* sums = reinterpret_cast<long long*>(smem + S::FIXED);
  Sequence* seqs = reinterpret_cast<Sequence*>(sums + a.pool.sequences);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int dim = a.cache.head_dim, group = a.group;
  const uint32_t q_tile = ptx::smem_u32(smem), stages = q_tile + S::TILES * S::QUERIES;

  if (tid == 0) {
    ring.init(PAIR ? 2 : 1);
    for (int j = 0; j < 2; ++j) {
      ptx::mbar_init(ptx::smem_u32(&q_full[j]), PAIR ? ROWS : COMPUTERS);
      ptx::mbar_init(ptx::smem_u32(&s_full[j][0]), 1);
      ptx::mbar_init(ptx::smem_u32(&s_full[j][1]), 1);
      ptx::mbar_init(ptx::smem_u32(&p_full[j][0]), ROWS);
      ptx::mbar_init(ptx::smem_u32(&p_full[j][1]), ROWS);
      ptx::mbar_init(ptx::smem_u32(&o_done[j][0]), 1);
      ptx::mbar_init(ptx::smem_u32(&o_done[j][1]), 1);
      ptx::mbar_init(ptx::smem_u32(&drained[j]), 1);
      bad[j][0] = bad[j][1] = 0;
    }
    ptx::fence_barrier_init();
    abort_flag = 0;
    ptx::prefetch_tensormap(&km);
    ptx::prefetch_tensormap(&vm);
  }
  ptx::griddep_wait();
  // Tensor memory, while the others read the batch's lengths.  (Not before the predecessor is done, which may still need its own; and
  // before the successor may come: one that takes all of it while this block still waits for its share would wait for this block's end.)
  if (warp == MAKERS) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), S::COLUMNS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  const long long total = lay_out<BLOCK, GROWS>(a, TILE_ROWS, ITEM_COST, seqs, sums, scan_buf);
  const Line<GROWS> line{seqs, a.pool.sequences, a.cache.heads, group, TILE_ROWS, ITEM_COST};
  const long long run = run_of(total);
  const long long u0 = (long long)blockIdx.x * run, u1 = u0 + run < total ? u0 + run : total;
  if (tid == 0) a.items[blockIdx.x].parts = 0;
  ptx::tc_fence_after_sync();   // (lay_out ends with the block's barrier)
  ptx::griddep_launch_dependents();
  const uint32_t tmem = tmem_slot;
  if (u0 >= u1) {
    if (warp == MAKERS) ptx::tmem_dealloc(tmem, S::COLUMNS);
    return;
  }

  Place<GROWS> at;
  at.find(line, sums, u0);
  // A wait that runs out ends all waiting: the roles go on without (or stop, where they would load or multiply), and the status says
  // so.
  bool dead = false;
  auto wait = [&](uint64_t* bar, uint32_t parity, int where) { return warp_wait(bar, parity, dead, &abort_flag, where, a.wait_ns); };

  if (warp == COMPUTERS / 32) {
    load_units<DIM>(a, &km, line, at, u1, stages, ring, 0, wait);
  } else if (warp == COMPUTERS / 32 + 1) {
    load_units<DIM>(a, &vm, line, at, u1, stages, ring, 1, wait);
  } else if (warp >= MAKERS) {
    // ---------------------------------------------------------------- products of a stream
    // Scores are asked for one step ahead, within an item.
    constexpr uint32_t FORMAT = F16 ? 0 : 1;
    constexpr uint32_t idesc_s = ptx::make_idesc(1, FORMAT, FORMAT, ROWS, UNIT);
    constexpr uint32_t idesc_o = ptx::make_idesc(1, FORMAT, FORMAT, ROWS, DIM) | IDESC_B_MN;
    const uint32_t j = warp - MAKERS, columns = tmem + j * S::STREAM;
    const uint64_t q_desc = ptx::make_smem_desc_kmajor(q_tile + (PAIR ? j * S::QUERIES : 0), 1024, 2);
    uint32_t asked = 0, made = 0, items = 0;      // steps whose scores were asked for, whose products were; items with steps so far
    uint32_t unit0 = 0;                           // units of the run before the item
    auto unit_of = [&](uint32_t step) { return PAIR ? step : 2 * step + j; };   // the unit of the run that a step takes
    auto scores = [&]() {
      // The buffer held the weights of the step before the last: its products have to be done.  (Those of the last step, at a new item.)
      if (made && !wait(&o_done[j][(made - 1) & 1], (made - 1) >> 1 & 1, 6)) return;
      const uint32_t u = unit_of(asked);
      if (!wait(&ring.full[u % RING], u / RING & 1, 3)) return;
      ptx::tc_fence_after_sync();
      const uint64_t k_desc = ptx::make_smem_desc_kmajor(stages + u % RING * 2 * S::TILE, 1024, 2);
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
        umma_qk(columns + (asked & 1) * UNIT, (uint32_t)q_desc + h * (ROWS * 128 >> 4), (uint32_t)(q_desc >> 32),
                (uint32_t)k_desc + h * (UNIT * 128 >> 4), (uint32_t)(k_desc >> 32), idesc_s, h > 0);
      commit(&s_full[j][asked & 1]);
      ++asked;
    };
    while (at.pos < u1 && !dead) {
      // an item, or this block's part of one, and the steps up to its end
      const long long left = u1 - at.pos;
      const uint32_t units = (uint32_t)(left < at.units - at.unit ? left : at.units - at.unit);
      const uint32_t first = made, end = PAIR ? unit0 + units : (unit0 + units + 1 - j) / 2;
      if (made < end) wait(&q_full[j], items++ & 1, 5);
      while (made < end && !dead) {
        if (asked == made) scores();
        if (asked < end && !dead) scores();
        if (dead || !wait(&p_full[j][made & 1], made >> 1 & 1, 7)) break;
        ptx::tc_fence_after_sync();
        const uint32_t u = unit_of(made);
        const uint64_t v_desc = make_smem_desc_mnmajor(stages + (u % RING * 2 + 1) * S::TILE, UNIT * 128);
        umma_pv(columns + S::O, columns + (made & 1) * UNIT, (uint32_t)v_desc, (uint32_t)(v_desc >> 32), idesc_o, made > first);
        commit(&ring.empty[u % RING]);
        commit(&o_done[j][made & 1]);
        ++made;
      }
      unit0 += units;
      at.skip(line, units);
    }
    if (dead) {
      // products that are still running end before tensor memory is given back
      int flag = 0;
      commit(&drained[j]);
      ptx::mbar_wait_bounded_fast<20>(ptx::smem_u32(&drained[j]), 0, &flag, 1, a.wait_ns);
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- a row a thread
    const int stream = warp >> 2, row_in = tid & (ROWS - 1);
    const int bar_rows = PAIR ? 3 : 1 + stream;
    uint32_t* const bad_rows = bad[PAIR ? 0 : stream];
    const uint16_t* vp = static_cast<const uint16_t*>(a.cache.v) + a.io.layer * a.cache.layer_stride;
    const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21) + stream * S::STREAM;   // this warp's 32 lanes of its stream's columns
    constexpr int STEP = (PAIR ? ROWS : COMPUTERS) / PIECES;   // rows between a thread's pieces of the queries
    const int step_t = STEP / group, step_h = STEP - step_t * group;
    const int64_t step_from = step_t * a.io.q_row_stride + step_h * a.io.q_head_stride, carry_from = a.io.q_row_stride - group * a.io.q_head_stride;
    uint32_t done = 0;    // steps of this stream so far
    uint32_t unit = 0;    // units of the run so far
    while (at.pos < u1) {
      // ---- an item (or this block's part of one).  All products with the old queries are done: o_done of both streams was waited for
      const long long left = u1 - at.pos;
      const int started = at.unit, units = (int)(left < at.units - at.unit ? left : at.units - at.unit);
      const long long first = at.pos - at.unit;   // where the item's units start in the line
      const int r0 = at.tile * TILE_ROWS + (PAIR ? stream * ROWS : 0), rows = at.nodes * group;
      {
        // 16 bytes a thread and copy, all of them in flight together (loaded and stored one after the other they took 6000 clocks and more)
        const int at0 = PAIR ? row_in : tid, piece = at0 % PIECES, row0 = at0 / PIECES;
        const uint32_t dst = q_tile + (PAIR ? stream * S::QUERIES : 0) + (piece >> 3) * (ROWS * 128);
        const uint16_t* src = static_cast<const uint16_t*>(a.io.q) + (int64_t)at.first_row * a.io.q_row_stride + (int64_t)at.head * group * a.io.q_head_stride;
        // One division for (node, head of the group), then STEP rows further each: a division a row took as long as the loads.  Addresses go on
        // by sums or by products, whichever the rest of the loop came out better with (PAIR: 512 rows x 8 sequences 81.3 and 88.0 us; not
        // PAIR: 96 rows 41.3 and 38.4).
        int t = (unsigned)(r0 + row0) / (unsigned)group, h = r0 + row0 - t * group;
        int64_t from = (int64_t)t * a.io.q_row_stride + h * a.io.q_head_stride;
#pragma unroll
        for (int i = 0; i < ROWS / STEP; ++i) {
          const int row = row0 + i * STEP;
          const bool in = r0 + row < rows && piece * 8 < dim;
          cp_async16(dst + row * 128 + (((piece & 7) ^ (row & 7)) * 16),
                     in ? src + (PAIR ? from : (int64_t)t * a.io.q_row_stride + h * a.io.q_head_stride) + piece * 8 : src, in);
          h += step_h;
          t += step_t;
          from += step_from;
          if (h >= group) {
            h -= group;
            ++t;
            from += carry_from;
          }
        }
        cp_async_wait_all();
      }
      ptx::fence_proxy_async_smem();
      // (not PAIR: an item of one unit is one stream's alone)
      if (PAIR) {
        ptx::mbar_arrive(ptx::smem_u32(&q_full[stream]));
      } else {
        for (int j = 0; j < 2; ++j)
          if (units > 1 || (unit & 1) == j) ptx::mbar_arrive(ptx::smem_u32(&q_full[j]));
      }
      const int r = r0 + row_in, node = (unsigned)r / (unsigned)group;
      const bool real = r < rows;
      if (a.io.mask && a.io.mask_stride && real) prefetch(a.io.mask + (int64_t)(at.first_row + node) * a.io.mask_stride);
      float m = -INFINITY, l = 0.f;
      bool fresh = true;

      for (int u = 0; u < units; ++u, ++unit) {
        if (!PAIR && (unit & 1) != stream) continue;
        // ---- scores
        wait(&s_full[stream][done & 1], (done >> 1) & 1, 8);
        ptx::tc_fence_after_sync();
        const uint32_t s_tmem = mine + (done & 1) * UNIT;
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
        const int p0 = (started + u) * UNIT;
        const uint64_t in_pool = ring.there[unit % ring.NOTES];
        const int unseen = at.unseen(line);
        const bool drafted = p0 > unseen - UNIT;   // or past the sequence's end: what lies there is anybody's
        uint64_t see = ~0ull;
        bool fix = false;
        if (drafted || in_pool != ~0ull) {
          see = in_pool & sees(a, at.first_row + (real ? node : 0), node, at.length, p0);
#pragma unroll
          for (int j = 0; j < UNIT; ++j)
            if (!(see >> j & 1)) s[j] = -INFINITY;
          if (drafted) {
            // infinite and NaN values of drafted nodes leave the tile: rows that do not see them would become NaN (tree_attention.cu)
            wait(&ring.full[unit % RING], unit / RING & 1, 9);
            const bool found = clean_values<F16, PIECES>(smem + (stages - q_tile) + (unit % RING * 2 + 1) * S::TILE, unseen > p0 ? unseen - p0 : 0,
                                                         PAIR ? tid : row_in, SHARERS, bad_rows);
            if (found) ptx::fence_proxy_async_smem();
            fix = rows_or<SHARERS>(bar_rows, found);
          }
        }
        // ---- running maximum
        float t0 = s[0], t1 = s[1], t2 = s[2], t3 = s[3];
#pragma unroll
        for (int j = 4; j < UNIT; j += 4) {
          t0 = fmaxf(t0, s[j]);
          t1 = fmaxf(t1, s[j + 1]);
          t2 = fmaxf(t2, s[j + 2]);
          t3 = fmaxf(t3, s[j + 3]);
        }
        const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * a.scale_log2;
        const bool grown = top > m + SLACK;   // (-inf: any score)
        if (__any_sync(0xffffffffu, grown)) {
          const float now = grown ? top : m;
          const float alpha = grown ? exp2_approx(m - now) : 1.f;
          m = now;
          l *= alpha;
          if (!fresh) {
            wait(&o_done[stream][(done - 1) & 1], (done - 1) >> 1 & 1, 10);
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
        // ---- The streams exponentiate in turn, step by step: left alone they fall into step, share the exponential unit and then both leave
        // it idle (8 trees of 64 nodes: 124.6 us where this took 114.5).
        const uint32_t turn = PAIR ? 2 * unit + stream : unit;
        if (turn) rows_sync<COMPUTERS>(4 + (turn & 1));
        // ---- weights (rounded to the 16-bit type: what the tensor cores take; the rounding is unbiased and averages out over positions)
        const float base = (m == -INFINITY ? 0.f : m) - lift<F16>();
        uint32_t p[2][16];   // two weights a word
        const float2 scale2 = make_float2(a.scale_log2, a.scale_log2), base2 = make_float2(-base, -base);
        float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < UNIT; j += 2) {
          const float2 y = fma2(make_float2(s[j], s[j + 1]), scale2, base2);
          const float2 x = make_float2(exp2_approx(y.x), exp2_approx(y.y));
          sum2 = add2(sum2, x);
          p[j / 32][j / 2 % 16] = pack_pair<F16>(x.x, x.y);
        }
        rows_arrive<COMPUTERS>(4 + (turn + 1 & 1));
        l += sum2.x + sum2.y;
        ptx::tmem_st_32x32b_x16(s_tmem, p[0]);
        ptx::tmem_st_32x32b_x16(s_tmem + 16, p[1]);
        ptx::tmem_st_wait();
        ptx::tc_fence_before_sync();
        ptx::mbar_arrive(ptx::smem_u32(&p_full[stream][done & 1]));
        if (fix) {
          wait(&o_done[stream][done & 1], done >> 1 & 1, 11);
          ptx::tc_fence_after_sync();
          for (int row = 0; row < UNIT; ++row) {
            if (!(bad_rows[row >> 5] >> (row & 31) & 1)) continue;
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
          rows_sync<SHARERS>(bar_rows);
          if (tid < 2 || (!PAIR && row_in < 2)) bad_rows[row_in] = 0;
          rows_sync<SHARERS>(bar_rows);
        }
        ++done;
        fresh = false;
      }

      // ---- the end of the item, or of this block's part
      if (!fresh) wait(&o_done[stream][(done - 1) & 1], (done - 1) >> 1 & 1, 12);
      ptx::tc_fence_after_sync();
      const bool whole = started == 0 && units == at.units;
      // not PAIR: both streams know both halves of the row, and each takes half of the columns out
      float f0 = 1.f, f1 = 0.f;   // factors on this stream's sums and on the other's
      if (!PAIR) {
        other_ml[stream][row_in] = make_float2(m, l);
        ptx::tc_fence_before_sync();
        rows_sync<COMPUTERS>(3);
        ptx::tc_fence_after_sync();
        const float2 ml = other_ml[stream ^ 1][row_in];
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top;
        f0 = exp2_approx(m - base);
        f1 = exp2_approx(ml.x - base);
        l = l * f0 + ml.y * f1;
        m = top;
      }
      const bool had0 = !fresh, had1 = !PAIR && (units > 1 || fresh);   // this stream, the other: had a unit at all
      // (a finite score that scale * log2(e) took past fp32 leaves a maximum of infinity and no weights: not a row that sees nothing)
      const float inv = m == INFINITY ? NAN : l == 0.f ? 0.f : 1.f / l;
      uint16_t* dst = static_cast<uint16_t*>(a.io.out) + (int64_t)(at.first_row + (real ? node : 0)) * a.io.out_row_stride +
                      (at.head * group + r - node * group) * a.io.out_head_stride;
      float* part = a.partial + (blockIdx.x * 2 + (started == 0)) * part_size(TILE_ROWS, DIM);
      const int part_row = (PAIR ? stream * ROWS : 0) + row_in;
      const uint32_t theirs = mine ^ S::STREAM;   // (the allocation starts at a multiple of its size)
#pragma unroll
      for (int c0 = 0; c0 < (PAIR ? DIM : DIM / 2); c0 += 32) {
        const int c = (PAIR ? 0 : stream * (DIM / 2)) + c0;
        uint32_t x[32], y[32];
        __syncwarp();   // (loads from tensor memory are the whole warp's)
        ptx::tmem_ld_32x32b_x32(mine + S::O + c, x);
        if (!PAIR) ptx::tmem_ld_32x32b_x32(theirs + S::O + c, y);
        if (PAIR) tmem_ld_wait_32(x);
        else tmem_ld_wait_64(x, y);
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          // (a stream without a unit left what tensor memory held)
          o[e] = had0 ? __uint_as_float(x[e]) * f0 : 0.f;
          if (!PAIR && had1) o[e] += __uint_as_float(y[e]) * f1;
        }
        if (!real) {
        } else if (whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8)
            if (c + e < dim)
              *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(pack_pair<F16>(o[e] * inv, o[e + 1] * inv), pack_pair<F16>(o[e + 2] * inv, o[e + 3] * inv),
                                                                  pack_pair<F16>(o[e + 4] * inv, o[e + 5] * inv), pack_pair<F16>(o[e + 6] * inv, o[e + 7] * inv));
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(part + part_at(TILE_ROWS, part_row, (c + e) / 4)) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      if (real && !whole && (PAIR || stream == 0)) *reinterpret_cast<float2*>(part + part_at(TILE_ROWS, part_row, DIM / 4)) = make_float2(m, l);
      ptx::tc_fence_before_sync();
      if (!PAIR) rows_sync<COMPUTERS>(3);   // the sums are out of tensor memory, and what was told is read, before either goes on
      if (tid == 0 && started == 0 && !whole)
        a.items[blockIdx.x] =
            SplitItem{(int)((first + at.units - 1) / run) - (int)blockIdx.x + 1, at.first_row, at.tile * TILE_ROWS, at.nodes * group, at.head};
      at.skip(line, units);
    }
  }
  if (dead && lane == 0 && a.io.status) atomicMax(a.io.status, abort_flag);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  if (warp == MAKERS) ptx::tmem_dealloc(tmem, S::COLUMNS);
}

template <bool F16, int DIM, bool PAIR, bool GROWS>
int launch(const AttnArgs& a, int sms, cudaStream_t s) {
  using S = Shape<DIM, PAIR>;
  auto kernel = tree_attention_umma_kernel<F16, DIM, PAIR, GROWS>;
  CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::bytes(KV_MAX_SEQUENCES)));
  CUtensorMap km, vm;
  B200Q_TRY(make_map(&km, a, a.cache.k));
  B200Q_TRY(make_map(&vm, a, a.cache.v));
  B200Q_TRY(launch_dependent(kernel, dim3(sms), dim3(BLOCK), S::bytes(a.pool.sequences), s, km, vm, a));
  return launch_join(a, sms, S::TILES * ROWS, DIM, s);
}
template <bool F16, int DIM>
int launch_form(const AttnArgs& a, bool pair, bool grows, int sms, cudaStream_t s) {
  if (grows) return launch<F16, DIM, true, true>(a, sms, s);
  return pair ? launch<F16, DIM, true, false>(a, sms, s) : launch<F16, DIM, false, false>(a, sms, s);
}
template <bool F16>
int launch_dim(const AttnArgs& a, bool pair, bool grows, int sms, cudaStream_t s) {
  return a.cache.head_dim <= 64 ? launch_form<F16, 64>(a, pair, grows, sms, s) : launch_form<F16, 128>(a, pair, grows, sms, s);
}

}  // namespace

namespace attn {
int launch_umma(const AttnArgs& a, bool pair, bool grows, int sms, cudaStream_t s) {
  return a.cache.dtype == B200Q_DT_F16 ? launch_dim<true>(a, pair, grows, sms, s) : launch_dim<false>(a, pair, grows, sms, s);
}
}  // namespace attn
}  // namespace b200q
