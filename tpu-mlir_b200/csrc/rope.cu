// Rotary positions of 16-bit heads, alone and joined with the write of keys and values into the paged cache.
//
// Pair i of a row at position p is turned by a = p * f_i: (x0, x1) -> m (x0 cos a - x1 sin a, x1 cos a + x0 sin a).  The angle is
// formed and brought into one turn in 64 bits (at position 131072 a 32-bit product is off by 2^-8 of a radian), and its sine and cosine are
// taken once for a (row, pair) and shared by all heads of the row through shared memory.
//
// What bounds it: HBM for prompts, where every element is read and written once (16 bytes a thread and access): 3 prompts of 1300 to 3900 tokens
// appended, 195 MB, in 36.3 us, 5.4 TB/s, 0.82 of the measured copy rate; 8000 rows of 48 heads of 128 rotated alone, 197 MB, in 33.6 us,
// 5.85 TB/s, 0.89.  For a token, launch and one row's chain sequence -> length -> page -> write (3.4 us).  Occupancy counts for more than loads in
// flight a thread: four pieces a thread at once, at 64 registers, took 45 us for the prompts that took 37.
// Not WIDE (half of the rotated part no multiple of 8 without interleaving, rows off 16 bytes): 2 bytes an access, in all of the head.  8000 rows of 64
// heads of 96 with 24 rotated take 106 us where the bytes would take 30.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "kv_cache.h"
#include "ptx_sm100.cuh"

namespace b200q {
namespace {

constexpr int ROPE_THREADS = 256, ROPE_ROWS = 8;   // most rows of a block: a warp finds each one's sequence

struct RopeArgs {
  b200q_rope_plan plan;
  b200q_kv_cache cache;
  b200q_kv_pool pool;
  b200q_rope_append io;   // k == nullptr: queries only
  int heads;              // q heads, then (with k) the cache's heads twice: keys and values
  int rows_per_block, heads_per_block;
};

template <bool F16>
__device__ __forceinline__ float to_f32(uint32_t bits16) {
  return F16 ? __half2float(__ushort_as_half((unsigned short)bits16)) : __uint_as_float(bits16 << 16);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where a pair's cosine and sine stand in a row's table: neighbouring threads take neighbouring pieces, so what they read together stands
// side by side (two pairs of a piece of eight, one of a piece of four; in the pairs' own order four threads met on a bank).
template <bool INTERLEAVED, bool WIDE>
__device__ __forceinline__ int turn_at(int pair, int half) {
  if (!WIDE) return pair;
  if (INTERLEAVED) return (pair & 3) * ((half + 3) / 4) + (pair >> 2);
  return ((pair >> 1 & 3) * (half / 8) + (pair >> 3)) * 2 + (pair & 1);
}
__host__ __device__ __forceinline__ int turn_size(int half) { return (half + 3) / 4 * 4; }

// WIDE: 16 bytes at a time (aligned rows and heads; the two halves of a non-interleaved head start on 16 bytes), else one pair.
template <bool F16, bool INTERLEAVED, bool WIDE>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const __grid_constant__ RopeArgs a) {
  extern __shared__ __align__(16) float2 turn[];   // [rows_per_block][turn_size] (cos, sin), the magnitude in both
  __shared__ int row_seq[ROPE_ROWS];
  __shared__ double row_pos[ROPE_ROWS];   // (past 31 bits where a length is near them)
  __shared__ int64_t row_entry[ROPE_ROWS];
  const b200q_rope_append& io = a.io;
  const int half = a.plan.rotary_dim / 2, dim = a.plan.head_dim;
  const int64_t r0 = (int64_t)blockIdx.x * a.rows_per_block;
  const int rows = (int)(io.rows - r0 < a.rows_per_block ? io.rows - r0 : a.rows_per_block);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();

  if (warp < rows) {
    const int64_t r = r0 + warp;
    int seq = 0;
    int64_t pos = 0, entry = -1;
    if (io.row_start) {
      // the last sequence that starts at or before the row (the starts ascend)
      int before = 0;
      for (int s = lane; s < a.pool.sequences; s += 32) before += io.row_start[s] <= r;
      seq = __reduce_add_sync(0xffffffffu, before) - 1;
      if (seq >= 0 && r < io.row_start[seq + 1]) {
        // (the length as it is: one past the table's row has no page, but it is where the row belongs)
        const int length = a.pool.length[seq];
        pos = (length < 0 ? 0 : length) + (r - io.row_start[seq]);
        if (pos <= 0x7fffffff) entry = kv_entry(a.cache, a.pool, seq, (int)pos);
      } else {
        seq = -1;
      }
    }
    if (io.positions) pos = io.positions[r];
    if (lane == 0) {
      row_seq[warp] = seq;
      row_pos[warp] = (double)pos;
      row_entry[warp] = entry;
    }
  }
  __syncthreads();
  if (half) {
    // a thread keeps to one pair (its frequency is read once) and goes through rows
    const int at_once = ROPE_THREADS / half, pair = threadIdx.x % half;
    const double turns_per_position = a.plan.frequency[pair] * 0.15915494309189533577;
    for (int row = threadIdx.x / half; row < rows && (int)threadIdx.x < at_once * half; row += at_once) {
      double t = row_pos[row] * turns_per_position;
      t -= rint(t);
      float s, c;
      sincospif(2.f * (float)t, &s, &c);
      turn[row * turn_size(half) + turn_at<INTERLEAVED, WIDE>(pair, half)] = make_float2(c * a.plan.magnitude, s * a.plan.magnitude);
    }
  }
  __syncthreads();

  const int h0 = blockIdx.y * a.heads_per_block, heads = min(a.heads - h0, a.heads_per_block);
  // pieces of a head: WIDE and not interleaved: rotary / 16 pieces of eight pairs, then the rest by eight elements;
  // WIDE and interleaved: eight elements; else: a pair, then the rest by two elements (dim is even)
  const int turned = WIDE ? (INTERLEAVED ? dim / 8 : half / 8) : half;
  const int pieces = turned + (WIDE ? (INTERLEAVED ? 0 : (dim - 2 * half) / 8) : (dim - 2 * half) / 2);
  // pieces ROPE_THREADS apart: (row, head, piece) goes on by the step's own three digits, with carries (two divisions a piece took longer
  // than its arithmetic)
  const int step_piece = ROPE_THREADS % pieces, step_head = ROPE_THREADS / pieces % heads, step_row = ROPE_THREADS / pieces / heads;
  int piece = threadIdx.x % pieces, head = threadIdx.x / pieces % heads, row = threadIdx.x / pieces / heads;
  auto go_on = [&]() {
    piece += step_piece;
    head += step_head;
    row += step_row;
    if (piece >= pieces) {
      piece -= pieces;
      ++head;
    }
    if (head >= heads) {
      head -= heads;
      ++row;
    }
  };
  for (; row < rows; go_on()) {
    int h = h0 + head;
    if (row_seq[row] < 0) continue;
    const int64_t r = r0 + row;
    const uint16_t* x;
    uint16_t* y;
    bool turns = true;
    if (h < io.q_heads) {
      x = static_cast<const uint16_t*>(io.q) + r * io.q_row_stride + h * io.q_head_stride;
      y = static_cast<uint16_t*>(io.q_out) + r * io.q_out_row_stride + h * io.q_out_head_stride;
    } else {
      if (row_entry[row] < 0) continue;
      h -= io.q_heads;
      turns = h < a.cache.heads;
      if (!turns) h -= a.cache.heads;
      x = turns ? static_cast<const uint16_t*>(io.k) + r * io.k_row_stride + h * io.k_head_stride
                : static_cast<const uint16_t*>(io.v) + r * io.v_row_stride + h * io.v_head_stride;
      y = static_cast<uint16_t*>(turns ? a.cache.k : a.cache.v) + io.layer * a.cache.layer_stride + row_entry[row] + h * a.cache.head_stride;
    }
    const float2* t = turn + row * turn_size(half);
    if (WIDE && INTERLEAVED) {
      uint4 v = *reinterpret_cast<const uint4*>(x + piece * 8);
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int pair = piece * 4 + j;
        if (turns && pair < half) {
          const float2 cs = t[turn_at<true, true>(pair, half)];
          const float p = to_f32<F16>(w[j] & 0xffffu), q = to_f32<F16>(w[j] >> 16);
          w[j] = pack2<F16>(p * cs.x - q * cs.y, q * cs.x + p * cs.y);
        }
      }
      *reinterpret_cast<uint4*>(y + piece * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if (WIDE) {
      if (piece < turned) {
        const uint4 vp = *reinterpret_cast<const uint4*>(x + piece * 8), vq = *reinterpret_cast<const uint4*>(x + half + piece * 8);
        uint32_t wp[4] = {vp.x, vp.y, vp.z, vp.w}, wq[4] = {vq.x, vq.y, vq.z, vq.w};
        if (turns) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 cs = *reinterpret_cast<const float4*>(t + turn_at<false, true>(piece * 8 + 2 * j, half));   // two pairs
            const float2 c0 = make_float2(cs.x, cs.y), c1 = make_float2(cs.z, cs.w);
            const float p0 = to_f32<F16>(wp[j] & 0xffffu), p1 = to_f32<F16>(wp[j] >> 16);
            const float q0 = to_f32<F16>(wq[j] & 0xffffu), q1 = to_f32<F16>(wq[j] >> 16);
            wp[j] = pack2<F16>(p0 * c0.x - q0 * c0.y, p1 * c1.x - q1 * c1.y);
            wq[j] = pack2<F16>(q0 * c0.x + p0 * c0.y, q1 * c1.x + p1 * c1.y);
          }
        }
        *reinterpret_cast<uint4*>(y + piece * 8) = make_uint4(wp[0], wp[1], wp[2], wp[3]);
        *reinterpret_cast<uint4*>(y + half + piece * 8) = make_uint4(wq[0], wq[1], wq[2], wq[3]);
      } else {
        const int e = 2 * half + (piece - turned) * 8;
        *reinterpret_cast<uint4*>(y + e) = *reinterpret_cast<const uint4*>(x + e);
      }
    } else {
      const int e0 = piece < turned ? (INTERLEAVED ? 2 * piece : piece) : 2 * half + 2 * (piece - turned);
      const int e1 = piece < turned && !INTERLEAVED ? piece + half : e0 + 1;
      uint32_t p = x[e0], q = x[e1];
      if (turns && piece < turned) {
        const float2 cs = t[piece];
        const float fp = to_f32<F16>(p), fq = to_f32<F16>(q);
        const uint32_t w = pack2<F16>(fp * cs.x - fq * cs.y, fq * cs.x + fp * cs.y);
        p = w & 0xffffu;
        q = w >> 16;
      }
      y[e0] = (uint16_t)p;
      y[e1] = (uint16_t)q;
    }
  }
}

int check_plan(const char* who, const b200q_rope_plan* p) {
  if (!p) return set_error(B200Q_ERR_INVALID, "%s: null plan", who);
  if (p->head_dim < 2 || p->head_dim > KV_MAX_HEAD_DIM || (p->head_dim & 1) || p->rotary_dim < 0 || p->rotary_dim > p->head_dim || (p->rotary_dim & 1))
    return set_error(B200Q_ERR_INVALID, "%s: head_dim and rotary_dim must be even, rotary_dim <= head_dim <= %d", who, KV_MAX_HEAD_DIM);
  return B200Q_OK;
}

int launch_rope(RopeArgs& a, bool f16, bool wide, int sms, cudaStream_t s) {
  const bool interleaved = a.plan.interleaved != 0;
  const int half = a.plan.rotary_dim / 2;
  wide = wide && a.plan.head_dim % 8 == 0 && (interleaved || half % 8 == 0);
  const int pieces = wide ? (interleaved ? a.plan.head_dim / 8 : half / 8 + (a.plan.head_dim - 2 * half) / 8) : a.plan.head_dim / 2;
  // Rows of a block: three pieces a thread (8000 rows of 48 heads of 128: 33.5 us with two rows, 34.8 with four, 39.3 with eight, 36.8 with one:
  // sines are taken once for a row of a block, but short blocks hide each other's start), fewer where that leaves no four blocks an SM.  With still
  // fewer rows the heads are spread over blocks until a thread has one piece, and every block takes the row's sines for itself.
  int rows = 1;
  while (rows < ROPE_ROWS && (int64_t)rows * a.heads * pieces < 3 * ROPE_THREADS) rows *= 2;
  while (rows > 1 && (a.io.rows + rows - 1) / rows < 4LL * sms) rows /= 2;
  int splits = 1;
  while (a.io.rows * splits < 4LL * sms && (int64_t)rows * ((a.heads + splits - 1) / splits) * pieces > ROPE_THREADS && splits < a.heads) splits *= 2;
  a.rows_per_block = rows;
  a.heads_per_block = (a.heads + splits - 1) / splits;
  const int64_t blocks = (a.io.rows + rows - 1) / rows;
  if (blocks > 0x7fffffffLL) return set_error(B200Q_ERR_UNSUPPORTED, "rope: too many rows");
  const dim3 grid((unsigned)blocks, (a.heads + a.heads_per_block - 1) / a.heads_per_block);
  const size_t smem = (size_t)rows * turn_size(half) * sizeof(float2);
#define B200Q_ROPE(F, I, W) return launch_dependent(rope_kernel<F, I, W>, grid, dim3(ROPE_THREADS), smem, s, a)
  if (f16) {
    if (interleaved) { if (wide) B200Q_ROPE(true, true, true); else B200Q_ROPE(true, true, false); }
    else { if (wide) B200Q_ROPE(true, false, true); else B200Q_ROPE(true, false, false); }
  } else {
    if (interleaved) { if (wide) B200Q_ROPE(false, true, true); else B200Q_ROPE(false, true, false); }
    else { if (wide) B200Q_ROPE(false, false, true); else B200Q_ROPE(false, false, false); }
  }
#undef B200Q_ROPE
}

bool aligned16(const void* p, int64_t row_stride, int64_t head_stride) {
  return !(((uintptr_t)p & 15) | ((row_stride | head_stride) & 7));
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_rope_plan_init(b200q_rope_plan* plan, int32_t head_dim, int32_t rotary_dim, int32_t interleaved, double base,
                         const b200q_rope_scaling* scaling) {
  if (!plan) return set_error(B200Q_ERR_INVALID, "rope_plan_init: null plan");
  b200q_rope_plan p{};
  p.head_dim = head_dim;
  p.rotary_dim = rotary_dim;
  p.interleaved = interleaved != 0;
  p.magnitude = 1.f;
  B200Q_TRY(check_plan("rope_plan_init", &p));
  if (!(base > 1.0) || !isfinite(base)) return set_error(B200Q_ERR_INVALID, "rope_plan_init: base must be above 1");
  const int kind = scaling ? scaling->kind : B200Q_ROPE_SCALING_NONE;
  const double factor = kind == B200Q_ROPE_SCALING_NONE ? 1.0 : scaling->factor, r = rotary_dim;
  if (kind < B200Q_ROPE_SCALING_NONE || kind > B200Q_ROPE_SCALING_BANDED) return set_error(B200Q_ERR_INVALID, "rope_plan_init: unknown scaling %d", kind);
  if (!(factor >= 1.0) || !isfinite(factor)) return set_error(B200Q_ERR_INVALID, "rope_plan_init: the factor must be at least 1");
  const bool two_ends = kind == B200Q_ROPE_SCALING_YARN || kind == B200Q_ROPE_SCALING_BANDED;
  if (two_ends && (!(scaling->original_positions > 0) || !isfinite(scaling->original_positions) || !(scaling->low_turns > 0) ||
                   !(scaling->high_turns > scaling->low_turns) || !isfinite(scaling->high_turns)))
    return set_error(B200Q_ERR_INVALID, "rope_plan_init: original_positions must be positive and 0 < low_turns < high_turns");
  const double two_pi = 6.283185307179586476925;
  if (kind == B200Q_ROPE_SCALING_STRETCHED && r > 2) base *= pow(factor, r / (r - 2));
  double first = 0, last = 0;
  if (kind == B200Q_ROPE_SCALING_YARN) {
    // the pairs (not rounded) that turn high_turns and low_turns times over original_positions, rounded outwards
    const double span = scaling->original_positions / two_pi;
    first = fmax(floor(r * log(span / scaling->high_turns) / (2 * log(base))), 0.0);
    last = fmin(ceil(r * log(span / scaling->low_turns) / (2 * log(base))), r - 1);
    p.magnitude = (float)(0.1 * log(factor) + 1.0);
  }
  for (int i = 0; i < rotary_dim / 2; ++i) {
    double f = pow(base, -2.0 * i / r);
    if (kind == B200Q_ROPE_SCALING_LINEAR) {
      f /= factor;
    } else if (kind == B200Q_ROPE_SCALING_YARN) {
      const double mix = fmin(fmax((i - first) / fmax(last - first, 0.001), 0.0), 1.0);
      f = f / factor * mix + f * (1 - mix);
    } else if (kind == B200Q_ROPE_SCALING_BANDED) {
      const double turns = scaling->original_positions * f / two_pi;
      const double mix = fmin(fmax((turns - scaling->low_turns) / (scaling->high_turns - scaling->low_turns), 0.0), 1.0);
      f *= (1 - mix) / factor + mix;
    }
    p.frequency[i] = f;
  }
  *plan = p;
  return B200Q_OK;
}

int b200q_rope_dev(const b200q_rope_plan* plan, const void* x, void* y, const int32_t* positions, int64_t rows, int32_t heads,
                   int64_t x_row_stride, int64_t x_head_stride, int64_t y_row_stride, int64_t y_head_stride, int32_t dtype, void* stream) {
  B200Q_TRY(check_plan("rope", plan));
  if (!x || !y || !positions) return set_error(B200Q_ERR_INVALID, "rope: null argument");
  if (rows < 0 || heads < 0) return set_error(B200Q_ERR_INVALID, "rope: bad shape");
  if (heads > 65535) return set_error(B200Q_ERR_UNSUPPORTED, "rope: at most 65535 heads");
  if (dtype != B200Q_DT_BF16 && dtype != B200Q_DT_F16) return set_error(B200Q_ERR_UNSUPPORTED, "rope: dtype must be bf16 or f16");
  if (((uintptr_t)x | (uintptr_t)y) & 1) return set_error(B200Q_ERR_INVALID, "rope: x and y must be 2-byte aligned");
  if ((uintptr_t)positions & 3) return set_error(B200Q_ERR_INVALID, "rope: positions must be 4-byte aligned");
  if (x == y && (x_row_stride != y_row_stride || x_head_stride != y_head_stride))
    return set_error(B200Q_ERR_INVALID, "rope: in place, the strides of x and y must be the same");
  if (rows == 0 || heads == 0) return B200Q_OK;
  OnDeviceOf dev("rope", x);
  B200Q_TRY(dev.rc);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  RopeArgs a{};
  a.plan = *plan;
  a.io.q = x;
  a.io.q_out = y;
  a.io.positions = positions;
  a.io.q_row_stride = x_row_stride;
  a.io.q_head_stride = x_head_stride;
  a.io.q_out_row_stride = y_row_stride;
  a.io.q_out_head_stride = y_head_stride;
  a.io.rows = rows;
  a.io.q_heads = a.heads = heads;
  const bool wide = aligned16(x, x_row_stride, x_head_stride) && aligned16(y, y_row_stride, y_head_stride);
  return launch_rope(a, dtype == B200Q_DT_F16, wide, sms, static_cast<cudaStream_t>(stream));
}

int b200q_rope_append_dev(const b200q_rope_plan* plan, const b200q_kv_cache* cache, const b200q_kv_pool* pool,
                          const b200q_rope_append* args, void* stream) {
  B200Q_TRY(check_plan("rope_append", plan));
  B200Q_TRY(kv_check_cache("rope_append", cache));
  B200Q_TRY(kv_check_pool("rope_append", pool));
  if (!args) return set_error(B200Q_ERR_INVALID, "rope_append: null args");
  const b200q_rope_append& io = *args;
  if (!io.q || !io.q_out || !io.k || !io.v || !io.row_start) return set_error(B200Q_ERR_INVALID, "rope_append: null argument");
  if (plan->head_dim != cache->head_dim) return set_error(B200Q_ERR_INVALID, "rope_append: the plan's head_dim is not the cache's");
  if (io.rows < 0 || io.q_heads < 0) return set_error(B200Q_ERR_INVALID, "rope_append: bad shape");
  if (io.q_heads > 65535) return set_error(B200Q_ERR_UNSUPPORTED, "rope_append: at most 65535 heads");
  if (io.layer < 0 || io.layer >= cache->layers) return set_error(B200Q_ERR_INVALID, "rope_append: no layer %d in the cache", io.layer);
  if (((uintptr_t)io.q | (uintptr_t)io.q_out | (uintptr_t)io.k | (uintptr_t)io.v) & 1)
    return set_error(B200Q_ERR_INVALID, "rope_append: q, q_out, k and v must be 2-byte aligned");
  if (((uintptr_t)io.row_start | (uintptr_t)io.positions) & 3)
    return set_error(B200Q_ERR_INVALID, "rope_append: row_start and positions must be 4-byte aligned");
  if (io.q == io.q_out && (io.q_row_stride != io.q_out_row_stride || io.q_head_stride != io.q_out_head_stride))
    return set_error(B200Q_ERR_INVALID, "rope_append: in place, the strides of q and q_out must be the same");
  if (io.rows == 0 || pool->sequences == 0) return B200Q_OK;
  OnDeviceOf dev("rope_append", pool->table);
  B200Q_TRY(dev.rc);
  const int sms = sm_count(dev.device);
  if (sms < 0) return sms;
  RopeArgs a{};
  a.plan = *plan;
  a.cache = *cache;
  a.pool = *pool;
  a.io = io;
  a.heads = io.q_heads + 2 * cache->heads;
  const bool wide = aligned16(io.q, io.q_row_stride, io.q_head_stride) && aligned16(io.q_out, io.q_out_row_stride, io.q_out_head_stride) &&
                    aligned16(io.k, io.k_row_stride, io.k_head_stride) && aligned16(io.v, io.v_row_stride, io.v_head_stride);
  return launch_rope(a, cache->dtype == B200Q_DT_F16, wide, sms, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
