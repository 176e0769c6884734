// The step between two blocks of a transformer, with 8-bit checkpoints of what its backward pass needs:
//   n = N_post(block)                     (or block itself)
//   y = round(alpha x + gate * n)         the residual stream, rounded to its type
//   h = N_pre(y)                          the next block's input
// N is an RMS norm  v r w  or a layer norm  (v - m) r w + b,  r = 1 / sqrt(mean (v - m)^2 + eps); a gate is a row of
// factors for every token or for every token of a sequence.  Kept: checkpoints y~ of y and (with N_post or a gate) b~
// of block, and the fp32 statistics m, r of both norms, which are those of the unrounded-to-8-bits values.
//
// Backward, from dh and (where the stream goes on) dy, with y^ = (y~ - m) r and b^ = (b~ - m) r:
//   c = dh w,  t = r (c - mean(c) - y^ mean(c y^))            (RMS: without mean(c))
//   g = t + dy,  dx = alpha g,  e = gate g
//   dblock = e, or the same norm backward of e w_post at b^
//   dw = sum dh y^, db = sum dh;  G1 = sum g b^, G0 = sum g over a sequence, from which
//   dw_post = sum gate G1, db_post = sum gate G0, dgate = w_post G1 + b_post G0 follow, since a sequence has one gate.
//
// Both passes are bound by memory: forward 4 tensors of the type's width and 1 or 2 checkpoints, 10 bytes an element for
// bf16 with everything, backward the same; 7 and 5 for "add and norm" alone, whose stream nobody reads.  A row is held
// in registers, sixteen columns a thread, by one warp or several, so that statistics and results take one pass over
// memory; small rows share a CTA.  A CTA walks a run of rows that belong to one
// sequence: its parameters and its gate stay in shared memory (fetched anew for every row, from L2, they cost three
// times what the row does), and the next row's loads are under way while this one is reduced and written.
// Sums over tokens: a CTA keeps its columns' sums in registers over its run and stores them once; a second kernel
// adds the runs' sums in a fixed order (no atomics: the same bits on every run).
// Measured, bf16, L2 cold: RMS sandwich with a gate a sequence, 16384 x 4096: forward 124 us (5.4 TB/s), backward 164 us
// (4.1 TB/s) and 15 us for the sums (forward with a residual factor that fp32 does not hold 2 us more); "add and norm" 4096 x
// 1024: 11.8, 10.8 and 5.6 us.  The backward pass is short of
// registers: 128 a thread allow two CTAs, whose 16 warps an SM leave a third of the issue slots empty.  A variant without
// the ragged forms of loads and stores, and one that fetched the next row into shared memory, took 14 % longer.  Rows off 16-byte
// boundaries are accessed by single elements: bf16 16384 x 4095 against x 4096, RMS norm alone, with the launch, forward 825
// and 85 us, backward 454 and 79.
// A run never crosses from one sequence to the next where each has a gate, so a number of sequences just above the number of
// places for runs (two CTAs an SM at 4096 columns) leaves most of a second wave empty, and the workspace of the sums, 16 bytes a
// column for each run, is at least that for each sequence.
#include <algorithm>

#include "act8.cuh"
#include "act8.h"
#include "common.cuh"
#include "gradio.cuh"

namespace grace {
namespace {

// Columns col .. col + 3 of a row of parameters, fp32 or of the activations' type; past the end, or without such parameters:
// `none`.  Loading and converting are two steps, so that the loads of all parameters are under way together: one after
// the other they took most of a small call's time.
template <class T>
struct Param4 {
  unsigned w[4];
  __device__ __forceinline__ void load(const BlockNormArgs& a, const void* p, int col) {
    w[0] = w[1] = w[2] = w[3] = 0u;
    if (p == nullptr || col >= a.cols) return;
    if (a.params_vec) {       // (then columns come in fours)
      if (sizeof(T) == 4 || a.params_f32) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const float*>(p) + col));
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + col));
        w[0] = v.x & 0xffffu; w[1] = v.x >> 16; w[2] = v.y & 0xffffu; w[3] = v.y >> 16;
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < a.cols) w[j] = sizeof(T) == 4 || a.params_f32 ? __ldg(static_cast<const unsigned*>(p) + col + j) : __ldg(static_cast<const unsigned short*>(p) + col + j);
  }
  __device__ __forceinline__ float4 get(const BlockNormArgs& a, const void* p, int col, float none) const {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (p == nullptr || col + j >= a.cols) {
        v[j] = none;
      } else if (sizeof(T) == 4 || a.params_f32) {
        v[j] = __uint_as_float(w[j]);
      } else {
        const unsigned short bits = (unsigned short)w[j];
        v[j] = to_f32<T>(*reinterpret_cast<const T*>(&bits));
      }
    }
    return make_float4(v[0], v[1], v[2], v[3]);
  }
};

// A row of parameters in shared memory, fp32, for `chunks` chunks of sixteen columns: the first quarters of all chunks,
// then the second ones, and so on, so that a quarter warp's 16-byte accesses are consecutive.
struct SharedRow {
  float4* at;
  int chunks;
  __device__ __forceinline__ void put(int i, float4 v) const { at[(i & 3) * chunks + (i >> 2)] = v; }   // columns 4 i .. 4 i + 3
  __device__ __forceinline__ void get(int chunk, float (&v)[16]) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 x = at[q * chunks + chunk];
      v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
    }
  }
};
__device__ __forceinline__ float4 times(float4 a, float4 b) { return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w); }
__device__ __forceinline__ float4 first_of(float4 v, int n) {    // its first n numbers, then zeros
  return make_float4(n > 0 ? v.x : 0.f, n > 1 ? v.y : 0.f, n > 2 ? v.z : 0.f, n > 3 ? v.w : 0.f);
}

// The rows of this CTA's run: run = sequence * parts + part, rows [part * L / parts, (part + 1) * L / parts) of the
// sequence, L = gate_rows (all rows are one sequence where no gate belongs to a sequence).
struct Run {
  long long row0, row1, seq;
};
__device__ __forceinline__ Run run_of(const BlockNormArgs& a) {
  const long long run = blockIdx.x, seq = run / a.parts, part = run - seq * a.parts, length = a.gate_rows ? a.gate_rows : a.rows;
  return {seq * length + part * length / a.parts, seq * length + (part + 1) * length / a.parts, seq};
}
template <class T>
__device__ __forceinline__ const void* gate_of(const BlockNormArgs& a, const Run& run) {
  if (!a.gate || !a.gate_rows) return a.gate;
  return static_cast<const char*>(a.gate) + run.seq * a.cols * (a.params_f32 ? 4 : (long long)sizeof(T));
}

constexpr int kMaxSums = 7;                      // values that one reduction may add up
constexpr int kSumFloats = 2 * kMaxSums * 32;    // shared memory of the reductions

// Sums over the `tpr` threads (whole warps) that share a row, the same value in all of them: shuffles within a warp, then
// every thread adds the warps' sums from shared memory (a few 16-byte broadcasts take less time than five more
// shuffles).  Every thread of the CTA calls it.  Two buffers alternate: a warp cannot be two reductions ahead of another.
struct RowSum {
  float* buf;
  int parity, warps, first, warp;   // warps of a row, the first of this row's, this one
  __device__ __forceinline__ RowSum(float* b, int tpr) : buf(b), parity(0), warps(tpr >> 5), warp(threadIdx.x >> 5) { first = warp / warps * warps; }
  __device__ __forceinline__ float* next() {
    float* const b = buf + parity * (kMaxSums * 32);
    parity ^= 1;
    return b;
  }
  // w[warp] = x of each of the row's warps, visible after the next barrier; the same for all of the row's threads
  __device__ __forceinline__ float total(const float* w) const {
    float s = 0.f;
    if ((warps & 3) == 0) {
      for (int i = 0; i < warps; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(w + first + i);
        s += (x.x + x.y) + (x.z + x.w);
      }
    } else {
      for (int i = 0; i < warps; ++i) s += w[first + i];
    }
    return s;
  }
  template <int N>
  __device__ __forceinline__ void operator()(float (&v)[N]) {
    static_assert(N <= kMaxSums, "");
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (warps == 1) return;
    float* const b = next();
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) b[i * 32 + warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = total(b + i * 32);
  }
};

// sum of a[j] b[j], in four chains
__device__ __forceinline__ float dot16(const float (&a)[16], const float (&b)[16]) {
  F2 s = mul2(pair(a, 0), pair(b, 0)), t = mul2(pair(a, 1), pair(b, 1));
#pragma unroll
  for (int i = 2; i < 8; i += 2) {
    s = fma2(pair(a, i), pair(b, i), s);
    t = fma2(pair(a, i + 1), pair(b, i + 1), t);
  }
  return s.sum() + t.sum();
}
__device__ __forceinline__ float sum16(const float (&a)[16]) {
  F2 s = pair(a, 0), t = pair(a, 1);
#pragma unroll
  for (int i = 2; i < 8; i += 2) {
    s = add2(s, pair(a, i));
    t = add2(t, pair(a, i + 1));
  }
  return s.sum() + t.sum();
}
// v = v * w, v * w + u and the like, for sixteen columns
__device__ __forceinline__ void mul16(float (&v)[16], const float (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) put(v, i, mul2(pair(v, i), pair(w, i)));
}
__device__ __forceinline__ void add16(float (&v)[16], const float (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) put(v, i, add2(pair(v, i), pair(w, i)));
}
__device__ __forceinline__ void add_product16(float (&v)[16], const float (&a)[16], const float (&b)[16]) {      // v += a b
#pragma unroll
  for (int i = 0; i < 8; ++i) put(v, i, fma2(pair(a, i), pair(b, i), pair(v, i)));
}
__device__ __forceinline__ void add_scaled16(float (&v)[16], float c, const float (&a)[16]) {      // v += c a
#pragma unroll
  for (int i = 0; i < 8; ++i) put(v, i, fma2(F2(c), pair(a, i), pair(v, i)));
}
// (v - mean) * r: the difference first, since a mean far from zero must not cost digits
template <bool LAYER>
__device__ __forceinline__ void normalise16(float (&v)[16], float mean, float r) {
#pragma unroll
  for (int i = 0; i < 8; ++i) put(v, i, mul2(LAYER ? add2(pair(v, i), F2(-mean)) : pair(v, i), F2(r)));
}

// 1 / sqrt(sum / cols + eps): the quotient and the hardware's root each with one correction by their remainder.  An error
// here is one of the whole row, all of whose values it would push the same way across the borders of their rounding.
__device__ __forceinline__ float inv_deviation(float sum, float cols, float inv_cols, float eps) {
  float x = sum * inv_cols;
  x = fmaf(fmaf(-x, cols, sum), inv_cols, x) + eps;
  const float r = rsqrtf(x), h = x * r;
  return fmaf(0.5f * r, fmaf(-h, r, 1.f), r);
}

// (mean, 1 / deviation) of a row, sixteen columns a thread.  Layer norm: each warp's mean and squared deviations from
// it, joined over the warps by Chan, Golub and LeVeque's formula, so that one barrier does and nothing cancels.
template <bool LAYER>
__device__ __forceinline__ float2 row_stats(const float (&v)[16], int valid, int cols, float inv_cols, float eps, RowSum& sum) {
  if (!LAYER) {
    float s[1] = {dot16(v, v)};      // (columns past the end are zeros)
    sum(s);
    return make_float2(0.f, inv_deviation(s[0], (float)cols, inv_cols, eps));
  }
  const float n = (float)min(512, max(0, cols - (sum.warp - sum.first) * 512));
  const float inv_n = n > 0.f ? __fdividef(1.f, n) : 0.f;
  float m = warp_sum(sum16(v)) * inv_n, d;
  float x[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = j < valid ? v[j] - m : 0.f;
  d = warp_sum(dot16(x, x));
  if (sum.warps > 1) {
    float* const b = sum.next();
    if ((threadIdx.x & 31) == 0) {
      b[sum.warp] = m;
      b[32 + sum.warp] = d;
    }
    __syncthreads();
    float total = 0.f;
    for (int i = 0; i < sum.warps; ++i) total = fmaf((float)min(512, max(0, cols - i * 512)), b[sum.first + i], total);
    m = total * inv_cols;
    d = 0.f;
    for (int i = 0; i < sum.warps; ++i) {
      const float off = b[sum.first + i] - m;
      d += fmaf((float)min(512, max(0, cols - i * 512)) * off, off, b[32 + sum.first + i]);
    }
  }
  return make_float2(m, inv_deviation(d, (float)cols, inv_cols, eps));
}

// The codes at columns col .. col + 15 of a row and, from the lane with a group's first columns, its scale byte.
__device__ __forceinline__ void put_codes(const Held& h, long long row, int col, uint4 codes, unsigned s) {
  *reinterpret_cast<uint4*>(h.codes + row * h.pitch + col) = codes;
  if ((col & 31) == 0) h.scales[row * h.spitch + (col >> 5)] = (unsigned char)s;
}

// v += alpha x, where alpha is the sum of two fp32 numbers (a caller's 2.63 is none) of which the second is mostly zero.  Where
// x or the product is infinite the second part says nothing, and of the other sign it would make a NaN of the sum.
__device__ __forceinline__ void add_scaled(float alpha, float alpha_low, const float (&x)[16], float (&v)[16]) {
  constexpr float kMax = 3.4028235e38f;
  if (alpha_low != 0.f) {
    float top = max_abs(x[0], x[1], x[2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) top = max_abs(top, x[j], x[j + 1]);
    top = max_abs(top, x[15], 0.f);
    if (fabsf(alpha_low) * top <= kMax) {      // (not where one of them is a NaN)
      add_scaled16(v, alpha_low, x);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float low = alpha_low * x[j];
        v[j] += fabsf(low) <= kMax ? low : 0.f;      // (a NaN comes with the other part)
      }
    }
  }
  add_scaled16(v, alpha, x);
}

// T: the stream's type, TB: the block's.  THREADS: 256 where a row takes no more, three CTAs an SM; 512
template <class T, class TB, bool PRE_LAYER, int POST, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1) block_norm_forward_kernel(const BlockNormArgs a, int tpr) {
  __shared__ __align__(16) float buf[kSumFloats];
  extern __shared__ float4 params[];
  const int rpb = blockDim.x / tpr, lane_row = threadIdx.x / tpr, t = threadIdx.x - lane_row * tpr;
  const int col = t * 16, valid = min(16, max(0, a.cols - col)), chunks = a.held_y.pitch / 16;
  const bool owns = col < a.held_y.pitch;      // (threads past the last group of 32 only take part in the sums)
  const int chunk = owns ? t : 0;
  const float inv_cols = 1.f / (float)a.cols;
  const Run run = run_of(a);
  RowSum sum(buf, tpr);
  Chunk16<TB> cb;
  Chunk16<T> cx;
  auto load = [&](long long row) {
    if (row < run.row1) {
      cb.load(static_cast<const TB*>(a.block) + row * a.block_stride, col, a.cols, a.block_vec);
      cx.load(static_cast<const T*>(a.x) + row * a.x_stride, col, a.cols, a.x_vec);
    } else {
      cb.zero();
      cx.zero();
    }
  };
  load(run.row0 + lane_row);
  // The norm after the block and the gate as one factor (and one summand) for each column.
  constexpr bool BIAS = POST == kNormLayer;
  const bool scaled = POST || a.gate;
  const SharedRow pre_w{params, chunks}, pre_b{params + 4 * chunks, chunks};
  const SharedRow u_row{params + (PRE_LAYER ? 8 : 4) * chunks, chunks}, ub_row{u_row.at + 4 * chunks, chunks};
  const void* const g = gate_of<T>(a, run);
  for (int i = threadIdx.x; i < 4 * chunks; i += blockDim.x) {
    Param4<T> w, b, u, ub, f;
    w.load(a, a.pre_weight, i * 4);
    if (PRE_LAYER) b.load(a, a.pre_bias, i * 4);
    if (POST) u.load(a, a.post_weight, i * 4);
    if (BIAS) ub.load(a, a.post_bias, i * 4);
    f.load(a, g, i * 4);
    pre_w.put(i, w.get(a, a.pre_weight, i * 4, 1.f));
    if (PRE_LAYER) pre_b.put(i, b.get(a, a.pre_bias, i * 4, 0.f));
    if (scaled) {
      const float4 gate = f.get(a, g, i * 4, 1.f);
      if (POST) u_row.put(i, times(u.get(a, a.post_weight, i * 4, 1.f), gate));
      else u_row.put(i, gate);
      if (BIAS) ub_row.put(i, times(ub.get(a, a.post_bias, i * 4, 0.f), gate));
    }
  }
  __syncthreads();

  for (long long base = run.row0; base < run.row1; base += rpb) {
    const long long row = base + lane_row;
    const bool in = row < run.row1;
    float v[16], w[16];
    cb.get(v);
    unsigned s;
    if (a.held_b.codes) {
      const uint4 codes = act8_encode(v, s);
      if (in && owns) put_codes(a.held_b, row, col, codes, s);
    }
    float2 post = make_float2(0.f, 1.f);
    if (POST) post = row_stats<POST == kNormLayer>(v, valid, a.cols, inv_cols, a.eps, sum);
    if (scaled) {
      u_row.get(chunk, w);
      if (POST) normalise16<POST == kNormLayer>(v, post.x, post.y);
      mul16(v, w);
      if (BIAS) {
        ub_row.get(chunk, w);
        add16(v, w);
      }
    }
    cx.get(w);
    add_scaled(a.alpha, a.alpha_low, w, v);
    load(row + rpb);       // the next row's loads are under way during the rest of this one
    if (valid < 16) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = j < valid ? v[j] : 0.f;
    }
    Chunk16<T> cy;
    cy.set(v);       // the stream as it is rounded to its type
    cy.get(v);
    if (in && a.y) store16(v, static_cast<T*>(a.y) + row * a.cols, col, a.cols, a.out_vec);
    if (a.held_y.codes) {
      const uint4 codes = act8_encode(v, s);
      if (in && owns) put_codes(a.held_y, row, col, codes, s);
    }
    const float2 pre = row_stats<PRE_LAYER>(v, valid, a.cols, inv_cols, a.eps, sum);
    pre_w.get(chunk, w);
    normalise16<PRE_LAYER>(v, pre.x, pre.y);
    mul16(v, w);
    if (PRE_LAYER) {
      pre_b.get(chunk, w);
      add16(v, w);
    }
    if (in) store16(v, static_cast<T*>(a.h) + row * a.cols, col, a.cols, a.out_vec);
    if (a.held_h.codes) {
      if (valid < 16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = j < valid ? v[j] : 0.f;
      }
      cy.set(v);
      cy.get(v);
      const uint4 codes = act8_encode(v, s);
      if (in && owns) put_codes(a.held_h, row, col, codes, s);
    }
    if (in && t == 0 && a.stats) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(pre.x, pre.y, post.x, post.y);
  }
}

// What a thread loads of a row in the backward pass: sixteen columns.
template <class T, bool TWO>
struct RowLoads {
  Chunk16<T> dh, dy;
  uint4 qy, qb;
  unsigned sy, sb;
  float4 stats;
  __device__ __forceinline__ void load(const BlockNormArgs& a, long long row, int col, bool in) {
    qy = qb = make_uint4(0u, 0u, 0u, 0u);
    sy = sb = 1u;
    dh.zero();
    dy.zero();
    stats = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!in) return;
    dh.load(static_cast<const T*>(a.grad_h) + row * a.grad_h_stride, col, a.cols, a.grad_h_vec);
    if (a.grad_y) dy.load(static_cast<const T*>(a.grad_y) + row * a.grad_y_stride, col, a.cols, a.grad_y_vec);
    stats = __ldg(reinterpret_cast<const float4*>(a.stats + row * 4));
    if (col < a.held_y.pitch) {
      qy = __ldg(reinterpret_cast<const uint4*>(a.held_y.codes + row * a.held_y.pitch + col));
      sy = __ldg(a.held_y.scales + row * a.held_y.spitch + (col >> 5));
      if (TWO) {
        qb = __ldg(reinterpret_cast<const uint4*>(a.held_b.codes + row * a.held_b.pitch + col));
        sb = __ldg(a.held_b.scales + row * a.held_b.spitch + (col >> 5));
      }
    }
  }
};

// (value - mean) * rstd of held values; the difference first: a mean far from zero must not cost digits
template <bool LAYER>
__device__ __forceinline__ void decode_normed(uint4 codes, unsigned s, float mean, float rstd, float (&v)[16]) {
  const float step = act8_step(s);      // (a code times a step is exact, so these round as often as the formula)
  const F2 scale(LAYER ? step : step * rstd), off(-mean), r(rstd);
  act8_codes(codes, [&](int i, F2 q) { put(v, i, LAYER ? mul2(fma2(q, scale, off), r) : mul2(q, scale)); });
}

// POST: what b~ is read for.  kNoBlock: nothing (neither a norm after the block nor a gate); kGateOnly; an RMS norm, a
// layer norm, each with or without a gate.
//
// The norm backward after the block needs sums over g, which itself needs sums over the row.  One reduction does for
// both: with f = r c + dy and u = gate w_post,
//   g = f - k1 y^ - k0,  k1 = r mean(c y^),  k0 = r mean(c) (layer norm before the next block, else 0),
//   sum u g b^ = sum f u b^ - k1 sum y^ u b^ - k0 sum u b^,      sum u g = sum f u - k1 sum y^ u - k0 sum u,
// where every sum on the right is known before k1 and k0 are; a second round through the barrier cost a quarter of the
// kernel.
enum BlockUse : int { kNoBlock = 0, kGateOnly = 1, kBlockRms = 2, kBlockLayer = 3 };

template <class T, class TB, bool PRE_LAYER, int POST>
__global__ void __launch_bounds__(512) block_norm_backward_kernel(const BlockNormArgs a, int tpr) {
  constexpr bool TWO = POST != kNoBlock, NORM = POST >= kBlockRms, LAYER = POST == kBlockLayer;
  constexpr int B = TWO ? 16 : 1, L = PRE_LAYER ? 16 : 1, Z = LAYER ? 16 : 1;
  // the sums of a row: c y^ | c | f u b^, y^ u b^ | u b^ | f u, y^ u
  constexpr int kC = 1, kB = kC + (PRE_LAYER ? 1 : 0), kD = kB + (NORM ? 2 : 0), kE = kD + (NORM && PRE_LAYER ? 1 : 0), kN = kE + (LAYER ? 2 : 0);
  __shared__ __align__(16) float buf[kSumFloats];
  extern __shared__ float4 params[];
  const int rpb = blockDim.x / tpr, lane_row = threadIdx.x / tpr, t = threadIdx.x - lane_row * tpr;
  const int chunks = a.held_y.pitch / 16, chunk = t < chunks ? t : 0, col = t * 16;
  const float inv_cols = 1.f / (float)a.cols;
  const Run run = run_of(a);
  RowSum sum(buf, tpr);
  float dw[16] = {}, db[L] = {}, g1[B] = {}, g0[Z] = {};

  cudaTriggerProgrammaticLaunchCompletion();     // (the sums kernel's blocks take an SM as soon as one is left; it waits for all)
  RowLoads<T, TWO> r;
  r.load(a, run.row0 + lane_row, col, run.row0 + lane_row < run.row1);
  const SharedRow pre_w{params, chunks}, u_row{params + 4 * chunks, chunks};
  const void* const gate = gate_of<T>(a, run);
  for (int i = threadIdx.x; i < 4 * chunks; i += blockDim.x) {
    Param4<T> w, u, f;
    w.load(a, a.pre_weight, i * 4);
    if (NORM) u.load(a, a.post_weight, i * 4);
    if (TWO) f.load(a, gate, i * 4);
    pre_w.put(i, w.get(a, a.pre_weight, i * 4, 1.f));
    if (TWO) {
      float4 v = f.get(a, gate, i * 4, 1.f);
      if (NORM) v = times(v, u.get(a, a.post_weight, i * 4, 1.f));
      u_row.put(i, first_of(v, a.cols - i * 4));
    }
  }
  __syncthreads();
  float sum_u = 0.f;
  if constexpr (LAYER && PRE_LAYER) {
    float u[16], s[1];
    u_row.get(chunk, u);
    s[0] = t < chunks ? sum16(u) : 0.f;
    sum(s);
    sum_u = s[0];
  }

  for (long long base = run.row0; base < run.row1; base += rpb) {
    const long long row = base + lane_row;
    const bool in = row < run.row1;
    float f[16], hat[16], bh[B], w[16], s[kN];
    const float4 stats = r.stats;
    r.dh.get(f);
    decode_normed<PRE_LAYER>(r.qy, r.sy, stats.x, stats.y, hat);
    pre_w.get(chunk, w);
    add_product16(dw, f, hat);
    if constexpr (PRE_LAYER) add16(db, f);
    mul16(f, w);                                     // c
    s[0] = dot16(f, hat);
    if constexpr (PRE_LAYER) s[kC] = sum16(f);
    r.dy.get(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) put(f, i, fma2(F2(stats.y), pair(f, i), pair(w, i)));
    if constexpr (TWO) decode_normed<LAYER>(r.qb, r.sb, stats.z, stats.w, bh);
    r.load(a, row + rpb, col, row + rpb < run.row1);     // the next row's loads are under way during the sums
    if constexpr (NORM) {
      u_row.get(chunk, w);
      if constexpr (LAYER) {
        s[kE] = dot16(f, w);
        s[kE + 1] = dot16(hat, w);
      }
      mul16(w, bh);      // (u is zero past the end of the row)
      s[kB] = dot16(f, w);
      s[kB + 1] = dot16(hat, w);
      if constexpr (PRE_LAYER) s[kD] = sum16(w);
      if (t >= chunks) {
#pragma unroll
        for (int i = kB; i < kN; ++i) s[i] = 0.f;      // (a thread past the row's end holds another chunk's u)
      }
    }
    sum(s);
    const float k1 = stats.y * s[0] * inv_cols, k0 = PRE_LAYER ? stats.y * s[PRE_LAYER ? kC : 0] * inv_cols : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) put(f, i, fma2(F2(-k1), pair(hat, i), PRE_LAYER ? add2(pair(f, i), F2(-k0)) : pair(f, i)));   // g
    if (in && a.dx) {
#pragma unroll
      for (int i = 0; i < 8; ++i) put(w, i, mul2(F2(a.alpha), pair(f, i)));
      store16(w, static_cast<T*>(a.dx) + row * a.cols, col, a.cols, a.out_vec);
    }
    if constexpr (TWO) {
      if (!in || col + 16 > a.cols) {   // what does not exist adds nothing
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = in && col + j < a.cols ? f[j] : 0.f;
      }
      u_row.get(chunk, w);
      add_product16(g1, f, bh);
      if constexpr (LAYER) add16(g0, f);
      mul16(f, w);
      if constexpr (NORM) {
        const float p1 = (s[kB] - k1 * s[kB + 1] - (PRE_LAYER ? k0 * s[PRE_LAYER ? kD : 0] : 0.f)) * inv_cols;
        const float p0 = LAYER ? (s[LAYER ? kE : 0] - k1 * s[LAYER ? kE + 1 : 0] - k0 * sum_u) * inv_cols : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) put(f, i, mul2(F2(stats.w), fma2(pair(bh, i), F2(-p1), LAYER ? add2(pair(f, i), F2(-p0)) : pair(f, i))));
      }
    }
    if (in) store16(f, static_cast<TB*>(a.dblock) + row * a.cols, col, a.cols, a.dblock_vec);
  }
  if (!a.sums) return;
  // This run's sums: [4][pitch] floats.  The CTA's row lanes are added in order, each on top of the one before it.
  const long long pitch = a.held_y.pitch;
  float4* const out = reinterpret_cast<float4*>(a.sums + (long long)blockIdx.x * 4 * pitch);
  float4* const part = params;                       // the parameters are not needed any more
  for (int l = 0; l < rpb; ++l) {
    __syncthreads();
    if (lane_row != l || t >= chunks) continue;
    int n = 0;
    auto put = [&](int which, const float (&v)[16]) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float4 x = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        float4* const p = part + (n * 4 + q) * chunks + t;
        if (l > 0) {
          const float4 y = *p;
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
        }
        if (l + 1 < rpb) *p = x;
        else out[which * (pitch / 4) + t * 4 + q] = x;
      }
      ++n;
    };
    put(0, dw);
    if constexpr (PRE_LAYER) put(1, db);
    if constexpr (TWO) put(2, g1);
    if constexpr (LAYER) put(3, g0);
  }
}

// Adds the runs' sums.  Block: 32 columns x LANES lanes of runs.  blockIdx.y 0 .. 3: one of the norms' parameters, over all
// runs; 4 + s: the gate of sequence s.  LANES: 32 where that many blocks run at once (two an SM), since each thread's
// chain of loads is then what takes the time; 8 where there are more blocks, for a quarter of the joining.  Of 296 runs,
// 1024 columns and no gate 5.4 us with 32 lanes, 10.4 with 8; 4096 columns and eight gates 20 and 15.4.
template <class T, int LANES>
__global__ void __launch_bounds__(32 * LANES) block_norm_sums_kernel(const BlockNormArgs a, int runs, int gates) {
  __shared__ float part[2][LANES][33];
  const int col = blockIdx.x * 32 + threadIdx.x, lane = threadIdx.y;
  const long long pitch = a.held_y.pitch;
  const bool for_gate = blockIdx.y >= 4;
  const int seq = (int)blockIdx.y - 4, per_gate = runs / gates, which = for_gate ? 2 : (int)blockIdx.y;
  void* const grads[4] = {a.pre_weight_grad, a.pre_bias_grad, a.post_weight_grad, a.post_bias_grad};
  if (!for_gate && grads[which] == nullptr) return;
  const int first = for_gate ? seq * per_gate : 0, last = for_gate ? first + per_gate : runs;
  const bool second = for_gate && a.post_bias;
  auto param = [&](const void* p, long long at) {
    return a.params_f32 ? static_cast<const float*>(p)[at] : to_f32<T>(static_cast<const T*>(p)[at]);
  };
  const bool weigh = !for_gate && which >= 2 && a.gate && col < a.cols;     // sum of gate * G over the sequences
  cudaGridDependencySynchronize();
  float v = 0.f, z = 0.f;
  const float* p = a.sums + (long long)(first + lane) * 4 * pitch + which * pitch + col;
#pragma unroll 8
  for (int u = first + lane; u < last; u += LANES, p += LANES * 4 * pitch) {
    float x = *p;
    if (weigh && a.gate_rows) x *= param(a.gate, (long long)(u / per_gate) * a.cols + col);
    v += x;
    if (second) z += p[pitch];
  }
  part[0][lane][threadIdx.x] = v;
  part[1][lane][threadIdx.x] = z;
  __syncthreads();
  if (lane != 0 || col >= a.cols) return;
  v = z = 0.f;
#pragma unroll
  for (int l = 0; l < LANES; ++l) {
    v += part[0][l][threadIdx.x];
    z += part[1][l][threadIdx.x];
  }
  auto put = [&](void* to, long long i, float x) {
    if (a.params_f32) static_cast<float*>(to)[i] = x;
    else static_cast<T*>(to)[i] = from_f32<T>(x);
  };
  if (for_gate) put(a.gate_grad, (long long)seq * a.cols + col, (a.post_weight ? param(a.post_weight, col) : 1.f) * v + (second ? param(a.post_bias, col) * z : 0.f));
  else put(grads[which], col, weigh && !a.gate_rows ? v * param(a.gate, col) : v);
}

template <class K>
cudaError_t launch_shared(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const BlockNormArgs& a, int tpr) {
  if (smem > 40 * 1024) {   // (48 KB with the static part need no leave)
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return err;
  }
  kernel<<<grid, block, smem, stream>>>(a, tpr);
  return cudaGetLastError();
}

// Whether every row of parameters starts where four of its elements do, and ends after a multiple of four.
bool params_vec(const BlockNormArgs& a, size_t es) {
  uintptr_t all = 0;
  for (const void* p : {a.pre_weight, a.pre_bias, a.post_weight, a.post_bias, a.gate}) all |= reinterpret_cast<uintptr_t>(p);
  return a.cols % 4 == 0 && all % (4 * (a.params_f32 ? 4 : es)) == 0;
}

template <class T, class TB>
cudaError_t forward_typed(BlockNormArgs a, int sms, cudaStream_t stream) {
  a.x_vec = row_align(a.x, a.x_stride, sizeof(T));
  a.block_vec = row_align(a.block, a.block_stride, sizeof(TB));
  a.params_vec = params_vec(a, sizeof(T));
  a.out_vec = std::min(row_align(a.h, a.cols, sizeof(T)), row_align(a.y, a.cols, sizeof(T)));
  const BlockNormShape shape = block_norm_shape(a.rows, a.cols, a.gate_rows, sms, false);
  a.parts = shape.parts;
  const dim3 block(shape.tpr * shape.rpb), grid(shape.runs);
  const bool layer = a.pre == kNormLayer;
  const int rows = 1 + (layer ? 1 : 0) + (a.post || a.gate ? 1 : 0) + (a.post == kNormLayer ? 1 : 0);
  const size_t smem = (size_t)rows * a.held_y.pitch * 4;
  auto go = [&](auto kernel) { return launch_shared(kernel, grid, block, smem, stream, a, shape.tpr); };
  if (block.x > 256) {
    switch (a.post * 2 + (layer ? 1 : 0)) {
      case 0: return go(block_norm_forward_kernel<T, TB, false, kNormNone, 512>);
      case 1: return go(block_norm_forward_kernel<T, TB, true, kNormNone, 512>);
      case 2: return go(block_norm_forward_kernel<T, TB, false, kNormRms, 512>);
      case 3: return go(block_norm_forward_kernel<T, TB, true, kNormRms, 512>);
      case 4: return go(block_norm_forward_kernel<T, TB, false, kNormLayer, 512>);
      default: return go(block_norm_forward_kernel<T, TB, true, kNormLayer, 512>);
    }
  }
  switch (a.post * 2 + (layer ? 1 : 0)) {
    case 0: return go(block_norm_forward_kernel<T, TB, false, kNormNone, 256>);
    case 1: return go(block_norm_forward_kernel<T, TB, true, kNormNone, 256>);
    case 2: return go(block_norm_forward_kernel<T, TB, false, kNormRms, 256>);
    case 3: return go(block_norm_forward_kernel<T, TB, true, kNormRms, 256>);
    case 4: return go(block_norm_forward_kernel<T, TB, false, kNormLayer, 256>);
    default: return go(block_norm_forward_kernel<T, TB, true, kNormLayer, 256>);
  }
}

template <class T, class TB>
cudaError_t backward_launch(const BlockNormArgs& a, const BlockNormShape& shape, cudaStream_t stream) {
  const dim3 block(shape.tpr * shape.rpb), grid(shape.runs);
  const int use = a.held_b.codes == nullptr ? kNoBlock : (a.post == kNormNone ? kGateOnly : (a.post == kNormRms ? kBlockRms : kBlockLayer));
  const bool layer = a.pre == kNormLayer;
  // the parameters, or (several row lanes) the sums on their way from lane to lane
  int rows = 1 + (use ? 1 : 0);
  const int sums = 1 + (layer ? 1 : 0) + (use ? 1 : 0) + (use == kBlockLayer ? 1 : 0);
  if (shape.rpb > 1 && sums > rows) rows = sums;
  const size_t smem = (size_t)rows * a.held_y.pitch * 4;
  auto go = [&](auto kernel) { return launch_shared(kernel, grid, block, smem, stream, a, shape.tpr); };
  switch (use * 2 + (layer ? 1 : 0)) {
    case 0: return go(block_norm_backward_kernel<T, TB, false, kNoBlock>);
    case 1: return go(block_norm_backward_kernel<T, TB, true, kNoBlock>);
    case 2: return go(block_norm_backward_kernel<T, TB, false, kGateOnly>);
    case 3: return go(block_norm_backward_kernel<T, TB, true, kGateOnly>);
    case 4: return go(block_norm_backward_kernel<T, TB, false, kBlockRms>);
    case 5: return go(block_norm_backward_kernel<T, TB, true, kBlockRms>);
    case 6: return go(block_norm_backward_kernel<T, TB, false, kBlockLayer>);
    default: return go(block_norm_backward_kernel<T, TB, true, kBlockLayer>);
  }
}

template <class T, class TB>
cudaError_t backward_typed(BlockNormArgs a, const BlockNormShape& shape, int sms, cudaStream_t stream) {
  a.grad_h_vec = row_align(a.grad_h, a.grad_h_stride, sizeof(T));
  a.grad_y_vec = row_align(a.grad_y, a.grad_y_stride, sizeof(T));
  a.params_vec = params_vec(a, sizeof(T));
  a.out_vec = row_align(a.dx, a.cols, sizeof(T));
  a.dblock_vec = row_align(a.dblock, a.cols, sizeof(TB));
  a.parts = shape.parts;
  const cudaError_t err = backward_launch<T, TB>(a, shape, stream);
  const bool params = a.pre_weight_grad || a.pre_bias_grad || a.post_weight_grad || a.post_bias_grad || a.gate_grad;
  if (err != cudaSuccess || !a.sums || !params) return err;
  cudaLaunchConfig_t cfg{};     // (set up while the first kernel still runs; it waits for that one's end before it reads)
  cfg.gridDim = dim3((a.cols + 31) / 32, 4 + (a.gate_grad ? shape.sequences : 0));
  const bool few = (long long)cfg.gridDim.x * cfg.gridDim.y <= 2 * sms;
  cfg.blockDim = dim3(32, few ? 32 : 8);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, few ? block_norm_sums_kernel<T, 32> : block_norm_sums_kernel<T, 8>, a, shape.runs, shape.sequences);
}

}  // namespace

// How a pass covers [rows, cols]: a thread takes sixteen columns, an SM as many threads as the pass's registers allow.
BlockNormShape block_norm_shape(long long rows, int cols, long long gate_rows, int sms, bool backward) {
  BlockNormShape s{};
  s.tpr = ((cols + 31) / 32 * 2 + 31) / 32 * 32;
  s.rpb = s.tpr >= 256 ? 1 : 256 / s.tpr;
  const long long length = gate_rows ? gate_rows : rows;
  s.sequences = (int)(length ? rows / length : 0);
  const long long target = (long long)sms * (backward || s.tpr > 256 ? 512 : 768) / (s.tpr * s.rpb);
  long long parts = s.sequences ? target / s.sequences : 1;
  const long long most = (length + s.rpb - 1) / s.rpb;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  s.parts = (int)parts;
  s.runs = s.sequences * s.parts;
  return s;
}

namespace {

// f(the stream's type, the block's)
template <class F>
cudaError_t by_types(int dtype, int block_dtype, F f) {
  if (dtype == kGradF32) {
    switch (block_dtype) {
      case kGradF32: return f(float{}, float{});
      case kGradBF16: return f(float{}, __nv_bfloat16{});
      case kGradF16: return f(float{}, __half{});
    }
  } else if (dtype == block_dtype) {
    switch (dtype) {
      case kGradBF16: return f(__nv_bfloat16{}, __nv_bfloat16{});
      case kGradF16: return f(__half{}, __half{});
    }
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_block_norm_forward(const BlockNormArgs& a, int dtype, int block_dtype, int sms, cudaStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  if (a.cols > kBlockNormMaxCols || a.rows > 0x7fffffffll) return cudaErrorInvalidValue;
  return by_types(dtype, block_dtype, [&](auto t, auto b) { return forward_typed<decltype(t), decltype(b)>(a, sms, stream); });
}

cudaError_t launch_block_norm_backward(const BlockNormArgs& a, int dtype, int block_dtype, int sms, cudaStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  if (a.cols > kBlockNormMaxCols || a.rows > 0x7fffffffll) return cudaErrorInvalidValue;
  const BlockNormShape shape = block_norm_shape(a.rows, a.cols, a.gate_rows, sms, true);
  if (shape.sequences > 65531) return cudaErrorInvalidValue;
  return by_types(dtype, block_dtype, [&](auto t, auto b) { return backward_typed<decltype(t), decltype(b)>(a, shape, sms, stream); });
}

}  // namespace grace
