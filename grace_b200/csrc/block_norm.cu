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
// in registers, eight columns a thread (16 columns in the backward pass beyond 4096), by one warp or several, so that
// the mean, the squared deviations from it and the results take one pass over memory; small rows share a CTA.  Sums
// over tokens: a CTA walks a run of rows of one sequence with its columns' sums in registers and stores them once; a
// second kernel adds the runs' sums in a fixed order (no atomics: the same bits on every run).
#include "act8.cuh"
#include "act8.h"
#include "common.cuh"
#include "gradio.cuh"

namespace grace {
namespace {

// Columns col .. col + 7 of a row of parameters, fp32 or of the activations' type; null, or past the end: `none`.
template <class T>
__device__ __forceinline__ void load_param(const BlockNormArgs& a, const void* p, int col, float none, float (&v)[8]) {
  if (p != nullptr && a.param_vec && col + 8 <= a.cols) {
    if (a.params_f32) {
      Chunk8<float> c;
      c.load(static_cast<const float*>(p) + col);
      c.get(v);
    } else {
      Chunk8<T> c;
      c.load(static_cast<const T*>(p) + col);
      c.get(v);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    v[j] = p == nullptr || col + j >= a.cols ? none
                                              : (a.params_f32 ? static_cast<const float*>(p)[col + j] : to_f32<T>(static_cast<const T*>(p)[col + j]));
}

// Sums over the `tpr` threads (whole warps) that share a row, the same value in all of them.  Every thread of the CTA
// calls it.  The two buffers alternate: a warp cannot be two reductions ahead of another.
template <int N>
struct RowSum {
  float* buf;      // [2][32][N]
  int parity, tpr;
  __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if (tpr == 32) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = tpr >> 5, first = warp / warps * warps;
    float* const b = buf + parity * 32 * N;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) b[warp * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? b[(first + lane) * N + i] : 0.f);
    parity ^= 1;
  }
};

__device__ __forceinline__ void put_codes(const Held& h, size_t row, int col, uint2 codes, unsigned s) {
  *reinterpret_cast<uint2*>(h.codes + row * h.pitch + col) = codes;
  if ((col & 31) == 0) h.scales[row * h.spitch + (col >> 5)] = (unsigned char)s;
}

__device__ __forceinline__ float2 row_stats(const float (&v)[8], int valid, int kind, float inv_cols, float eps, RowSum<1>& sum) {
  float s[1] = {0.f};
  float mean = 0.f;
  if (kind == kNormLayer) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[0] += v[j];   // (columns past the end are zeros)
    sum(s);
    mean = s[0] * inv_cols;
  }
  s[0] = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d = j < valid ? v[j] - mean : 0.f;
    s[0] = fmaf(d, d, s[0]);
  }
  sum(s);
  return make_float2(mean, rsqrtf(fmaf(s[0], inv_cols, eps)));
}

template <class T>
__global__ void __launch_bounds__(1024) block_norm_forward_kernel(const BlockNormArgs a, int tpr) {
  __shared__ float buf[2 * 32];
  const int rpb = blockDim.x / tpr, lane_row = threadIdx.x / tpr, t = threadIdx.x - lane_row * tpr;
  const int col = t * 8, valid = min(8, max(0, a.cols - col));
  const bool owns = col < a.held_y.pitch;      // (threads past the last group of 32 only take part in the sums)
  const float inv_cols = 1.f / (float)a.cols;
  const long long row = (long long)blockIdx.x * rpb + lane_row;
  const bool in = row < a.rows;
  RowSum<1> sum{buf, 0, tpr};
  Chunk8<T> cb, cx;
  cb.zero();
  cx.zero();
  if (in) {
    load_chunk(cb, static_cast<const T*>(a.block) + row * a.block_stride, col, a.cols, a.block_vec);
    load_chunk(cx, static_cast<const T*>(a.x) + row * a.x_stride, col, a.cols, a.x_vec);
  }
  float v[8], w[8], x[8];
  cb.get(v);
  unsigned s;
  if (a.held_b.codes) {
    const uint2 codes = act8_encode(v, s);
    if (in && owns) put_codes(a.held_b, row, col, codes, s);
  }
  float2 post = make_float2(0.f, 1.f);
  if (a.post != kNormNone) {
    post = row_stats(v, valid, a.post, inv_cols, a.eps, sum);
    load_param<T>(a, a.post_weight, col, 1.f, w);
    load_param<T>(a, a.post_bias, col, 0.f, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf((v[j] - post.x) * post.y, w[j], x[j]);
  }
  if (a.gate) {
    const char* gate = static_cast<const char*>(a.gate);
    if (in && a.gate_rows) gate += (row / a.gate_rows) * a.cols * (a.params_f32 ? 4 : sizeof(T));
    load_param<T>(a, gate, col, 0.f, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= w[j];
  }
  cx.get(x);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < valid ? fmaf(a.alpha, x[j], v[j]) : 0.f;
  cx.set(v);       // the stream as it is rounded to its type
  cx.get(v);
  if (in && a.y) store_chunk(v, static_cast<T*>(a.y) + row * a.cols, col, a.cols, a.out_vec);
  {
    const uint2 codes = act8_encode(v, s);
    if (in && owns && a.held_y.codes) put_codes(a.held_y, row, col, codes, s);
  }
  const float2 pre = row_stats(v, valid, a.pre, inv_cols, a.eps, sum);
  load_param<T>(a, a.pre_weight, col, 1.f, w);
  load_param<T>(a, a.pre_bias, col, 0.f, x);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < valid ? fmaf((v[j] - pre.x) * pre.y, w[j], x[j]) : 0.f;
  if (in) store_chunk(v, static_cast<T*>(a.h) + row * a.cols, col, a.cols, a.out_vec);
  if (a.held_h.codes) {
    cx.set(v);
    cx.get(v);
    const uint2 codes = act8_encode(v, s);
    if (in && owns) put_codes(a.held_h, row, col, codes, s);
  }
  if (in && t == 0 && a.stats) *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(pre.x, pre.y, post.x, post.y);
}

// What a thread loads of a row: eight columns.
template <class T, bool TWO>
struct RowLoads {
  Chunk8<T> dh, dy;
  uint2 qy, qb;
  unsigned sy, sb;
  __device__ __forceinline__ void load(const BlockNormArgs& a, long long row, int col, bool in) {
    qy = qb = make_uint2(0u, 0u);
    sy = sb = 1u;
    dh.zero();
    dy.zero();
    if (!in) return;
    load_chunk(dh, static_cast<const T*>(a.grad_h) + row * a.grad_h_stride, col, a.cols, a.grad_h_vec);
    if (a.grad_y) load_chunk(dy, static_cast<const T*>(a.grad_y) + row * a.grad_y_stride, col, a.cols, a.grad_y_vec);
    if (col < a.held_y.pitch) {
      qy = __ldg(reinterpret_cast<const uint2*>(a.held_y.codes + (size_t)row * a.held_y.pitch + col));
      sy = __ldg(a.held_y.scales + (size_t)row * a.held_y.spitch + (col >> 5));
      if (TWO) {
        qb = __ldg(reinterpret_cast<const uint2*>(a.held_b.codes + (size_t)row * a.held_b.pitch + col));
        sb = __ldg(a.held_b.scales + (size_t)row * a.held_b.spitch + (col >> 5));
      }
    }
  }
};

// A CTA walks the rows of one run: run = sequence * parts + part, rows [part * L / parts, (part + 1) * L / parts) of the
// sequence, L = a.gate_rows (all rows are one sequence where no gate belongs to a sequence).  VPT chunks of eight columns
// a thread, tpr * 8 columns apart.  TWO: N_post or a gate, so that b~ is read.
template <class T, int VPT, bool TWO>
__global__ void __launch_bounds__(512) block_norm_backward_kernel(const BlockNormArgs a, int tpr) {
  __shared__ float buf[2 * 32 * 2];
  const int rpb = blockDim.x / tpr, lane_row = threadIdx.x / tpr, t = threadIdx.x - lane_row * tpr;
  const float inv_cols = 1.f / (float)a.cols;
  const long long run = blockIdx.x, seq = run / a.parts, part = run - seq * a.parts;
  const long long length = a.gate_rows ? a.gate_rows : a.rows;
  const long long row0 = seq * length + part * length / a.parts, row1 = seq * length + (part + 1) * length / a.parts;
  RowSum<2> sum{buf, 0, tpr};
  const bool post = TWO && a.post != kNormNone, layer = a.pre == kNormLayer, post_layer = a.post == kNormLayer;
  float dw[VPT][8] = {}, db[VPT][8] = {}, g1[TWO ? VPT : 1][8] = {}, g0[TWO ? VPT : 1][8] = {};
  const char* gate = static_cast<const char*>(a.gate);
  if (gate && a.gate_rows) gate += seq * a.cols * (a.params_f32 ? 4 : (int)sizeof(T));

  RowLoads<T, TWO> r[VPT];
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  {
    const long long row = row0 + lane_row;
    const bool in = row < row1;
#pragma unroll
    for (int i = 0; i < VPT; ++i) r[i].load(a, row, (i * tpr + t) * 8, in);
    if (in) st = __ldg(reinterpret_cast<const float4*>(a.stats + row * 4));
  }
  for (long long base = row0; base < row1; base += rpb) {
    const long long row = base + lane_row;
    const bool in = row < row1;
    float c[VPT][8], hat[VPT][8], bh[TWO ? VPT : 1][8];
    Chunk8<T> dy[VPT];
    float s[2] = {0.f, 0.f};
    const float4 stats = st;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = (i * tpr + t) * 8;
      float w[8], d[8];
      r[i].dh.get(d);
      act8_decode(r[i].qy, r[i].sy, hat[i]);
      load_param<T>(a, a.pre_weight, col, 1.f, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        hat[i][j] = (hat[i][j] - stats.x) * stats.y;
        dw[i][j] = fmaf(d[j], hat[i][j], dw[i][j]);
        db[i][j] += d[j];
        c[i][j] = d[j] * w[j];
        s[0] += c[i][j];
        s[1] = fmaf(c[i][j], hat[i][j], s[1]);
      }
      dy[i] = r[i].dy;
      if (TWO) {
        act8_decode(r[i].qb, r[i].sb, bh[TWO ? i : 0]);
#pragma unroll
        for (int j = 0; j < 8; ++j) bh[TWO ? i : 0][j] = (bh[TWO ? i : 0][j] - stats.z) * stats.w;
      }
    }
    {   // the next row's loads are under way during the sums
      const bool next = row + rpb < row1;
#pragma unroll
      for (int i = 0; i < VPT; ++i) r[i].load(a, row + rpb, (i * tpr + t) * 8, next);
      st = next ? __ldg(reinterpret_cast<const float4*>(a.stats + (row + rpb) * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    sum(s);
    const float m0 = layer ? s[0] * inv_cols : 0.f, m1 = s[1] * inv_cols;
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = (i * tpr + t) * 8;
      float d[8], w[8];
      dy[i].get(d);
#pragma unroll
      for (int j = 0; j < 8; ++j) c[i][j] = fmaf(stats.y, c[i][j] - m0 - hat[i][j] * m1, d[j]);   // g
      if (in && a.dx) {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = a.alpha * c[i][j];
        store_chunk(d, static_cast<T*>(a.dx) + row * a.cols, col, a.cols, a.out_vec);
      }
      if (TWO) {
        constexpr int z = TWO ? 1 : 0;
        const bool some = in;   // a row that does not exist adds nothing
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float g = some && col + j < a.cols ? c[i][j] : 0.f;
          g1[i * z][j] = fmaf(g, bh[i * z][j], g1[i * z][j]);
          g0[i * z][j] += g;
          c[i][j] = g;
        }
        if (gate) {
          load_param<T>(a, gate, col, 0.f, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) c[i][j] *= w[j];
        }
        if (post) {
          load_param<T>(a, a.post_weight, col, 1.f, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            c[i][j] *= w[j];
            s[0] += c[i][j];
            s[1] = fmaf(c[i][j], bh[i * z][j], s[1]);
          }
        }
      }
    }
    float p0 = 0.f, p1 = 0.f;
    if (post) {
      sum(s);
      p0 = post_layer ? s[0] * inv_cols : 0.f;
      p1 = s[1] * inv_cols;
    }
    if (in) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int col = (i * tpr + t) * 8;
        if (post) {
#pragma unroll
          for (int j = 0; j < 8; ++j) c[i][j] = stats.w * (c[i][j] - p0 - bh[TWO ? i : 0][j] * p1);
        }
        store_chunk(c[i], static_cast<T*>(a.dblock) + row * a.cols, col, a.cols, a.out_vec);
      }
    }
  }
  // this run's sums: [4][pitch] floats for each row lane of the CTA
  if (a.sums) {
    float* const out = a.sums + (run * rpb + lane_row) * 4 * (long long)a.held_y.pitch;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int col = (i * tpr + t) * 8;
      if (col >= a.held_y.pitch) continue;
      auto put = [&](int which, const float (&v)[8]) {
        float4* p = reinterpret_cast<float4*>(out + (long long)which * a.held_y.pitch + col);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
      };
      put(0, dw[i]);
      if (layer) put(1, db[i]);
      if (TWO) {
        put(2, g1[TWO ? i : 0]);
        put(3, g0[TWO ? i : 0]);
      }
    }
  }
}

// Adds the runs' sums.  Block: 32 columns x 8 lanes of runs.  blockIdx.y 0: the norms' parameters, over all runs; 1 + s:
// the gate of sequence s.
constexpr int kLanes = 8;
template <class T>
__global__ void __launch_bounds__(32 * kLanes) block_norm_sums_kernel(const BlockNormArgs a, int sum_rows, int gates) {
  __shared__ float part[4][kLanes][33];
  const int col = blockIdx.x * 32 + threadIdx.x, lane = threadIdx.y;
  const long long pitch = a.held_y.pitch;
  const bool for_gate = blockIdx.y > 0;
  const long long seq = (long long)blockIdx.y - 1;
  const long long runs = (long long)sum_rows;                         // rows of sums in all
  const long long per_gate = runs / gates;
  const long long first = for_gate ? seq * per_gate : 0, last = for_gate ? first + per_gate : runs;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (long long u = first + lane; u < last; u += kLanes) {
    const float* p = a.sums + u * 4 * pitch + col;
    float g = 1.f;
    if (!for_gate) {
      if (a.pre_weight_grad) v[0] += p[0];
      if (a.pre_bias_grad) v[1] += p[pitch];
      if (a.gate && col < a.cols) {
        const long long at = a.gate_rows ? u / per_gate * a.cols + col : col;
        g = a.params_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
      }
    }
    if (for_gate || a.post_weight_grad) v[2] = fmaf(g, p[2 * pitch], v[2]);
    if (for_gate ? a.post_bias != nullptr : a.post_bias_grad != nullptr) v[3] = fmaf(g, p[3 * pitch], v[3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[i][lane][threadIdx.x] = v[i];
  __syncthreads();
  if (lane != 0 || col >= a.cols) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = 0.f;
    for (int l = 0; l < kLanes; ++l) v[i] += part[i][l][threadIdx.x];
  }
  auto put = [&](void* p, long long at, float x) {
    if (!p) return;
    if (a.params_f32) static_cast<float*>(p)[at] = x;
    else static_cast<T*>(p)[at] = from_f32<T>(x);
  };
  auto get = [&](const void* p, float none) {
    return p == nullptr ? none : (a.params_f32 ? static_cast<const float*>(p)[col] : to_f32<T>(static_cast<const T*>(p)[col]));
  };
  if (for_gate) {
    put(a.gate_grad, seq * a.cols + col, get(a.post_weight, 1.f) * v[2] + get(a.post_bias, 0.f) * v[3]);
  } else {
    put(a.pre_weight_grad, col, v[0]);
    put(a.pre_bias_grad, col, v[1]);
    put(a.post_weight_grad, col, v[2]);
    put(a.post_bias_grad, col, v[3]);
  }
}

bool aligned(const void* p, long long stride, int es) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * es % 16 == 0; }

bool params_aligned(const BlockNormArgs& a) {
  const void* all[] = {a.pre_weight, a.pre_bias, a.post_weight, a.post_bias, a.gate};
  for (const void* p : all)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return a.cols % 8 == 0;
}

template <class T>
cudaError_t forward_typed(BlockNormArgs a, cudaStream_t stream) {
  a.x_vec = aligned(a.x, a.x_stride, sizeof(T));
  a.block_vec = aligned(a.block, a.block_stride, sizeof(T));
  a.out_vec = aligned(a.h, a.cols, sizeof(T)) && aligned(a.y, a.cols, sizeof(T));
  a.param_vec = params_aligned(a);
  const int tpr = (a.held_y.pitch / 8 + 31) / 32 * 32, rpb = tpr >= 256 ? 1 : 256 / tpr;
  const long long grid = (a.rows + rpb - 1) / rpb;
  block_norm_forward_kernel<T><<<(unsigned)grid, tpr * rpb, 0, stream>>>(a, tpr);
  return cudaGetLastError();
}

template <class T>
cudaError_t backward_typed(BlockNormArgs a, const BlockNormShape& shape, cudaStream_t stream) {
  a.grad_h_vec = aligned(a.grad_h, a.grad_h_stride, sizeof(T));
  a.grad_y_vec = a.grad_y && aligned(a.grad_y, a.grad_y_stride, sizeof(T));
  a.out_vec = aligned(a.dblock, a.cols, sizeof(T)) && aligned(a.dx, a.cols, sizeof(T));
  a.param_vec = params_aligned(a);
  a.parts = shape.parts;
  const dim3 block(shape.tpr * shape.rpb), grid(shape.runs);
  const bool two = a.held_b.codes != nullptr;
  if (shape.vpt == 1) {
    if (two) block_norm_backward_kernel<T, 1, true><<<grid, block, 0, stream>>>(a, shape.tpr);
    else block_norm_backward_kernel<T, 1, false><<<grid, block, 0, stream>>>(a, shape.tpr);
  } else {
    if (two) block_norm_backward_kernel<T, 2, true><<<grid, block, 0, stream>>>(a, shape.tpr);
    else block_norm_backward_kernel<T, 2, false><<<grid, block, 0, stream>>>(a, shape.tpr);
  }
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess || !a.sums) return err;
  const bool params = a.pre_weight_grad || a.pre_bias_grad || a.post_weight_grad || a.post_bias_grad || a.gate_grad;
  if (!params) return cudaSuccess;
  const int gates = a.gate_grad ? shape.sequences : 0;
  block_norm_sums_kernel<T><<<dim3((a.cols + 31) / 32, 1 + gates), dim3(32, kLanes), 0, stream>>>(a, shape.runs * shape.rpb,
                                                                                                 shape.sequences);
  return cudaGetLastError();
}

}  // namespace

// How the backward pass covers [rows, cols]: about two CTAs of 512 threads, or four of 256, for each SM.
BlockNormShape block_norm_shape(long long rows, int cols, long long gate_rows, int sms) {
  BlockNormShape s{};
  const int chunks = (cols + 31) / 32 * 4;
  s.vpt = chunks > 512 ? 2 : 1;
  s.tpr = ((chunks + s.vpt - 1) / s.vpt + 31) / 32 * 32;
  s.rpb = s.tpr >= 256 ? 1 : 256 / s.tpr;
  const long long length = gate_rows ? gate_rows : rows;
  s.sequences = (int)(length ? rows / length : 0);
  const long long target = (long long)sms * 1024 / (s.tpr * s.rpb);
  long long parts = s.sequences ? target / s.sequences : 1;
  const long long most = (length + s.rpb - 1) / s.rpb;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  s.parts = (int)parts;
  s.runs = s.sequences * s.parts;
  return s;
}

cudaError_t launch_block_norm_forward(const BlockNormArgs& a, int dtype, cudaStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  if (a.cols > kBlockNormMaxCols || a.rows > 0x7fffffffll) return cudaErrorInvalidValue;
  switch (dtype) {
    case kGradF32: return forward_typed<float>(a, stream);
    case kGradBF16: return forward_typed<__nv_bfloat16>(a, stream);
    case kGradF16: return forward_typed<__half>(a, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_block_norm_backward(const BlockNormArgs& a, int dtype, int sms, cudaStream_t stream) {
  if (a.rows <= 0 || a.cols <= 0) return cudaSuccess;
  if (a.cols > kBlockNormMaxCols || a.rows > 0x7fffffffll) return cudaErrorInvalidValue;
  const BlockNormShape shape = block_norm_shape(a.rows, a.cols, a.gate_rows, sms);
  if (shape.sequences > 65534) return cudaErrorInvalidValue;
  switch (dtype) {
    case kGradF32: return backward_typed<float>(a, shape, stream);
    case kGradBF16: return backward_typed<__nv_bfloat16>(a, shape, stream);
    case kGradF16: return backward_typed<__half>(a, shape, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace grace
