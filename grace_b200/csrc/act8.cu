// 8-bit activation checkpoints: writing them, reading them back, and the activation functions of a feed-forward layer
// that write them in the forward pass and read them in the backward pass.
//
//   pack      codes, scales = checkpoint(x)                               es + 1 1/32 bytes an element
//   unpack    x~ = value of the checkpoint                                1 1/32 + es
//   forward   y = f(x), checkpoint(x), optionally checkpoint(y)           2 es + 1 1/32 (+ 1 1/32)
//             gated: x = [a | b], y = f(a) b, checkpoints of a and b      3 es + 2 1/16 (+ 1 1/32), for an element of y
//   backward  dx = dy f'(x~);  gated: da = dy b~ f'(a~), db = dy f(a~)    2 es + 1 1/32;  3 es + 2 1/16
//
// All four are bound by memory where rows start on 16-byte boundaries (others: below), the GELU forward pass with both
// checkpoints by its issue slots: a thread takes a chunk of sixteen neighbouring elements (32 bytes of a 16-bit type in, 16
// bytes of codes out; with eight, half of both, pack took a fifth longer), two lanes share a group of 32 and agree on its
// largest magnitude by one shuffle.  What hides the latency is
// the number of threads: with two chunks each, all loads first, the gated backward pass took 89 us for 77, the others as
// long as with one.  At 6.5 TB/s an SM has about 16 issue slots an element of a bf16 pack and 25 of a forward pass, so
// arithmetic is on pairs of numbers, the encoder clamps only where a group needs it (together 34.6 -> 29.2 us for
// pack), and the functions take one exponential and one reciprocal.
// Measured, bf16 16384 x 4096 (L2 cold): pack 29.2 us, 7.0 TB/s; unpack 28.8 us, 7.1 TB/s; gated SiLU forward 78 us, 6.9
// TB/s, and backward 77 us, 7.0 TB/s; 4096 x 4096 GELU forward with both checkpoints 19.9 us, 5.1 TB/s, backward 16.4 us,
// 5.2 TB/s.  (Above the copy rate of 6.5 where the last writes are still in L2.)  fp32 16384 x 4096, with the launch: pack 57,
// unpack 55, GELU forward 170 and backward 270 us (CUDA's erfc).
// Rows off 16-byte boundaries (a width that is no multiple of 8 of a 16-bit type, a slice that starts between) are read and
// written by single elements, 32 bytes apart from lane to lane: 16384 x 4095 against x 4096, with the launch, pack 74 and 37 us,
// unpack 371 and 35, gated forward 371 and 85, gated backward 766 and 86.
//
// f is GELU (erf form), GELU (tanh form) or SiLU.  For 16-bit tensors the exponential and the reciprocal are the hardware's,
// and the normal distribution function of the erf form is, for x <= 0,
//   P(x) = erfc(z) / 2 = t (c1 + t (c2 + ... + t c6)) exp(-z^2),   z = -x / sqrt 2,  t = 1 / (1 + 0.424 z),
// whose exponential is also the density that the derivative needs.  The form is that of Hastings' approximations; the
// coefficients were fitted by linear programming for the least largest error relative to the value, weighted 1 : 3 : 8 : 16 : 30 at
// z = 0, 1.5, 3, 5, 9.4, since what a 16-bit result shows is that.  Relative error with its roundings: 1.4e-6 for x >= -1, 3.6e-6 to
// -3, 1e-5 to -6, 2.2e-5 to -13 (half a step is at least 2^-12 of a normal fp16 value, 2^-9 of a bf16 one); from -13.2 on, where
// the result is below 2^-126, it is zero.  The other two forms are the logistic function's, accurate relative to the value as well,
// and zero where that function is below 2^-126 (SiLU: x < -87.3).  For fp32 tensors erfc and exp are CUDA's.
#include <algorithm>

#include "act8.cuh"
#include "act8.h"
#include "gradio.cuh"

namespace grace {
namespace {

constexpr int kBlock = 256;

// n / d for 0 <= n < 2^31 as a multiplication: m = ceil(2^p / d) with p = 31 + ceil(log2 d) (Granlund and Montgomery)
struct FastDiv {
  unsigned d, m;
  int p;
};
FastDiv make_div(unsigned d) {
  int l = 0;
  while ((1ull << l) < d) ++l;
  const unsigned long long p = 31 + l;
  return {d, (unsigned)(((1ull << p) + d - 1) / d), (int)p};
}
__device__ __forceinline__ void divmod(const FastDiv& f, unsigned n, unsigned& q, unsigned& r) {
  q = (unsigned)(((unsigned long long)n * f.m) >> f.p);
  r = n - q * f.d;
}

struct Rows {          // which chunks a launch covers
  unsigned chunks;     // of sixteen columns: rows * (pitch / 16), below 2^28; a multiple of 2
  FastDiv per_row;     // pitch / 16
  int cols;
};

__device__ __forceinline__ void put_held(const Held& h, size_t row, int col, uint4 codes, unsigned s) {
  *reinterpret_cast<uint4*>(h.codes + row * h.pitch + col) = codes;
  if ((col & 31) == 0) h.scales[row * h.spitch + (col >> 5)] = (unsigned char)s;
}
struct HeldChunk {
  uint4 codes;
  unsigned s;
  __device__ __forceinline__ void load(const Held& h, size_t row, int col) {
    codes = __ldg(reinterpret_cast<const uint4*>(h.codes + row * h.pitch + col));
    s = __ldg(h.scales + row * h.spitch + (col >> 5));
  }
  __device__ __forceinline__ void get(float (&v)[16]) const { act8_decode(codes, s, v); }
};

// ---- the functions: f and f' at x ----
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float kInvSqrt2Pi = 0.3989422804f, kLog2e = 1.4426950409f;
constexpr float kTanhC = 0.7978845608f, kTanhA = 0.044715f;

__device__ __forceinline__ F2 exp2_fast(F2 x) {
  float a, b;
  x.get(a, b);
  return F2(exp2_fast(a), exp2_fast(b));
}
__device__ __forceinline__ F2 rcp_fast(F2 x) {
  float a, b;
  x.get(a, b);
  return F2(rcp_fast(a), rcp_fast(b));
}
__device__ __forceinline__ F2 one_minus(F2 x) { return fma2(x, F2(-1.f), F2(1.f)); }

// f and f' at two numbers, for 16-bit tensors
template <int KIND>
__device__ __forceinline__ void function(F2 x, F2& f, F2& d) {
  const F2 one(1.f);
  F2 p;
  if (KIND == kActGelu) {   // p: the normal distribution function, e: exp(-x^2 / 2)
    float a, b, qa, qb;
    x.get(a, b);
    const F2 t = rcp_fast(F2(fmaf(0.29981327f, fabsf(a), 1.f), fmaf(0.29981327f, fabsf(b), 1.f)));
    const F2 e = exp2_fast(mul2(mul2(x, x), F2(-0.5f * kLog2e)));
    F2 poly = fma2(t, F2(-0.081011303f), F2(0.22808936f));
    poly = fma2(t, poly, F2(-0.030255733f));
    poly = fma2(t, poly, F2(0.15101245f));
    poly = fma2(t, poly, F2(0.11201961f));
    poly = fma2(t, poly, F2(0.12014519f));
    mul2(mul2(t, poly), e).get(qa, qb);      // erfc(|x| / sqrt 2) / 2
    p = F2(a < 0.f ? qa : 1.f - qa, b < 0.f ? qb : 1.f - qb);
    d = fma2(mul2(x, F2(kInvSqrt2Pi)), e, p);
  } else if (KIND == kActGeluTanh) {
    float a, b;
    mul2(x, x).get(a, b);
    const F2 xx(fminf(a, 1e4f), fminf(b, 1e4f));      // past |x| = 100 the sigmoid is 0 or 1 to the last bit
    const F2 u = mul2(mul2(x, F2(-2.f * kTanhC * kLog2e)), fma2(xx, F2(kTanhA), one));
    p = rcp_fast(add2(exp2_fast(u), one));            // (1 + tanh) / 2
    d = fma2(mul2(mul2(mul2(x, F2(2.f * kTanhC)), p), one_minus(p)), fma2(xx, F2(3.f * kTanhA), one), p);
  } else {
    p = rcp_fast(add2(exp2_fast(mul2(x, F2(-kLog2e))), one));
    d = mul2(p, fma2(x, one_minus(p), one));
  }
  f = mul2(x, p);
}
// the same with CUDA's functions, for fp32 tensors
template <int KIND>
__device__ __forceinline__ float2 function(float x) {
  if (KIND == kActGelu) {
    const float e = expf(-0.5f * x * x), p = 0.5f * erfcf(-0.70710678f * x);
    return make_float2(x * p, fmaf(x * kInvSqrt2Pi, e, p));
  }
  if (KIND == kActGeluTanh) {
    const float xx = fminf(x * x, 1e4f), p = 1.f / (1.f + expf(-2.f * kTanhC * x * fmaf(kTanhA, xx, 1.f)));
    return make_float2(x * p, fmaf(2.f * kTanhC * x * p * (1.f - p), fmaf(3.f * kTanhA, xx, 1.f), p));
  }
  const float p = 1.f / (1.f + expf(-x));
  return make_float2(x * p, p * fmaf(x, 1.f - p, 1.f));
}
// f(x) and f'(x) of sixteen
template <class T, int KIND>
__device__ __forceinline__ void function16(const float (&x)[16], float (&f)[16], float (&d)[16]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      F2 y, z;
      function<KIND>(pair(x, i), y, z);
      put(f, i, y);
      put(d, i, z);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 y = function<KIND>(x[j]);
      f[j] = y.x;
      d[j] = y.y;
    }
  }
}
__device__ __forceinline__ void mul16(float (&v)[16], const float (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) put(v, i, mul2(pair(v, i), pair(w, i)));
}

// ---- kernels: thread t of block b takes chunk 256 b + t ----
// Blocks an SM of the gated 16-bit kernels, 5 forward and 4 backward, is what measured best (SiLU, 16384 x 4096): forward 78 us with
// 5 (48 registers, a few of them spilled) and 80 with 4; backward 77 with 4, 81 with 5; with 6 they spill and take 100 and 118.
template <class T, bool GATED> constexpr int blocks_an_sm(int gated) { return sizeof(T) == 4 ? 1 : (GATED ? gated : 6); }

struct Place {
  unsigned row, col;
  bool in;
};
__device__ __forceinline__ Place place_of(const Rows& r) {
  const unsigned at = blockIdx.x * kBlock + threadIdx.x;
  Place p{0, 0, at < r.chunks};
  if (p.in) divmod(r.per_row, at, p.row, p.col);
  p.col *= 16;
  return p;
}

template <class T>
__global__ void __launch_bounds__(kBlock) pack_kernel(const T* __restrict__ x, long long stride, int vec, Rows r, Held held) {
  const Place p = place_of(r);
  Chunk16<T> c;
  c.zero();
  if (p.in) c.load(x + (long long)p.row * stride, (int)p.col, r.cols, vec);
  float v[16];
  unsigned s;
  c.get(v);
  const uint4 codes = act8_encode(v, s);      // (all lanes take part)
  if (p.in) put_held(held, p.row, (int)p.col, codes, s);
}

template <class T>
__global__ void __launch_bounds__(kBlock) unpack_kernel(Held held, T* __restrict__ out, long long stride, int vec, Rows r) {
  const Place p = place_of(r);
  if (!p.in) return;
  HeldChunk c;
  c.load(held, p.row, (int)p.col);
  float v[16];
  c.get(v);
  store16(v, out + (long long)p.row * stride, (int)p.col, r.cols, vec);
}

template <class T, int KIND, bool GATED>
__global__ void __launch_bounds__(kBlock, blocks_an_sm<T, GATED>(5)) forward_kernel(const T* __restrict__ x, long long stride, int vec_x, T* __restrict__ y,
                                                        int vec_y, Rows r, Held held, Held held_b, Held held_y) {
  const Place p = place_of(r);
  const int col = (int)p.col;
  Chunk16<T> ca, cb;
  ca.zero();
  cb.zero();
  if (p.in) {
    const T* const row = x + (long long)p.row * stride;
    ca.load(row, col, r.cols, vec_x);
    if (GATED) cb.load(row + r.cols, col, r.cols, vec_x);
  }
  float v[16], w[16];
  unsigned s;
  uint4 codes;
  ca.get(v);
  if (held.codes) {
    codes = act8_encode(v, s);
    if (p.in) put_held(held, p.row, col, codes, s);
  }
  function16<T, KIND>(v, v, w);
  if (GATED) {
    cb.get(w);
    if (held_b.codes) {
      codes = act8_encode(w, s);
      if (p.in) put_held(held_b, p.row, col, codes, s);
    }
    mul16(v, w);
  }
  if (p.in) store16(v, y + (size_t)p.row * r.cols, col, r.cols, vec_y);
  if (held_y.codes) {
    Chunk16<T> cy;   // the checkpoint is of y as the next layer sees it
    cy.set(v);
    cy.get(v);
    codes = act8_encode(v, s);
    if (p.in) put_held(held_y, p.row, col, codes, s);
  }
}

template <class T, int KIND, bool GATED>
__global__ void __launch_bounds__(kBlock, blocks_an_sm<T, GATED>(4)) backward_kernel(const T* __restrict__ grad, long long stride, int vec_g, T* __restrict__ dx,
                                                         int vec_x, Rows r, Held held, Held held_b) {
  const Place p = place_of(r);
  if (!p.in) return;
  const int col = (int)p.col;
  Chunk16<T> c;
  HeldChunk qa, qb;
  c.load(grad + (long long)p.row * stride, col, r.cols, vec_g);
  qa.load(held, p.row, col);
  if (GATED) qb.load(held_b, p.row, col);
  float g[16], a[16], b[16], d[16];
  c.get(g);
  qa.get(a);
  function16<T, KIND>(a, a, d);
  mul16(d, g);
  T* const out = dx + (size_t)p.row * (GATED ? 2 : 1) * r.cols;
  if (GATED) {
    qb.get(b);
    mul16(d, b);
    mul16(a, g);
    store16(a, out + r.cols, col, r.cols, vec_x);
  }
  store16(d, out, col, r.cols, vec_x);
}

Held rows_from(Held h, long long row) {
  if (h.codes) {
    h.codes += (size_t)row * h.pitch;
    h.scales += (size_t)row * h.spitch;
  }
  return h;
}

// Calls f(first row, Rows, grid) for slabs of rows of less than 2^28 chunks (2^32 elements; only the rows' offsets need 64 bits).
template <class F>
cudaError_t over_slabs(long long rows, int cols, F f) {
  const long long per_row = ((long long)cols + 31) / 32 * 2;
  const long long slab = ((1ll << 28) - 1) / per_row;
  for (long long at = 0; at < rows; at += slab) {
    const long long n = rows - at < slab ? rows - at : slab;
    Rows r{(unsigned)(n * per_row), make_div((unsigned)per_row), cols};
    f(at, r, (unsigned)((n * per_row + kBlock - 1) / kBlock));
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

template <class T>
cudaError_t pack_typed(const void* x, long long stride, long long rows, int cols, Held held, cudaStream_t st) {
  const T* p = static_cast<const T*>(x);
  const int vec = row_align(x, stride, sizeof(T));
  return over_slabs(rows, cols, [&](long long at, Rows r, unsigned grid) {
    pack_kernel<T><<<grid, kBlock, 0, st>>>(p + at * stride, stride, vec, r, rows_from(held, at));
  });
}
template <class T>
cudaError_t unpack_typed(Held held, void* out, long long stride, long long rows, int cols, cudaStream_t st) {
  T* p = static_cast<T*>(out);
  const int vec = row_align(out, stride, sizeof(T));
  return over_slabs(rows, cols, [&](long long at, Rows r, unsigned grid) {
    unpack_kernel<T><<<grid, kBlock, 0, st>>>(rows_from(held, at), p + at * stride, stride, vec, r);
  });
}
template <class T, int KIND, bool GATED>
cudaError_t forward_typed(const void* x, long long stride, void* y, long long rows, int cols, Held a, Held b, Held hy, cudaStream_t st) {
  const T* p = static_cast<const T*>(x);
  T* q = static_cast<T*>(y);
  const int vec_y = row_align(y, cols, sizeof(T));
  const int vec_x = std::min(row_align(x, stride, sizeof(T)), GATED ? row_align(x, cols, sizeof(T)) : (int)kRow32);
  return over_slabs(rows, cols, [&](long long at, Rows r, unsigned grid) {
    forward_kernel<T, KIND, GATED><<<grid, kBlock, 0, st>>>(p + at * stride, stride, vec_x, q + at * cols, vec_y, r,
                                                                     rows_from(a, at), rows_from(b, at), rows_from(hy, at));
  });
}
template <class T, int KIND, bool GATED>
cudaError_t backward_typed(const void* grad, long long stride, void* dx, long long rows, int cols, Held a, Held b, cudaStream_t st) {
  const T* p = static_cast<const T*>(grad);
  T* q = static_cast<T*>(dx);
  const int vec_g = row_align(grad, stride, sizeof(T)), vec_x = row_align(dx, cols, sizeof(T));
  return over_slabs(rows, cols, [&](long long at, Rows r, unsigned grid) {
    backward_kernel<T, KIND, GATED><<<grid, kBlock, 0, st>>>(p + at * stride, stride, vec_g, q + at * cols * (GATED ? 2 : 1),
                                                                      vec_x, r, rows_from(a, at), rows_from(b, at));
  });
}

template <class F>
cudaError_t by_type(int dtype, F f) {
  switch (dtype) {
    case kGradF32: return f(float{});
    case kGradBF16: return f(__nv_bfloat16{});
    case kGradF16: return f(__half{});
  }
  return cudaErrorInvalidValue;
}
template <int V> struct Int { static constexpr int value = V; };
template <class F>
cudaError_t by_kind(int kind, int gated, F f) {
  switch (kind * 2 + (gated ? 1 : 0)) {
    case 0: return f(Int<kActGelu>{}, Int<0>{});
    case 1: return f(Int<kActGelu>{}, Int<1>{});
    case 2: return f(Int<kActGeluTanh>{}, Int<0>{});
    case 3: return f(Int<kActGeluTanh>{}, Int<1>{});
    case 4: return f(Int<kActSilu>{}, Int<0>{});
    case 5: return f(Int<kActSilu>{}, Int<1>{});
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_act8_pack(const void* x, long long x_stride, long long rows, int cols, int dtype, Held held, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  return by_type(dtype, [&](auto t) { return pack_typed<decltype(t)>(x, x_stride, rows, cols, held, stream); });
}

cudaError_t launch_act8_unpack(Held held, void* out, long long out_stride, long long rows, int cols, int dtype, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  return by_type(dtype, [&](auto t) { return unpack_typed<decltype(t)>(held, out, out_stride, rows, cols, stream); });
}

cudaError_t launch_act8_forward(const void* x, long long x_stride, void* y, long long rows, int cols, int dtype, int kind, int gated,
                                Held held, Held held_b, Held held_y, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  return by_type(dtype, [&](auto t) {
    return by_kind(kind, gated, [&](auto k, auto g) {
      return forward_typed<decltype(t), decltype(k)::value, decltype(g)::value != 0>(x, x_stride, y, rows, cols, held, held_b, held_y, stream);
    });
  });
}

cudaError_t launch_act8_backward(const void* grad, long long grad_stride, void* dx, long long rows, int cols, int dtype, int kind,
                                 int gated, Held held, Held held_b, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return cudaSuccess;
  return by_type(dtype, [&](auto t) {
    return by_kind(kind, gated, [&](auto k, auto g) {
      return backward_typed<decltype(t), decltype(k)::value, decltype(g)::value != 0>(grad, grad_stride, dx, rows, cols, held, held_b, stream);
    });
  });
}

}  // namespace grace
