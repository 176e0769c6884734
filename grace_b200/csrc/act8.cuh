// The 8-bit activation checkpoint format, shared by the kernels that write and read it.
//
// A row is cut into groups of 32 neighbouring elements.  With E the biased fp32 exponent of the group's largest
// magnitude, the group's scale byte is s = clamp(E, 7, 252) - 6 and stands for 2^(s - 127) (E8M0); an element x is
// held as the int8 code  q = rint(x * 2^(127 - s))  (ties to even), kept within [-127, 127], and reads back as
// q * 2^(s - 127).  This is the MXINT8 format of the OCP Microscaling Formats specification 1.0.  Scaling by a power
// of two is exact, so the only rounding is the one to an integer, and 7 bits of magnitude fit bf16's significand: a
// held value is exact in fp32 and in bf16 (in fp16 too unless it is subnormal there).  The largest error is half a
// code step, 2^-7 of the group's leading power of two (one step, 2^-6, within the last 1/128 below the next power).
// A group that holds an infinity or a NaN has s = 255 and reads back as NaN throughout, so an overflow in the forward
// pass still shows in the gradients.  Magnitudes of 2^126 and more saturate; below 2^-120 the step stays 2^-126.
//
// Why a power of two and not amax / 127: the division's scale would be at most twice finer (on average half a bit), but
// costs a correctly rounded division per element to be well defined, and its values would be rounded again on the
// way into a 16-bit tensor-core operand.  Groups of 32 (a byte of scale each, 3 %) win most of it back over longer ones.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace grace {

constexpr int kActGroup = 32;

__device__ __forceinline__ unsigned act8_scale_byte(unsigned top_bits) {   // bits of the largest magnitude (fp32)
  const unsigned e = top_bits >> 23;
  return e == 255u ? 255u : min(max(e, 7u), 252u) - 6u;
}
// 2^(127 - s); 0 for a group that reads back as NaN, whose codes are therefore 0
__device__ __forceinline__ float act8_inverse(unsigned s) { return __uint_as_float(s == 255u ? 0u : (254u - s) << 23); }
__device__ __forceinline__ float act8_step(unsigned s) { return __uint_as_float(s == 255u ? 0x7fffffffu : s << 23); }

__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN where either is one (its sign bit clear)
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight values of a group whose other 24 are held by the neighbouring three lanes (lanes 4i .. 4i + 3, all of them
// active): their codes, and the group's scale byte.
__device__ __forceinline__ uint2 act8_encode(const float (&v)[8], unsigned& s) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
  unsigned top = __float_as_uint(m);     // from here on as integers: a NaN is the largest
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  s = act8_scale_byte(top);
  const float inv = act8_inverse(s);
  unsigned u[8];
  constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: the sum's low byte is the integer nearest to x * inv, ties to even
#pragma unroll
  for (int j = 0; j < 8; ++j)
    u[j] = __float_as_uint(fminf(fmaxf(__fmaf_rn(v[j], inv, kMagic), kMagic - 127.f), kMagic + 127.f));
  if (s == 255u) return make_uint2(0u, 0u);   // (an infinity times 0 is a NaN, which the clamp above turns into a bound)
  const unsigned a = __byte_perm(u[0], u[1], 0x0040), b = __byte_perm(u[2], u[3], 0x0040);
  const unsigned c = __byte_perm(u[4], u[5], 0x0040), d = __byte_perm(u[6], u[7], 0x0040);
  return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410));
}

__device__ __forceinline__ void act8_decode(uint2 codes, unsigned s, float (&v)[8]) {
  const float step = act8_step(s);
  codes.x ^= 0x80808080u;   // code + 128, an unsigned byte
  codes.y ^= 0x80808080u;
#pragma unroll
  for (int j = 0; j < 4; ++j) {   // a byte in the low bits of 2^23 is the number 2^23 + byte
    v[j] = (__uint_as_float(__byte_perm(codes.x, 0x4b000000u, 0x7540 + j)) - 8388736.f) * step;
    v[j + 4] = (__uint_as_float(__byte_perm(codes.y, 0x4b000000u, 0x7540 + j)) - 8388736.f) * step;
  }
}

// ---- eight neighbouring elements of a row of fp32, bf16 or fp16, as fp32 ----
template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

// two neighbours in a register: one or two instructions each way
template <class T> __device__ __forceinline__ float2 unpack2(unsigned w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <class T> __device__ __forceinline__ unsigned pack2(float lo, float hi);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&v);
}

template <class T> struct Chunk8 {   // 16-bit types: 16 bytes
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ static unsigned bits(T x) { return (unsigned)*reinterpret_cast<unsigned short*>(&x); }
  __device__ __forceinline__ void load_some(const T* p, int n) {
    unsigned h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = j < n ? bits(p[j]) : 0u;
    w = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2<T>(u[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    w = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
};
template <> struct Chunk8<float> {   // 32 bytes
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = a;
    reinterpret_cast<float4*>(p)[1] = b;
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load_some(const float* p, int n) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.f;
    set(v);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
};

// Elements col .. col + 7 of a row of `cols` (zeros past its end).  `vec`: the row starts on a 16-byte boundary.
template <class T>
__device__ __forceinline__ void load_chunk(Chunk8<T>& c, const T* __restrict__ row, int col, int cols, bool vec) {
  if (vec && col + 8 <= cols) c.load(row + col);
  else if (col < cols) c.load_some(row + col, cols - col);
  else c.zero();
}
template <class T>
__device__ __forceinline__ void store_chunk(const float (&v)[8], T* __restrict__ row, int col, int cols, bool vec) {
  if (vec && col + 8 <= cols) {
    Chunk8<T> c;
    c.set(v);
    c.store(row + col);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols) row[col + j] = from_f32<T>(v[j]);
  }
}

}  // namespace grace
