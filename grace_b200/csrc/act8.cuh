// The 8-bit activation checkpoint format, shared by the kernels that write and read it.
//
// A row is cut into groups of 32 neighbouring elements.  With E the biased fp32 exponent of the group's largest
// magnitude, the group's scale byte is s = clamp(E, 7, 252) - 6 and stands for 2^(s - 127) (E8M0); an element x is
// held as the int8 code  q = rint(x * 2^(127 - s))  (ties to even), kept within [-127, 127], and reads back as
// q * 2^(s - 127).  The codes are those of MXINT8 of the OCP Microscaling Formats specification 1.0; the scale byte is that
// format's less 6, since its elements carry an implied factor of 2^-6 that is part of the scale here (who reads these bytes as
// MXINT8 gets values 64 times too small).  Scaling by a power
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

__device__ __forceinline__ float max_abs(float a, float b, float c) {   // a NaN where one of them is one
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two fp32 numbers in a register pair, and arithmetic on both in one instruction, each rounded as by itself.  The kernels
// that use these are short of issue slots before they are short of arithmetic.
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ explicit F2(float x) : F2(x, x) {}
  F2() = default;
  __device__ __forceinline__ void get(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
  __device__ __forceinline__ float sum() const {
    float x, y;
    get(x, y);
    return x + y;
  }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
template <int N> __device__ __forceinline__ F2 pair(const float (&v)[N], int i) { return F2(v[2 * i], v[2 * i + 1]); }
template <int N> __device__ __forceinline__ void put(float (&v)[N], int i, F2 x) { x.get(v[2 * i], v[2 * i + 1]); }

// Sixteen values of a group whose other half is held by the neighbouring lane (lanes 2i and 2i + 1, both active): their
// codes, and the group's scale byte.
__device__ __forceinline__ uint4 act8_encode(const float (&v)[16], unsigned& s) {
  float m[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) m[j] = max_abs(v[3 * j], v[3 * j + 1], v[3 * j + 2]);
  unsigned top = __float_as_uint(max_abs(max_abs(m[0], m[1], m[2]), max_abs(m[3], m[4], v[15]), 0.f)) & 0x7fffffffu;     // from here on as integers: a NaN is the largest
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  s = act8_scale_byte(top);
  const float inv = act8_inverse(s);
  constexpr float kMagic = 12582912.f;   // 1.5 * 2^23: the sum's low byte is the integer nearest to x * inv, ties to even
  float x[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) put(x, i, fma2(pair(v, i), F2(inv), F2(kMagic)));
  if (__uint_as_float(top) * inv >= 127.5f) {     // one group in two hundred: without the clamp all others take two instructions an element less
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = fminf(fmaxf(x[j], kMagic - 127.f), kMagic + 127.f);
  }
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = __float_as_uint(x[4 * i + j]);
    w[i] = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
  }
  return s == 255u ? make_uint4(0u, 0u, 0u, 0u) : make_uint4(w[0], w[1], w[2], w[3]);
}

// f(i, codes 2 i and 2 i + 1 as numbers) of sixteen codes
template <class F>
__device__ __forceinline__ void act8_codes(uint4 codes, F f) {
  const unsigned w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned c = w[i / 2] ^ 0x80808080u;   // code + 128, an unsigned byte; in the low bits of 2^23 it is the number 2^23 + byte
    const int j = i % 2 * 2;
    f(i, add2(F2(__uint_as_float(__byte_perm(c, 0x4b000000u, 0x7540 + j)), __uint_as_float(__byte_perm(c, 0x4b000000u, 0x7541 + j))), F2(-8388736.f)));
  }
}
// The values of sixteen codes.
__device__ __forceinline__ void act8_decode(uint4 codes, unsigned s, float (&v)[16]) {
  const F2 step(act8_step(s));
  act8_codes(codes, [&](int i, F2 q) { put(v, i, mul2(q, step)); });
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

// How a row may be accessed: its start, and the distance to the next row, on no boundary, on 16 or on 32 bytes.
enum RowAlign : int { kRowAny = 0, kRow16 = 1, kRow32 = 2 };
inline int row_align(const void* p, long long stride_elems, int es) {
  const unsigned long long both = reinterpret_cast<uintptr_t>(p) | (unsigned long long)(stride_elems * es);
  return both % 32 == 0 ? kRow32 : (both % 16 == 0 ? kRow16 : kRowAny);
}

// 32 bytes in one access
__device__ __forceinline__ void load32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
}
__device__ __forceinline__ void store32(void* p, uint4 a, uint4 b) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y),
               "r"(b.z), "r"(b.w) : "memory");
}
__device__ __forceinline__ uint4 as_u4(float4 v) { return make_uint4(__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)); }
__device__ __forceinline__ float4 as_f4(uint4 v) { return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)); }

// Sixteen neighbouring elements, as kernels hold and move them: elements col .. col + 15 of a row of `cols` (zeros past
// its end), col a multiple of 16.
template <class T>
struct Chunk16 {
  Chunk8<T> lo, hi;
  __device__ __forceinline__ void zero() {
    lo.zero();
    hi.zero();
  }
  __device__ __forceinline__ void load(const T* __restrict__ row, int col, int cols, int align) {
    if (align == kRow32 && col + 16 <= cols) {
      if constexpr (sizeof(T) == 2) {
        load32(row + col, lo.w, hi.w);
      } else {
        uint4 a, b;
        load32(row + col, a, b);
        lo.a = as_f4(a);
        lo.b = as_f4(b);
        load32(row + col + 8, a, b);
        hi.a = as_f4(a);
        hi.b = as_f4(b);
      }
    } else if (align == kRow16 && col + 16 <= cols) {
      lo.load(row + col);
      hi.load(row + col + 8);
    } else {
      zero();
      if (col < cols) lo.load_some(row + col, cols - col);
      if (col + 8 < cols) hi.load_some(row + col + 8, cols - col - 8);
    }
  }
  __device__ __forceinline__ void store(T* __restrict__ row, int col, int align) const {
    if (align == kRow32) {
      if constexpr (sizeof(T) == 2) {
        store32(row + col, lo.w, hi.w);
      } else {
        store32(row + col, as_u4(lo.a), as_u4(lo.b));
        store32(row + col + 8, as_u4(hi.a), as_u4(hi.b));
      }
    } else {
      lo.store(row + col);
      hi.store(row + col + 8);
    }
  }
  __device__ __forceinline__ void get(float (&v)[16]) const {
    float x[8];
    lo.get(x);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[j];
    hi.get(x);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[8 + j] = x[j];
  }
  __device__ __forceinline__ void set(const float (&v)[16]) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = v[j];
    lo.set(x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = v[8 + j];
    hi.set(x);
  }
};
template <class T>
__device__ __forceinline__ void store16(const float (&v)[16], T* __restrict__ row, int col, int cols, int align) {
  if (align != kRowAny && col + 16 <= cols) {
    Chunk16<T> c;
    c.set(v);
    c.store(row, col, align);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (col + j < cols) row[col + j] = from_f32<T>(v[j]);
  }
}

}  // namespace grace
