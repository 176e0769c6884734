// Host side of the 8-bit activation checkpoint kernels (act8.cu, act8_wgrad.cu) and of the residual-and-norm kernels
// (block_norm.cu).  Element types are GradType values (gradio.cuh): 0 fp32, 1 bf16, 2 fp16.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace grace {

// A checkpoint of [rows, cols]: codes int8 with `pitch` bytes a row (cols rounded up to 32), one scale byte for each 32
// codes, `spitch` bytes a row (the number of groups rounded up to 8).
struct Held {
  signed char* codes;
  unsigned char* scales;
  int pitch, spitch;
};

enum ActKind : int { kActGelu = 0, kActGeluTanh = 1, kActSilu = 2 };

cudaError_t launch_act8_pack(const void* x, long long x_stride, long long rows, int cols, int dtype, Held held, cudaStream_t stream);
cudaError_t launch_act8_unpack(Held held, void* out, long long out_stride, long long rows, int cols, int dtype, cudaStream_t stream);

// y = f(x), or with `gated` x = [a | b] and y = f(a) b.  `held`: checkpoint of x (of a), `held_b`: of b, `held_y`: of
// y as it is rounded to its type (codes null, each: not wanted).
cudaError_t launch_act8_forward(const void* x, long long x_stride, void* y, long long rows, int cols, int dtype, int kind, int gated,
                                Held held, Held held_b, Held held_y, cudaStream_t stream);
cudaError_t launch_act8_backward(const void* grad, long long grad_stride, void* dx, long long rows, int cols, int dtype, int kind,
                                 int gated, Held held, Held held_b, cudaStream_t stream);

// dW [outs, ins] = dY^T x~ and (bias not null) db [outs] = column sums of dY, both of grad's type or, with out_f32, fp32.
// grad: 16-bit, rows `grad_stride` elements apart, base and rows on 16-byte boundaries (launch_act8_repitch makes
// such a copy: [rows, ceil(cols / 8) * 8]).
cudaError_t launch_act8_wgrad(const void* grad, long long grad_stride, Held held, long long tokens, int outs, int ins, int dtype,
                              int out_f32, void* out, void* bias, int sms, cudaStream_t stream);
// The current device's status block of the bounded waits (16 words, the first 0 if none ran out), cleared if one did.
cudaError_t act8_wgrad_status(unsigned* words);
cudaError_t launch_act8_repitch(const void* src, long long stride, void* dst, long long rows, int cols, cudaStream_t stream);

}  // namespace grace
