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
// such a copy: [rows, ceil(cols / 8) * 8]).  work: act8_wgrad_work_bytes of scratch, often none.
cudaError_t launch_act8_wgrad(const void* grad, long long grad_stride, Held held, long long tokens, int outs, int ins, int dtype,
                              int out_f32, void* out, void* bias, void* work, int sms, cudaStream_t stream);
size_t act8_wgrad_work_bytes(long long tokens, int outs, int ins, int out_f32, int sms);
// Waits for the current device, all of its streams: its status block of the bounded waits (16 words, the first 0 if none ran
// out), cleared if one did.
cudaError_t act8_wgrad_status(unsigned* words);
cudaError_t act8_wgrad_status_block(void** block);      // where it is in the device's memory
cudaError_t launch_act8_repitch(const void* src, long long stride, void* dst, long long rows, int cols, cudaStream_t stream);

// ---- residual and norm step between two blocks (block_norm.cu) ----
enum NormKind : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
constexpr int kBlockNormMaxCols = 8192;

struct BlockNormArgs {
  long long rows;
  int cols;
  int pre, post;             // NormKind (pre: not kNormNone)
  int params_f32;            // parameters, gate and their gradients are fp32 (else of the activations' type)
  float alpha, alpha_low, eps;         // the residual's factor as the sum of two fp32 numbers
  long long gate_rows;       // rows of a sequence with a gate of its own; 0: one gate for all rows, or none
  const void *pre_weight, *pre_bias, *post_weight, *post_bias, *gate;   // null: ones, zeros, ones, zeros, no gate
  Held held_y, held_b, held_h;   // held_b: with N_post or a gate; held_h: on request; codes null: not kept (pitch is set all the same)
  float* stats;              // [rows][4]: mean and rstd of y, mean and rstd of block; null: not kept
  // forward
  const void *x, *block;
  long long x_stride, block_stride;
  void *h, *y;               // contiguous; y null: not wanted
  // (block and dblock may be of a 16-bit type where all else is fp32)
  // backward
  const void *grad_h, *grad_y;   // grad_y null: nothing reads the stream
  long long grad_h_stride, grad_y_stride;
  void *dx, *dblock;         // contiguous; dx null: it equals dblock
  void *pre_weight_grad, *pre_bias_grad, *post_weight_grad, *post_bias_grad, *gate_grad;   // null: not wanted
  float* sums;               // [runs of the backward pass][4][pitch] scratch (BlockNormShape)
  // filled in by the launchers
  int x_vec, block_vec, out_vec, dblock_vec, grad_h_vec, grad_y_vec;   // RowAlign (act8.cuh)
  int params_vec;                // the parameters may be read in fours
  int parts;
};

struct BlockNormShape {
  int tpr, rpb;              // threads a row, rows a CTA
  int sequences, parts, runs;
};
BlockNormShape block_norm_shape(long long rows, int cols, long long gate_rows, int sms, bool backward);
// block_dtype: of block and dblock; dtype's own, or one of 16 bits beside fp32
cudaError_t launch_block_norm_forward(const BlockNormArgs& a, int dtype, int block_dtype, int sms, cudaStream_t stream);
cudaError_t launch_block_norm_backward(const BlockNormArgs& a, int dtype, int block_dtype, int sms, cudaStream_t stream);

}  // namespace grace
