"""The step between two blocks of a transformer as one kernel each way: the norm after a block, its gate, the scaled
residual, and the norm before the next block, with 8-bit checkpoints (``ops/act8.py``) for the backward pass.

    n = N_post(block)                          (post=None: block)
    y = residual_scale * x + gate * n          the residual stream, rounded to its type
    h = N_pre(y)                               the next block's input

``pre`` and ``post`` are ``"rms"`` (``v / sqrt(mean v^2 + eps) * weight``) or ``"layer"`` (``(v - mean) / sqrt(var + eps) * weight +
bias``); a missing weight is ones.  ``gate`` is ``[cols]`` or, for ``x`` of three axes and more, ``[x.shape[0], cols]``: a row for
each sequence.  "Add and norm" of a post-norm layer is ``pre="layer"`` with nothing else and ``return_stream=False``; DeepNorm's is the same with
``residual_scale``; a sandwich norm has both.

What the forward pass keeps: a checkpoint of ``y``, with ``post`` or a gate one of ``block``, and four fp32 statistics a row.
Gradients are those of the formulas above at the checkpoints' values of ``y`` and ``block`` with the statistics of the full-precision
ones; parameter gradients are fp32 sums in a fixed order, rounded once to the parameter's type.
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Tuple

import torch

from . import native
from .act8 import Act8, _at, _autocast_type, _check_tensor, _decode_cpu, _encode_cpu, _launch, _new_like, _ptrs, _sms, empty_like, pitch_of
from .exchange import GRAD_DTYPE

NORMS = {None: 0, "rms": 1, "layer": 2}
MAX_COLS = 8192      # a row is held in the registers of one CTA (block_norm.cu: kBlockNormMaxCols)
MAX_ROWS = (1 << 31) - 1
MAX_SEQUENCES = 65531
PARAMS = ("pre_weight", "pre_bias", "post_weight", "post_bias", "gate")


class Saved:
    """What the backward pass takes from the forward pass: one allocation with the checkpoints and the statistics, the parameters, and the
    forms of the norms."""

    __slots__ = ("data", "shape", "dtype", "block_dtype", "rows", "pitch", "spitch", "two", "params", "pre", "post", "residual_scale", "return_stream", "held_h")

    def __init__(self, data: Optional[torch.Tensor], shape, dtype, device, params, pre, post, residual_scale, return_stream, held_h=None,
                 keep=True, block_dtype=None):
        self.shape, self.dtype, self.rows = shape, dtype, math.prod(shape[:-1])
        self.block_dtype = block_dtype or dtype
        self.pitch, self.spitch = pitch_of(shape[-1])
        self.two = post is not None or params[4] is not None       # a checkpoint of block too
        self.params, self.pre, self.post = params, pre, post
        self.residual_scale, self.return_stream, self.held_h = residual_scale, return_stream, held_h
        self.data = torch.empty(self._stats_at() + 16 * self.rows, dtype=torch.uint8, device=device) if data is None and keep else data

    def _held(self) -> int:     # bytes of a checkpoint, a multiple of 16
        return (self.rows * (self.pitch + self.spitch) + 15) // 16 * 16

    def _stats_at(self) -> int:
        return self._held() * (2 if self.two else 1)

    def ptrs(self) -> Tuple[int, int, int, int, int]:
        """Addresses: codes and scales of y, of block (0, 0 without), the statistics."""
        at, n, codes = self.data.data_ptr(), self._held(), self.rows * self.pitch
        if self.two:
            return at, at + codes, at + n, at + n + codes, at + 2 * n
        return at, at + codes, 0, 0, at + n

    @property
    def held_y(self) -> Act8:
        return Act8._over(self.data, 0, self.shape, self.dtype)

    @property
    def held_block(self) -> Optional[Act8]:
        return Act8._over(self.data, self._held(), self.shape, self.block_dtype) if self.two else None

    @property
    def stats(self) -> torch.Tensor:
        """fp32 ``[rows, 4]``: mean and 1 / deviation of ``y``, then of ``block`` (0 and 1 without ``post``)."""
        return self.data[self._stats_at() :].view(torch.float32).view(-1, 4)


def _check(x, block, pre, post, params, residual_scale, eps, mixed) -> int:
    """Rows of a sequence (0: the gate, if any, is the same for all rows).  ``mixed``: ``block`` may be of 16 bits beside ``x`` in fp32."""
    _check_tensor(x, "residual_norm: x")
    _check_tensor(block, "residual_norm: block")
    shape, dtype, device = x.shape, x.dtype, x.device
    if shape != block.shape or (dtype != block.dtype and not (mixed and dtype == torch.float32)) or device != block.device:
        raise ValueError("residual_norm: x %s %s on %s and block %s %s on %s have to be alike"
                         % (tuple(shape), dtype, device, tuple(block.shape), block.dtype, block.device))
    if pre not in ("rms", "layer") or post not in NORMS:
        raise ValueError("residual_norm: pre is 'rms' or 'layer', post one of them or None, not %r and %r" % (pre, post))
    cols, rows = shape[-1], math.prod(shape[:-1])
    if cols > MAX_COLS or rows > MAX_ROWS:
        raise ValueError("residual_norm: at most %d columns and 2^31 - 1 rows, not %d and %d" % (MAX_COLS, cols, rows))
    if not (abs(residual_scale) < 3e38 and 0 <= eps < 3e38):      # (fp32 numbers in the kernels)
        raise ValueError("residual_norm: residual_scale and eps >= 0 within fp32's range, not %r and %r" % (residual_scale, eps))
    if post is None and (params[2] is not None or params[3] is not None):
        raise ValueError("residual_norm: post_weight or post_bias without a norm after the block")
    if (pre == "rms" and params[1] is not None) or (post == "rms" and params[3] is not None):
        raise ValueError("residual_norm: an RMS norm has no bias")
    kind = None
    gate_rows = 0
    for name, p in zip(PARAMS, params):
        if p is None:
            continue
        if p.dtype != kind:
            if kind is not None or p.dtype not in (dtype, torch.float32):
                raise TypeError("residual_norm: parameters are all %s or all fp32, not %s" % (dtype, [str(q.dtype) for q in params if q is not None]))
            kind = p.dtype
        if p.device != device:
            raise ValueError("residual_norm: %s is on %s, x on %s" % (name, p.device, device))
        if name == "gate" and p.dim() == 2:
            if len(shape) < 3 or p.shape != (shape[0], cols):
                raise ValueError("residual_norm: a gate of two axes has a row for each entry of the first of x's three or more axes, "
                                 "not %s for x %s" % (tuple(p.shape), tuple(shape)))
            if p.shape[0] > MAX_SEQUENCES:
                raise ValueError("residual_norm: a gate has at most %d rows" % MAX_SEQUENCES)
            gate_rows = rows // max(1, p.shape[0])
        elif p.shape != (cols,):
            raise ValueError("residual_norm: %s is %s for %d columns" % (name, tuple(p.shape), cols))
    return gate_rows


def _param_ptrs(params):
    """The parameters' addresses, and the tensors that have to live until the launch."""
    kept = [p if p is None or (p.is_contiguous() and not p.is_neg()) else p.detach().resolve_neg().contiguous() for p in params]
    return [0 if p is None else p.data_ptr() for p in kept], kept


def residual_norm_forward(x: torch.Tensor, block: torch.Tensor, *, pre: str = "layer", pre_weight: Optional[torch.Tensor] = None,
                          pre_bias: Optional[torch.Tensor] = None, post: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                          post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                          eps: float = 1e-5, return_stream: bool = True, checkpoint_output: bool = False, checkpoint: bool = True
                          ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Saved]:
    """``(h, y, saved)`` (``y`` None without ``return_stream``); with ``checkpoint_output`` ``saved.held_h`` is what ``act8.pack(h)`` gives.  With
    ``checkpoint=False``, where no backward pass follows, ``saved`` holds nothing else.  A row of which the squares' sum passes fp32's
    range has no deviation: NaN on the GPU."""
    return _forward(x, block, pre, post, (pre_weight, pre_bias, post_weight, post_bias, gate), residual_scale, eps, return_stream,
                    checkpoint_output, checkpoint, False)


def _forward(x, block, pre, post, params, residual_scale, eps, return_stream, checkpoint_output, checkpoint, mixed):
    gate_rows = _check(x, block, pre, post, params, residual_scale, eps, mixed)
    shape, dtype, device = x.shape, x.dtype, x.device
    cols, rows = shape[-1], math.prod(shape[:-1])
    held_h = empty_like(shape, dtype, device) if checkpoint_output else None
    saved = Saved(None, shape, dtype, device, params, pre, post, float(residual_scale), return_stream, held_h, checkpoint,
                  block.dtype)
    if not x.is_cuda:
        return _forward_cpu(x, block, saved, float(eps)) + (saved,)
    h = _new_like(x)
    y = _new_like(x) if return_stream else None
    vx, x_at, x_stride = _at(x)
    vb, b_at, b_stride = _at(block)
    ptrs, kept = _param_ptrs(params)
    *held, stats = saved.ptrs() if checkpoint else (0,) * 5
    _launch(device, native().block_norm_forward, x_at, x_stride, b_at, b_stride, h.data_ptr(), 0 if y is None else y.data_ptr(), stats, rows,
            cols, GRAD_DTYPE[dtype], GRAD_DTYPE[block.dtype], NORMS[pre], NORMS[post], _f32(params), float(residual_scale), float(eps), gate_rows, ptrs,
            (*held, *_ptrs(held_h)), saved.pitch, saved.spitch, _sms(device))
    del kept
    return h, y, saved


def _f32(params) -> int:
    for p in params:
        if p is not None:      # (they are all of one type)
            return int(p.dtype == torch.float32)
    return 0


def residual_norm_backward(grad_h: torch.Tensor, grad_y: Optional[torch.Tensor], saved: Saved, needs=(True,) * 5
                           ) -> Dict[str, Optional[torch.Tensor]]:
    """The gradients of ``x``, ``block`` and the parameters (``PARAMS``), by name; None where there is no such parameter or ``needs`` (as
    ``PARAMS``) does not ask for it.  ``grad_y`` is that of the stream, None where nothing reads it.  Without ``post`` and gate and with a
    ``residual_scale`` of 1, ``x`` and ``block`` have one gradient: both names give the same tensor."""
    if saved.data is None:
        raise ValueError("residual_norm: the forward pass ran with checkpoint=False")
    params, shape, dtype, device = saved.params, saved.shape, saved.dtype, saved.data.device
    for name, g in (("grad_h", grad_h), ("grad_y", grad_y)):
        if g is None and name == "grad_y":
            continue
        _check_tensor(g, "residual_norm: " + name)
        if tuple(g.shape) != shape or g.dtype != dtype or g.device != device:
            raise ValueError("residual_norm: %s %s %s on %s for %s %s on %s" % (name, tuple(g.shape), g.dtype, g.device, shape, dtype, device))
    gate = params[4]
    want = [p is not None and n for p, n in zip(params, needs)]
    cols, rows = shape[-1], math.prod(shape[:-1])
    if device.type != "cuda" and rows and cols:
        return _backward_cpu(grad_h, grad_y, saved, want)
    if rows == 0 or cols == 0:
        empty = torch.empty(shape, dtype=dtype, device=device)
        return dict(zip(("x", "block") + PARAMS, [empty, empty.to(saved.block_dtype)] + [torch.zeros_like(p) if w else None for p, w in zip(params, want)]))
    one = not saved.two and saved.residual_scale == 1.0 and saved.block_dtype == dtype
    block = _new_like(grad_h) if saved.block_dtype == dtype else torch.empty(shape, dtype=saved.block_dtype, device=device)
    dx = None if one else _new_like(grad_h)
    grads = [(torch.empty_like(p) if p.is_contiguous() else torch.empty(p.shape, dtype=p.dtype, device=device)) if w else None
             for p, w in zip(params, want)]
    gate_rows = rows // gate.shape[0] if gate is not None and gate.dim() == 2 else 0
    C, sms = native(), _sms(device)
    g, g_at, g_stride = _at(grad_h)
    gy, gy_at, gy_stride = (None, 0, 0) if grad_y is None else _at(grad_y)
    ptrs, kept = _param_ptrs(params)
    *held, stats = saved.ptrs()
    sums = torch.empty(C.block_norm_sum_rows(rows, cols, gate_rows, sms) * 4 * saved.pitch, dtype=torch.float32, device=device) if any(want) else None
    _launch(device, C.block_norm_backward, g_at, g_stride, gy_at, gy_stride, 0 if dx is None else dx.data_ptr(), block.data_ptr(), stats,
            0 if sums is None else sums.data_ptr(), rows, cols, GRAD_DTYPE[dtype], GRAD_DTYPE[saved.block_dtype],
            NORMS[saved.pre], NORMS[saved.post], _f32(params), saved.residual_scale, gate_rows, ptrs, [0 if t is None else t.data_ptr() for t in grads], held, saved.pitch, saved.spitch, sms)
    del kept
    got = dict(zip(PARAMS, grads))
    got["x"], got["block"] = block if dx is None else dx, block
    return got


# ------------------------------------------------------------------------------------------------------------- on CPU
def _wide(p: Optional[torch.Tensor], shape, none: float) -> torch.Tensor:
    if p is None:
        return torch.full((), none)
    p = p.detach().float()
    return p if p.dim() == 1 else p.view((p.shape[0],) + (1,) * (len(shape) - 2) + (p.shape[1],))


def _stats_cpu(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    if kind is None:
        return mean, torch.ones_like(mean)
    return mean, ((v - mean).square().mean(-1, keepdim=True) + eps).rsqrt()


def _forward_cpu(x, block, saved: Saved, eps: float):
    if x.numel() == 0:
        return torch.empty_like(x), torch.empty_like(x) if saved.return_stream else None
    pre_w, pre_b, post_w, post_b, gate = saved.params
    b = block.detach().float()
    mb, rb = _stats_cpu(b, saved.post, eps)
    n = b if saved.post is None else (b - mb) * rb * _wide(post_w, x.shape, 1.0) + _wide(post_b, x.shape, 0.0)
    if gate is not None:
        n = n * _wide(gate, x.shape, 1.0)
    y = (saved.residual_scale * x.detach().double() + n).to(x.dtype)
    v = y.float()
    m, r = _stats_cpu(v, saved.pre, eps)
    h = ((v - m) * r * _wide(pre_w, x.shape, 1.0) + _wide(pre_b, x.shape, 0.0)).to(x.dtype)
    if saved.held_h is not None:
        _encode_cpu(h, saved.held_h)
    if saved.data is not None:
        saved.stats.copy_(torch.stack([t.reshape(-1) for t in (m, r, mb, rb)], -1))
        _encode_cpu(y, saved.held_y)
        if saved.two:
            _encode_cpu(block.detach(), saved.held_block)
    return h, y if saved.return_stream else None


def _norm_grad_cpu(c, hat, r, kind):
    return r * (c - (c.mean(-1, keepdim=True) if kind == "layer" else 0.0) - hat * (c * hat).mean(-1, keepdim=True))


def _backward_cpu(grad_h, grad_y, saved: Saved, want):
    shape, dtype = saved.held_y.shape, saved.held_y.dtype
    pre_w, _, post_w, post_b, gate = saved.params
    m, r, mb, rb = (t.reshape(shape[:-1] + (1,)) for t in saved.stats.unbind(-1))
    leading = tuple(range(len(shape) - 1))
    over = lambda t, axes: t.sum(axes) if axes else t  # noqa: E731  (no axes would mean all of them)
    got = dict.fromkeys(PARAMS)
    dh = grad_h.detach().float()
    hat = (_decode_cpu(saved.held_y) - m) * r
    got["pre_weight"], got["pre_bias"] = over(dh * hat, leading), over(dh, leading)
    g = _norm_grad_cpu(dh * _wide(pre_w, shape, 1.0), hat, r, saved.pre)
    if grad_y is not None:
        g = g + grad_y.detach().float()
    e = g if gate is None else g * _wide(gate, shape, 1.0)
    if saved.held_block is not None:
        b = _decode_cpu(saved.held_block)
        bh = b if saved.post is None else (b - mb) * rb
        if gate is not None:
            n = bh * _wide(post_w, shape, 1.0) + _wide(post_b, shape, 0.0)
            got["gate"] = over(g * n, leading if gate.dim() == 1 else leading[1:])
        if saved.post is not None:
            got["post_weight"], got["post_bias"] = over(e * bh, leading), over(e, leading)
            e = _norm_grad_cpu(e * _wide(post_w, shape, 1.0), bh, rb, saved.post)
    got = {k: got[k].to(p.dtype) if w else None for k, p, w in zip(PARAMS, saved.params, want)}
    got["x"], got["block"] = (saved.residual_scale * g).to(dtype), e.to(saved.block_dtype)
    return got


# ------------------------------------------------------------------------------------------------------ with autograd
class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, block, pre_weight, pre_bias, post_weight, post_bias, gate, pre, post, residual_scale, eps, return_stream,
                checkpoint_output, mixed, box):
        ctx.set_materialize_grads(False)
        h, y, saved = _forward(x, block, pre, post, (pre_weight, pre_bias, post_weight, post_bias, gate), residual_scale, eps, return_stream,
                               checkpoint_output, True, mixed)
        box.append(saved.held_h)
        ctx.save_for_backward(*saved.params, saved.data)
        ctx.kinds, ctx.shape, ctx.dtype, ctx.block_dtype = (pre, post, saved.residual_scale, return_stream), x.shape, x.dtype, block.dtype
        return (h, y) if return_stream else h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_h, grad_y=None):
        t = ctx.saved_tensors
        saved = Saved(t[5], ctx.shape, ctx.dtype, t[5].device, tuple(t[:5]), *ctx.kinds, block_dtype=ctx.block_dtype)
        if not saved.return_stream:
            grad_y = None
        if grad_h is None and grad_y is None:
            return (None,) * 15
        if grad_h is None:
            grad_h = torch.zeros(ctx.shape, dtype=ctx.dtype, device=t[5].device)
        got = residual_norm_backward(grad_h, grad_y, saved, ctx.needs_input_grad[2:7])
        return (got["x"], got["block"]) + tuple(got[k] for k in PARAMS) + (None,) * 8


def residual_norm(x: torch.Tensor, block: torch.Tensor, *, pre: str = "layer", pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, post: Optional[str] = None, post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                  eps: float = 1e-5, return_stream: bool = True, checkpoint_output: bool = False):
    """``residual_norm_forward`` with autograd: ``h``, then ``y`` with ``return_stream``, then the ``Act8`` of ``h`` with ``checkpoint_output``; one of them
    alone comes as it is, several as a tuple.  Under autocast ``x`` and results are of the wider type of ``x`` and ``block``, as their sum
    is: a stream in fp32 stays in fp32 where the blocks compute in 16 bits."""
    mixed = _autocast_type(x) is not None
    if mixed:
        t = torch.promote_types(x.dtype, block.dtype)
        t = t if t in GRAD_DTYPE else torch.float32
        x = x.to(t)
        if block.dtype != t and block.dtype not in GRAD_DTYPE:
            block = block.to(t)
        pre_weight, pre_bias, post_weight, post_bias, gate = (
            p if p is None or p.dtype in (t, torch.float32) else p.to(t) for p in (pre_weight, pre_bias, post_weight, post_bias, gate))
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, block, pre_weight, pre_bias, post_weight, post_bias, gate))):
        h, y, saved = _forward(x, block, pre, post, (pre_weight, pre_bias, post_weight, post_bias, gate), residual_scale, eps, return_stream,
                               checkpoint_output, False, mixed)
        out = (h,) + ((y,) if return_stream else ()) + ((saved.held_h,) if checkpoint_output else ())
        return out[0] if len(out) == 1 else out
    box = []
    out = _ResidualNorm.apply(x, block, pre_weight, pre_bias, post_weight, post_bias, gate, pre, post, float(residual_scale), float(eps),
                              return_stream, checkpoint_output, mixed, box)
    if not checkpoint_output:
        return out
    return (out if return_stream else (out,)) + (box[0],)
