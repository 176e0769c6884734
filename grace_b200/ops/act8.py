"""8-bit activation checkpoints: what the forward pass keeps for the backward pass, at a byte an element.

The exchange kernels shrink what ranks send to each other; these shrink what a rank keeps to itself between forward
and backward, which is what bounds its batch.  A checkpoint holds groups of 32 neighbours of the last axis as int8
codes with one power-of-two scale (MXINT8 of the OCP Microscaling specification but for the scale byte, which is 6 less, see
``csrc/act8.cuh``): 33 bytes for 32 values.  The forward pass computes with the full-precision tensors; only the backward pass sees the
rounded ones, so outputs are untouched and gradients carry an error of at most half a code step (2^-7 of the leading
power of two of a value's group) in the values they are made of.

* ``pack(x)`` / ``unpack(held)``: write a checkpoint, read it back.
* ``weight_grad(grad, held)``: the weight (and bias) gradient of a linear layer straight from the checkpoint of its
  input; the tensor cores' operand tiles are decoded on chip (``csrc/act8_wgrad.cu``).
* ``activation_forward`` / ``activation_backward``: GELU (erf or tanh form) and SiLU, plain or gated, with the checkpoint of their
  input (and, for the layer after them, of their output) written in the same pass.
* ``linear`` and ``activation``: the same with autograd.

CUDA tensors run the kernels, CPU tensors the same arithmetic in torch ops.  Every call allocates what it returns and
what it needs from torch's allocator on the current stream of the tensor's device, and keeps nothing between calls.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
import torch.nn.functional as F

from . import native
from .exchange import GRAD_DTYPE, GraceCommError, _stream_ptr

GROUP = 32
KINDS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}
MAX_COLS = 1 << 30     # columns of a row: the kernels index within a row in 32 bits
MAX_TOKENS = (1 << 31) - 64


def pitch_of(cols: int) -> Tuple[int, int]:
    """Bytes of a row of codes (whole groups) and of a row of scales (whole eights of groups)."""
    groups = -(-cols // GROUP)
    return groups * GROUP, -(-groups // 8) * 8


class Act8:
    """A checkpoint of a tensor of ``shape`` and ``dtype``: ``codes`` int8 ``[rows, pitch]`` and ``scales`` uint8
    ``[rows, spitch]`` (``pitch_of``), rows being the product of all axes but the last.  A scale byte is 1 to 246 or, for a group that reads
    as NaN, 255; bytes past a row's groups are not specified."""

    __slots__ = ("shape", "dtype", "rows", "pitch", "spitch", "_data", "_at", "_codes", "_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, dtype: torch.dtype):
        shape = tuple(shape)
        if not shape:
            raise ValueError("Act8: a checkpoint has at least one axis")
        if dtype not in GRAD_DTYPE:
            raise TypeError("Act8: fp32, bf16 or fp16, not %s" % dtype)
        if shape[-1] > MAX_COLS:
            raise ValueError("Act8: at most 2^30 columns")
        pitch, spitch = pitch_of(shape[-1])
        rows = math.prod(shape[:-1])
        if codes.dtype != torch.int8 or scales.dtype != torch.uint8:
            raise TypeError("Act8: int8 codes and uint8 scales")
        if codes.shape != (rows, pitch) or scales.shape != (rows, spitch):
            raise ValueError("Act8: a checkpoint of %s has codes %s and scales %s, not %s and %s"
                             % (shape, (rows, pitch), (rows, spitch), tuple(codes.shape), tuple(scales.shape)))
        if codes.device != scales.device:
            raise ValueError("Act8: codes and scales are on different devices")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16 or scales.data_ptr() % 8:
            raise ValueError("Act8: codes and scales are contiguous, and start on 16- and 8-byte boundaries")
        self.shape, self.dtype, self.rows, self.pitch, self.spitch = shape, dtype, rows, pitch, spitch
        self._data, self._at, self._codes, self._scales = None, 0, codes, scales

    @classmethod
    def _over(cls, data: torch.Tensor, at: int, shape, dtype: torch.dtype) -> "Act8":
        """A checkpoint in ``data`` (uint8) from byte ``at``, a multiple of 16, on: the codes, then the scales.  One allocation holds it,
        or several of them, because allocating costs a small call more than computing."""
        held = cls.__new__(cls)
        pitch, spitch = pitch_of(shape[-1])
        held.shape, held.dtype, held.rows, held.pitch, held.spitch = shape, dtype, math.prod(shape[:-1]), pitch, spitch
        held._data, held._at, held._codes, held._scales = data, at, None, None
        return held

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            n = self.rows * self.pitch
            self._codes = self._data[self._at : self._at + n].view(torch.int8).view(self.rows, self.pitch)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            at = self._at + self.rows * self.pitch
            self._scales = self._data[at : at + self.rows * self.spitch].view(self.rows, self.spitch)
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._codes if self._data is None else self._data).device

    @property
    def nbytes(self) -> int:
        return self.rows * (self.pitch + self.spitch)

    def _tensors(self) -> Tuple[torch.Tensor, ...]:
        return (self._data,) if self._data is not None else (self._codes, self._scales)

    def _with(self, tensors) -> "Act8":
        """This checkpoint over ``_tensors()`` as autograd gives them back."""
        held = Act8.__new__(Act8)
        for name in ("shape", "dtype", "rows", "pitch", "spitch", "_at"):
            setattr(held, name, getattr(self, name))
        held._data, held._codes, held._scales = (tensors[0], None, None) if len(tensors) == 1 else (None,) + tuple(tensors)
        return held

    def _shell(self) -> "Act8":
        """Its description without its tensors, for a context that saves those with autograd's own means."""
        return self._with((None,))

    def __repr__(self):
        return "Act8(shape=%s, dtype=%s, device=%s, nbytes=%d)" % (self.shape, self.dtype, self.device, self.nbytes)


def held_bytes(shape) -> int:
    """Bytes of a checkpoint of a tensor of ``shape``, rounded up to a multiple of 16."""
    pitch, spitch = pitch_of(shape[-1])
    return (math.prod(shape[:-1]) * (pitch + spitch) + 15) // 16 * 16


def empty_like(shape, dtype: torch.dtype, device) -> Act8:
    """An Act8 for a tensor of ``shape`` whose contents are yet to be written."""
    return Act8._over(torch.empty(held_bytes(shape), dtype=torch.uint8, device=device), 0, shape, dtype)


# ---------------------------------------------------------------------------------------------------- shared checks
def _launch(device: torch.device, launch, *args) -> None:
    """``launch(*args, stream)`` on the current stream of ``device``, which is made current for the call if it is not."""
    index = device.index
    if index == torch.cuda.current_device():
        launch(*args, _stream_ptr(index))
    else:
        with torch.cuda.device(index):
            launch(*args, _stream_ptr(index))


def _autocast_type(x: torch.Tensor) -> Optional[torch.dtype]:
    """The type that products are computed in on ``x``'s device, None without autocast."""
    kind = "cuda" if x.is_cuda else "cpu"
    return torch.get_autocast_dtype(kind) if torch.is_autocast_enabled(kind) else None


def _check_tensor(x, what: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s: a tensor, not %s" % (what, type(x).__name__))
    if x.dtype not in GRAD_DTYPE:
        raise TypeError("%s: fp32, bf16 or fp16, not %s" % (what, x.dtype))
    if x.layout != torch.strided:
        raise TypeError("%s: a dense tensor, not %s" % (what, x.layout))
    if x.dim() == 0:
        raise ValueError("%s: at least one axis" % what)
    if x.shape[-1] > MAX_COLS:
        raise ValueError("%s: at most 2^30 columns" % what)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as ``[rows, cols]`` with neighbouring columns; a copy only where its strides leave no other way."""
    if x.dim() != 2:
        x = x.detach().reshape(math.prod(x.shape[:-1]), x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] > 1:
        x = x.detach().contiguous()
    return x


def _at(x: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """``_rows`` for a launch: the tensor to keep until then, its address, and the distance between its rows."""
    if x.is_neg():             # a view that changes the sign (``z.conj().imag``): memory has the other one
        x = x.detach().resolve_neg()
    if x.is_contiguous():      # no view is made: that would take longer than the checks of the whole call
        return x, x.data_ptr(), x.shape[-1]
    x = _rows(x)
    return x, x.data_ptr(), x.stride(0)


def _new_like(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of ``x``'s shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _ptrs(held: Optional[Act8]) -> Tuple[int, int]:
    """Addresses of a checkpoint's codes and scales."""
    if held is None:
        return 0, 0
    if held._data is None:
        return held._codes.data_ptr(), held._scales.data_ptr()
    at = held._data.data_ptr() + held._at
    return at, at + held.rows * held.pitch


# -------------------------------------------------------------------------------------------- the arithmetic on CPU
def _encode_cpu(x: torch.Tensor, held: Act8) -> None:
    rows, pitch = held.codes.shape
    groups = pitch // GROUP
    v = F.pad(_rows(x).float(), (0, pitch - x.shape[-1])).view(rows, groups, GROUP)
    finite = torch.isfinite(v).all(-1)
    top = v.abs().amax(-1) if v.numel() else v.new_zeros(rows, groups)
    e = torch.frexp(torch.where(finite, top, torch.zeros_like(top))).exponent.clamp(-119, 126)
    q = torch.ldexp(v, (7 - e).unsqueeze(-1)).round().clamp(-127, 127)
    held.codes.copy_(torch.where(finite.unsqueeze(-1), q, torch.zeros_like(q)).view(rows, pitch))
    held.scales.zero_()
    held.scales[:, :groups] = torch.where(finite, e + 120, torch.full_like(e, 255)).to(torch.uint8)


def _decode_cpu(held: Act8) -> torch.Tensor:
    rows, pitch = held.codes.shape
    groups = pitch // GROUP
    s = held.scales[:, :groups].int()
    v = torch.ldexp(held.codes.float().view(rows, groups, GROUP), (s - 127).unsqueeze(-1))
    v = torch.where((s == 255).unsqueeze(-1), torch.full_like(v, math.nan), v)
    return v.view(rows, pitch)[:, : held.shape[-1]].reshape(held.shape)


def _operand_cpu(held: Act8, dtype: torch.dtype) -> torch.Tensor:
    """``_decode_cpu`` as the product with a gradient of ``dtype`` takes it."""
    v = _decode_cpu(held)
    if dtype != torch.float16:
        return v
    wide = (held.scales[:, : held.pitch // GROUP] > 136).repeat_interleave(GROUP, 1)[:, : held.shape[-1]].reshape(held.shape)
    return torch.where(wide, torch.full_like(v, math.nan), v.half().float())


def _function_cpu(x: torch.Tensor, kind: str) -> Tuple[torch.Tensor, torch.Tensor]:
    if kind == "gelu":
        p = 0.5 * torch.erfc(-x * math.sqrt(0.5))
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        c, a = math.sqrt(2 / math.pi), 0.044715
        xx = (x * x).clamp_max(1e4)
        p = torch.sigmoid(2 * c * x * (1 + a * xx))
        return x * p, p + 2 * c * x * p * (1 - p) * (1 + 3 * a * xx)
    p = torch.sigmoid(x)
    return x * p, p * (1 + x * (1 - p))


# ------------------------------------------------------------------------------------------------------- checkpoints
def pack(x: torch.Tensor) -> Act8:
    """The checkpoint of ``x`` (fp32, bf16 or fp16, any shape and strides)."""
    _check_tensor(x, "act8.pack")
    device = x.device
    held = empty_like(x.shape, x.dtype, device)
    if x.is_cuda:
        v, at, stride = _at(x)
        _launch(device, native().act8_pack, at, stride, held.rows, held.shape[-1], GRAD_DTYPE[x.dtype], *_ptrs(held),
                held.pitch, held.spitch)
    else:
        _encode_cpu(x, held)
    return held


def unpack(held: Act8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``held`` stands for, contiguous, as its own or another of the three types."""
    dtype = held.dtype if dtype is None else dtype
    if dtype not in GRAD_DTYPE:
        raise TypeError("act8.unpack: fp32, bf16 or fp16, not %s" % dtype)
    device = held.device
    if device.type == "cuda":
        out, cols = torch.empty(held.shape, dtype=dtype, device=device), held.shape[-1]
        _launch(device, native().act8_unpack, *_ptrs(held), held.pitch, held.spitch, out.data_ptr(), cols, held.rows, cols, GRAD_DTYPE[dtype])
        return out
    return _decode_cpu(held).to(dtype)


# --------------------------------------------------------------------------------------------------- weight gradient
_sm_count = {}


def _sms(device: torch.device) -> int:
    n = _sm_count.get(device.index)
    if n is None:
        n = _sm_count[device.index] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


def weight_grad(grad: torch.Tensor, held: Act8, bias: bool = False, dtype: Optional[torch.dtype] = None
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``(dW, db)`` of ``y = x W^T + b``: ``dW [outs, ins] = sum over rows of grad^T x~`` with ``x~`` the values of ``held``, and with
    ``bias`` the column sums of ``grad`` (else None).  ``grad`` is ``[..., outs]`` with ``held``'s leading axes and, on the GPU, bf16 or
    fp16; the results are of ``grad``'s type or, with ``dtype=torch.float32``, not rounded below fp32.  With an fp16 gradient ``x~`` is
    taken in fp16: a checkpoint of another type is rounded where fp16 is subnormal, and a group of it with a value of 2^16 or more is NaN."""
    _check_tensor(grad, "act8.weight_grad: grad")
    outs, ins, rows = grad.shape[-1], held.shape[-1], held.rows
    if grad.shape[:-1] != held.shape[:-1]:
        raise ValueError("act8.weight_grad: grad %s and the checkpoint %s differ in their leading axes"
                         % (tuple(grad.shape), held.shape))
    if grad.device != held.device:
        raise ValueError("act8.weight_grad: grad is on %s, the checkpoint on %s" % (grad.device, held.device))
    dtype = grad.dtype if dtype is None else dtype
    if dtype not in (grad.dtype, torch.float32):
        raise TypeError("act8.weight_grad: results in grad's type or fp32, not %s" % dtype)
    if not grad.is_cuda:
        g = _rows(grad).float()
        with torch.autocast("cpu", enabled=False):      # (the product is one of fp32 numbers whatever the caller's)
            dw = g.t() @ _operand_cpu(held, grad.dtype).reshape(rows, ins)
        return dw.to(dtype), g.sum(0).to(dtype) if bias else None
    if grad.dtype == torch.float32:
        raise TypeError("act8.weight_grad: the tensor cores take bf16 or fp16 gradients; run the layer in one of them")
    if rows > MAX_TOKENS or outs * 2 > 1 << 31:
        raise ValueError("act8.weight_grad: at most 2^31 - 64 rows and 2^30 output features")
    if rows == 0 or outs == 0 or ins == 0:
        return (torch.zeros((outs, ins), dtype=dtype, device=grad.device),
                torch.zeros(outs, dtype=dtype, device=grad.device) if bias else None)
    C, device = native(), grad.device
    g, at, stride = _at(grad)
    if at % 16 or stride % 8 or stride < outs:   # not what a TMA load takes
        wide = torch.empty((rows, -(-outs // 8) * 8), dtype=g.dtype, device=device)
        _launch(device, C.act8_repitch, at, stride, wide.data_ptr(), rows, outs)
        g, at, stride = wide, wide.data_ptr(), wide.shape[1]
    out = torch.empty((outs, ins), dtype=dtype, device=device)
    db = torch.empty(outs, dtype=dtype, device=device) if bias else None
    f32, sms = int(dtype == torch.float32), _sms(device)
    nbytes = C.act8_wgrad_work_bytes(rows, outs, ins, f32, sms)
    work = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _launch(device, C.act8_wgrad, at, stride, *_ptrs(held), held.pitch, held.spitch, rows, outs, ins, GRAD_DTYPE[g.dtype],
            f32, out.data_ptr(), db.data_ptr() if bias else 0, 0 if work is None else work.data_ptr(), sms)
    return out, db


def check(device=None) -> None:
    """Waits for the device, all of its streams, and raises ``GraceCommError`` if a bounded wait of a ``weight_grad`` kernel ran out since the last
    check (its results are NaN)."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    with torch.cuda.device(device):
        words = native().act8_wgrad_status()
    if words[0]:
        raise GraceCommError(words[0], words[1], words[2], 0)


# ----------------------------------------------------------------------------------------------- activation functions
Held = Union[Act8, Tuple[Act8, Act8]]


def _kind(kind: str) -> int:
    if kind not in KINDS:
        raise ValueError("act8: unknown function %r (one of %s)" % (kind, ", ".join(KINDS)))
    return KINDS[kind]


def activation_forward(x: torch.Tensor, kind: str = "gelu", gated: bool = False, checkpoint_output: bool = False,
                       checkpoint: bool = True) -> Tuple[torch.Tensor, Optional[Held], Optional[Act8]]:
    """``(y, held, held_y)``: ``y = f(x)``, or for a gated function ``x = [a | b]`` and ``y = f(a) * b``; ``held`` is the checkpoint of
    ``x`` (a pair of them, of ``a`` and of ``b``; None with ``checkpoint=False``, where no backward pass follows), ``held_y`` with
    ``checkpoint_output`` that of ``y`` (what ``pack(y)`` gives), else None."""
    k = _kind(kind)
    _check_tensor(x, "act8.activation")
    if gated and x.shape[-1] % 2:
        raise ValueError("act8.activation: a gated function takes two halves, not %d columns" % x.shape[-1])
    cols, device, dtype = x.shape[-1] // 2 if gated else x.shape[-1], x.device, x.dtype
    shape = x.shape[:-1] + (cols,)
    a = b = out = None
    parts = (2 if gated else 1) if checkpoint else 0
    if parts:
        n = held_bytes(shape)
        data = torch.empty(parts * n, dtype=torch.uint8, device=device)
        a = Act8._over(data, 0, shape, dtype)
        b = Act8._over(data, n, shape, dtype) if gated else None
    if checkpoint_output:
        out = empty_like(shape, dtype, device)
    if x.is_cuda:
        y = torch.empty(shape, dtype=dtype, device=device) if gated else _new_like(x)
        v, at, stride = _at(x)
        _launch(device, native().act8_forward, at, stride, y.data_ptr(), math.prod(shape[:-1]), cols, GRAD_DTYPE[dtype], k, int(gated),
                *_ptrs(a), *_ptrs(b), *_ptrs(out), *pitch_of(cols))
    else:
        v = x.detach()
        y = _function_cpu(v[..., :cols].float(), kind)[0]
        if gated:
            y = y * v[..., cols:].float()
        y = y.to(x.dtype)
        for part, into in ((v[..., :cols], a), (v[..., cols:], b), (y, out)):
            if into is not None:
                _encode_cpu(part, into)
    return y, (a, b) if b is not None else a, out


def activation_backward(grad: torch.Tensor, held: Held, kind: str = "gelu", gated: bool = False) -> torch.Tensor:
    """The gradient of ``activation_forward``'s ``x`` from that of ``y``, at the values that ``held`` stands for."""
    k = _kind(kind)
    _check_tensor(grad, "act8.activation: grad")
    if gated != isinstance(held, tuple):
        raise ValueError("act8.activation: a gated function has a pair of checkpoints, another one of them")
    a, b = held if gated else (held, None)
    if tuple(grad.shape) != a.shape or (gated and b.shape != a.shape):
        raise ValueError("act8.activation: grad %s for a checkpoint of %s" % (tuple(grad.shape), a.shape))
    if grad.device != a.device or (gated and b.device != a.device):
        raise ValueError("act8.activation: grad is on %s, the checkpoint on %s" % (grad.device, a.device))
    cols, device = a.shape[-1], grad.device
    if grad.is_cuda:
        dx = torch.empty(grad.shape[:-1] + (2 * cols,), dtype=grad.dtype, device=device) if gated else _new_like(grad)
        g, at, stride = _at(grad)
        _launch(device, native().act8_backward, at, stride, dx.data_ptr(), a.rows, cols, GRAD_DTYPE[grad.dtype], k, int(gated),
                *_ptrs(a), *_ptrs(b), a.pitch, a.spitch)
        return dx
    g = grad.detach().float()
    f, d = _function_cpu(_decode_cpu(a), kind)
    return (torch.cat([g * _decode_cpu(b) * d, g * f], -1) if gated else g * d).to(grad.dtype)


# ------------------------------------------------------------------------------------------------------ with autograd
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, held):
        ctx.save_for_backward(weight, *held._tensors())
        ctx.held, ctx.has_bias = held._shell(), bias is not None
        return F.linear(x, weight, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        weight, *tensors = ctx.saved_tensors
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = grad @ weight
        want_bias = ctx.has_bias and ctx.needs_input_grad[2]
        if ctx.needs_input_grad[1]:
            dw, db = weight_grad(grad, ctx.held._with(tensors), bias=want_bias)
        elif want_bias:
            db = grad.reshape(-1, grad.shape[-1]).sum(0)
        return dx, dw, db, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, checkpoint: Optional[Act8] = None
           ) -> torch.Tensor:
    """``x W^T + b`` whose backward pass keeps an 8-bit checkpoint of ``x`` in the place of ``x``.  ``checkpoint``: that of ``x``, where
    the operation that made ``x`` wrote it already (``activation`` and ``residual_norm`` do on request)."""
    t = _autocast_type(x)
    if t is not None:
        x, weight, bias = x.to(t), weight.to(t), None if bias is None else bias.to(t)
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return F.linear(x, weight, bias)       # nothing reads x again
    _check_tensor(x, "act8.linear")
    if weight.dim() != 2:      # (the library's layer takes a vector too; its gradient is no product of matrices)
        raise ValueError("act8.linear: a weight of [outs, ins], not %s" % (tuple(weight.shape),))
    if x.is_cuda and x.dtype == torch.float32:
        raise TypeError("act8.linear: bf16 or fp16 on the GPU (or fp32 under autocast): the weight gradient runs on the tensor cores")
    if checkpoint is None:
        checkpoint = pack(x)
    elif checkpoint.shape != tuple(x.shape) or checkpoint.device != x.device:
        raise ValueError("act8.linear: a checkpoint of %s on %s for x %s on %s"
                         % (checkpoint.shape, checkpoint.device, tuple(x.shape), x.device))
    return _Linear.apply(x, weight, bias, checkpoint)


class _Activation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind, gated, checkpoint_output, box):
        y, held, out = activation_forward(x, kind, gated, checkpoint_output)
        box.append(out)
        a = held[0] if gated else held       # (of a pair, both are in one allocation)
        ctx.save_for_backward(a._data)
        ctx.kind, ctx.held = kind, tuple(h._shell() for h in held) if gated else (a._shell(),)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        held = tuple(h._with(ctx.saved_tensors) for h in ctx.held)
        gated = len(held) == 2
        return activation_backward(grad, held if gated else held[0], ctx.kind, gated), None, None, None, None


def activation(x: torch.Tensor, kind: str = "gelu", gated: bool = False, checkpoint_output: bool = False):
    """``activation_forward`` with autograd: ``y``, or with ``checkpoint_output`` the pair ``(y, Act8 of y)`` for the ``linear`` after it."""
    if torch.is_grad_enabled() and x.requires_grad:
        box = []
        y = _Activation.apply(x, kind, gated, checkpoint_output, box)
        held_y = box[0]
    else:
        y, _, held_y = activation_forward(x, kind, gated, checkpoint_output, checkpoint=False)
    return (y, held_y) if checkpoint_output else y
