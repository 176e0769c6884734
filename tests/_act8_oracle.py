"""The 8-bit activation checkpoint operators in plain 64-bit arithmetic, for the tests."""
import math

import torch


def held_value(x):
    """What a checkpoint of x reads back as (float64): groups of 32, scale 2^(floor(log2 of the largest magnitude) - 6)."""
    rows, cols, groups = math.prod(x.shape[:-1]), x.shape[-1], -(-x.shape[-1] // 32)
    v = torch.nn.functional.pad(x.double().reshape(rows, cols), (0, -cols % 32)).view(rows, groups, 32)
    finite = torch.isfinite(v).all(-1, keepdim=True)
    top = torch.where(finite, v.abs().amax(-1, keepdim=True) if v.numel() else v[..., :1], torch.zeros_like(v[..., :1]))
    exponent = torch.frexp(top)[1].clamp(-119, 126).double() - 1
    step = torch.exp2(exponent - 6)
    q = torch.round(v / step).clamp(-127, 127) * step
    return torch.where(finite, q, torch.full_like(q, math.nan)).view(rows, groups * 32)[:, :cols].reshape(x.shape)


def function(x, kind):
    """(f, f') in float64."""
    x = x.double().requires_grad_()
    with torch.enable_grad():
        if kind == "gelu":
            y = 0.5 * x * torch.special.erfc(-x / math.sqrt(2))
        elif kind == "gelu_tanh":
            y = x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
        else:
            y = x * torch.sigmoid(x)
        d, = torch.autograd.grad(y.sum(), x)
    return y.detach(), d


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, tol, what=""):
    """Every element within its tolerance (a tensor or a number); NaN exactly where the other has it."""
    got, want = got.double().cpu(), want.cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu().expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN in other places"
    off = (got - want).abs() - tol
    off = torch.where(torch.isnan(want), torch.full_like(off, -1), off)
    off = torch.where(got == want, torch.full_like(off, -1), off)
    if off.numel() and off.max() > 0:
        i = int(off.argmax())
        raise AssertionError("%s: element %d is %r, want %r within %r (%d of %d off)" % (
            what, i, got.flatten()[i].item(), want.flatten()[i].item(), tol.flatten()[i].item(), int((off > 0).sum()), off.numel()))
