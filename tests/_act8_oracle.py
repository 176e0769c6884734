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


# ------------------------------------------------------------------------------------- the residual-and-norm step
def wide(p, dims, none):
    """A parameter [cols], or a gate [sequences, cols], against [sequences, ..., cols]."""
    if p is None:
        return torch.full((), none, dtype=torch.float64)
    p = p.double()
    return p if p.dim() == 1 else p.view((p.shape[0],) + (1,) * (dims - 2) + (p.shape[1],))


def norm_stats(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps) if kind is not None else torch.ones_like(mean)
    return mean, rstd


def stream(x, block, post, post_weight, post_bias, gate, alpha, eps):
    """y before its rounding, and the size of the terms it is made of."""
    b = block.double()
    m, r = norm_stats(b, post, eps)
    n = (b - m) * r * wide(post_weight, b.dim(), 1.0) + wide(post_bias, b.dim(), 0.0)
    size = (b.abs() + m.abs()) * r * wide(post_weight, b.dim(), 1.0).abs() + wide(post_bias, b.dim(), 0.0).abs()
    g = wide(gate, b.dim(), 1.0)
    return alpha * x.double() + g * n, abs(alpha) * x.double().abs() + g.abs() * size


def normed(y, kind, weight, bias, eps):
    """h and the size of its terms."""
    v = y.double()
    m, r = norm_stats(v, kind, eps)
    w, b = wide(weight, v.dim(), 1.0), wide(bias, v.dim(), 0.0)
    return (v - m) * r * w + b, (v.abs() + m.abs()) * r * w.abs() + b.abs()


def _norm_back(c, size, hat, r, kind):
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    out = r * (c - (mean(c) if kind == "layer" else 0.0) - hat * mean(c * hat))
    return out, r * (size + (mean(size) if kind == "layer" else 0.0) + hat.abs() * mean(size * hat.abs()))


def block_norm_gradients(dh, dy, y, y_stats, b, b_stats, pre, post, pre_weight, post_weight, post_bias, gate, alpha):
    """{name: (gradient, size of its terms)} at the values y and b (b None: not kept) with the given (mean, rstd) of both."""
    dims, lead = dh.dim(), tuple(range(dh.dim() - 1))
    dh = dh.double()
    (m, r), got = y_stats, {}
    hat = (y - m) * r
    got["pre_weight"], got["pre_bias"] = ((dh * hat).sum(lead), (dh * hat).abs().sum(lead)), (dh.sum(lead), dh.abs().sum(lead))
    c = dh * wide(pre_weight, dims, 1.0)
    g, size = _norm_back(c, c.abs(), hat, r, pre)
    if dy is not None:
        g, size = g + dy.double(), size + dy.double().abs()
    got["x"] = (alpha * g, abs(alpha) * size)
    gw = wide(gate, dims, 1.0)
    e, e_size = g * gw, size * gw.abs()
    if b is not None:
        bm, br = b_stats
        bh = b if post is None else (b - bm) * br
        pw, pb = wide(post_weight, dims, 1.0), wide(post_bias, dims, 0.0)
        if gate is not None:
            over = lead if gate.dim() == 1 else lead[1:]
            got["gate"] = ((g * (bh * pw + pb)).sum(over), (size * ((bh * pw).abs() + pb.abs())).sum(over))
        if post is not None:
            got["post_weight"], got["post_bias"] = ((e * bh).sum(lead), (e_size * bh.abs()).sum(lead)), (e.sum(lead), e_size.sum(lead))
            e, e_size = _norm_back(e * pw, e_size * pw.abs(), bh, br, post)
    got["block"] = (e, e_size)
    return got
