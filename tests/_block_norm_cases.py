"""Checks of the residual-and-norm step that the CPU and the GPU tests share."""
import torch

from _act8_oracle import block_norm_gradients, close, half_step, held_value, norm_stats, normed, stream
from grace_b200.ops import act8, block_norm
from grace_b200.ops.block_norm import PARAMS

#: fp32 arithmetic relative to the size of the terms: a row's sums (a tree over up to 8192 values: 13 levels and 8 in order, 2^-24 each), the
#: reciprocal root and the products, about 40 roundings in all
REL = 40 * 2.0 ** -24


def make(shape, dtype, pre, post, gate, param_dtype=None, seed=0, device="cpu", bias=True):
    g = torch.Generator().manual_seed(seed)
    cols, pd = shape[-1], param_dtype or dtype

    def rand(*s, scale=1.0, add=0.0, dt=dtype):
        return (torch.randn(*s, generator=g) * scale + add).to(dt).to(device)

    d = dict(x=rand(*shape, scale=2.0), block=rand(*shape, scale=1.5, add=0.3))
    p = dict(pre=pre, post=post, pre_weight=rand(cols, scale=0.3, add=1.0, dt=pd))
    if pre == "layer" and bias:
        p["pre_bias"] = rand(cols, scale=0.2, dt=pd)
    if post:
        p["post_weight"] = rand(cols, scale=0.3, add=1.0, dt=pd)
        if post == "layer" and bias:
            p["post_bias"] = rand(cols, scale=0.2, dt=pd)
    if gate:
        p["gate"] = rand(*((cols,) if gate == "channel" else (shape[0], cols)), scale=0.4, add=0.5, dt=pd)
    d["dh"], d["dy"] = rand(*shape, scale=0.1), rand(*shape, scale=0.1)
    return d, p


def check(d, p, alpha=1.0, eps=1e-5, with_stream=True):
    """Forward and backward of one call against the 64-bit formulas, each step from what the one before it really gave."""
    dtype = d["x"].dtype
    half, least = half_step(dtype), 2.0 ** -25 if dtype == torch.float16 else 0.0
    h, y, saved = block_norm.residual_norm_forward(d["x"], d["block"], residual_scale=alpha, eps=eps, return_stream=with_stream,
                                                   checkpoint_output=True, **p)
    # the stream is known from its checkpoint alone where it is not returned: ask for it once more
    full = y if with_stream else block_norm.residual_norm_forward(d["x"], d["block"], residual_scale=alpha, eps=eps, **p)[1]
    assert (y is None) != with_stream and h.dtype == dtype and h.shape == d["x"].shape
    cpu = {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    get = cpu.get
    xb = d["x"].cpu(), d["block"].cpu()
    want, size = stream(*xb, get("post"), get("post_weight"), get("post_bias"), get("gate"), alpha, eps)
    close(full, want, half * want.abs() + REL * size + least, "y")
    yc = full.cpu()
    want, size = normed(yc, p["pre"], get("pre_weight"), get("pre_bias"), eps)
    close(h, want, half * want.abs() + REL * size + least, "h")
    two = get("post") is not None or get("gate") is not None
    for held, of in ((saved.held_y, full), (saved.held_block, d["block"] if two else None), (saved.held_h, h)):
        assert (held is None) == (of is None)
        if held is not None:
            ref = act8.pack(of)
            groups = -(-of.shape[-1] // 32)
            assert torch.equal(held.codes, ref.codes) and torch.equal(held.scales[:, :groups], ref.scales[:, :groups])
    stats = saved.stats.cpu().double()
    at = lambda i: stats[:, i].reshape(yc.shape[:-1] + (1,))  # noqa: E731
    for i, v, kind in ((0, yc, p["pre"]), (2, xb[1], get("post"))):
        if kind is not None:
            m, r = norm_stats(v.double(), kind, eps)
            close(at(i), m, REL * v.double().abs().mean(-1, keepdim=True), "mean")
            close(at(i + 1), r, REL * r * (1 + m.abs() * r), "rstd")
    dy = d["dy"] if with_stream else None
    got = block_norm.residual_norm_backward(d["dh"], dy, saved)
    want = block_norm_gradients(d["dh"].cpu(), None if dy is None else dy.cpu(), held_value(yc), (at(0), at(1)),
                                held_value(xb[1]) if two else None, (at(2), at(3)), p["pre"], get("post"), get("pre_weight"),
                                get("post_weight"), get("post_bias"), get("gate"), alpha)
    rows = yc[..., 0].numel()
    for name in ("x", "block") + block_norm.PARAMS:
        if name not in ("x", "block") and get(name) is None:
            assert got[name] is None
            continue
        w, size = want[name]
        out = got[name]
        own = half_step(out.dtype)
        # (sums over rows: in order within a run, at most `rows` additions; the terms themselves twice REL)
        rel = 2 * REL if name in ("x", "block") else 2 * REL + rows * 2.0 ** -24
        close(out, w, own * w.abs() + rel * size + (2.0 ** -25 if out.dtype == torch.float16 else 0.0), name)
    return h, y, got


def check_mixed(shape, kind, pre, post, gate, alpha, with_stream, device):
    """A block in 16 bits beside a stream in fp32, under autocast: to the bit what the block gives in fp32, its gradient rounded once."""
    d, p = make(shape, torch.float32, pre, post, gate, seed=27, device=device)
    block = d["block"].to(kind)
    q = dict(p, residual_scale=alpha, return_stream=with_stream, checkpoint_output=True)
    wanted = [k for k in PARAMS if k in p]

    def run(b, mixed):
        leaves = [d["x"].clone().requires_grad_(), b.clone().requires_grad_()] + [p[k].clone().requires_grad_() for k in wanted]
        with torch.autocast(device, dtype=kind, enabled=mixed):
            out = block_norm.residual_norm(leaves[0], leaves[1], **dict(q, **dict(zip(wanted, leaves[2:]))))
            with torch.no_grad():
                again = block_norm.residual_norm(leaves[0], leaves[1], **dict(q, **dict(zip(wanted, leaves[2:]))))
        assert all(torch.equal(a, b) for a, b in zip(out[:-1], again[:-1])) and torch.equal(out[-1].codes, again[-1].codes)
        grads = torch.autograd.grad(out[:-1], leaves, (d["dh"], d["dy"])[: len(out) - 1])
        return out, grads

    got, grads = run(block, True)
    want, ref = run(block.float(), False)
    assert len(got) == (3 if with_stream else 2)
    for a, b in zip(got[:-1], want[:-1]):
        assert a.dtype == torch.float32 and torch.equal(a, b)
    assert got[-1].dtype == torch.float32 and torch.equal(got[-1].codes, want[-1].codes)
    for i, (a, b) in enumerate(zip(grads, ref)):
        assert a.dtype == (kind if i == 1 else torch.float32) and torch.equal(a, b.to(a.dtype)), i


def check_one_row(device):
    """A row without leading axes gives what it gives as the one row of a matrix."""
    for pre, post, gate in (("layer", None, None), ("rms", "layer", "channel"), ("layer", "rms", "channel")):
        d, p = make((1, 72), torch.float32, pre, post, gate, seed=30, device=device)
        want = block_norm.residual_norm_forward(d["x"], d["block"], **p)
        got = block_norm.residual_norm_forward(d["x"][0], d["block"][0], **p)
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[1][0])
        want = block_norm.residual_norm_backward(d["dh"], d["dy"], want[2])
        got = block_norm.residual_norm_backward(d["dh"][0], d["dy"][0], got[2])
        for k, v in want.items():
            assert (got[k] is None) == (v is None) and (v is None or torch.equal(got[k], v[0] if k in ("x", "block") else v)), k
        leaves = [d["x"][0].requires_grad_(), d["block"][0].requires_grad_(), p["pre_weight"].requires_grad_()]
        h, y = block_norm.residual_norm(*leaves[:2], **p)
        grads = torch.autograd.grad((h, y), leaves, (d["dh"][0], d["dy"][0]))
        assert all(torch.equal(a, b) for a, b in zip(grads, (got["x"], got["block"], got["pre_weight"])))
