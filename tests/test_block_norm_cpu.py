"""The residual-and-norm step on the CPU: against the 64-bit formulas, which are themselves checked by differences, and its refusals."""
import pytest
import torch

from _act8_oracle import block_norm_gradients, norm_stats, normed, stream
from _block_norm_cases import check, check_mixed, check_one_row, make
from grace_b200.ops import act8, block_norm


@pytest.mark.parametrize("pre", ["layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("gate", [None, "channel", "sequence"])
def test_oracle_gradients_are_those_of_differences(pre, post, gate):
    d, p = make((2, 3, 5), torch.float64, pre, post, gate, seed=1)
    names = [k for k, v in p.items() if isinstance(v, torch.Tensor)]
    tensors = [d["x"], d["block"]] + [p[k] for k in names]
    get = lambda q, k: q.get(k)  # noqa: E731

    def loss(*t):
        q = dict(zip(names, t[2:]))
        y, _ = stream(t[0], t[1], post, get(q, "post_weight"), get(q, "post_bias"), get(q, "gate"), 1.7, 1e-5)
        h, _ = normed(y, pre, get(q, "pre_weight"), get(q, "pre_bias"), 1e-5)
        return (h * d["dh"]).sum() + (y * d["dy"]).sum()

    y, _ = stream(d["x"], d["block"], post, get(p, "post_weight"), get(p, "post_bias"), get(p, "gate"), 1.7, 1e-5)
    got = block_norm_gradients(d["dh"], d["dy"], y, norm_stats(y, pre, 1e-5), d["block"], norm_stats(d["block"], post, 1e-5), pre, post,
                               get(p, "pre_weight"), get(p, "post_weight"), get(p, "post_bias"), get(p, "gate"), 1.7)
    for i, name in enumerate(["x", "block"] + names):
        for at in range(0, tensors[i].numel(), max(1, tensors[i].numel() // 3)):
            diff = []
            for s in (1e-5, -1e-5):
                t = [v.clone() for v in tensors]
                t[i].view(-1)[at] += s
                diff.append(loss(*t).item())
            # differences: h^2 f'''/6 with f''' of the order of r^3 (10 at most here), and 1e-16 / h of rounding
            assert abs((diff[0] - diff[1]) / 2e-5 - got[name][0].reshape(-1)[at].item()) < 1e-7, name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pre,post,gate,alpha,with_stream", [
    ("layer", None, None, 1.0, False), ("rms", None, None, 2.63, True), ("rms", "rms", "sequence", 1.0, True),
    ("layer", "layer", "channel", 0.5, True), ("layer", "rms", None, 1.0, True), ("rms", None, "sequence", 1.0, False)])
@pytest.mark.parametrize("shape", [(2, 3, 70), (1, 1, 1), (3, 4, 32)])
def test_against_formulas(shape, pre, post, gate, alpha, with_stream, dtype):
    d, p = make(shape, dtype, pre, post, gate, seed=2)
    check(d, p, alpha=alpha, with_stream=with_stream)
    if dtype != torch.float32:
        d, p = make(shape, dtype, pre, post, gate, param_dtype=torch.float32, seed=3, bias=False)
        check(d, p, alpha=alpha, with_stream=with_stream)


def test_exact_values_give_exact_gradients():
    """Integers of a step of one are held exactly: the gradients are those of the plain module."""
    g = torch.Generator().manual_seed(4)
    x = torch.randint(-50, 50, (6, 64), generator=g).float()
    b = torch.randint(-50, 50, (6, 64), generator=g).float()
    x[:, ::32], b[:, ::32] = 40.0, 30.0
    w, bias = torch.randn(64, generator=g), torch.randn(64, generator=g)
    leaves = [t.requires_grad_() for t in (x, b, w, bias)]
    h = block_norm.residual_norm(x, b, pre="layer", pre_weight=w, pre_bias=bias, return_stream=False)
    dh = torch.randn(6, 64, generator=g)
    h.backward(dh)
    ref = [t.detach().clone().requires_grad_() for t in leaves]
    torch.nn.functional.layer_norm(ref[0] + ref[1], (64,), ref[2], ref[3], 1e-5).backward(dh)
    for p, q in zip(leaves, ref):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-5, atol=1e-6)


def test_autograd_outputs_and_unused_ones():
    d, p = make((2, 4, 40), torch.float32, "rms", "rms", "sequence", seed=5)
    x, b, gate = d["x"].requires_grad_(), d["block"].requires_grad_(), p.pop("gate").requires_grad_()
    h, y, held = block_norm.residual_norm(x, b, gate=gate, checkpoint_output=True, **p)
    assert isinstance(held, act8.Act8) and torch.equal(held.codes, act8.pack(h).codes)
    _, _, saved = block_norm.residual_norm_forward(x, b, gate=gate, **p)
    zero = torch.zeros_like(h)
    for out, grads in (((h, y), (d["dh"], d["dy"])), ((y,), (d["dy"],)), ((h,), (d["dh"],))):
        dh = grads[0] if out[0] is h else zero
        dy = grads[-1] if out[-1] is y else None
        want = block_norm.residual_norm_backward(dh, dy, saved)
        got = torch.autograd.grad(out, (x, b, gate), grads, retain_graph=True)
        for a, k in zip(got, ("x", "block", "gate")):
            assert torch.equal(a, want[k])


def test_refusals():
    d, p = make((2, 4, 40), torch.float32, "layer", "layer", "sequence", seed=6)
    f, x, b = block_norm.residual_norm_forward, d["x"], d["block"]
    bad = [dict(p, pre="batch"), dict(p, pre=None), dict(p, post=None), dict(p, post="rms"), dict(p, pre="rms"),
           dict(p, gate=p["gate"][:1]), dict(p, gate=p["gate"][0, :39]), dict(p, pre_weight=p["pre_weight"][:39]),
           dict(p, pre_weight=p["pre_weight"].view(1, 40)), dict(p, residual_scale=float("nan")), dict(p, eps=-1.0),
           dict(p, residual_scale=-1e39), dict(p, eps=1e39)]
    for q in bad:
        with pytest.raises(ValueError):
            f(x, b, **q)
    with pytest.raises(ValueError):
        f(x, b[:1], **p)
    with pytest.raises(ValueError):
        f(x, b.bfloat16(), **p)
    with pytest.raises(ValueError):
        f(x[0], b[0], **p)                                   # a gate of two axes needs sequences
    with pytest.raises(TypeError):
        f(x, b, **dict(p, pre_weight=p["pre_weight"].bfloat16()))
    with pytest.raises(TypeError):
        f(x.double(), b.double(), **p)
    with pytest.raises(ValueError):
        f(torch.zeros(1, 8193), torch.zeros(1, 8193))
    saved = f(x, b, **p)[2]
    with pytest.raises(ValueError):
        block_norm.residual_norm_backward(d["dh"][:1], None, saved)
    with pytest.raises(ValueError):
        block_norm.residual_norm_backward(d["dh"], d["dy"].bfloat16(), saved)


@pytest.mark.parametrize("pre,post,gate", [("layer", None, None), ("rms", "rms", "sequence"), ("layer", "layer", "channel")])
@pytest.mark.parametrize("with_stream", [False, True])
def test_without_a_backward_pass(pre, post, gate, with_stream):
    """The same results, and nothing kept."""
    d, p = make((2, 5, 72), torch.bfloat16, pre, post, gate, seed=21)
    q = dict(p, return_stream=with_stream, checkpoint_output=True)
    h, y, saved = block_norm.residual_norm_forward(d["x"], d["block"], **q)
    h2, y2, kept = block_norm.residual_norm_forward(d["x"], d["block"], checkpoint=False, **q)
    with torch.no_grad():
        out = block_norm.residual_norm(d["x"].requires_grad_(), d["block"], **q)
    assert kept.data is None and torch.equal(h, h2) and torch.equal(h, out[0]) and torch.equal(kept.held_h.codes, saved.held_h.codes)
    assert torch.equal(out[-1].scales[:, :3], saved.held_h.scales[:, :3]) and len(out) == (3 if with_stream else 2)
    if with_stream:
        assert torch.equal(y, y2) and torch.equal(y, out[1])
    with pytest.raises(ValueError):
        block_norm.residual_norm_backward(d["dh"], d["dy"], kept)


@pytest.mark.parametrize("alpha", [2.63, 0.1, 1 / 3])
def test_residual_factor_is_not_rounded(alpha):
    """y = alpha x to half a step (and 2^-20 of one for the part of alpha that 48 bits do not hold)."""
    x = torch.randn(7, 96, generator=torch.Generator().manual_seed(22))
    y = block_norm.residual_norm_forward(x, torch.zeros_like(x), pre="rms", residual_scale=alpha)[1].double()
    want = alpha * x.double()
    assert bool(((y - want).abs() <= 2 ** -24 * (1 + 2 ** -20) * torch.exp2(torch.floor(torch.log2(want.abs())) + 1)).all())


def test_autocast_keeps_the_stream():
    """A stream in fp32 next to blocks in 16 bits: the sum is fp32's own, to the bit."""
    g = torch.Generator().manual_seed(25)
    x, b, w = torch.randn(6, 72, generator=g), torch.randn(6, 72, generator=g).bfloat16().requires_grad_(), torch.randn(72, generator=g)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        h, y, held = block_norm.residual_norm(x, b, pre="rms", pre_weight=w, checkpoint_output=True)
        assert block_norm.residual_norm(x.bfloat16(), b.detach(), pre="rms", pre_weight=w)[1].dtype == torch.bfloat16
    assert h.dtype == y.dtype == held.dtype == torch.float32 and torch.equal(y, x + b)
    h.sum().backward()
    assert b.grad.dtype == torch.bfloat16 and b.grad.isfinite().all()


@pytest.mark.parametrize("pre,post,gate,alpha,with_stream", [
    ("layer", None, None, 1.0, False), ("rms", "rms", "sequence", 1.0, True), ("layer", "layer", "channel", 0.5, True), ("rms", None, "sequence", 1.0, False)])
def test_a_block_in_16_bits_beside_an_fp32_stream(pre, post, gate, alpha, with_stream):
    check_mixed((2, 3, 70), torch.bfloat16, pre, post, gate, alpha, with_stream, "cpu")


def test_one_row_without_leading_axes():
    check_one_row("cpu")


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 32), (3, 0), (0,)])
def test_empty(shape):
    x, w = torch.empty(shape).requires_grad_(), torch.ones(shape[-1]).requires_grad_()
    h, y, held = block_norm.residual_norm(x, x.detach(), pre="layer", pre_weight=w, pre_bias=w, checkpoint_output=True)
    assert h.shape == y.shape == held.shape == shape
    (h.sum() + y.sum()).backward()
    assert x.grad.shape == shape and w.grad.shape == w.shape and not w.grad.any()
    with torch.no_grad():
        assert block_norm.residual_norm(x, x, pre="rms", return_stream=False).shape == shape
