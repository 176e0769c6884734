"""The kernels of the residual-and-norm step against the 64-bit formulas."""
import math

import pytest
import torch

from _act8_oracle import half_step
from _block_norm_cases import check, check_mixed, check_one_row, make
from grace_b200.ops import act8, block_norm

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
FORMS = [("layer", None, None, 1.0, False), ("rms", None, None, 2.63, True), ("rms", "rms", "sequence", 1.0, True),
         ("layer", "layer", "channel", 0.5, True), ("layer", "rms", None, 1.0, True), ("rms", None, "sequence", 1.0, False)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("pre,post,gate,alpha,with_stream", FORMS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 70), (3, 37, 256), (2, 5, 1000), (1, 33, 1003), (5, 7, 4096), (2, 9, 5001), (1, 3, 8192)])
def test_against_formulas(shape, pre, post, gate, alpha, with_stream, dtype):
    d, p = make(shape, dtype, pre, post, gate, seed=2, device="cuda")
    check(d, p, alpha=alpha, with_stream=with_stream)


@pytest.mark.parametrize("pre,post,gate,alpha,with_stream", FORMS)
def test_fp32_parameters(pre, post, gate, alpha, with_stream):
    for dtype in (BF16, FP16):
        d, p = make((2, 11, 136), dtype, pre, post, gate, param_dtype=FP32, seed=3, device="cuda", bias=False)
        check(d, p, alpha=alpha, with_stream=with_stream)


@pytest.mark.parametrize("shape", [(1, 3000, 64), (40, 100, 96), (700, 2, 40), (1, 1200, 1024)])
@pytest.mark.parametrize("gate", [None, "sequence"])
def test_many_rows(shape, gate):
    d, p = make(shape, BF16, "layer", "rms", gate, param_dtype=FP32, seed=4, device="cuda")
    check(d, p)


def test_no_parameters_at_all():
    d, p = make((2, 5, 72), BF16, "rms", "layer", None, seed=5, device="cuda")
    check(d, dict(pre="rms", post="layer"))


def test_strides():
    d, p = make((4, 6, 96), BF16, "rms", "rms", "sequence", seed=6, device="cuda")
    want = block_norm.residual_norm_forward(d["x"], d["block"], **p)
    back = block_norm.residual_norm_backward(d["dh"], d["dy"], want[2])
    wide = {}
    for k, off in (("x", 3), ("block", 8), ("dh", 1), ("dy", 16)):     # rows off their boundaries, and transposed
        t = torch.zeros(4, 6, 130, dtype=BF16, device="cuda")
        t[..., off:off + 96] = d[k]
        wide[k] = t[..., off:off + 96]
    turned = {k: d[k].transpose(0, 2).contiguous().transpose(0, 2) for k in d}
    q = dict(p, gate=torch.stack([p["gate"], p["gate"]], 1)[:, 0], pre_weight=torch.stack([p["pre_weight"]] * 2, 1)[:, 0])
    for e in (wide, turned):
        got = block_norm.residual_norm_forward(e["x"], e["block"], **q)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        grads = block_norm.residual_norm_backward(e["dh"], e["dy"], got[2])
        assert all(torch.equal(grads[k], back[k]) for k in back if back[k] is not None)


def test_parameters_off_their_boundaries():
    d, p = make((2, 3, 64), BF16, "layer", "layer", "channel", seed=7, device="cuda")
    q = {k: torch.cat([v[:1], v])[1:] if isinstance(v, torch.Tensor) else v for k, v in p.items()}
    a, b = block_norm.residual_norm_forward(d["x"], d["block"], **p), block_norm.residual_norm_forward(d["x"], d["block"], **q)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(d, q)


def test_non_finite_rows_stay_by_themselves():
    d, p = make((1, 6, 64), BF16, "rms", "rms", None, seed=8, device="cuda")
    d["x"][0, 2, 5], d["block"][0, 4, 7] = math.inf, math.nan
    h, y, saved = block_norm.residual_norm_forward(d["x"], d["block"], **p)
    rows = [0, 1, 3, 5]
    assert h[0, rows].isfinite().all() and h[0, 4].isnan().all() and not h[0, 2].isfinite().all()
    got = block_norm.residual_norm_backward(d["dh"], d["dy"], saved)
    for k in ("x", "block"):
        assert got[k][0, rows].isfinite().all() and got[k][0, 2].isnan().any()
    assert got["pre_weight"].isnan().any()


def test_constant_rows():
    """A row without variance: 1 / sqrt(eps) times nothing."""
    x, b = torch.full((3, 40), 2.0, dtype=BF16, device="cuda"), torch.full((3, 40), -0.5, dtype=BF16, device="cuda")
    h, y, saved = block_norm.residual_norm_forward(x, b, pre="layer", post="layer", eps=1e-6)
    assert not h.any() and torch.equal(y, x)
    got = block_norm.residual_norm_backward(torch.ones_like(x), None, saved)
    assert got["x"].isfinite().all() and got["block"].isfinite().all()


def test_empty():
    for shape in ((0, 64), (2, 0, 32), (3, 0)):
        x = torch.empty(shape, dtype=BF16, device="cuda")
        w = torch.ones(shape[-1], dtype=BF16, device="cuda")
        h, y, saved = block_norm.residual_norm_forward(x, x, pre="rms", pre_weight=w)
        got = block_norm.residual_norm_backward(x, x, saved)
        assert h.shape == y.shape == got["x"].shape == shape and not got["pre_weight"].any()


def test_same_bits_twice():
    d, p = make((8, 300, 520), BF16, "layer", "layer", "sequence", seed=9, device="cuda")
    _, _, saved = block_norm.residual_norm_forward(d["x"], d["block"], **p)
    a, b = (block_norm.residual_norm_backward(d["dh"], d["dy"], saved) for _ in range(2))
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_only_what_is_asked_for():
    d, p = make((2, 50, 64), BF16, "layer", "layer", "channel", seed=10, device="cuda")
    _, _, saved = block_norm.residual_norm_forward(d["x"], d["block"], **p)
    full = block_norm.residual_norm_backward(d["dh"], d["dy"], saved)
    for needs in ((True, False, False, False, False), (False, False, False, False, True), (False,) * 5, (False, True, False, True, False)):
        got = block_norm.residual_norm_backward(d["dh"], d["dy"], saved, needs)
        for n, k in zip(needs, block_norm.PARAMS):
            assert (got[k] is not None) == n and (not n or torch.equal(got[k], full[k]))
        assert torch.equal(got["x"], full["x"]) and torch.equal(got["block"], full["block"])


def test_graph_replay():
    d, p = make((2, 64, 256), BF16, "rms", "rms", "sequence", seed=11, device="cuda")

    def step():
        h, y, saved = block_norm.residual_norm_forward(d["x"], d["block"], checkpoint_output=True, **p)
        dw, _ = act8.weight_grad(d["dy"], saved.held_h)
        got = block_norm.residual_norm_backward(d["dh"], d["dy"], saved)
        return [h, y, dw] + [v for v in got.values() if v is not None]

    step()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    d2, _ = make((2, 64, 256), BF16, "rms", "rms", "sequence", seed=12, device="cuda")
    for k in d:
        d[k].copy_(d2[k])
    graphs[0].replay()
    want = step()
    graphs[1].replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("pre,post,gate", [("layer", None, None), ("rms", "rms", "sequence"), ("layer", "layer", "channel")])
@pytest.mark.parametrize("with_stream", [False, True])
def test_without_a_backward_pass(pre, post, gate, with_stream):
    """The same results, and nothing kept."""
    d, p = make((2, 5, 72), torch.bfloat16, pre, post, gate, seed=21, device="cuda")
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
    x = torch.randn(7, 96, generator=torch.Generator().manual_seed(22)).cuda()
    y = block_norm.residual_norm_forward(x, torch.zeros_like(x), pre="rms", residual_scale=alpha)[1].double()
    want = alpha * x.double()
    assert bool(((y - want).abs() <= 2 ** -24 * (1 + 2 ** -20) * torch.exp2(torch.floor(torch.log2(want.abs())) + 1)).all())


@pytest.mark.parametrize("cols", [96, 90])
def test_parameters_off_their_boundaries_by_one_and_by_four(cols):
    """Slices that start where no four elements do, and rows of a gate that do."""
    d, p = make((3, 5, cols), BF16, "layer", "layer", "sequence", seed=23, device="cuda")
    want = block_norm.residual_norm_forward(d["x"], d["block"], **p)
    back = block_norm.residual_norm_backward(d["dh"], d["dy"], want[2])
    for off in (1, 4):
        q = dict(p)
        for k in ("pre_weight", "pre_bias", "post_weight", "post_bias", "gate"):
            t = torch.zeros(p[k].numel() + off, dtype=BF16, device="cuda")
            t[off:] = p[k].reshape(-1)
            q[k] = t[off:].view(p[k].shape)
        got = block_norm.residual_norm_forward(d["x"], d["block"], **q)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        grads = block_norm.residual_norm_backward(d["dh"], d["dy"], got[2])
        assert all(torch.equal(grads[k], back[k]) for k in back)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("alpha", [2.63, 0.1, -1 / 3, 1.0])
def test_infinite_stream_keeps_its_sign(alpha, dtype):
    """alpha x is infinite where x is, whatever the part of alpha that fp32 does not hold, as on the CPU."""
    x = torch.randn(4, 96, generator=torch.Generator().manual_seed(24)).to(dtype)
    x[1, 3], x[1, 50], x[2, 7], x[3, 9] = math.inf, -math.inf, -math.inf, math.nan
    b = torch.full_like(x, 0.25)
    want = block_norm.residual_norm_forward(x, b, pre="rms", residual_scale=alpha)[1]
    y = block_norm.residual_norm_forward(x.cuda(), b.cuda(), pre="rms", residual_scale=alpha)[1].cpu()
    assert torch.equal(y.isnan(), x.isnan()) and torch.equal(want.isnan(), x.isnan())
    assert torch.equal(y.isinf(), x.isinf()) and torch.equal(y[x.isinf()], (x * math.copysign(1, alpha))[x.isinf()])
    # b + alpha_low x and the sum with alpha x are each rounded to fp32 (2^-24 of themselves, the first at most 0.25 and 2^-24 of the product),
    # then y to its type; equal bits are not owed, since the CPU rounds a 64-bit sum once
    finite = x.isfinite()
    exact = (alpha * x.double() + 0.25)[finite]
    part = 0.25 + 2.0 ** -24 * (alpha * x.double()).abs()[finite]
    least = 2.0 ** -25 if dtype == FP16 else 0.0
    assert ((y[finite].double() - exact).abs() <= (half_step(dtype) + 2.0 ** -24) * exact.abs() + 2.0 ** -24 * (1 + 2.0 ** -20) * part + least).all()


@pytest.mark.parametrize("alpha", [1.1e30, -2.7e37])
def test_a_product_beyond_the_range_is_infinite(alpha):
    x = torch.tensor([[1e38, -1e38, 3e20, 1.0]])
    y = block_norm.residual_norm_forward(x.cuda(), torch.zeros_like(x).cuda(), pre="rms", residual_scale=alpha)[1].cpu()
    want = (alpha * x.double()).float()
    assert torch.equal(y.isinf(), want.isinf()) and torch.equal(y[want.isinf()], want[want.isinf()])
    assert ((y - want)[~want.isinf()].abs() <= 2.0 ** -23 * want[~want.isinf()].abs()).all()


@pytest.mark.parametrize("kind", [BF16, FP16])
def test_autocast_keeps_the_stream(kind):
    """A stream in fp32 next to blocks in 16 bits: the sum is fp32's own, to the bit, and the norm of it that of fp32."""
    g = torch.Generator().manual_seed(25)
    x, b, w = (torch.randn(*s, generator=g).cuda() for s in ((6, 72), (6, 72), (72,)))
    b = b.to(kind).requires_grad_()
    x.requires_grad_()
    with torch.autocast("cuda", dtype=kind):
        h, y, held = block_norm.residual_norm(x, b, pre="rms", pre_weight=w, checkpoint_output=True)
    assert h.dtype == y.dtype == held.dtype == FP32 and torch.equal(y, x + b)
    want = torch.nn.functional.rms_norm((x + b).double(), (72,), w.double(), 1e-5)
    assert ((h - want).abs() <= 1e-6 * (1 + want.abs())).all()
    torch.autograd.backward((h, y), (torch.ones_like(h), torch.ones_like(y)))
    assert x.grad.dtype == FP32 and b.grad.dtype == kind and torch.equal(b.grad, x.grad.to(kind))
    with torch.autocast("cuda", dtype=kind):       # a stream in 16 bits stays in 16 bits; one without gradients is treated alike
        assert block_norm.residual_norm(x.detach().to(kind), b.detach(), pre="rms", pre_weight=w)[1].dtype == kind
        assert torch.equal(block_norm.residual_norm(x.detach(), b.detach(), pre="rms", pre_weight=w.to(kind))[1], y.detach())
        assert block_norm.residual_norm(x.detach().double(), b.detach(), pre="rms", pre_weight=w)[1].dtype == FP32
    with pytest.raises(ValueError):
        block_norm.residual_norm(x.detach(), b.detach(), pre="rms", pre_weight=w)


def test_views_that_change_the_sign():
    """The imaginary part of a conjugate is a view of memory with the other sign, in rows of one column without a stride to show it."""
    z = torch.randn(6, 40, dtype=torch.complex64, generator=torch.Generator().manual_seed(26)).cuda()
    for v in (z.conj().imag, z[:, :1].conj().imag, torch._neg_view(z.real.contiguous())):
        assert v.is_neg()
        c = v.clone()
        assert not c.is_neg() and torch.equal(act8.unpack(act8.pack(v)), act8.unpack(act8.pack(c)))
        assert torch.equal(act8.activation(v, "silu"), act8.activation(c, "silu"))
        w = v[0]
        h, y, saved = block_norm.residual_norm_forward(v, v, pre="rms", pre_weight=w)
        h2, y2, saved2 = block_norm.residual_norm_forward(c, c, pre="rms", pre_weight=c[0])
        assert torch.equal(h, h2) and torch.equal(y, y2)
        a, b = block_norm.residual_norm_backward(v, v, saved), block_norm.residual_norm_backward(c, c, saved2)
        assert torch.equal(a["x"], b["x"]) and torch.equal(a["pre_weight"], b["pre_weight"])


@pytest.mark.parametrize("kind", [BF16, FP16])
@pytest.mark.parametrize("pre,post,gate,alpha,with_stream", FORMS)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 70), (3, 37, 256), (2, 5, 1000), (2, 9, 5001), (1, 3, 8192)])
def test_a_block_in_16_bits_beside_an_fp32_stream(shape, pre, post, gate, alpha, with_stream, kind):
    check_mixed(shape, kind, pre, post, gate, alpha, with_stream, "cuda")


def test_a_block_in_16_bits_without_rows_and_as_slices():
    with torch.autocast("cuda", dtype=BF16):
        x, b = torch.empty(0, 64, device="cuda").requires_grad_(), torch.empty(0, 64, dtype=BF16, device="cuda").requires_grad_()
        gx, gb = torch.autograd.grad(block_norm.residual_norm(x, b, pre="rms", return_stream=False), (x, b), torch.empty(0, 64, device="cuda"))
        assert gx.shape == gb.shape == (0, 64) and gx.dtype == FP32 and gb.dtype == BF16
        wide = torch.randn(6, 130, generator=torch.Generator().manual_seed(28)).to("cuda", BF16)
        x = torch.randn(6, 96, generator=torch.Generator().manual_seed(29)).cuda()
        for off in (0, 1, 8, 16):        # rows off their boundaries
            a = block_norm.residual_norm(x, wide[:, off:off + 96], pre="layer")
            c = block_norm.residual_norm(x, wide[:, off:off + 96].contiguous(), pre="layer")
            assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_one_row_without_leading_axes():
    check_one_row("cuda")
