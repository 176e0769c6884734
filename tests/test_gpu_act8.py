"""The kernels of 8-bit activation checkpoints against 64-bit arithmetic."""
import math

import pytest
import torch

from _act8_oracle import close, function, half_step, held_value
from test_act8_cpu import check_fp16_operand
from grace_b200.ops import act8, native
from grace_b200.ops.exchange import GraceCommError

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def rand(*shape, seed=0, dtype=FP32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ---------------------------------------------------------------------------------------------------------- checkpoints
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (1, 33), (3, 7), (5, 64), (2, 3, 100), (37, 1003), (300, 256), (1, 8200), (2049, 40)])
def test_round_trip(shape, dtype):
    x = rand(*shape, dtype=dtype, scale=3.0)
    held = act8.pack(x)
    host = act8.pack(x.cpu())
    groups = -(-shape[-1] // 32)
    assert torch.equal(held.codes.cpu(), host.codes) and torch.equal(held.scales[:, :groups].cpu(), host.scales[:, :groups])
    close(act8.unpack(held).cpu(), held_value(x.cpu()), 2.0 ** -25 if dtype == FP16 else 0.0, "unpack")
    assert torch.equal(act8.unpack(held, FP32).cpu().double(), held_value(x.cpu()))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_strides_and_offsets(dtype):
    wide = rand(40, 210, dtype=dtype, seed=1)
    for x in (wide[:, 3:103], wide[::2, :96], wide.t(), wide[:, 5], wide[0].expand(6, 210), wide.view(8, 5, 210)[:, 1:3, 8:40],
              wide[:, ::2]):
        assert torch.equal(act8.unpack(act8.pack(x)), act8.unpack(act8.pack(x.contiguous())))
        assert torch.equal(act8.unpack(act8.pack(x), FP32).cpu().double(), held_value(x.cpu()))


def test_empty():
    for shape in ((0, 64), (4, 0), (0,), (0, 0)):
        x = torch.empty(shape, device="cuda", dtype=BF16)
        assert act8.unpack(act8.pack(x)).shape == shape
        assert act8.activation(x, "silu").shape == shape


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_extremes(dtype):
    top = float(torch.finfo(dtype).max)
    x = torch.zeros(8, 64)
    x[0, 3], x[1, 40], x[2, 5], x[3, 6] = math.inf, math.nan, -math.inf, top
    x[4, :2] = torch.tensor([float(torch.finfo(dtype).tiny), -float(torch.finfo(dtype).tiny) / 4])
    x[5, 32:] = 1.0
    x[6, :8] = torch.tensor([64.0, 0.5, 1.5, 2.5, -0.5, -1.5, 127.5, -126.5])
    x = x.to(dtype)
    got = act8.unpack(act8.pack(x.cuda()), FP32).cpu()
    assert got[0, :32].isnan().all() and got[1, 32:].isnan().all() and got[2, :32].isnan().all() and not got[:3].isnan().all(-1).any()
    close(got, held_value(x), 0.0)


def test_more_elements_than_a_launch_takes():
    """More than 2^32 elements: offsets past 32 bits, and a second launch for the last rows (which are compared)."""
    rows, cols = (1 << 32) // 4096 + 3, 4096
    x = torch.zeros(rows, cols, dtype=FP16, device="cuda")
    x[-3:] = rand(3, cols, dtype=FP16, seed=2)
    held = act8.pack(x)
    assert torch.equal(act8.unpack(act8.Act8(held.codes[-3:], held.scales[-3:], (3, cols), FP16)), act8.unpack(act8.pack(x[-3:])))
    del x
    assert torch.equal(act8.unpack(held)[-3:], act8.unpack(act8.Act8(held.codes[-3:], held.scales[-3:], (3, cols), FP16)))


# ------------------------------------------------------------------------------------------------- activation functions
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", [(1, 32), (3, 45), (65, 264)])
def test_activation(shape, kind, gated, dtype):
    rows, f = shape
    x = rand(rows, f * (2 if gated else 1), dtype=dtype, seed=3, scale=2.5)
    g = rand(rows, f, dtype=dtype, seed=4)
    y, held, out = act8.activation_forward(x, kind, gated=gated, checkpoint_output=True)
    dx = act8.activation_backward(g, held, kind, gated=gated)
    v, gd = x.cpu().double(), g.cpu().double()
    a, b = v[:, :f], v[:, f:]
    # the functions: 1.5e-7 / 2 of the error function's approximation and a few fp32 roundings, times |x|; then one rounding
    eps, least = half_step(dtype), 2.0 ** -25 if dtype == FP16 else 0.0
    want = function(a, kind)[0] * (b if gated else 1)
    f_err = 1e-6 * (1 + a.abs())
    close(y, want, eps * want.abs() + f_err * (b.abs() if gated else 1) + least, "y")
    assert torch.equal(act8.unpack(out, FP32).cpu().double(), held_value(y.cpu()))
    assert torch.equal(out.codes, act8.pack(y).codes)
    ha, hb = held_value(x[:, :f].cpu()), held_value(x[:, f:].cpu())
    fa, da = function(ha, kind)
    f_err = 1e-6 * (1 + ha.abs())
    if gated:
        want = torch.cat([gd * hb * da, gd * fa], -1)
        tol = torch.cat([gd.abs() * hb.abs() * f_err, gd.abs() * f_err], -1)
    else:
        want, tol = gd * da, gd.abs() * f_err
    close(dx, want, eps * want.abs() + tol + 3 * 2.0 ** -24 * want.abs() + least, "dx")


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activation_far_out(kind):
    x = torch.tensor([-3e38, -1e30, -200.0, -90.0, -13.0, -8.0, 0.0, 8.0, 13.0, 90.0, 200.0, 1e30]).view(-1, 1).to(BF16)
    y, held, _ = act8.activation_forward(x.cuda(), kind)
    dx = act8.activation_backward(torch.ones_like(x).cuda(), held, kind)
    f, _ = function(x, kind)
    d = torch.where(x.double() > 9, 1.0, torch.where(x.double() < -20, 0.0, function(held_value(x).clamp(-20, 20), kind)[1]))
    close(y, f, half_step(BF16) * f.abs() + 2e-5, "y")
    close(dx, d, half_step(BF16) * d.abs() + 2e-5, "dx")


def test_activation_strided_and_autograd():
    wide = rand(6, 5, 200, dtype=BF16, seed=5)
    x = wide[:, :, 4:132].requires_grad_()
    y, held = act8.activation(x, "silu", gated=True, checkpoint_output=True)
    g = rand(6, 64, 5, dtype=BF16, seed=6).transpose(1, 2)
    dx, = torch.autograd.grad(y, x, g)
    y2, held2, _ = act8.activation_forward(x.detach().contiguous(), "silu", gated=True)
    assert torch.equal(y, y2) and torch.equal(dx, act8.activation_backward(g.contiguous(), held2, "silu", gated=True))
    with torch.no_grad():
        assert torch.equal(act8.activation(x, "silu", gated=True), y)


# ------------------------------------------------------------------------------------------------------ weight gradient
def check_weight_grad(tokens, outs, ins, dtype, out, bias=True, seed=7, x=None, g=None):
    x = rand(tokens, ins, dtype=dtype, seed=seed) if x is None else x
    g = rand(tokens, outs, dtype=dtype, seed=seed + 1, scale=0.1) if g is None else g
    dw, db = act8.weight_grad(g, act8.pack(x), bias=bias, dtype=out)
    assert dw.dtype == out and dw.shape == (outs, ins)
    gd, xd = g.cpu().double(), held_value(x.cpu())
    want, size = gd.t() @ xd, gd.abs().t() @ xd.abs()
    # one truncated fp32 addition for 16 tokens and the joins of up to 8 partial sums, then one rounding to the type
    least = 2.0 ** -25 if out == FP16 else 0.0
    tail = 2.0 ** -25 * gd.abs().sum(0).view(-1, 1) if dtype == FP16 else 0.0     # fp16 operands: subnormal values are rounded
    close(dw, want, half_step(out) * want.abs() + (tokens / 16 + 24) * 2.0 ** -23 * size + least + tail, "dW")
    if bias:
        want, size = gd.sum(0), gd.abs().sum(0)
        close(db, want, half_step(out) * want.abs() + (tokens + 8) * 2.0 ** -24 * size + least, "db")
    else:
        assert db is None
    return dw, db


@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 200, 513, 1100])
@pytest.mark.parametrize("outs,ins", [(64, 32), (8, 128), (256, 128), (264, 160), (1000, 96)])
def test_weight_grad(tokens, outs, ins):
    check_weight_grad(tokens, outs, ins, BF16, BF16)


@pytest.mark.parametrize("dtype,out", [(BF16, FP32), (FP16, FP16), (FP16, FP32)])
@pytest.mark.parametrize("tokens,outs,ins", [(1, 1, 1), (100, 72, 40), (777, 101, 1003), (2000, 600, 257)])
def test_weight_grad_types_and_odd_sizes(tokens, outs, ins, dtype, out):
    check_weight_grad(tokens, outs, ins, dtype, out)


@pytest.mark.parametrize("tokens,outs,ins", [(4096, 1024, 1024), (16384, 512, 640), (300, 4096, 2500), (5000, 1000, 99), (9000, 2100, 2700)])
def test_weight_grad_larger(tokens, outs, ins):
    check_weight_grad(tokens, outs, ins, BF16, FP32, bias=True)
    check_weight_grad(tokens, outs, ins, BF16, BF16, bias=False)


def test_weight_grad_one_column_of_tiles_has_every_bias_column():
    check_weight_grad(130, 700, 20, BF16, FP32)          # one tile along the inputs: a CTA adds up all 256 columns
    check_weight_grad(130, 30, 128 * 130, BF16, FP32)    # 130 of them: two columns each, most CTAs none


def test_weight_grad_strides():
    g, x = rand(3, 70, 200, dtype=BF16, seed=8), rand(3, 70, 64, dtype=BF16, seed=9)
    held = act8.pack(x)
    for part in (g[..., 8:136], g[..., 1:130], g.transpose(0, 1).contiguous().transpose(0, 1)[..., :64], g[:, :1].expand(3, 70, 200)):
        a, b = act8.weight_grad(part, held, bias=True), act8.weight_grad(part.contiguous(), held, bias=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_weight_grad_scales_differ_by_group_and_token():
    x = torch.zeros(96, 96)
    x[:, :32] = torch.exp2(torch.arange(96) % 60 - 30.0).view(-1, 1) * torch.randn(96, 32, generator=torch.Generator().manual_seed(1))
    x[:, 64:] = torch.randn(96, 32, generator=torch.Generator().manual_seed(2)) * 1e-3
    check_weight_grad(96, 64, 96, BF16, FP32, x=x.to(BF16).cuda())


def test_weight_grad_non_finite_values_reach_their_rows_and_columns_only():
    x, g = rand(100, 96, dtype=BF16, seed=10), rand(100, 64, dtype=BF16, seed=11)
    x[7, 40] = math.inf
    dw, db = act8.weight_grad(g, act8.pack(x), bias=True)
    assert dw[:, 32:64].isnan().all() and dw[:, :32].isfinite().all() and dw[:, 64:].isfinite().all() and db.isfinite().all()
    g[3, 5] = math.nan
    dw, db = act8.weight_grad(g, act8.pack(rand(100, 96, dtype=BF16)), bias=True)
    assert dw[5].isnan().all() and dw[:5].isfinite().all() and dw[6:].isfinite().all() and db.isnan().sum() == 1


def test_weight_grad_same_bits_twice_and_no_failure():
    x, g = rand(2500, 300, dtype=BF16, seed=12), rand(2500, 280, dtype=BF16, seed=13)
    held = act8.pack(x)
    a, b = act8.weight_grad(g, held, bias=True), act8.weight_grad(g, held, bias=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    act8.check()


def test_weight_grad_refusals():
    held = act8.pack(rand(8, 64, dtype=BF16))
    with pytest.raises(TypeError):
        act8.weight_grad(rand(8, 64), held)
    with pytest.raises(TypeError):
        act8.weight_grad(rand(8, 64, dtype=BF16), held, dtype=FP16)
    with pytest.raises(ValueError):
        act8.weight_grad(rand(9, 64, dtype=BF16), held)
    with pytest.raises(ValueError):
        act8.weight_grad(rand(8, 64, dtype=BF16).cpu(), held)
    with pytest.raises(TypeError):
        act8.linear(rand(8, 64).requires_grad_(), rand(4, 64).requires_grad_())
    dw, db = act8.weight_grad(torch.empty(0, 16, dtype=BF16, device="cuda"), act8.pack(torch.empty(0, 64, dtype=BF16, device="cuda")), bias=True)
    assert dw.shape == (16, 64) and not dw.any() and not db.any()


# ----------------------------------------------------------------------------------------------------------- as a layer
def test_linear_and_activation_together():
    x, w1, b1, w2 = (rand(50, 64, dtype=BF16, seed=14), rand(128, 64, dtype=BF16, seed=15, scale=0.2), rand(128, dtype=BF16, seed=16),
                     rand(64, 128, dtype=BF16, seed=17, scale=0.2))
    leaves = [t.requires_grad_() for t in (x, w1, b1, w2)]
    h = act8.linear(x, w1, b1)
    a, held = act8.activation(h, "gelu", checkpoint_output=True)
    y = act8.linear(a, w2, checkpoint=held)
    g = rand(50, 64, dtype=BF16, seed=18)
    y.backward(g)
    da = g @ w2
    dh = act8.activation_backward(da, act8.pack(h), "gelu")
    dw1, db1 = act8.weight_grad(dh, act8.pack(x), bias=True)
    assert torch.equal(w2.grad, act8.weight_grad(g, act8.pack(a))[0])
    assert torch.equal(w1.grad, dw1) and torch.equal(b1.grad, db1) and torch.equal(x.grad, dh @ w1)
    ref = [t.detach().clone().requires_grad_() for t in leaves]
    full = torch.nn.functional.gelu(torch.nn.functional.linear(ref[0], ref[1], ref[2])) @ ref[3].t()
    full.backward(g)
    for p, q in zip(leaves, ref):     # against the layer that keeps everything: the codes' steps, 2^-7 of their group's leading power at most
        assert (p.grad - q.grad).float().norm() < 0.05 * q.grad.float().norm()


def test_autocast():
    x, w, b = rand(40, 64, seed=19).requires_grad_(), rand(32, 64, seed=20).requires_grad_(), rand(32, seed=21).requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        y = act8.linear(x, w, b)
    assert y.dtype == BF16
    y.float().sum().backward()
    assert w.grad.dtype == FP32 and x.grad.dtype == FP32 and torch.equal(b.grad, torch.full_like(b, 40.0))


def test_graph_replay_and_two_graphs():
    """Captured calls replay on new values; two graphs and eager calls in between do not share anything."""
    x, g = rand(700, 256, dtype=BF16, seed=22), rand(700, 520, dtype=BF16, seed=23)

    def step():
        a, held, out = act8.activation_forward(x, "gelu", checkpoint_output=True)
        dw, db = act8.weight_grad(g, out, bias=True)
        return a, dw, db, act8.activation_backward(a, held, "gelu")

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in (24, 25):
        x.copy_(rand(700, 256, dtype=BF16, seed=seed))
        g.copy_(rand(700, 520, dtype=BF16, seed=seed + 10))
        graphs[0].replay()
        want = step()
        graphs[1].replay()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_side_stream():
    x, g = rand(3000, 512, dtype=BF16, seed=26), rand(3000, 512, dtype=BF16, seed=27)
    want = act8.weight_grad(g, act8.pack(x))[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.zeros(1 << 28, device="cuda")      # the side stream is busy when the calls are made
        big.add_(1)
        y = x * 1
        got = act8.weight_grad(g, act8.pack(y))[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_weight_grad_fp16_over_its_whole_range():
    """Groups from fp16's smallest subnormal to its largest value, each against weights of one: the decoded operand itself."""
    tokens, cols = 41, 64
    x = torch.zeros(tokens, cols)
    g = torch.Generator().manual_seed(28)
    for t in range(tokens):
        x[t] = (torch.rand(cols, generator=g) * 2 - 1) * 2.0 ** (t - 24)
        x[t, 0] = 2.0 ** (t - 24) * (1 if t < 40 else 0.99)
    x = x.clamp(-65504, 65504).to(FP16)
    eye = torch.eye(tokens, dtype=FP16)
    dw, _ = act8.weight_grad(eye.cuda(), act8.pack(x.cuda()), dtype=FP32)
    close(dw, held_value(x), 2.0 ** -25, "decoded")       # exact but for subnormals, half a step of 2^-24
    x = torch.zeros(2, 64)
    x[0, :32], x[1, 32:] = 1e5, 1.0                          # beyond fp16: the group is NaN, the others are not
    dw, _ = act8.weight_grad(eye[:2, :2].cuda(), act8.Act8(*(lambda h: (h.codes, h.scales))(act8.pack(x.cuda())), (2, 64), FP16))
    assert dw[0, :32].isnan().all() and (dw[1, 32:] == 1).all()


def test_weight_grad_with_a_cold_cache():
    """Loads that miss L2 land out of order: the stages' barriers have to keep the steps apart, over runs that end inside a tile."""
    x, g = rand(8192, 1024, dtype=BF16, seed=29), rand(8192, 512, dtype=BF16, seed=30)
    held = act8.pack(x)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    want, _ = act8.weight_grad(g, held, dtype=FP32)
    ref = g.double().t() @ held_value(x.cpu()).cuda()
    assert ((want.double() - ref).norm() / ref.norm()).item() < 2e-6
    for _ in range(12):
        flush.zero_()
        assert torch.equal(act8.weight_grad(g, held, dtype=FP32)[0], want)
    act8.check()


def test_largest_magnitude_anywhere():
    """Each place of a group in turn holds its largest magnitude, of either sign, finite or not."""
    for dtype in (BF16, FP16, FP32):
        x = rand(96 * 4, 32, dtype=dtype, seed=31)
        rows = torch.arange(96 * 4, device="cuda")
        x[rows, rows % 32] = torch.where(rows % 96 < 48, 9.0, -9.0).to(dtype)
        x[rows[96:192], rows[96:192] % 32] *= math.inf
        x[rows[192:288], rows[192:288] % 32] = math.nan
        held, host = act8.pack(x), act8.pack(x.cpu())
        assert torch.equal(held.codes.cpu(), host.codes) and torch.equal(held.scales[:, :1].cpu(), host.scales[:, :1])


def test_codes_at_their_bounds():
    """Values that round to +-128 steps are kept at +-127, and only those."""
    steps = torch.tensor([127.0, 127.25, 127.49999, 127.5, 127.75, 127.99999, 126.5, 125.5])
    x = torch.cat([steps, -steps, steps / 3, -steps / 7]).repeat(40, 1) * torch.exp2(torch.arange(-20.0, 20.0)).unsqueeze(1)
    x[::2, 3:6] = 0.25
    x[::4, 11:14] = -0.125
    held = act8.pack(x.cuda())
    assert torch.equal(held.codes.cpu(), act8.pack(x).codes) and held.codes.abs().max() == 127
    assert torch.equal(act8.unpack(held).cpu().double(), held_value(x))


def test_one_row_without_leading_axes():
    x = rand(72, dtype=BF16, seed=41).requires_grad_()
    w, b = rand(40, 72, dtype=BF16, seed=42).requires_grad_(), rand(40, dtype=BF16, seed=43).requires_grad_()
    y, held = act8.activation(x, "silu", checkpoint_output=True)
    act8.linear(y, w, b, checkpoint=held).backward(rand(40, dtype=BF16, seed=44))
    g = rand(40, dtype=BF16, seed=44).double()
    want = g.unsqueeze(1) * act8.unpack(held, FP32).double()
    close(w.grad, want, half_step(BF16) * want.abs(), "weight")      # one product, exact in fp32, and one rounding, relative to the value
    assert torch.equal(b.grad, g.to(BF16)) and x.grad.shape == (72,)


def test_calls_on_two_streams_at_once():
    """Products that fill the GPU, each with its partial sums, next to each other and to a step of the other kernels."""
    x, g = rand(6000, 1000, dtype=BF16, seed=45), rand(6000, 1032, dtype=BF16, seed=46)
    held = act8.pack(x)
    want = act8.weight_grad(g, held, bias=True, dtype=FP32)
    y = act8.activation_forward(x, "gelu", checkpoint_output=True)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams * 8:
        with torch.cuda.stream(s):
            got.append((act8.weight_grad(g, held, bias=True, dtype=FP32), act8.activation_forward(x, "gelu", checkpoint_output=True)))
    torch.cuda.synchronize()
    for (dw, db), (z, a, out) in got:
        assert torch.equal(dw, want[0]) and torch.equal(db, want[1]) and torch.equal(z, y[0])
        assert torch.equal(a.codes, y[1].codes) and torch.equal(out.codes, y[2].codes)
    act8.check()


@pytest.mark.parametrize("dtype,out", [(FP16, FP16), (BF16, FP32)])
def test_weight_grad_over_a_quarter_of_a_million_tokens(dtype, out):
    """Terms of one sign: a sum that stayed in the tensor core's truncating accumulator all along would be short by about 2^-11.5 of itself, with
    the rounding to fp16 more than half a step for many results."""
    tokens, n = 1 << 18, 9 * 256                                      # more tiles than pairs of CTAs: none is cut along its tokens
    g = (torch.rand(tokens, n, generator=torch.Generator(device="cuda").manual_seed(47), device="cuda") * 2 ** -8 + 2 ** -9).to(dtype)
    x = (torch.rand(tokens, n, generator=torch.Generator(device="cuda").manual_seed(48), device="cuda") + 0.5).to(dtype)
    held = act8.pack(x)
    dw, _ = act8.weight_grad(g, held, dtype=out)
    at = torch.arange(0, n, 67, device="cuda")
    want = (g[:, at].double().t() @ act8.unpack(held, FP32)[:, at].double()).cpu()
    # what is truncated is at most a step (2^-23) for each of the 4 x 32 products between two emptyings, each of those rounds once (2^-24)
    close(dw[at][:, at], want, half_step(out) * want + (128 + tokens / 1536 + 24) * 2.0 ** -23 * want, "dW")


def test_check_waits_for_side_streams():
    """A failure that a kernel on a side stream records only after check() was called is reported, once."""
    class Block:      # the device's status block as an array
        __cuda_array_interface__ = dict(shape=(16,), typestr="<i4", data=(native().act8_wgrad_status_block(), False), version=3)

    status, fail = torch.as_tensor(Block(), device="cuda"), torch.zeros(16, dtype=torch.int32, device="cuda")
    fail[:3] = torch.tensor([6, 300, 0], dtype=torch.int32)      # (a bounded wait at a barrier)
    act8.check()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(100_000_000)                              # some 50 ms
        status.copy_(fail)
    assert not s.query()
    with pytest.raises(GraceCommError):
        act8.check()
    assert s.query() and not status.any()
    act8.check()


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gelu_in_its_negative_tail(dtype):
    """Relative to the value, down to where it leaves fp32's normal range: the approximation of the distribution function (2.2e-5), the exponent's
    rounding (x^2 / 2 times a few 2^-24) and the rounding to the type."""
    x = -torch.linspace(0.01, 13.0, 4001).to(dtype).view(-1, 1)
    y, held, _ = act8.activation_forward(x.cuda(), "gelu")
    dx = act8.activation_backward(torch.ones_like(x).cuda(), held, "gelu")
    least = 2.0 ** -25 if dtype == FP16 else 0.0
    rel = lambda v: 2.2e-5 + (v * v / 2 + 2) * 2.0 ** -22  # noqa: E731
    f, _ = function(x, "gelu")
    close(y, f, (half_step(dtype) + rel(x.double())) * f.abs() + least, "y")
    h = held_value(x)
    _, d = function(h, "gelu")
    p, density = 0.5 * torch.special.erfc(-h / math.sqrt(2)), torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)
    close(dx, d, half_step(dtype) * d.abs() + rel(h) * (p + h.abs() * density) + least, "dx")


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_weight_grad_with_an_fp16_gradient_of_another_types_checkpoint(dtype):
    check_fp16_operand(dtype, "cuda")
