"""8-bit activation checkpoints on the CPU: the format, its refusals, and the autograd functions against the 64-bit oracle."""
import math

import pytest
import torch

from _act8_oracle import close, function, half_step, held_value
from grace_b200.ops import act8

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (31,), (32,), (3, 33), (2, 5, 100), (0, 64), (4, 0), (1, 257)])
def test_round_trip(shape, dtype):
    x = rand(*shape, dtype=dtype, scale=3.0)
    held = act8.pack(x)
    assert held.codes.dtype == torch.int8 and held.scales.dtype == torch.uint8
    got = act8.unpack(held)
    assert got.dtype == dtype and got.shape == x.shape
    # the value is exact in fp32 and bf16; in fp16 unless it is subnormal there (half a step of 2^-24)
    close(got, held_value(x), 2.0 ** -25 if dtype == torch.float16 else 0.0, "unpack")


def test_error_bound_and_ties():
    x = rand(64, 96, seed=1)
    top = x.abs().view(64, 3, 32).amax(-1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(top)) - 6)
    err = (act8.unpack(act8.pack(x)) - x).abs().view(64, 3, 32)
    assert (err <= step).all() and (err[x.abs().view(64, 3, 32) <= 127.5 * step] <= (step / 2).expand(64, 3, 32)[x.abs().view(64, 3, 32) <= 127.5 * step]).all()
    # steps of 1: ties go to the even code, 127.5 and above saturate
    v = torch.zeros(32)
    v[:8] = torch.tensor([64.0, 0.5, 1.5, 2.5, -0.5, -1.5, 127.5, -127.9])
    assert act8.unpack(act8.pack(v))[:8].tolist() == [64, 0, 2, 2, 0, -2, 127, -127]


def test_extremes():
    x = torch.zeros(6, 32)
    x[0, 3] = math.inf
    x[1, 4] = math.nan
    x[2, :2] = torch.tensor([3.4e38, 1.0])
    x[3, :2] = torch.tensor([1e-45, 2.0 ** -121])
    x[4, :2] = torch.tensor([2.0 ** -119, 2.0 ** -126])
    got = act8.unpack(act8.pack(x))
    assert got[:2].isnan().all()                        # an overflow is kept visible
    assert got[2, 0] == 127 * 2.0 ** 119                # saturates
    assert got[3, 0] == 0 and got[3, 1] == 2.0 ** -121  # the step never goes below 2^-126
    assert got[4, 0] == 2.0 ** -119 and (got[5] == 0).all()
    close(got, held_value(x), 0.0)


def test_refusals():
    x = rand(4, 64)
    held = act8.pack(x)
    with pytest.raises(TypeError):
        act8.pack(torch.zeros(4, dtype=torch.int32))
    with pytest.raises(TypeError):
        act8.pack(torch.zeros(4, dtype=torch.float64))
    with pytest.raises(TypeError):
        act8.pack([1.0])
    with pytest.raises(ValueError):
        act8.pack(torch.tensor(1.0))
    with pytest.raises(TypeError):
        act8.pack(x.to_sparse())
    with pytest.raises(TypeError):
        act8.unpack(held, torch.float64)
    with pytest.raises(ValueError):
        act8.Act8(held.codes, held.scales, (4, 65), torch.float32)
    with pytest.raises(ValueError):
        act8.Act8(held.codes[:, :32], held.scales, (4, 32), torch.float32)      # not contiguous
    with pytest.raises(TypeError):
        act8.Act8(held.codes.view(torch.uint8), held.scales, (4, 64), torch.float32)
    with pytest.raises(TypeError):
        act8.Act8(held.codes, held.scales, (4, 64), torch.int32)
    with pytest.raises(ValueError):
        act8.weight_grad(rand(5, 8), held)
    with pytest.raises(TypeError):
        act8.weight_grad(rand(4, 8, dtype=torch.bfloat16), held, dtype=torch.float16)
    with pytest.raises(ValueError):
        act8.activation_forward(x, "relu")
    with pytest.raises(ValueError):
        act8.activation_forward(rand(4, 65), "silu", gated=True)
    with pytest.raises(ValueError):
        act8.activation_backward(x, held, "silu", gated=True)
    with pytest.raises(ValueError):
        act8.activation_backward(x[:3], held, "silu")
    with pytest.raises(ValueError):
        act8.linear(x.requires_grad_(), rand(8, 64).requires_grad_(), checkpoint=act8.pack(rand(3, 64)))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activation(kind, gated):
    x = rand(7, 2, 90, seed=2, scale=2.0).requires_grad_()
    f = 45 if gated else 90
    y, held_y = act8.activation(x, kind, gated=gated, checkpoint_output=True)
    g = rand(*y.shape, seed=3)
    y.backward(g)
    v = x.detach().double()
    a, b = v[..., :f], v[..., f:]
    want = function(a, kind)[0] * (b if gated else 1)
    close(y.detach(), want, 1e-6 * (1 + a.abs()) * (1 + b.abs() if gated else 1), "y")
    assert torch.equal(act8.unpack(held_y).double(), held_value(y.detach()))
    ha, hb = held_value(x.detach()[..., :f]), held_value(x.detach()[..., f:])
    fa, da = function(ha, kind)
    want = torch.cat([g * hb * da, g * fa], -1) if gated else g * da
    close(x.grad, want, 1e-5, "dx")


def test_linear_gradients_and_differences():
    x, w, b = rand(6, 5, 40, seed=4).requires_grad_(), rand(24, 40, seed=5).requires_grad_(), rand(24, seed=6).requires_grad_()
    g = rand(6, 5, 24, seed=7)
    y = act8.linear(x, w, b)
    assert torch.equal(y, torch.nn.functional.linear(x, w, b))
    y.backward(g)
    held = held_value(x.detach()).reshape(-1, 40)
    close(w.grad, g.reshape(-1, 24).double().t() @ held, 1e-4, "dW")
    close(b.grad, g.reshape(-1, 24).double().sum(0), 1e-5, "db")
    close(x.grad, g.double() @ w.detach().double(), 1e-4, "dx")
    # on values that the checkpoint holds exactly, the gradient is that of differences
    x = act8.unpack(act8.pack(rand(4, 32, seed=8))).requires_grad_()
    w = rand(3, 32, seed=9).requires_grad_()
    g = rand(4, 3, seed=10)
    act8.linear(x, w).backward(g)
    for i, j in ((0, 0), (2, 31)):
        d = torch.zeros(3, 32, dtype=torch.float64)
        d[i, j] = 1e-3
        f = lambda v: (torch.nn.functional.linear(x.detach().double(), v) * g.double()).sum()  # noqa: E731
        assert abs((f(w.detach().double() + d) - f(w.detach().double() - d)).item() / 2e-3 - w.grad[i, j].item()) < 1e-5


def test_activation_gradient_is_that_of_differences():
    x = act8.unpack(act8.pack(rand(2, 64, seed=11))).requires_grad_()
    for kind in act8.KINDS:
        x.grad = None
        act8.activation(x, kind).sum().backward()
        v, h = x.detach().double(), 1e-5
        num = (function(v + h, kind)[0] - function(v - h, kind)[0]) / (2 * h)
        close(x.grad, num, 1e-5, kind)      # differences: h^2 f'''/6 and rounding 1e-16 / h; fp32 f' 1e-6


def test_no_gradient_keeps_nothing():
    x, w = rand(3, 32), rand(4, 32)
    assert not act8.linear(x, w).requires_grad and not act8.activation(x).requires_grad
    y, held = act8.activation(x, checkpoint_output=True)
    assert torch.equal(act8.unpack(held).double(), held_value(y))


def test_weight_shared_by_two_layers():
    x, w = rand(4, 32, seed=12).requires_grad_(), rand(32, 32, seed=13).requires_grad_()
    act8.linear(act8.linear(x, w), w).sum().backward()
    h = torch.nn.functional.linear(x.detach(), w.detach())
    ones = torch.ones(4, 32, dtype=torch.float64)
    want = ones.t() @ held_value(h) + (ones @ w.detach().double()).t() @ held_value(x.detach())
    close(w.grad, want, 1e-3, "dW")
    assert half_step(torch.float32) == 2.0 ** -24


def test_a_checkpoint_too_wide_is_refused():
    with pytest.raises(ValueError, match="2\\^30 columns"):
        act8.Act8(torch.empty(0, 0, dtype=torch.int8), torch.empty(0, 0, dtype=torch.uint8), (0, (1 << 30) + 1), torch.bfloat16)


@pytest.mark.parametrize("given", [None, "act8"])
def test_linear_under_autocast(given):
    """As the library's layer: computed in autocast's type, gradients in the leaves' own."""
    x, w, b = rand(6, 40, seed=14).requires_grad_(), rand(24, 40, seed=15).requires_grad_(), rand(24, seed=16).requires_grad_()
    g = rand(6, 24, seed=17, dtype=torch.bfloat16)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = act8.linear(x, w, b, checkpoint=None if given is None else act8.pack(x.detach()))
        assert torch.equal(y, torch.nn.functional.linear(x, w, b))
        with torch.no_grad():
            assert torch.equal(act8.linear(x, w, b), y)
    assert y.dtype == torch.bfloat16
    y.backward(g)
    assert x.grad.dtype == w.grad.dtype == b.grad.dtype == torch.float32
    held, gd = held_value(x.detach() if given else x.detach().bfloat16()), g.double()
    half = half_step(torch.bfloat16)
    want, size = gd.t() @ held, gd.abs().t() @ held.abs()
    close(w.grad, want, half * want.abs() + 6 * 2.0 ** -24 * size, "dW")
    close(b.grad, gd.sum(0), half * gd.sum(0).abs() + 6 * 2.0 ** -24 * gd.abs().sum(0), "db")
    wd = w.detach().bfloat16().double()
    want, size = gd @ wd, gd.abs() @ wd.abs()
    close(x.grad, want, half * want.abs() + 24 * 2.0 ** -24 * size, "dx")


def test_weight_grad_sums_in_fp32_under_autocast():
    x, g = rand(50, 32, seed=18), rand(50, 8, seed=19)
    want = act8.weight_grad(g, act8.pack(x), bias=True)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = act8.weight_grad(g, act8.pack(x), bias=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def check_fp16_operand(dtype, device):
    """A checkpoint of a wider type meets an fp16 gradient as its values rounded to fp16, half a step of 2^-24 at most where they are
    subnormal; a group with a value of 2^16 or more is NaN, and with it its columns."""
    g = torch.Generator().manual_seed(20)
    x = torch.zeros(50, 128)
    x[:, :64] = (torch.rand(50, 64, generator=g) * 2 - 1) * torch.exp2(torch.arange(50) - 34.0).unsqueeze(1)      # groups from 2^-35 to 2^15
    x[:, 64:] = torch.randn(50, 64, generator=g)
    x[7, 70], x[9, 100] = 65536.0, 65000.0
    held = act8.pack(x.to(device, dtype))
    dw = act8.weight_grad(torch.eye(50, dtype=torch.float16, device=device), held, dtype=torch.float32)[0].cpu()
    want = act8.unpack(held, torch.float32).cpu().half().float()
    assert dw[:, 64:96].isnan().all()
    keep = [c for c in range(128) if not 64 <= c < 96]
    assert torch.equal(dw[:, keep], want[:, keep]) and (want[:12, :64] != 0).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weight_grad_with_an_fp16_gradient_of_another_types_checkpoint(dtype):
    check_fp16_operand(dtype, "cpu")


def test_linear_refuses_a_vector_for_its_weight():
    """Before the forward pass, not in the backward pass."""
    with pytest.raises(ValueError, match="outs, ins"):
        act8.linear(rand(4, 64), rand(64).requires_grad_())
