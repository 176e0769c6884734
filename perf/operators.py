"""Cases that measure the 8-bit activation checkpoint operators: the checkpoint itself, the weight gradient that reads it, the
activation functions and the residual-and-norm step that write it in the forward and read it in the backward pass.

``run`` computes them in plain torch operations (``own`` false) or by the package's calls (``own`` true).

A checkpoint holds groups of 32 neighbours of the last axis as 8-bit integers with one power-of-two scale (the MXINT8 format
of the OCP microscaling specification): the scale comes from the exponent of the group's largest magnitude, the code is
the value over the scale, rounded to the nearest integer (ties to even) and kept within +-127.
"""
import math

import torch

own = False

GROUP = 32
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence of 128 tokens, hidden size 1024: the smallest checkpoint of a fine-tuning step, a matter of latency
        dict(name="checkpoint 128x1024", op="checkpoint", dtype="bf16", rows=128, cols=1024),
        # 32 sequences of 512 tokens, the feed-forward width 4096: a whole micro-batch's widest tensor
        dict(name="checkpoint 16384x4096", op="checkpoint", dtype="bf16", rows=16384, cols=4096),
        # attention output projection of the BERT-large workload, 32 x 128 tokens, with its bias
        dict(name="weight_grad 4096t 1024x1024", op="weight_grad", dtype="bf16", out="bf16", tokens=4096, outs=1024, ins=1024, bias=True),
        # its first feed-forward layer, gradients kept in 32 bits for accumulation over micro-batches
        dict(name="weight_grad 4096t 4096x1024 f32", op="weight_grad", dtype="bf16", out="fp32", tokens=4096, outs=4096, ins=1024, bias=True),
        # a wide layer over a long batch: the largest product
        dict(name="weight_grad 16384t 4096x4096", op="weight_grad", dtype="bf16", out="bf16", tokens=16384, outs=4096, ins=4096, bias=False),
        # odd sizes throughout, fp16
        dict(name="weight_grad 777t 1000x1003 fp16", op="weight_grad", dtype="fp16", out="fp16", tokens=777, outs=1000, ins=1003, bias=True),
        # GELU of the BERT-large feed-forward layer, with the checkpoint of its output for the layer after it
        dict(name="gelu 4096x4096", op="activation", dtype="bf16", kind="gelu", gated=False, rows=4096, cols=4096, output=True),
        # gated SiLU of a wide feed-forward layer, 16384 tokens
        dict(name="silu gated 16384x4096", op="activation", dtype="bf16", kind="silu", gated=True, rows=16384, cols=4096, output=False),
        # odd sizes, tanh form of the GELU, fp16
        dict(name="gelu_tanh 333x1003 fp16", op="activation", dtype="fp16", kind="gelu_tanh", gated=False, rows=333, cols=1003, output=False),
        # add and LayerNorm after a sub-layer of the BERT-large workload (32 x 128 tokens): nothing but the normalised stream goes on
        dict(name="add layer norm 4096x1024", op="residual_norm", dtype="bf16", seqs=32, length=128, cols=1024, post="none", pre="layer",
             gate="none", alpha=1.0, stream=False),
        # sandwich: RMS norm after the block, a gate for each sequence, scaled residual, RMS norm before the next block
        dict(name="sandwich rms gated 16384x4096", op="residual_norm", dtype="bf16", seqs=8, length=2048, cols=4096, post="rms", pre="rms",
             gate="sequence", alpha=1.0, stream=True),
        # scaled residual (2.63 = 48 ** 0.25), layer norms with a gate of each channel, odd sizes
        dict(name="sandwich layer 3x67x1000 fp16", op="residual_norm", dtype="fp16", seqs=3, length=67, cols=1000, post="layer", pre="layer",
             gate="channel", alpha=2.63, stream=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["checkpoint", "weight_grad", "activation", "residual_norm"])
    if op == "checkpoint":
        cols = _log(rng, 32, 8192)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), cols=cols, rows=_log(rng, 1, min(65536, (1 << 25) // cols)))
    if op == "weight_grad":
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        outs, ins = _log(rng, 64, 4096), _log(rng, 64, 4096)
        if rng.random() < 0.7:
            outs, ins = (outs + 7) // 8 * 8, (ins + 31) // 32 * 32
        return dict(op=op, dtype=dtype, out=rng.choice([dtype, "fp32"]), tokens=_log(rng, 1, 16384), outs=outs, ins=ins, bias=rng.random() < 0.5)
    if op == "activation":
        cols, gated = _log(rng, 32, 8192), rng.random() < 0.4
        if rng.random() < 0.7:
            cols = (cols + 31) // 32 * 32
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        # (the layer after it takes a checkpoint of the output where it computes in 16 bits)
        return dict(op=op, dtype=dtype, kind=rng.choice(["gelu", "gelu_tanh", "silu"]), gated=gated, cols=cols, rows=_log(rng, 1, min(65536, (1 << 25) // cols)),
                    output=dtype != "fp32" and rng.random() < 0.5)
    cols = _log(rng, 32, 8192)
    if rng.random() < 0.7:
        cols = (cols + 31) // 32 * 32
    seqs = rng.randint(1, 32)
    length = _log(rng, 1, max(1, min(4096, (1 << 25) // (cols * seqs))))
    pre, gate = rng.choice(["layer", "rms"]), rng.choice(["none", "channel", "sequence"])
    return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), seqs=seqs, length=length, cols=cols, post=rng.choice(["none", "rms", "layer"]), pre=pre,
                gate=gate, alpha=rng.choice([1.0, 0.5, 2.63]), stream=rng.random() < 0.6)


def work(case):
    es = _BYTES[case["dtype"]]
    op, held = case["op"], 1 + 1 / GROUP      # bytes of a value, and of a value in a checkpoint
    if op == "checkpoint":
        n = case["rows"] * case["cols"]
        return {"bytes": n * 2 * (es + held), "flops": n * 4}
    if op == "weight_grad":
        t, n, k = case["tokens"], case["outs"], case["ins"]
        return {"bytes": t * n * es + t * k * held + n * k * _BYTES[case["out"]], "flops": 2 * t * n * k + (t * n if case["bias"] else 0)}
    if op == "activation":
        n = case["rows"] * case["cols"]
        wide = 2 if case["gated"] else 1
        # forward: x in, y and the checkpoints out; backward: dy and the checkpoint in, dx out
        forward = n * (wide * es + es + wide * held + (held if case["output"] else 0))
        return {"bytes": forward + n * (es + wide * held + wide * es), "flops": n * 40}
    n = case["seqs"] * case["length"] * case["cols"]
    two = case["post"] != "none" or case["gate"] != "none"      # the block's own values are needed again for these
    forward = 2 * es + es + (es if case["stream"] else 0) + held * (2 if two else 1)
    one_out = not two and case["alpha"] == 1.0                   # both inputs have the same gradient
    backward = es + (es if case["stream"] else 0) + held * (2 if two else 1) + (es if one_out else 2 * es)
    return {"bytes": n * (forward + backward), "flops": n * 50}


# ------------------------------------------------------------------------------------------------------------ inputs
def _hidden(g, rows, cols, dtype):
    """Values as hidden states have them: normal, with a few channels an order of magnitude larger."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    wide = 1 + 15 * (torch.rand(cols, generator=g, device="cuda") < 0.004).float()
    return (x * wide).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = _TYPES[case["dtype"]], case["op"]

    def grad(rows, cols):
        return (torch.randn(rows, cols, generator=g, device="cuda") * 0.05).to(dtype)

    s = dict(case)
    if op == "checkpoint":
        s["x"] = _hidden(g, case["rows"], case["cols"], dtype)
    elif op == "weight_grad":
        x = _hidden(g, case["tokens"], case["ins"], dtype)
        s["grad"] = grad(case["tokens"], case["outs"])
        s["codes"], s["scales"] = _held(x)      # the forward pass left them
    elif op == "activation":
        wide = 2 if case["gated"] else 1
        s["x"] = (torch.randn(case["rows"], wide * case["cols"], generator=g, device="cuda") * 1.5).to(dtype)
        s["grad"] = grad(case["rows"], case["cols"])
    else:
        rows, cols = case["seqs"] * case["length"], case["cols"]
        shape = (case["seqs"], case["length"], cols)
        s["x"], s["block"] = _hidden(g, rows, cols, dtype).view(shape), _hidden(g, rows, cols, dtype).view(shape)
        s["grad_h"] = grad(rows, cols).view(shape)
        s["grad_y"] = grad(rows, cols).view(shape) if case["stream"] else None
        for side in ("post", "pre"):
            w = 1 + 0.2 * torch.randn(cols, generator=g, device="cuda")
            b = 0.1 * torch.randn(cols, generator=g, device="cuda")
            s[side + "_weight"] = None if case[side] == "none" else w.to(dtype)
            s[side + "_bias"] = b.to(dtype) if case[side] == "layer" else None
        gates = {"none": None, "channel": (cols,), "sequence": (case["seqs"], cols)}[case["gate"]]
        s["gate"] = None if gates is None else (0.3 + 0.2 * torch.randn(gates, generator=g, device="cuda")).to(dtype)
    return s


def _held(x):
    """The checkpoint's two arrays: int8 codes, a row's length rounded up to whole groups, and a byte of scale for each group, a
    row's scales rounded up to eight bytes."""
    rows, cols = x.shape
    groups = -(-cols // GROUP)
    v = torch.zeros(rows, groups * GROUP, device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, groups, GROUP)
    codes, byte = _codes(v)
    scales = torch.zeros(rows, -(-groups // 8) * 8, dtype=torch.uint8, device=x.device)
    scales[:, :groups] = byte
    return codes.to(torch.int8).view(rows, groups * GROUP), scales


def _codes(v):
    """(codes as floats, scale bytes) of fp32 groups [rows, groups, 32]; every step but the rounding to an integer is exact."""
    top = v.abs().amax(-1)
    exponent = torch.frexp(top).exponent.clamp(-119, 126)        # top = mantissa * 2 ** exponent, mantissa in [0.5, 1)
    q = torch.ldexp(v, (7 - exponent).unsqueeze(-1)).round().clamp(-127, 127)
    return q, (exponent + 120).to(torch.uint8)


# -------------------------------------------------------------------------------------------------------- plain form
def _through(x):
    """What a checkpoint of x reads back as, in 32 bits."""
    shape, cols = x.shape, x.shape[-1]
    groups = -(-cols // GROUP)
    v = torch.nn.functional.pad(x.float().reshape(-1, cols), (0, groups * GROUP - cols)).view(-1, groups, GROUP)
    q, byte = _codes(v)
    v = torch.ldexp(q, (byte.int() - 127).unsqueeze(-1))
    return v.view(-1, groups * GROUP)[:, :cols].reshape(shape)


def _from_parts(codes, scales, cols):
    groups = codes.shape[1] // GROUP
    v = torch.ldexp(codes.float().view(-1, groups, GROUP), (scales[:, :groups].int() - 127).unsqueeze(-1))
    return v.view(codes.shape)[:, :cols]


def _function(x, kind):
    """(f(x), f'(x)) in x's own precision."""
    if kind == "silu":
        p = 1 / (1 + torch.exp(-x))
        return x * p, p * (1 + x * (1 - p))
    if kind == "gelu":
        p = 0.5 * torch.erfc(-x * math.sqrt(0.5))
        return x * p, p + x * torch.exp(-0.5 * x * x) * (1 / math.sqrt(2 * math.pi))
    c, a = math.sqrt(2 / math.pi), 0.044715
    p = 1 / (1 + torch.exp(-2 * c * (x + a * x * x * x)))        # (1 + tanh) / 2
    return x * p, p + x * 2 * p * (1 - p) * c * (1 + 3 * a * x * x)


def _norm(v, kind, weight, bias, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    n = (v - mean) * rstd * weight.float()
    return (n if bias is None else n + bias.float()), mean, rstd


def _norm_grad(c, hat, rstd, kind):
    c = c - hat * (c * hat).mean(-1, keepdim=True) - (c.mean(-1, keepdim=True) if kind == "layer" else 0)
    return c * rstd


EPS = 1e-6


def _plain_norm(s):
    x, block, dtype = s["x"], s["block"], s["x"].dtype
    post, pre, gate = s["post"], s["pre"], s["gate"]
    wide = gate.float().view((-1, 1, gate.shape[-1])) if gate is not None else None
    b = block.float()
    n = b
    if post != "none":
        n, b_mean, b_rstd = _norm(b, post, s["post_weight"], s["post_bias"], EPS)
    y = (x.double() * s["alpha"] + (n if wide is None else n * wide).double()).to(dtype)
    h, mean, rstd = _norm(y.float(), pre, s["pre_weight"], s["pre_bias"], EPS)
    out = {"h": h.to(dtype)}
    # backward, from what the checkpoints hold of y and of the block's output
    dh = s["grad_h"].float()
    hat = (_through(y) - mean) * rstd
    g = _norm_grad(dh * s["pre_weight"].float(), hat, rstd, pre)
    out["pre_weight"] = (dh * hat).sum((0, 1)).to(dtype)
    if pre == "layer":
        out["pre_bias"] = dh.sum((0, 1)).to(dtype)
    if s["stream"]:
        out["y"] = y
        g = g + s["grad_y"].float()
    out["x"] = (g * s["alpha"]).to(dtype)
    e = g if wide is None else g * wide
    held = _through(block) if post != "none" or gate is not None else None
    if post != "none":
        b_hat = (held - b_mean) * b_rstd
        out["post_weight"] = (e * b_hat).sum((0, 1)).to(dtype)
        if post == "layer":
            out["post_bias"] = e.sum((0, 1)).to(dtype)
        n = b_hat * s["post_weight"].float()
        n = n + s["post_bias"].float() if post == "layer" else n
        e = _norm_grad(e * s["post_weight"].float(), b_hat, b_rstd, post)
    else:
        n = held
    if gate is not None:
        out["gate"] = (g * n).sum(1 if gate.dim() == 2 else (0, 1)).to(dtype)
    out["block"] = e.to(dtype)
    return out


def _plain(s):
    op = s["op"]
    if op == "checkpoint":
        return {"x": _through(s["x"]).to(s["x"].dtype)}
    if op == "weight_grad":
        out = _TYPES[s["out"]]
        g = s["grad"].float()
        got = {"weight": (g.t() @ _from_parts(s["codes"], s["scales"], s["ins"])).to(out)}
        if s["bias"]:
            got["bias"] = g.sum(0).to(out)
        return got
    if op == "activation":
        x, g, dtype = s["x"], s["grad"].float(), s["x"].dtype
        f = s["cols"]
        v, t = x.float(), _through_halves(x, f) if s["gated"] else _through(x)
        y = _function(v[:, :f], s["kind"])[0]
        fa, da = _function(t[:, :f], s["kind"])
        if s["gated"]:
            y = y * v[:, f:]
            dx = torch.cat([g * t[:, f:] * da, g * fa], 1)
        else:
            dx = g * da
        got = {"y": y.to(dtype), "x": dx.to(dtype)}
        if s["output"]:
            got["held"] = _through(got["y"]).to(dtype)
        return got
    return _plain_norm(s)


def _through_halves(x, f):
    """A gated input's halves [a | b] are held as two tensors beside each other."""
    return torch.cat([_through(x[:, :f]), _through(x[:, f:])], 1)


# ------------------------------------------------------------------------------------------------- the package's calls
def _own(s):
    from grace_b200.ops import act8, block_norm

    op = s["op"]
    if op == "checkpoint":
        return {"x": act8.unpack(act8.pack(s["x"]))}
    if op == "weight_grad":
        held = act8.Act8(s["codes"], s["scales"], (s["tokens"], s["ins"]), s["grad"].dtype)
        weight, bias = act8.weight_grad(s["grad"], held, bias=s["bias"], dtype=_TYPES[s["out"]])
        return {"weight": weight, "bias": bias} if s["bias"] else {"weight": weight}
    if op == "activation":
        y, held, out = act8.activation_forward(s["x"], s["kind"], gated=s["gated"], checkpoint_output=s["output"])
        got = {"y": y, "x": act8.activation_backward(s["grad"], held, s["kind"], gated=s["gated"])}
        if s["output"]:
            got["held"] = act8.unpack(out)
        return got
    h, y, saved = block_norm.residual_norm_forward(
        s["x"], s["block"], pre=s["pre"], pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], post=None if s["post"] == "none" else s["post"],
        post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"], residual_scale=s["alpha"], eps=EPS, return_stream=s["stream"])
    got = block_norm.residual_norm_backward(s["grad_h"], s["grad_y"], saved)
    got = {k: v for k, v in got.items() if v is not None}
    got["h"] = h
    if s["stream"]:
        got["y"] = y
    return got


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---------------------------------------------------------------------------------------------------- 64-bit results
def _held64(x):
    """What the checkpoint of x reads back as, from the definition: the scale is two to the (exponent of the group's largest magnitude - 6)."""
    x = x.double()
    cols = x.shape[-1]
    parts = []
    flat = x.reshape(-1, cols)
    whole = cols // GROUP * GROUP
    for part in (flat[:, :whole].reshape(flat.shape[0], -1, GROUP), flat[:, whole:].reshape(flat.shape[0], -1, max(1, cols - whole))):
        if part.numel():
            top = part.abs().max(-1, keepdim=True).values
            step = torch.exp2((torch.floor(torch.log2(top.clamp_min(2.0 ** -120))) - 6))
            step = torch.where(top >= step * 128, step * 2, step)          # log2 next to a power of two
            step = torch.where(top < step * 64, step / 2, step).clamp_min(2.0 ** -126)
            parts.append((torch.round(part / step).clamp(-127, 127) * step).reshape(flat.shape[0], -1))
    return torch.cat(parts, 1).reshape(x.shape)


def _function64(x, kind):
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x / math.sqrt(2)))
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def _norm64(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * weight.double()
    return v if bias is None else v + bias.double()


def _norm_back64(d, v, held, kind, weight):
    """Gradients of a norm's input, weight and bias for the incoming d, where the statistics are v's and the normalised values those of `held`."""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else 0
    sigma = torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + EPS)
    hat = (held - mean) / sigma
    dw = (d * hat).sum((0, 1))
    c = d * weight.double()
    c = (c - (c.mean(-1, keepdim=True) if kind == "layer" else 0) - hat * (c * hat).mean(-1, keepdim=True)) / sigma
    return c, dw, d.sum((0, 1)), hat


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "checkpoint":
        return {"x": _held64(s["x"])}
    if op == "weight_grad":
        q = s["codes"].double()
        x = q * torch.exp2(s["scales"][:, : q.shape[1] // GROUP].double() - 127).repeat_interleave(GROUP, 1)
        g = s["grad"].double()
        got = {"weight": torch.einsum("mn,mk->nk", g, x[:, : case["ins"]])}
        if case["bias"]:
            got["bias"] = g.sum(0)
        return got
    if op == "activation":
        f = case["cols"]
        parts = [s["x"][:, :f], s["x"][:, f:]] if case["gated"] else [s["x"]]
        held = [_held64(p).requires_grad_() for p in parts]
        y = _function64(parts[0].double(), case["kind"]) * (parts[1].double() if case["gated"] else 1)
        z = _function64(held[0], case["kind"]) * (held[1] if case["gated"] else 1)
        got = {"y": y, "x": torch.cat(torch.autograd.grad(z, held, s["grad"].double()), 1)}
        if case["output"]:
            got["held"] = _held64(y.to(s["x"].dtype))
        return got
    x, block, dtype = s["x"].double(), s["block"].double(), s["x"].dtype
    gate = 1 if s["gate"] is None else s["gate"].double().reshape(-1, 1, case["cols"])
    y = (case["alpha"] * x + gate * _norm64(block, case["post"], s["post_weight"], s["post_bias"])).to(dtype).double()
    got = {"h": _norm64(y, case["pre"], s["pre_weight"], s["pre_bias"])}
    g, got["pre_weight"], bias, _ = _norm_back64(s["grad_h"].double(), y, _held64(y), case["pre"], s["pre_weight"])
    if case["pre"] == "layer":
        got["pre_bias"] = bias
    if case["stream"]:
        got["y"] = y
        g = g + s["grad_y"].double()
    got["x"] = case["alpha"] * g
    n = held = _held64(block)
    e = g * gate
    if case["post"] != "none":
        e, got["post_weight"], bias, hat = _norm_back64(e, block, held, case["post"], s["post_weight"])
        n = hat * s["post_weight"].double()
        if case["post"] == "layer":
            got["post_bias"] = bias
            n = n + s["post_bias"].double()
    if s["gate"] is not None:
        got["gate"] = (g * n).sum(1) if case["gate"] == "sequence" else (g * n).sum((0, 1))
    got["block"] = e
    return got
