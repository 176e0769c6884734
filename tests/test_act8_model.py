"""BERT with 8-bit activation checkpoints against the same model without: outputs, gradients, parameters, a training step."""
import pytest
import torch
import torch.utils.checkpoint

from grace_b200.models import bert_tiny
from grace_b200.models.bert import BertForPreTraining

FORMS = [dict(), dict(post_norm="rms", layer_scale=0.7), dict(post_norm="layer", residual_scale=1.5), dict(residual_scale=0.5, layer_scale=0.3)]


def batch(device, b=4, s=16):
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 1000, (b, s), generator=g)
    labels = ids.clone()
    labels[torch.rand(b, s, generator=g) > 0.3] = -100
    return ids.to(device), labels.to(device), torch.randint(0, 2, (b,), generator=g).to(device)


def pair(device, dtype, **form):
    torch.manual_seed(1)
    full = bert_tiny(dropout=0.0, **form).to(device, dtype)
    held = bert_tiny(dropout=0.0, activation_checkpoint="int8", **form).to(device, dtype)
    held.load_state_dict(full.state_dict())
    return full, held


def losses_and_gradients(model, device, autocast=None):
    ids, labels, nsp = batch(device)
    with torch.autocast(device, dtype=autocast or torch.bfloat16, enabled=autocast is not None):
        loss = model(ids, mlm_labels=labels, nsp_labels=nsp)
    loss.backward()
    return loss.item(), {n: p.grad.float() for n, p in model.named_parameters()}


def compare(a, b, loss_tol, grad_tol):
    assert abs(a[0] - b[0]) <= loss_tol * abs(a[0]), (a[0], b[0])
    assert a[1].keys() == b[1].keys()
    for n, g in a[1].items():
        assert torch.isfinite(b[1][n]).all(), n
        assert (g - b[1][n]).norm() <= grad_tol * g.norm() + 1e-8, (n, ((g - b[1][n]).norm() / g.norm()).item())


# Held values are off by half a code step at most, 2^-7 of the leading power of two of their group: about 1 % of a usual value's size.
# Through one layer's product that is 1 % of a gradient's norm at most; two layers and a head add up to a few.
@pytest.mark.parametrize("form", FORMS)
def test_cpu(form):
    full, held = pair("cpu", torch.float32, **form)
    compare(losses_and_gradients(full, "cpu"), losses_and_gradients(held, "cpu"), 1e-5, 0.06)


def test_option_is_checked_and_state_is_the_same():
    with pytest.raises(ValueError):
        bert_tiny(activation_checkpoint="fp4")
    with pytest.raises(ValueError):
        bert_tiny(post_norm="batch")
    full, held = pair("cpu", torch.float32, post_norm="layer", layer_scale=1.0)
    assert list(full.state_dict()) == list(held.state_dict())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("autocast", [False, True])
def test_gpu(form, autocast):
    full, held = pair("cuda", torch.float32 if autocast else torch.bfloat16, **form)
    kind = torch.bfloat16 if autocast else None
    # both arms round to bf16 between kernels, at different places: 2^-8 each, some ten of them on the way to a gradient
    compare(losses_and_gradients(full, "cuda", kind), losses_and_gradients(held, "cuda", kind), 2e-2, 0.15)


@pytest.mark.gpu
def test_gpu_keeps_less():
    """What a step holds between forward and backward, in a model whose layers outweigh its head."""
    def peak(kind):
        torch.manual_seed(2)
        m = BertForPreTraining(1000, 256, 6, 4, 1024, 128, dropout=0.0, activation_checkpoint=kind).to("cuda", torch.bfloat16)
        ids, labels, nsp = batch("cuda", 32, 128)
        m(ids, mlm_labels=labels, nsp_labels=nsp).backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = m(ids, mlm_labels=labels, nsp_labels=nsp)
        after = torch.cuda.memory_allocated() - before
        del loss
        return after

    full, held = peak(None), peak("int8")
    # per token and layer, bf16 bytes over hidden: inputs of qkv, proj, fc1 (2 each), GELU and fc2 (8 each), two norms (2 each), q k v and the
    # attention's output (2 each, kept by both): 34; with checkpoints 5 1/6 halves of all but the attention's 8: 21.4
    assert held < 0.8 * full, (held, full)


@pytest.mark.gpu
@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_gpu_trains_with_the_compressed_exchange(checkpoint):
    """Both halves of a step at once: 8-bit checkpoints in the backward pass, the fused compressed exchange after it."""
    import grace_b200
    from grace_b200.optim import FusedSGD
    from grace_b200.parallel.flat import FlatParams

    torch.manual_seed(3)
    model = bert_tiny(dropout=0.0, activation_checkpoint=checkpoint).cuda()
    flat = FlatParams(model.named_parameters())
    opt = FusedSGD(model.parameters(), lr=0.05, momentum=0.9, flat=flat)
    grc = grace_b200.grace_from_params({"compressor": "qsgd", "memory": "residual", "communicator": "allgather", "quantum_num": 64,
                                        "world_size": 1, "fused": True})
    ids, labels, nsp = batch("cuda")
    for _ in range(3):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model(ids, mlm_labels=labels, nsp_labels=nsp)
        loss.backward()
        assert flat.flat_g.isfinite().all() and flat.flat_g.any()
        grc.step_flat(flat.flat_g, flat.layout)
        opt.step()
    grc.check()
    assert torch.isfinite(loss)


@pytest.mark.gpu
def test_gpu_dropout_and_graph_capture():
    """A whole forward and backward pass captured and replayed on new inputs gives the eager pass's gradients."""
    torch.manual_seed(4)
    model = bert_tiny(dropout=0.0, activation_checkpoint="int8").to("cuda", torch.bfloat16)
    ids, labels, nsp = batch("cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            model.zero_grad(set_to_none=True)
            model(ids, mlm_labels=labels, nsp_labels=nsp).backward()
    torch.cuda.current_stream().wait_stream(s)
    model.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = model(ids, mlm_labels=labels, nsp_labels=nsp)
        loss.backward()
    ids.copy_(ids.flip(0))
    labels.copy_(labels.flip(0))
    nsp.copy_(nsp.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    want = {}
    model.zero_grad(set_to_none=True)
    model(ids, mlm_labels=labels, nsp_labels=nsp).backward()
    for n, p in model.named_parameters():
        want[n] = p.grad
        # (embedding gradients are library atomics: their order may differ)
        assert (got[n].float() - p.grad.float()).norm() <= 0.02 * p.grad.float().norm() + 1e-6, n
    model.train()
    drop = bert_tiny(dropout=0.1, activation_checkpoint="int8").to("cuda", torch.bfloat16)
    drop(ids, mlm_labels=labels, nsp_labels=nsp).backward()
    assert all(torch.isfinite(p.grad).all() for p in drop.parameters())


def without_gradients(device, dtype):
    for form in FORMS:
        _, held = pair(device, dtype, **form)
        ids, labels, nsp = batch(device)
        want = held(ids, mlm_labels=labels, nsp_labels=nsp)
        with torch.no_grad():
            assert torch.equal(held(ids, mlm_labels=labels, nsp_labels=nsp), want.detach())


def test_cpu_without_gradients():
    without_gradients("cpu", torch.float32)


@pytest.mark.gpu
def test_gpu_without_gradients():
    without_gradients("cuda", torch.bfloat16)


def test_a_layer_without_the_option_returns_a_tensor():
    """Callers of a layer, its hooks and wrappers around it get the tensor itself; with the option the pair that the next layer takes."""
    full, held = pair("cpu", torch.float32)
    x, seen = torch.randn(2, 16, 64), []
    for model in (full, held):
        model.layers[0].register_forward_hook(lambda module, args, out: seen.append(out))
    ids, _, _ = batch("cpu")
    full(ids), held(ids)
    assert isinstance(seen[0], torch.Tensor) and seen[0].shape == (4, 16, 64)
    y = full.layers[0](x)
    assert isinstance(y, torch.Tensor) and y.shape == x.shape and torch.equal(torch.utils.checkpoint.checkpoint(full.layers[0], x, use_reentrant=False), y)
    z, kept = held.layers[0](x)
    assert kept.shape == x.shape and torch.allclose(y, z, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_gpu_autocast_has_the_same_stream(form):
    """Under autocast the stream of fp32 parameters is fp32 with and without the option, and one sub-layer's join on the same values gives
    the same to fp32's rounding."""
    full, held = pair("cuda", torch.float32, **form)
    g = torch.Generator().manual_seed(5)
    x, block = torch.randn(3, 16, 64, generator=g).cuda(), torch.randn(3, 16, 64, generator=g).to("cuda", torch.bfloat16)
    a, b = full.layers[0], held.layers[0]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want, _ = a._join(x, block.float(), a.ln1, a.post1, a.gate1)      # (a norm of a bf16 block would round to bf16 on its way)
        got, kept = b._join(x, block, b.ln1, b.post1, b.gate1)
        outs = a(x), b(x)[0]
    assert got.dtype == want.dtype == kept.dtype == outs[0].dtype == outs[1].dtype == torch.float32
    assert ((got - want).abs() <= 2e-6 * (1 + want.abs())).all()


@pytest.mark.parametrize("form", FORMS)
def test_cpu_autocast(form):
    full, held = pair("cpu", torch.float32, **form)
    # as on the GPU: both arms round to bf16 between the layers' products, at different places
    compare(losses_and_gradients(full, "cpu", torch.bfloat16), losses_and_gradients(held, "cpu", torch.bfloat16), 2e-2, 0.15)
