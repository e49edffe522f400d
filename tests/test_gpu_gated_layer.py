"""STACRGatedFeedForward against the block of two separate layers, and the example that trains with it."""
import os
import sys

import pytest
import torch
from torch import nn
from torch.nn import functional as F

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# u: largest relative rounding of the type.  Two forms of the same gradients from the same saved factors differ
# by the roundings of g, u, act(g), dg and du: five of them at most, 2-norms, independent
U = {"f32": 2.0 ** -19, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return torch.device("cuda:0")


def off(got, want):
    got, want = got.detach().double(), want.detach().double()
    return float((got - want).norm() / want.norm())


def layers(d, ff, dtype, dev, bias, seed=0):
    torch.manual_seed(seed)
    return [nn.Linear(d, ff, bias=bias).to(dev, DT[dtype]) for _ in range(2)]


@pytest.mark.parametrize("options", [dict(residual_budget=0.02), dict(residual_budget=0.02, residual_bits=4),
                                     dict(residual_budget=0.05, residual_bits=0, residual_mode="global_topk"),
                                     dict(residual_mode="none"), dict(residual_budget=0.05, residual_mode="uniform")],
                         ids=lambda o: "-".join(str(v) for v in o.values()))
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,d,ff,bias", [(96, 64, 48, True), (130, 72, 45, False)])
def test_against_two_layers(dev, rows, d, ff, bias, dtype, options):
    """Both forms fit the same basis to the same input, so they save the same factors."""
    import stacr_amd

    print("case", rows, d, ff, dtype, options, flush=True)
    a, b = layers(d, ff, dtype, dev, bias), layers(d, ff, dtype, dev, bias)
    block = stacr_amd.STACRGatedFeedForward.from_linears(*a, rank=4, **options)
    gate, up = (stacr_amd.STACRLinear.from_linear(m, rank=4, **options) for m in b)
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(2, rows // 2, d, generator=g, device=dev).to(DT[dtype])
    dh = torch.randn(2, rows // 2, ff, generator=g, device=dev).to(DT[dtype])
    xa, xb = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    ha = block(xa)
    hb = F.silu(gate(xb)) * up(xb)
    assert off(ha, hb) <= 4 * U[dtype]
    ha.backward(dh)
    hb.backward(dh)
    assert off(xa.grad, xb.grad) <= 5 * U[dtype]
    for m, n in zip(a, b):
        assert off(m.weight.grad, n.weight.grad) <= 5 * U[dtype]
        if bias:
            assert off(m.bias.grad, n.bias.grad) <= 5 * U[dtype]
    assert torch.equal(block.gate.basis, gate.basis)


def test_memory_and_schedule(dev):
    """One compressed input for both projections; set_step reaches the basis; eval is the exact operator."""
    import stacr_amd

    a = layers(256, 512, "bf16", dev, False)
    block = stacr_amd.STACRGatedFeedForward.from_linears(*a, rank=8, turbo_after_step=3)
    model = nn.Sequential(block)
    x = torch.randn(4096, 256, device=dev, dtype=torch.bfloat16)
    held = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        block(x.requires_grad_(True))
    kept = sum(t.numel() * t.element_size() for t in held if t.data_ptr() not in (a[0].weight.data_ptr(), a[1].weight.data_ptr()))
    stored = block.stored_bytes(4096)
    assert kept == stored["total"] - stored["persistent_basis"]
    assert all(t.data_ptr() != x.data_ptr() for t in held)
    before = block.gate.basis.clone()
    stacr_amd.set_step(model, 1)
    block(x)
    assert not torch.equal(block.gate.basis, before) and block.gate.step == 1
    stacr_amd.set_step(model, 3)
    held.clear()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(t) or t, lambda t: t):
        block(x)
    assert not any(t.dtype in (torch.int32, torch.int8) for t in held)  # Turbo: no residual
    model.eval()
    assert torch.equal(block(x), stacr_amd.gated_feed_forward(x, a[0].weight, a[1].weight))
    assert block(x[:0]).shape == (0, 512)


def test_refusals(dev):
    import stacr_amd

    a, b = layers(64, 32, "f32", dev, True)
    f = stacr_amd.STACRGatedFeedForward.from_linears
    with pytest.raises(TypeError, match="two nn.Linear"):
        f(a, nn.Identity())
    with pytest.raises(ValueError, match="activation"):
        f(a, b, activation="swish")
    with pytest.raises(ValueError, match="weights differ"):
        f(a, nn.Linear(64, 16).to(dev))
    with pytest.raises(ValueError, match="rank must be"):
        f(a, b, rank=0)
    with pytest.raises(ValueError, match="Expected last input dimension 64"):
        f(a, b)(torch.zeros(2, 63, device=dev))


def test_the_example_learns(dev):
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import train_gated_block

    losses, norms = train_gated_block.train(steps=150, report=50)
    assert all(v == v and v < float("inf") for v in losses + norms)
    # a uniform guess over 64 tokens is 4.16
    assert losses[0] > 4.0 and sum(losses[-5:]) / 5 < 2.0
