"""Rotary positions against their formula in 64 bits.

Tolerances (2-norm of the error over that of the result): products and sums in fp32 and one rounding, so
u = 2^-8 (bf16), 2^-11 (fp16), 2^-24 (fp32), of values of at most the pair's length, and three fp32
roundings of 2^-24 before it: 4 * 2^-24 in fp32.  Features past the turned ones are copied bit for bit.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOL = {"f32": 4 * 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return torch.device("cuda:0")


def announce(*what):
    print("case", *what, flush=True)


def tables64(length, rot, base=10000.0):
    j = torch.arange(rot // 2, dtype=torch.float64)
    t = torch.arange(length, dtype=torch.float64)[:, None] * base ** (-2 * j / rot)
    return t.cos(), t.sin()


def turn64(x, cos, sin, at, layout, sign=1.0):
    """The formula on the CPU in 64 bits; at: batch x seq positions."""
    y = x.detach().double().cpu().clone()
    rot = 2 * cos.shape[1]
    c, s = cos.double().cpu()[at][:, :, None], sign * sin.double().cpu()[at][:, :, None]
    ia = torch.arange(rot // 2) if layout == "half" else torch.arange(0, rot, 2)
    ib = ia + (rot // 2 if layout == "half" else 1)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def off(got, want):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape
    return float((got - want).norm() / want.norm())


# batch, seq, heads, kv heads, head, rot: one token, odd numbers of heads, heads that 64 lanes are no multiple
# of, rot and head off the vectors, one pair, more units than a wave has lanes
SHAPES = [(1, 1, 1, 1, 64, 64), (2, 5, 3, 1, 80, 80), (1, 33, 16, 4, 128, 32), (3, 7, 2, 2, 96, 24), (2, 9, 5, 5, 20, 6),
          (1, 3, 2, 1, 2, 2), (2, 4, 1, 1, 256, 256), (1, 5, 40, 8, 128, 128), (2, 3, 3, 2, 257, 130), (1, 2, 2, 1, 48, 16)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(dev, shape, dtype, layout):
    import stacr_amd

    b, t, hq, hk, head, rot = shape
    announce("rotary", shape, dtype, layout)
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, dq, dk = (torch.randn(b, t, h, head, generator=g, device=dev).to(DT[dtype]) for h in (hq, hk, hq, hk))
    cos, sin = stacr_amd.rotary_tables(t + 50, rot, device=dev)
    at = torch.randint(0, t + 50, (b, t), generator=g, device=dev)
    q.requires_grad_(True), k.requires_grad_(True)
    yq, yk = stacr_amd.rotary(q, k, cos, sin, positions=at, layout=layout)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    where = at.cpu()
    for got, x, sign in ((yq, q, 1.0), (yk, k, 1.0), (gq, dq, -1.0), (gk, dk, -1.0)):
        assert off(got, turn64(x, cos, sin, where, layout, sign)) <= TOL[dtype]
        assert torch.equal(got[..., rot:], x[..., rot:])


def test_layouts_in_memory_and_in_place(dev):
    """Views of a fused projection, heads before tokens, rows off 16 bytes, and the in-place form of each: the
    same bits as from packed tensors, and nothing else touched."""
    import stacr_amd

    announce("rotary layouts")
    b, t, hq, hk, head, rot = 2, 6, 4, 2, 64, 32
    cos, sin = stacr_amd.rotary_tables(64, rot, device=dev)
    base = torch.randn(b, t, hq + 2 * hk, head + 3, device=dev).bfloat16()
    fused = base[..., :head].contiguous()
    for whole, cut in ((fused, lambda w: (w[:, :, :hq], w[:, :, hq:hq + hk])),
                       (fused.transpose(1, 2).contiguous(), lambda w: (w[:, :hq].transpose(1, 2), w[:, hq:hq + hk].transpose(1, 2))),
                       (base, lambda w: (w[:, :, :hq, 1:head + 1], w[:, :, hq:hq + hk, 1:head + 1]))):
        q, k = cut(whole)
        want = stacr_amd.rotary(q.contiguous(), k.contiguous(), cos, sin, offset=7)
        got = stacr_amd.rotary(q, k, cos, sin, offset=7)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        work = whole.clone()
        qw, kw = cut(work)
        iq, ik = stacr_amd.rotary(qw, kw, cos, sin, offset=7, inplace=True)
        assert iq.data_ptr() == qw.data_ptr() and torch.equal(iq, want[0]) and torch.equal(ik, want[1])
        back = whole.clone()
        bq, bk = cut(back)
        bq.copy_(want[0]), bk.copy_(want[1])
        assert torch.equal(work, back)
    assert torch.equal(stacr_amd.rotary(q, None, cos, sin, offset=7), want[0])


def test_positions(dev):
    """Every way to give them, and positions that the tables do not have."""
    import stacr_amd

    announce("rotary positions")
    q = torch.randn(2, 5, 3, 16, device=dev)
    cos, sin = stacr_amd.rotary_tables(40, 16, device=dev)
    want, _ = stacr_amd.rotary(q, q, cos, sin, offset=3)
    at = torch.arange(3, 8, device=dev)
    for p in (at, at.int(), at[None].expand(2, 5), at.int()[None].repeat(2, 1), torch.stack((at, at), 1).t()):
        assert torch.equal(stacr_amd.rotary(q, None, cos, sin, positions=p), want)
    at = torch.tensor([0, -1, 39, 40, 1 << 40], device=dev)
    y = stacr_amd.rotary(q, None, cos, sin, positions=at)
    assert torch.equal(y.isnan().all(-1), torch.tensor([0, 1, 0, 1, 1], device=dev).bool()[None, :, None].expand(2, 5, 3))
    assert not y[:, [0, 2]].isnan().any()
    for shape in ((0, 5, 3, 16), (2, 0, 3, 16), (2, 5, 0, 16)):
        assert stacr_amd.rotary(torch.empty(shape, device=dev), None, cos, sin).shape == shape


def test_expanded_gradients_and_shared_heads(dev):
    """The gradient of a sum over keys that several query heads share: an expanded tensor without memory of
    its own."""
    import stacr_amd

    announce("rotary expanded")
    q = torch.randn(1, 4, 6, 32, device=dev, requires_grad=True)
    k = torch.randn(1, 4, 2, 32, device=dev, requires_grad=True)
    cos, sin = stacr_amd.rotary_tables(8, 32, device=dev)
    yq, yk = stacr_amd.rotary(q, k, cos, sin)
    gq, gk = torch.autograd.grad(yq.sum() + yk[:, :, :, None].expand(1, 4, 2, 3, 32).sum(), (q, k))
    at = torch.arange(4)[None]
    assert off(gq, turn64(torch.ones_like(q), cos, sin, at, "half", -1.0)) <= TOL["f32"]
    assert off(gk, turn64(3 * torch.ones_like(k), cos, sin, at, "half", -1.0)) <= TOL["f32"]
    # differences: the operator is linear, so one step of any length gives the slope but for its rounding
    v = torch.randn_like(q)
    f = [float(stacr_amd.rotary((q + s * v).detach(), None, cos, sin).double().sum()) for s in (1, -1)]
    assert abs((f[0] - f[1]) / 2 - float((gq * v).sum())) <= 1e-4 * float(gq.norm() * v.norm())


def test_a_long_sequence(dev):
    """More than 2^31 bytes of queries, far positions."""
    import stacr_amd

    announce("rotary long")
    t, h = 70000, 128
    cos, sin = stacr_amd.rotary_tables(t + 1000000, 128, device=dev)
    q = torch.empty(1, t, h, 128, device=dev, dtype=torch.bfloat16).normal_()
    y = stacr_amd.rotary(q, None, cos, sin, offset=1000000)
    rows = torch.tensor([0, 1, 32767, 65535, 69999])
    want = turn64(q[:, rows.to(dev)], cos, sin, (rows + 1000000)[None], "half")
    assert off(y[:, rows.to(dev)], want) <= TOL["bf16"]


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "by_parts"])
def test_tables(dev, scaling):
    """fp32 roundings of the 64-bit formula: 2^-24 of 1, and of the angle's own 64-bit error nothing."""
    import stacr_amd

    announce("rotary tables", scaling)
    length, rot, base, factor, original = 70000, 64, 10000.0, 8.0, 4096
    cos, sin = stacr_amd.rotary_tables(length, rot, base=base, scaling=scaling, factor=factor, original_length=original,
                                       device=dev)
    j = torch.arange(rot // 2, dtype=torch.float64)
    f, size = base ** (-2 * j / rot), 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ntk":
        f = (base * factor ** (rot / (rot - 2))) ** (-2 * j / rot)
    elif scaling == "by_parts":
        def pair(turns):  # the pair with so many turns over the original length
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = math.floor(pair(32.0)), math.ceil(pair(1.0))
        slow = ((j - low) / (high - low)).clamp(0, 1)
        f, size = f * (1 - slow) + f / factor * slow, 0.1 * math.log(factor) + 1
    t = torch.arange(length, dtype=torch.float64)[:, None] * f
    for got, want in ((cos, t.cos() * size), (sin, t.sin() * size)):
        assert float((got.double().cpu() - want).abs().max()) <= 1.3 * 2.0 ** -24
    assert stacr_amd.rotary_tables(0, 8, device=dev)[0].shape == (0, 4)


def test_refusals(dev):
    import stacr_amd

    q = torch.randn(1, 2, 2, 8, device=dev)
    cos, sin = stacr_amd.rotary_tables(4, 8, device=dev)
    f = stacr_amd.rotary
    with pytest.raises(ValueError, match="layout"):
        f(q, None, cos, sin, layout="pairs")
    with pytest.raises(ValueError, match="batch x seq"):
        f(q[0], None, cos, sin)
    with pytest.raises(ValueError, match="do not match"):
        f(q, q[:, :1], cos, sin)
    with pytest.raises(ValueError, match="do not fit"):
        f(q[..., :4], None, cos, sin)
    with pytest.raises(ValueError, match="outside tables"):
        f(q, None, cos, sin, offset=3)
    with pytest.raises(ValueError, match="positions must be"):
        f(q, None, cos, sin, positions=torch.zeros(3, dtype=torch.int64, device=dev))
    with pytest.raises(TypeError, match="int32 or int64"):
        f(q, None, cos, sin, positions=torch.zeros(2, device=dev))
    with pytest.raises(TypeError, match="float32"):
        f(q, None, cos.half(), sin.half())
    with pytest.raises(TypeError, match="keys are"):
        f(q, q.half(), cos, sin)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        f(q.cpu(), None, cos, sin)
    with pytest.raises(RuntimeError, match="tensors on cpu"):
        f(q, None, cos.cpu(), sin.cpu())
    with pytest.raises(ValueError, match="no gradient"):
        f(q.requires_grad_(True), None, cos, sin, inplace=True)
    with pytest.raises(ValueError, match="share memory"):
        f(q.detach()[:, :1].expand(1, 2, 2, 8), None, cos, sin, inplace=True)
    with pytest.raises(ValueError, match="scaling must be"):
        stacr_amd.rotary_tables(4, 8, scaling="dynamic")
    with pytest.raises(ValueError, match="even rot"):
        stacr_amd.rotary_tables(4, 7)
    with pytest.raises(ValueError, match="factor"):
        stacr_amd.rotary_tables(4, 8, scaling="linear", factor=0.5)
    with pytest.raises(ValueError, match="original_length"):
        stacr_amd.rotary_tables(4, 8, scaling="by_parts", factor=2.0)
