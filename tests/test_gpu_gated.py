"""The gated feed-forward block against its formulas in 64 bits.

Tolerances are 2-norms of the error over the 2-norm of the result, from the arithmetic alone.  With u
the largest relative rounding of the type (2^-8 bf16, 2^-11 fp16):
  h                u: one rounding of each value; the fp32 sums' own error is 2^-13 of that or less, 5 % room
  gradients        2 u: the rounding of the result and that of dg and du before the product, whose errors
                   are independent and so pass through it with at most their own relative size
  fp32             2^-21 (terms of the split that are left out) + sqrt(6 K) 2^-25 (K sums of six products,
                   each rounded at the running sum's size); K the longest sum on the way to the result, and
                   the gradients' factors carry the forward's error once more
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return torch.device("cuda:0")


def announce(*what):
    print("case", *what, flush=True)


def act64(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "sigmoid":
        return torch.sigmoid(g)
    if name == "relu":
        return torch.where(g > 0, g, torch.zeros_like(g))
    if name == "gelu":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))


def formula(tensors, dh, act):
    """(h, gradients) in 64 bits, the gradients by automatic differentiation."""
    wide = [None if t is None else t.detach().double().requires_grad_(True) for t in tensors]
    x, wg, wu, bg, bu = wide
    g, u = x @ wg.t(), x @ wu.t()
    if bg is not None:
        g = g + bg
    if bu is not None:
        u = u + bu
    h = act64(g, act) * u
    return h.detach(), torch.autograd.grad(h, [t for t in wide if t is not None], dh.double())


def make(rows, d, ff, dtype, dev, biases=(True, True), seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(DT[dtype])

    t = [normal(rows, d), normal(ff, d, scale=d ** -0.5), normal(ff, d, scale=d ** -0.5),
         normal(ff, scale=0.5) if biases[0] else None, normal(ff, scale=0.5) if biases[1] else None]
    return t, normal(rows, ff)


def off(got, want):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    norm = want.norm()
    return float((got - want).norm() / norm) if norm else float((got - want).norm())


def tolerance(dtype, sums, gradient):
    if dtype == "f32":
        return (2.0 ** -21 + math.sqrt(6 * sums) * 2.0 ** -25) * (2 if gradient else 1)
    u = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    return 2 * u if gradient else 1.05 * u


def check(tensors, dh, act, dtype):
    for recompute in (False, True):
        check_form(tensors, dh, act, dtype, recompute)


def check_form(tensors, dh, act, dtype, recompute):
    import stacr_amd

    h64, g64 = formula(tensors, dh, act)
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in tensors]
    h = stacr_amd.gated_feed_forward(*leaves, activation=act, recompute=recompute)
    rows, d, ff = h.shape[0], tensors[1].shape[1], tensors[1].shape[0]
    assert off(h.detach(), h64) <= tolerance(dtype, d, False)
    with torch.no_grad():  # the form without a backward is the same kernel
        assert torch.equal(stacr_amd.gated_feed_forward(*tensors, activation=act), h.detach())
    grads = torch.autograd.grad(h, [t for t in leaves if t is not None], dh)
    for name, a, b in zip(("dx", "dw_gate", "dw_up", "db", "db"), grads, g64):
        assert off(a, b) <= tolerance(dtype, max(d, ff, rows), True), name


# (rows, d, ff): one row and few rows (every block count), a row past them, features off every multiple, less
# than one step of K, one feature, several tiles with ragged edges
SHAPES = [(1, 64, 32), (1, 7, 5), (3, 1, 1), (16, 200, 48), (17, 129, 65), (33, 136, 264), (64, 264, 130), (65, 96, 40),
          (128, 64, 64), (130, 1000, 300), (257, 264, 392), (512, 513, 1031), (300, 1, 3)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,d,ff", SHAPES)
def test_against_the_formula(dev, rows, d, ff, dtype):
    announce("gated", rows, d, ff, dtype)
    tensors, dh = make(rows, d, ff, dtype, dev, biases=(rows % 2 == 0, rows % 3 == 0))
    check(tensors, dh, ACTS[(rows + d + ff) % len(ACTS)], dtype)


# enough tiles of 256 x 256 for the forward, the input's gradient and the weights' gradients in turn
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,d,ff", [(4100, 72, 2056), (8200, 2050, 40), (100, 2056, 4104)])
def test_large_tiles(dev, rows, d, ff, dtype):
    announce("gated large", rows, d, ff, dtype)
    tensors, dh = make(rows, d, ff, dtype, dev, biases=(False, False))
    check(tensors, dh, "silu", dtype)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_activations_over_their_range(dev, act, dtype):
    """Gates from -40 to 40: the tails of every activation, and 0 itself."""
    announce("gated activations", act, dtype)
    n = 161
    x = torch.linspace(-40, 40, n, device=dev).to(DT[dtype])[:, None].repeat(1, 8)
    x[n // 2] = 0
    wg = torch.full((8, 8), 0.125, device=dev, dtype=DT[dtype])
    wu = torch.eye(8, device=dev, dtype=DT[dtype])
    check([x, wg, wu, None, None], torch.ones(n, 8, device=dev, dtype=DT[dtype]), act, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_no_rows(dev, dtype):
    import stacr_amd

    announce("gated no rows", dtype)
    tensors, _ = make(0, 24, 16, dtype, dev)
    leaves = [t.requires_grad_(True) for t in tensors]
    h = stacr_amd.gated_feed_forward(*leaves)
    assert h.shape == (0, 16)
    for t, g in zip(leaves, torch.autograd.grad(h.sum(), leaves)):
        assert g.shape == t.shape and not g.any()


def test_leading_dimensions_strides_and_shared_gradients(dev):
    """A 3-D input that is a slice of a wider one, a transposed input, an expanded incoming gradient, weights
    that are views."""
    import stacr_amd

    announce("gated strides")
    wide = torch.randn(2, 40, 96, device=dev, dtype=torch.bfloat16)
    w = torch.randn(2, 56, 64, device=dev, dtype=torch.bfloat16) / 8
    for x in (wide[..., 16:80], wide[..., 3:67], wide[:, :, :64].transpose(0, 1), wide[:, ::2, :64],
              wide.transpose(1, 2)[:, :64].transpose(1, 2)):
        for wg, wu in ((w[0], w[1]), (w[0].t().contiguous().t(), w[1])):
            leaf = x.detach().requires_grad_(True)
            h = stacr_amd.gated_feed_forward(leaf, wg, wu)
            assert h.shape == (*x.shape[:-1], 56)
            flat = x.reshape(-1, 64)
            dh = torch.ones(1, device=dev, dtype=torch.bfloat16).expand(h.shape)
            h64, g64 = formula([flat, wg, wu, None, None], dh.reshape(-1, 56), "silu")
            assert off(h.detach().reshape(-1, 56), h64) <= tolerance("bf16", 64, False)
            dx, = torch.autograd.grad(h, leaf, dh)
            assert off(dx.reshape(-1, 64), g64[0]) <= tolerance("bf16", 64, True)


def test_only_the_gradients_asked_for(dev):
    import stacr_amd

    announce("gated partial gradients")
    tensors, dh = make(70, 64, 48, "bf16", dev)
    full = [t.detach().requires_grad_(True) for t in tensors]
    whole = torch.autograd.grad(stacr_amd.gated_feed_forward(*full), full, dh)
    for i in range(5):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(tensors)]
        got, = torch.autograd.grad(stacr_amd.gated_feed_forward(*some), some[i], dh)
        assert torch.equal(got, whole[i])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [5, 300])
def test_values_that_are_not_finite_stay_in_their_rows(dev, dtype, rows):
    import stacr_amd

    announce("gated non-finite", dtype, rows)
    (x, wg, wu, _, _), _ = make(rows, 40, 24, dtype, dev, biases=(False, False))
    clean = stacr_amd.gated_feed_forward(x, wg, wu)
    x = x.clone()
    x[1, 3], x[2, 0], x[4, 39] = float("inf"), float("nan"), float("-inf")
    h = stacr_amd.gated_feed_forward(x, wg, wu)
    keep = [i for i in range(rows) if i not in (1, 2, 4)]
    assert torch.equal(h[keep], clean[keep])
    want = act64(x.double() @ wg.double().t(), "silu") * (x.double() @ wu.double().t())
    assert torch.equal(h.isnan(), want.isnan()) and torch.equal(h.isinf(), want.isinf())
    assert torch.equal(h[h.isinf()].double(), want[want.isinf()])


def test_fp32_extremes(dev):
    """Products near the ends of fp32's range, and values whose low parts are below bf16's smallest."""
    import stacr_amd

    announce("gated fp32 extremes")
    big = torch.full((3, 8), 3.0e38, device=dev)
    one = torch.eye(8, device=dev)
    h = stacr_amd.gated_feed_forward(big, one * 0 + 0, one, torch.ones(8, device=dev), None, activation="relu")
    assert torch.equal(h, big)
    small = torch.full((3, 8), 1.2345e-30, device=dev)
    h = stacr_amd.gated_feed_forward(small, one * 0, one, torch.ones(8, device=dev), None, activation="relu")
    assert off(h, small) <= 2.0 ** -23


def test_gradient_against_differences(dev):
    """Central differences of sum(h * dh) in fp32 along random directions: with step e the third derivative
    leaves e^2 / 6 of the slope's size and fp32 sums leave 2^-23 sqrt(n) / e; e = 2^-6 makes both below 1e-3."""
    import stacr_amd

    announce("gated differences")
    for act in ACTS:
        if act == "relu":
            continue  # not smooth
        tensors, dh = make(24, 20, 12, "f32", dev)
        leaves = [t.requires_grad_(True) for t in tensors]
        grads = torch.autograd.grad(stacr_amd.gated_feed_forward(*leaves, activation=act), leaves, dh)
        e = 2.0 ** -6
        for i, (t, g) in enumerate(zip(tensors, grads)):
            v = g.detach() / g.norm()
            plus, minus = ([u.detach() + (s * e * v if j == i else 0) for j, u in enumerate(tensors)] for s in (1, -1))
            f = [float((stacr_amd.gated_feed_forward(*z, activation=act).double() * dh.double()).sum()) for z in (plus, minus)]
            slope = (f[0] - f[1]) / (2 * e)
            assert abs(slope - float(g.norm())) <= 5e-3 * float(g.norm()) + 1e-3, (act, i)


def test_another_stream(dev):
    import stacr_amd

    announce("gated stream")
    tensors, dh = make(300, 264, 392, "f32", dev)
    leaves = [t.requires_grad_(True) for t in tensors]
    want = torch.autograd.grad(stacr_amd.gated_feed_forward(*leaves), leaves, dh)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = torch.autograd.grad(stacr_amd.gated_feed_forward(*leaves), leaves, dh)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)  # and the same bits on every run


def test_autocast(dev):
    import stacr_amd

    announce("gated autocast")
    tensors, dh = make(70, 64, 48, "f32", dev)
    leaves = [t.requires_grad_(True) for t in tensors]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        h = stacr_amd.gated_feed_forward(*leaves)
    assert h.dtype == torch.bfloat16
    grads = torch.autograd.grad(h, leaves, dh.bfloat16())
    low = [t.detach().bfloat16().requires_grad_(True) for t in tensors]
    want = torch.autograd.grad(stacr_amd.gated_feed_forward(*low), low, dh.bfloat16())
    for a, b in zip(grads, want):
        assert a.dtype == torch.float32 and torch.equal(a, b.float())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,d,ff", [(5, 16, 13), (200, 136, 72)])
def test_kept_preactivations(dev, rows, d, ff, dtype):
    """The form that keeps g and u in the type: one more rounding of each in dg and du (3 u for three
    independent roundings), and [dg | du] given out."""
    from stacr_amd import kernels

    announce("gated kept", rows, d, ff, dtype)
    (x, wg, wu, bg, bu), dh = make(rows, d, ff, dtype, dev)
    h, kept = kernels.gated_forward(x, wg, wu, bg, bu, "silu", keep="type")
    pad = (ff + 7) // 8 * 8
    g = kept[:rows * pad * h.element_size()].view(h.dtype).view(rows, pad)
    assert torch.equal(h, kernels.gated_forward(x, wg, wu, bg, bu, "silu"))
    g64 = x.double() @ wg.double().t() + bg.double()
    assert off(g[:, :ff], g64) <= tolerance(dtype, d, False)
    half = dtype != "f32"
    dx, dwg, dwu, dbg, dbu, dgu = kernels.gated_backward(dh, x, wg, wu, bg, bu, "silu", kept=kept,
                                                         needs=(True, True, True, True), slopes=True)
    _, want = formula([x, wg, wu, bg, bu], dh, "silu")
    room = 1.5 if half else 1.0
    for a, b in zip((dx, dwg, dwu, dbg, dbu), want):
        assert off(a, b) <= room * tolerance(dtype, max(rows, d, ff), True)
    assert dgu.shape == (rows, 2 * pad) and not dgu[:, ff:pad].any() and not dgu[:, pad + ff:].any()
    assert off(dgu[:, :ff].double().t() @ x.double(), want[1]) <= room * tolerance(dtype, max(rows, d, ff), True)
    alone = kernels.gated_backward(dh, None, wg, wu, bg, bu, "silu", kept=kept, needs=(True, False, False, False),
                                   slopes=True)
    assert torch.equal(alone[0], dx) and torch.equal(alone[5], dgu)


def test_refusals(dev):
    import stacr_amd

    (x, wg, wu, bg, bu), _ = make(4, 16, 8, "bf16", dev)
    f = stacr_amd.gated_feed_forward
    with pytest.raises(ValueError, match="activation"):
        f(x, wg, wu, activation="swish")
    with pytest.raises(ValueError, match="Expected last input dimension 16"):
        f(x[:, :8], wg, wu)
    with pytest.raises(ValueError, match="one shape"):
        f(x, wg, wu[:4])
    with pytest.raises(ValueError, match="b_up"):
        f(x, wg, wu, bg, bu[:3])
    with pytest.raises(TypeError, match="one type"):
        f(x, wg.float(), wu)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        f(x.cpu(), wg.cpu(), wu.cpu())
    with pytest.raises(RuntimeError, match="w_up is on cpu"):
        f(x, wg, wu.cpu())
    with pytest.raises(TypeError, match="float32, bfloat16 and float16"):
        f(x.double(), wg.double(), wu.double())


def test_in_a_graph(dev):
    """Both passes captured once and replayed on other inputs, eager work between."""
    from stacr_amd import kernels

    announce("gated graph")
    for dtype in ("bf16", "f32"):
        (x, wg, wu, _, _), dh = make(200, 136, 72, dtype, dev)

        def both():
            h, kept = kernels.gated_forward(x, wg, wu, keep="full")
            return (h, *kernels.gated_backward(dh, x, wg, wu, kept=kept)[:3])

        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            both()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        for _ in range(3):
            x.normal_()
            dh.normal_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, both()):
                assert torch.equal(a, b)


def test_large_gates_have_finite_slopes(dev):
    """Gates whose squares fp32 cannot hold: the slope's tail is 0 or 1, not infinity times 0."""
    import stacr_amd

    announce("gated large gates")
    x = torch.full((3, 8), 3.0e19, device=dev)
    x[1] = -3.0e19
    w, one = torch.eye(8, device=dev), torch.zeros(8, 8, device=dev)
    for act in ACTS:
        leaf = x.clone().requires_grad_(True)
        h = stacr_amd.gated_feed_forward(leaf, w, one, None, torch.ones(8, device=dev), activation=act)
        dx, = torch.autograd.grad(h, leaf, torch.ones_like(h))
        want = 0.0 if act == "sigmoid" else 1.0
        assert torch.equal(dx[0], torch.full((8,), want, device=dev)), act
        assert not dx[1].any(), act
