"""The global gradient norm and clipping against 64 bits.

Tolerances: the norm is a 64-bit sum rounded once, 2^-24; a clipped gradient is the product with an fp32
factor (2^-24 off) rounded once to its type: u = 2^-8 (bf16), 2^-11 (fp16), 2^-23 (fp32, both roundings),
value by value.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8 * 1.001, torch.float16: 2.0 ** -11 * 1.001}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return torch.device("cuda:0")


def announce(*what):
    print("case", *what, flush=True)


def norm64(grads, p):
    flat = torch.cat([g.detach().double().reshape(-1) for g in grads]).abs()
    if not flat.numel():
        return 0.0
    return float(flat.max() if p == math.inf else flat.sum() if p == 1 else flat.square().sum().sqrt())


def check(grads, max_norm, p=2.0, eps=1e-6, out=None):
    import stacr_amd

    before = [g.clone() for g in grads]
    n = norm64(grads, p)
    norm = stacr_amd.clip_gradients(grads, max_norm, norm_type=p, eps=eps, out=out)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - n) <= 2.0 ** -24 * 1.001 * n
    f = min(1.0, max_norm / (n + eps))
    for g, b, o in zip(grads, before, out or grads):
        if out is not None:
            assert torch.equal(g, b)
        if f == 1.0:
            assert torch.equal(o, b)
        else:
            want = b.double() * f
            small = torch.finfo(b.dtype).smallest_normal  # below it roundings are absolute
            assert bool(((o.double() - want).abs() <= U[b.dtype] * want.abs() + U[b.dtype] * small).all())


SIZES = [[1], [7], [8191, 8192, 8193], [0, 5, 0], [16385, 3, 100000], [1] * 300, [40000] * 130]


@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_against_64_bits(dev, sizes, dtype, p):
    announce("clip", len(sizes), sizes[0], dtype, p)
    g = torch.Generator(device=dev).manual_seed(2)
    grads = [torch.randn(n, generator=g, device=dev).to(DT[dtype]) for n in sizes]
    n = norm64(grads, p)
    check([t.clone() for t in grads], 0.3 * n, p)
    check([t.clone() for t in grads], 2.0 * n, p)
    check(grads, 0.3 * n, p, out=[torch.empty_like(t) for t in grads])


def test_mixed_types_and_packed_views(dev):
    """Views of a bucket at every alignment, types mixed; values beside them stay."""
    announce("clip views")
    for shift in range(9):
        flat = torch.randn(60000, device=dev).bfloat16()
        wide = torch.randn(30000, device=dev)
        keep, keep_wide = flat.clone(), wide.clone()
        grads = [flat[shift:shift + 20011], wide[shift:shift + 9001].view(-1, 1), flat[20011 + shift:59990]]
        check(grads, 1.0)
        assert torch.equal(flat[:shift], keep[:shift]) and torch.equal(flat[59990:], keep[59990:])
        assert torch.equal(wide[:shift], keep_wide[:shift]) and torch.equal(wide[shift + 9001:], keep_wide[shift + 9001:])
        other = torch.zeros(60000, device=dev).bfloat16()  # another alignment than the gradient's
        check([flat[shift:shift + 20011]], 1.0, out=[other[1:20012]])
        assert not other[:1].any() and not other[20012:].any()


def test_orders_of_memory(dev):
    """Transposed, permuted and gapped tensors in place, and into outputs of another order."""
    announce("clip strides")
    a = torch.randn(30, 50, device=dev)
    for g in (a.clone().t(), torch.randn(4, 6, 10, device=dev).permute(2, 0, 1), torch.randn(30, 60, device=dev)[:, 5:40],
              torch.randn(30, 60, device=dev)[::2], torch.randn((), device=dev)):
        check([g], 0.01)
        check([g], 0.01, out=[torch.empty(g.shape, device=dev)])
        if g.dim() == 2:
            check([g], 0.01, out=[torch.empty(g.shape[::-1], device=dev).t()])
            check([g], 0.01, out=[torch.empty(g.shape[0], 2 * g.shape[1], device=dev)[:, ::2]])
            check([g], 100.0 * norm64([g], 2), out=[torch.empty(g.shape[0], 2 * g.shape[1], device=dev)[:, ::2]])


def test_extremes(dev):
    """Squares that fp32 could not hold, infinities, NaN, zeros."""
    import stacr_amd

    announce("clip extremes")
    for scale in (1e30, 1e-30):
        check([torch.full((5000,), scale, device=dev)], scale, eps=0.0)
    zero = torch.zeros(100, device=dev)
    check([zero], 1.0)
    check([torch.randn(100, device=dev)], 0.0)
    for p in (2.0, 1.0, math.inf):
        g = torch.randn(9000, device=dev)
        g[8500] = math.inf
        n = stacr_amd.clip_gradients([g], 1.0, norm_type=p)
        assert math.isinf(float(n)) and g[8500].isnan() and not g[:8500].any()
        for bad in (math.nan, -math.nan):
            g = torch.randn(9000, device=dev)
            g[8500], g[3] = bad, math.inf
            n = stacr_amd.clip_gradients([g, torch.ones(3, device=dev)], 1.0, norm_type=p)
            assert math.isnan(float(n)) and g.isnan().all()


def test_parameters_and_the_norm_alone(dev):
    import stacr_amd

    announce("clip parameters")
    model = torch.nn.Sequential(torch.nn.Linear(40, 30), torch.nn.Linear(30, 20)).to(dev)
    model[1].bias.requires_grad_(False)
    model(torch.randn(8, 40, device=dev)).square().sum().backward()
    grads = [p.grad for p in model.parameters() if p.grad is not None]
    n = norm64(grads, 2)
    before = [g.clone() for g in grads]
    assert abs(float(stacr_amd.grad_norm(grads)) - n) <= 2.0 ** -24 * 1.001 * n
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    norm = stacr_amd.clip_grad_norm(model.parameters(), 0.5 * n)
    assert abs(float(norm) - n) <= 2.0 ** -24 * 1.001 * n
    assert abs(norm64(grads, 2) - 0.5 * n) <= 1e-5 * n
    p = torch.nn.Parameter(torch.ones(3, device=dev))
    p.grad = torch.full((3,), 2.0, device=dev)
    stacr_amd.clip_grad_norm(p, 1.0)
    assert abs(float(p.grad.norm()) - 1.0) <= 1e-5
    assert float(stacr_amd.clip_grad_norm([torch.nn.Parameter(torch.ones(3, device=dev))], 1.0)) == 0.0


def test_same_bits_and_another_stream(dev):
    import stacr_amd

    announce("clip stream")
    g = [torch.randn(100003, device=dev).bfloat16(), torch.randn(77, device=dev)]
    out = [[torch.empty_like(t) for t in g] for _ in range(2)]
    a = stacr_amd.clip_gradients(g, 0.1, out=out[0])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b = stacr_amd.clip_gradients(g, 0.1, out=out[1])
    s.synchronize()
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(*out))


def test_in_a_graph(dev):
    """Captured once, replayed with other gradients in the same buffers, eager work between."""
    import stacr_amd

    announce("clip graph")
    g = [torch.randn(50000, device=dev), torch.randn(301, device=dev).bfloat16()]
    out = [torch.empty_like(t) for t in g]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        stacr_amd.clip_gradients(g, 1.0, out=out)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = stacr_amd.clip_gradients(g, 1.0, out=out)
    for i in range(4):
        for t in g:
            t.normal_()
            t.mul_(i + 0.01)
        graph.replay()
        torch.cuda.synchronize()
        want = [torch.empty_like(t) for t in g]
        n = stacr_amd.clip_gradients(g, 1.0, out=want)
        assert torch.equal(n, norm) and all(torch.equal(x, y) for x, y in zip(out, want))


def test_refusals(dev):
    import stacr_amd

    g = [torch.ones(4, device=dev)]
    f = stacr_amd.clip_gradients
    with pytest.raises(ValueError, match="norm_type"):
        f(g, 1.0, norm_type=3)
    with pytest.raises(ValueError, match="negative"):
        f(g, -1.0)
    with pytest.raises(ValueError, match="negative"):
        f(g, math.nan)
    with pytest.raises(ValueError, match="outputs"):
        f(g, 1.0, out=[])
    with pytest.raises(ValueError, match="an output of"):
        f(g, 1.0, out=[torch.ones(5, device=dev)])
    with pytest.raises(ValueError, match="an output of"):
        f(g, 1.0, out=[torch.ones(4, device=dev).half()])
    with pytest.raises(RuntimeError, match="GPU tensor"):
        f([torch.ones(4)], 1.0)
    with pytest.raises(RuntimeError, match="one GPU"):
        f([g[0], _Elsewhere(g[0])], 1.0)
    with pytest.raises(TypeError, match="float32"):
        f([torch.ones(4, device=dev, dtype=torch.float64)], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        f([torch.ones(1, device=dev).expand(4)], 1.0)
    with pytest.raises(RuntimeError, match="total norm"):
        f([torch.full((4,), math.inf, device=dev)], 1.0, error_if_nonfinite=True)
    assert float(f([], 1.0)) == 0.0


class _Elsewhere:
    """A gradient on another GPU, of which there may be none here."""

    def __init__(self, like):
        self.device, self.is_cuda, self.dtype, self.layout = torch.device("cuda:1"), True, like.dtype, like.layout

    def get_device(self):
        return 1
