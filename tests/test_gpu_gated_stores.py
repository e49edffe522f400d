"""Where the gated forward writes, and its GELU far below zero.

The outputs stand between guard bytes: nothing outside the rows, and in the kept planes nothing outside the
padded rows, may change, whatever the tile's overhang (rows and columns past the last, in wide and in narrow
pieces).  GELU is taken at gates that reach the product exactly (one term a sum), so its error is the rounding of
the type (2^-8 bf16, 2^-11 fp16 of the value) and that of the 16-bit types' own exponential and reciprocal, 1e-5
at these gates."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GUARD = 4096


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    return torch.device("cuda:0")


def guarded(nbytes, dev):
    return torch.full((nbytes + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=dev)


def outside(buf, nbytes):
    return bool((buf[:GUARD] == 0xA5).all()) and bool((buf[GUARD + nbytes:] == 0xA5).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,d,ff", [(3, 16, 24), (65, 40, 72), (130, 64, 200), (257, 72, 333), (300, 8, 8), (4100, 24, 2056)])
def test_nothing_outside_the_rows(dev, rows, d, ff, dtype):
    from stacr_amd import _lib, kernels

    print("case gated guards", rows, d, ff, dtype, flush=True)
    g = torch.Generator(device="cpu").manual_seed(rows + ff)
    x, wg, wu = (torch.randn(n, d, generator=g).to(dev, DT[dtype]) for n in (rows, ff, ff))
    code, size = _lib.__dict__["DTYPE_" + {"f32": "F32", "bf16": "BF16", "f16": "F16"}[dtype]], x.element_size()
    padded = (ff + 7) // 8 * 8
    h_bytes, kept_bytes, low_bytes = rows * ff * size, rows * padded * size, rows * padded
    h, gate, up = guarded(h_bytes, dev), guarded(kept_bytes, dev), guarded(kept_bytes, dev)
    low = [guarded(low_bytes, dev) for _ in range(2)] if code else [None, None]
    ws, nbytes = kernels._gated_workspace(x, code, rows, d, d, wg, wu, 0)

    def at(t):
        return None if t is None else t.data_ptr() + GUARD

    rc = _lib.load().stacr_gated_forward(x.data_ptr(), code, rows, d, d, wg.data_ptr(), wu.data_ptr(), ff, None, None, 0, at(h),
                                         at(gate), at(up), at(low[0]), at(low[1]), None if ws is None else ws.data_ptr(), nbytes,
                                         torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "stacr_gated_forward")
    torch.cuda.synchronize()
    assert outside(h, h_bytes)
    for t in (gate, up):
        assert outside(t, kept_bytes)
    for t in low:
        assert t is None or outside(t, low_bytes)
    # and every value inside is there: h = act(g) u of the kept g and u, to the rounding of the type
    exact = [x.double().cpu() @ w.double().cpu().t() for w in (wg, wu)]
    for t, l, want in ((gate, low[0], exact[0]), (up, low[1], exact[1])):
        v = t[GUARD:GUARD + kept_bytes].cpu()
        if l is not None:
            v = v.view(torch.int16).to(torch.int32) * 65536 + l[GUARD:GUARD + low_bytes].cpu().to(torch.int32) * 256
        got = v.view(torch.float32).view(rows, padded)[:, :ff].double()
        # 2^-16 for the 24 bits, 2^-21 for fp32's part products, and the sums' rounding at the size of their terms
        assert (got - want).norm() <= ((2.0 ** -16 if l is not None else 2.0 ** -21) + d ** 0.5 * 2.0 ** -23) * want.norm()
    got = h[GUARD:GUARD + h_bytes].view(DT[dtype]).view(rows, ff).double().cpu()
    want = exact[0] * torch.sigmoid(exact[0]) * exact[1]
    unit = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -18}[dtype]
    assert (got - want).norm() <= unit * want.norm()


@pytest.mark.parametrize("rows", [33, 97])
@pytest.mark.parametrize("dtype,least", [("bf16", -8.0), ("f16", -3.5)])
def test_gelu_keeps_its_digits_below_zero(dev, dtype, least, rows):
    import stacr_amd

    print("case gelu tail", dtype, rows, flush=True)
    x = torch.zeros(rows, 8, device=dev, dtype=DT[dtype])
    x[:, 0] = torch.linspace(least, 2.0, rows).to(DT[dtype])
    x[:, 1] = 1
    wg, wu = torch.zeros(16, 8, device=dev, dtype=DT[dtype]), torch.zeros(16, 8, device=dev, dtype=DT[dtype])
    wg[:, 0], wu[:, 1] = 1, 1
    h = stacr_amd.gated_feed_forward(x, wg, wu, activation="gelu")
    g = x[:, :1].double().cpu()
    want = (g * 0.5 * torch.special.erfc(-g / 2 ** 0.5)).expand(rows, 16)
    unit = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    assert ((h.double().cpu() - want).abs() <= (unit + 1e-5) * want.abs()).all()
