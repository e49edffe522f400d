"""Refusals of the gated block, rotary positions and clipping at the C ABI, and their workspace sizes: host
rules that end before any launch, so they need no GPU.  (The addresses given are never read.)"""
import ctypes
import os

import pytest

A = 1 << 12  # an aligned address


@pytest.fixture(scope="module")
def lib():
    from stacr_amd import _lib as L

    if not os.path.exists(L.LIB_PATH):
        pytest.skip("libstacr_amd.so not built")
    return L.load()


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


FORWARD = dict(x=A, dtype=1, rows=100, d=64, x_ld=64, w_gate=A, w_up=A, ff=128, b_gate=None, b_up=None, activation=0, h=A,
               gate=None, up=None, gate_low=None, up_low=None, workspace=None, nbytes=0, stream=None)


@pytest.mark.parametrize("change,code,words", [
    (dict(dtype=7), 1, "dtype"), (dict(dtype=-1), 1, "dtype"), (dict(rows=-1), 1, "rows"), (dict(d=0), 1, "d >= 1"),
    (dict(ff=0), 1, "ff >= 1"), (dict(x_ld=63), 1, "stride"), (dict(activation=5), 1, "activation"),
    (dict(activation=-1), 1, "activation"), (dict(ff=(1 << 20) + 1), 2, "2^20"), (dict(rows=1 << 24), 2, "2^24"),
    (dict(x=None), 1, "NULL"), (dict(w_gate=None), 1, "NULL"), (dict(w_up=None), 1, "NULL"), (dict(h=None), 1, "NULL"),
    (dict(gate=A), 1, "gate goes with up"), (dict(gate_low=A, up_low=A), 1, "gate goes with up"),
    (dict(gate=A, up=A, gate_low=A), 1, "gate goes with up"), (dict(gate=A + 8, up=A), 1, "16-byte"),
    (dict(gate=A, up=A, gate_low=A, up_low=A + 1), 1, "16-byte"),
    (dict(dtype=0, gate=A, up=A, gate_low=A, up_low=A), 1, "no low bytes"),
    (dict(dtype=0), 3, "needed"), (dict(d=60, x_ld=60), 3, "needed"), (dict(x=A + 2), 3, "needed")])
def test_forward_refuses(lib, change, code, words):
    rc = lib.stacr_gated_forward(*{**FORWARD, **change}.values())
    assert rc == code
    assert words in lib.stacr_last_error().decode()


def test_forward_of_no_rows(lib):
    assert lib.stacr_gated_forward(*{**FORWARD, "rows": 0, "x": None, "h": None}.values()) == 0


BACKWARD = dict(dh=A, x=A, dtype=1, rows=100, d=64, x_ld=64, w_gate=A, w_up=A, ff=128, b_gate=None, b_up=None, activation=0,
                gate=A, up=A, gate_low=None, up_low=None, dx=A, dw_gate=A, dw_up=A, db_gate=None, db_up=None, dgu=None,
                workspace=None, nbytes=0, stream=None)


@pytest.mark.parametrize("change,code,words", [
    (dict(dtype=3), 1, "dtype"), (dict(x_ld=1), 1, "stride"), (dict(activation=9), 1, "activation"),
    (dict(dw_up=None), 1, "dw_gate with dw_up"), (dict(dw_gate=None), 1, "dw_gate with dw_up"), (dict(dh=None), 1, "NULL"),
    (dict(up=None), 1, "gate goes with up"), (dict(dgu=A + 8), 1, "16-byte"), (dict(), 3, "needed")])
def test_backward_refuses(lib, change, code, words):
    rc = lib.stacr_gated_backward(*{**BACKWARD, **change}.values())
    assert rc == code
    assert words in lib.stacr_last_error().decode()


def test_workspace_grows_with_what_is_laid_out_anew(lib):
    def need(dtype, rows, d, ff, x=A, backward=0):
        n = ctypes.c_size_t()
        assert lib.stacr_gated_workspace_bytes(x, dtype, rows, d, d, A, A, ff, backward, ctypes.byref(n)) == 0
        return n.value

    assert need(1, 100, 64, 128) == 0  # multiplied as they are
    assert need(1, 12, 60, 128) == 0 and need(0, 12, 64, 128) == 0  # few rows: read in place in any form
    assert need(1, 100, 64, 128, x=A + 2) >= 100 * 64 * 2  # x alone
    assert need(1, 100, 60, 128) >= (100 + 2 * 128) * 64 * 2  # rows of 60 become rows of 64
    assert need(0, 100, 64, 128) >= 4 * (100 + 2 * 128) * 64 * 2  # four planes
    assert need(1, 100, 64, 128, backward=1) >= 100 * 2 * 128 * 2  # [dg | du]
    assert lib.stacr_gated_workspace_bytes(A, 1, 100, 64, 64, A, A, 128, 0, None) == 1


ROTARY = dict(q=A, q_strides=i64(8, 8, 8, 1), q_heads=2, k=A, k_strides=i64(8, 8, 8, 1), k_heads=1, dtype=1, batch=1, seq=3, head=64,
              rot=64, layout=0, cos=A, sin=A, length=16, positions=None, position_bytes=8, psb=0, pss=0, offset=0, inverse=0,
              q_out=A, q_out_strides=i64(8, 8, 8, 1), k_out=A, k_out_strides=i64(8, 8, 8, 1), stream=None)


@pytest.mark.parametrize("change,code,words", [
    (dict(dtype=4), 1, "dtype"), (dict(rot=3), 1, "even rot"), (dict(rot=0), 1, "even rot"), (dict(rot=66), 1, "even rot"),
    (dict(batch=-1), 1, "sizes"), (dict(length=-1), 1, "sizes"), (dict(layout=2), 1, "layout"),
    (dict(positions=A, position_bytes=2), 1, "4 or 8"), (dict(head=(1 << 16) + 2), 2, "2^16"), (dict(q=None), 1, "NULL"),
    (dict(k_out=None), 1, "NULL"), (dict(cos=None), 1, "NULL"), (dict(q_strides=None), 1, "NULL"),
    (dict(batch=1 << 16, seq=1 << 16), 2, "2^31")])
def test_rotary_refuses(lib, change, code, words):
    rc = lib.stacr_rotary(*{**ROTARY, **change}.values())
    assert rc == code
    assert words in lib.stacr_last_error().decode()


@pytest.mark.parametrize("change", [dict(batch=0), dict(seq=0), dict(q_heads=0, k_heads=0)])
def test_rotary_of_nothing(lib, change):
    assert lib.stacr_rotary(*{**ROTARY, **change}.values()) == 0


TABLES = dict(length=16, rot=64, base=10000.0, scaling=0, factor=1.0, original=0, fast=0.0, slow=0.0, cos=A, sin=A, stream=None)


@pytest.mark.parametrize("change", [
    dict(rot=3), dict(rot=0), dict(length=-1), dict(base=1.0), dict(base=float("nan")), dict(scaling=4), dict(scaling=1, factor=0.5),
    dict(scaling=2, factor=2.0, rot=2), dict(scaling=3, factor=2.0, original=0, fast=32.0, slow=1.0),
    dict(scaling=3, factor=2.0, original=8, fast=1.0, slow=32.0), dict(cos=None), dict(sin=None)])
def test_rotary_tables_refuse(lib, change):
    assert lib.stacr_rotary_tables(*{**TABLES, **change}.values()) == 1


def test_clipping_refuses(lib):
    need = ctypes.c_size_t()
    assert lib.stacr_clip_workspace_bytes(2, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.stacr_clip_workspace_bytes(-1, ctypes.byref(need)) == 1
    two = (ctypes.c_void_p * 2)(A, A)
    types = (ctypes.c_int * 2)(0, 1)

    def call(count=2, inp=two, out=two, sizes=i64(8, 8), dtypes=types, norm_type=2, most=1.0, eps=1e-6, norm=A, ws=A, nbytes=1 << 30):
        return lib.stacr_clip_gradients(count, inp, out, sizes, dtypes, norm_type, most, eps, norm, ws, nbytes, None)

    assert call(count=-1) == 1 and call(inp=None) == 1 and call(sizes=None) == 1 and call(dtypes=None) == 1
    assert call(norm=None) == 1 and call(norm_type=3) == 1 and call(norm_type=-1) == 1
    assert call(most=-1.0) == 1 and call(most=float("nan")) == 1 and call(eps=-1.0) == 1
    assert call(sizes=i64(8, -1)) == 1 and call(inp=(ctypes.c_void_p * 2)(A, None)) == 1
    assert call(out=(ctypes.c_void_p * 2)(None, A)) == 1 and call(dtypes=(ctypes.c_int * 2)(0, 3)) == 1
    assert call(sizes=i64(8, 1 << 60)) == 2
    assert call(ws=None) == 3 and call(nbytes=8) == 3
