"""Refusals of the grouped and 4-bit-weight calls, which the library settles
on the host before it touches a device (CPU only).

The handle is a block of zeroed bytes: the checks look at nothing in it."""
import ctypes

import pytest

OK, INVALID, UNSUPPORTED = 0, 3, 5
P = ctypes.c_void_p(256)  # an operand that is not NULL and is never read
NULL = None


@pytest.fixture(scope="module")
def lib():
    import b2blas

    return b2blas.load_library()


@pytest.fixture(scope="module")
def fake():
    block = ctypes.create_string_buffer(4096)
    yield ctypes.cast(block, ctypes.c_void_p)


def forward(lib, h, type=0, trans=0, groups=2, rows=8, n=8, k=8, a=P, b=P, c=P, off=P):
    return lib.b2b_hgemm_grouped(h, type, trans, groups, rows, n, k, 1.0, a, b, 0.0, c, off)


def wgrad(lib, h, type=0, c_type=2, groups=2, rows=8, m=8, n=8, a=P, b=P, c=P, off=P):
    return lib.b2b_hgemm_grouped_wgrad(h, type, c_type, groups, rows, m, n, 1.0, a, b, 0.0, c, off)


def quant(lib, h, type=0, m=4, n=64, group=32, w=P, p=P, s=P):
    return lib.b2b_quantize_w4(h, type, m, n, group, w, p, s, NULL)


def dequant(lib, h, type=0, m=4, n=64, group=32, w=P, p=P, s=P):
    return lib.b2b_dequantize_w4(h, type, m, n, group, p, s, NULL, w)


def gemv(lib, h, type=0, m=4, n=64, group=32, count=1, p=P, s=P, x=P, y=P):
    return lib.b2b_hgemv_w4(h, type, m, n, group, 1.0, p, s, NULL, x, count, 0.0, y)


def gemvg(lib, h, type=0, groups=2, m=4, n=64, group=32, count=1, fan=1, p=P, s=P, x=P, y=P, index=P):
    return lib.b2b_hgemv_w4_grouped(h, type, groups, m, n, group, 1.0, p, s, NULL, x, count, fan, index, 0.0, y)


@pytest.mark.parametrize("call", [forward, wgrad, quant, dequant, gemv, gemvg])
def test_null_handle_and_unknown_types(lib, fake, call):
    assert call(lib, NULL) == INVALID and b"NULL handle" in lib.b2b_last_error()
    for bad in (-1, 2, 3):
        assert call(lib, fake, type=bad) == INVALID and b"type" in lib.b2b_last_error()


@pytest.mark.parametrize("call,names", [(forward, ("a", "b", "c", "off")), (wgrad, ("a", "b", "c", "off")),
                                        (quant, ("w", "p", "s")), (dequant, ("w", "p", "s")),
                                        (gemv, ("p", "s", "x", "y")), (gemvg, ("p", "s", "x", "y", "index"))])
def test_null_operands(lib, fake, call, names):
    for name in names:
        assert call(lib, fake, **{name: NULL}) == INVALID and b"NULL operand" in lib.b2b_last_error()


@pytest.mark.parametrize("call,names", [(forward, ("a", "b", "c")), (wgrad, ("a", "b")), (quant, ("w", "s")),
                                        (dequant, ("w", "s")), (gemv, ("s", "x", "y")), (gemvg, ("s", "x", "y"))])
def test_misaligned_operands(lib, fake, call, names):
    for name in names:
        assert call(lib, fake, **{name: ctypes.c_void_p(257)}) == INVALID and b"aligned" in lib.b2b_last_error()
    for four in {forward: ("off",), wgrad: ("off", "c"), gemvg: ("index",)}.get(call, ()):
        assert call(lib, fake, **{four: ctypes.c_void_p(258)}) == INVALID and b"aligned" in lib.b2b_last_error()
    if call is wgrad:
        assert wgrad(lib, fake, c_type=0, c=ctypes.c_void_p(257)) == INVALID


@pytest.mark.parametrize("call,names", [(forward, ("groups", "rows", "n", "k")), (wgrad, ("groups", "m", "n")),
                                        (quant, ("m", "n")), (dequant, ("m", "n")), (gemv, ("m", "n", "count")),
                                        (gemvg, ("groups", "m", "n", "count"))])
def test_empty_sizes_return_without_a_launch(lib, fake, call, names):
    for name in names:
        assert call(lib, fake, **{name: 0}) == OK


def test_grouped_limits(lib, fake):
    for call, sizes in ((forward, ("rows", "n", "k")), (wgrad, ("rows", "m", "n"))):
        assert call(lib, fake, groups=1025) == UNSUPPORTED
        for name in sizes:
            assert call(lib, fake, **{name: 2 ** 31}) == UNSUPPORTED
    assert forward(lib, fake, groups=1024, n=2 ** 31 - 1, k=2 ** 31 - 1) == INVALID  # 2^73 bytes of B
    assert forward(lib, fake, trans=2) == INVALID
    assert wgrad(lib, fake, type=0, c_type=1) == INVALID and wgrad(lib, fake, type=1, c_type=0) == INVALID
    assert wgrad(lib, fake, rows=0, a=NULL, b=NULL, c=NULL) == INVALID


def test_w4_limits(lib, fake):
    for call in (quant, dequant, gemv, gemvg):
        for bad in (0, 1, 16, 33, 2 ** 64 - 1):
            assert call(lib, fake, group=bad) == INVALID and b"multiple of 32" in lib.b2b_last_error()
        for name in ("m", "n"):
            assert call(lib, fake, **{name: 2 ** 31}) == UNSUPPORTED
        assert call(lib, fake, group=2 ** 32) == UNSUPPORTED
    for call in (gemv, gemvg):
        assert call(lib, fake, count=2 ** 31) == UNSUPPORTED
    assert gemvg(lib, fake, fan=0) == INVALID
    assert gemvg(lib, fake, groups=2 ** 31) == UNSUPPORTED
    assert gemvg(lib, fake, groups=2 ** 31 - 1, m=2 ** 31 - 1, n=2 ** 31 - 1) == INVALID


class Fake:
    """A Handle whose library would fail if it were reached."""

    _h = None

    class _lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} reached the library")


def buf(n, dtype):
    import b2blas

    return b2blas.DeviceBuffer(None, 256, n, dtype, owned=False)


def test_python_checks_lengths_and_types():
    import numpy as np

    import b2blas

    h = b2blas.Handle.__new__(b2blas.Handle)
    h._h, h._lib = None, Fake._lib()
    u16, u8, i32, f32 = np.uint16, np.uint8, np.int32, np.float32
    cfg = b2blas.GemmConfig(10, 6, 4)
    good = dict(a=buf(40, u16), b=buf(2 * 24, u16), offsets=buf(3, i32), c=buf(60, u16))
    for name, bad, kind in [("a", buf(39, u16), "Dim"), ("b", buf(47, u16), "Dim"), ("offsets", buf(2, i32), "Dim"),
                            ("c", buf(59, u16), "Dim"), ("a", buf(40, f32), "Inv"), ("offsets", buf(3, np.int64), "Inv"),
                            ("c", buf(60, f32), "Inv")]:
        with pytest.raises(b2blas.CublasError) as e:
            h.hgemm_grouped(cfg, 2, **{**good, name: bad})
        assert e.value.kind.startswith(kind)
    cfg = b2blas.GemmConfig(4, 6, 10)
    good = dict(a=buf(40, u16), b=buf(60, u16), offsets=buf(3, i32), c=buf(48, f32))
    for name, bad, kind in [("a", buf(39, u16), "Dim"), ("b", buf(59, u16), "Dim"), ("c", buf(47, f32), "Dim"),
                            ("c", buf(47, u16), "Dim"), ("c", buf(48, np.float64), "Inv"), ("offsets", buf(2, i32), "Dim")]:
        with pytest.raises(b2blas.CublasError) as e:
            h.hgemm_grouped_wgrad(cfg, 2, **{**good, name: bad})
        assert e.value.kind.startswith(kind)
    w = dict(packed=buf(3 * 33, u8), scales=buf(9, u16), zeros=buf(9, u8))
    short = [("packed", buf(98, u8)), ("scales", buf(8, u16)), ("zeros", buf(8, u8))]
    for name, bad in short + [("w", buf(3 * 65 - 1, u16))]:
        args = {**w, "w": buf(3 * 65, u16), name: bad}
        for call in (h.quantize_w4, h.dequantize_w4):
            with pytest.raises(b2blas.CublasError) as e:
                call(3, 65, 32, **args)
            assert e.value.kind == "DimensionMismatch"
    for name, bad in short + [("x", buf(129, u16)), ("y", buf(5, u16))]:
        args = {**w, "x": buf(130, u16), "y": buf(6, u16), name: bad}
        with pytest.raises(b2blas.CublasError):
            h.hgemv_w4(3, 65, 32, 1.0, args["packed"], args["scales"], args["zeros"], args["x"], 0.0, args["y"], count=2)
    w = dict(packed=buf(6 * 33, u8), scales=buf(18, u16), zeros=buf(18, u8))
    for name, bad in [("packed", buf(197, u8)), ("scales", buf(17, u16)), ("zeros", buf(17, u8)), ("x", buf(129, u16)),
                      ("y", buf(8, u16)), ("index", buf(2, i32)), ("index", buf(3, np.int64))]:
        args = {**w, "x": buf(130, u16), "y": buf(9, u16), "index": buf(3, i32), name: bad}
        with pytest.raises(b2blas.CublasError):
            h.hgemv_w4_grouped(2, 3, 65, 32, 1.0, args["packed"], args["scales"], args["zeros"], args["x"], args["index"],
                               0.0, args["y"], count=3, fan=2)
