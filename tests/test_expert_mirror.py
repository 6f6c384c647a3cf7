"""What the Python mirror of the expert-layer calls settles itself (CPU only)."""
import numpy as np
import pytest

from test_expert_args import Fake, buf


@pytest.fixture
def h():
    import b2blas

    h = b2blas.Handle.__new__(b2blas.Handle)
    h._h, h._lib = None, Fake._lib()
    return h


@pytest.mark.parametrize("fan", [0, -1, -3, -2 ** 63])
@pytest.mark.parametrize("x", [0, 65, 130])
def test_fan_below_one_is_refused(h, fan, x):
    """A negative fan would reach the C ABI as a huge size_t, which stands for
    "all products share one vector", with x of unchecked length."""
    import b2blas

    with pytest.raises(b2blas.CublasError, match="fan") as e:
        h.hgemv_w4_grouped(2, 3, 65, 32, 1.0, buf(6 * 33, np.uint8), buf(18, np.uint16), None, buf(x, np.uint16),
                           buf(4, np.int32), 0.0, buf(12, np.uint16), count=4, fan=fan)
    assert e.value.kind == "InvalidArgument"


class Own:
    """A caller's own buffer: it has what the calls use, and is no DeviceBuffer."""

    def __init__(self, n, dtype):
        self.ptr, self.dtype, self.n = 256, np.dtype(dtype), n

    def __len__(self):
        return self.n


def test_buffers_of_the_callers_own_are_taken(h):
    """Every call asks a buffer for its dtype, its length by len() and its
    address, nothing else."""
    import b2blas

    with pytest.raises(b2blas.CublasError, match="expected 12, got 11"):
        h.saxpy(12, 1.0, Own(11, np.float32), Own(12, np.float32))
    with pytest.raises(AssertionError, match="b2b_saxpy reached the library"):
        h.saxpy(12, 1.0, Own(12, np.float32), Own(12, np.float32))
    with pytest.raises(AssertionError, match="b2b_hgemm_grouped reached the library"):
        h.hgemm_grouped(b2blas.GemmConfig(10, 6, 4), 2, Own(40, np.uint16), Own(48, np.uint16), Own(3, np.int32),
                        Own(60, np.uint16))


def test_every_expert_call_has_its_cpp_method():
    import os
    import re

    from conftest import PKG

    src = open(os.path.join(PKG, "cpp", "cublas_rs.hpp")).read()
    for name in ("hgemm_grouped", "hgemm_grouped_wgrad", "quantize_w4", "dequantize_w4", "hgemv_w4", "hgemv_w4_grouped"):
        assert re.search(rf"void {name}\(", src) and f"b2b_{name}(h_" in src
