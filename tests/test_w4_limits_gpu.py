"""The largest number of products that a 4-bit call accepts."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_gemv_of_two_billion_vectors(handle):
    """2^31 - 1 products of a 1 x 1 matrix: their number rounded up to whole
    sets of 8 passes 32 signed bits for the last seven counts."""
    import torch

    import b2blas

    count = 2 ** 31 - 1
    view = lambda t, d=np.uint16: b2blas.DeviceBuffer.from_ptr(handle, t.data_ptr(), t.numel(), d, t)  # noqa: E731
    x = torch.arange(count, dtype=torch.int32, device="cuda").bitwise_and_(1023).to(torch.float16)
    y = torch.full((count,), float("nan"), dtype=torch.float16, device="cuda")
    packed = torch.tensor([0x0B], dtype=torch.uint8, device="cuda")  # 11 - 8
    scale = torch.tensor([0.5], dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    handle.hgemv_w4(1, 1, 32, 1.0, view(packed, np.uint8), view(scale), None, view(x), 0.0, view(y), count=count)
    handle.synchronize()
    assert torch.equal(y, x.mul_(1.5))
    del x, y
    torch.cuda.empty_cache()
