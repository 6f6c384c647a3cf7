"""4-bit weights whose values or vectors are not finite, or next to a type's
largest value."""
import numpy as np
import pytest

import expert_ref as R
from test_w4_gpu import dequantize, gemv, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("n,shift", [(96, 0), (97, 0), (96, 2)])
def test_scales_that_are_not_finite_show(handle, t, with_zeros, n, shift):
    """W = scale (q - zero) for scales of infinity and NaN too; a finite scale
    that takes a value beyond the type gives its largest finite value."""
    import torch

    top = torch.finfo(R.HALF[t]).max
    rng = np.random.default_rng(n)
    packed, _, zeros = make(rng, t, 1, 8, n, 32, with_zeros)
    s = np.full((8, -(-n // 32)), 0.5)
    s[0, 0], s[1, 1], s[2, 2], s[3, 0], s[4, 1] = np.inf, -np.inf, np.nan, top, -top / 3
    scales = R.bits(s, t)
    got = R.value(dequantize(handle, t, n, 32, packed, scales, zeros, shift), t)
    with np.errstate(invalid="ignore"):
        want = R.w4_values(packed, scales, zeros, n, 32, t)
    finite = np.isfinite(s[:, np.arange(n) // 32])
    want = np.where(finite, np.clip(want, -top, top), want)
    want = R.value(R.bits(want, t), t)
    assert np.isinf(want).any() and np.isnan(want).any() and (np.abs(want) == top).any()
    assert np.array_equal(got, want, equal_nan=True)
