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


def same(got, want, t):
    """Bit patterns against float64 values, NaN for NaN."""
    got, want = R.value(got, t), R.value(R.bits(want, t), t)
    return np.array_equal(got, want, equal_nan=True)


def spoilt(rng, count, n):
    """Whole numbers, with an infinity and a NaN in vectors 1 and 4, and both
    infinities, first and last column, in vector 6."""
    x = rng.integers(-3, 4, (count, n)).astype(np.float64)
    x[1, n // 2], x[4, n - 1] = np.inf, np.nan
    x[6, 0], x[6, n - 1] = -np.inf, np.inf
    return x


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 512])
@pytest.mark.parametrize("n", [512, 520, 513])
def test_infinities_and_nan_stay_in_their_vector(handle, t, with_zeros, group, n):
    """One vector of a set of 8 that share their weights: what it holds shows
    in its own products alone, an infinity as one unless its weight is 0."""
    rng = np.random.default_rng(n + group)
    m = 70
    w = make(rng, t, 1, m, n, group, with_zeros)
    x = spoilt(rng, 9, n)
    got = gemv(handle, t, 1, m, n, group, w, x, np.zeros((9, m)), 9)
    with np.errstate(invalid="ignore"):
        want = reference(t, m, n, group, w, x, None, 9)
    assert np.isinf(want[1]).any() and np.isnan(want[1]).any() and np.isnan(want[4]).all()
    assert np.isfinite(want[[0, 2, 3, 5, 7, 8]]).all()
    assert same(got, want, t)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("n", [512, 513])
def test_infinities_and_nan_stay_in_their_product(handle, t, n):
    rng = np.random.default_rng(n)
    m, index = 70, np.array([2, 0, 2, 1, 2, 2, 0, -1, 2], np.int32)
    w = make(rng, t, 3, m, n, 64, True)
    x = spoilt(rng, 9, n)
    got = gemv(handle, t, 3, m, n, 64, w, x, np.zeros((9, m)), 9, index)
    with np.errstate(invalid="ignore"):
        want = reference(t, m, n, 64, w, x, None, 9, index)
    assert (want[7] == 0).all() and same(got, want, t)


@pytest.mark.parametrize("group", [32, 128, 512, 96])
@pytest.mark.parametrize("n", [1024, 1021])
def test_large_bfloat16_vectors(handle, group, n):
    """A group's columns, at most 256 at a time, are summed before their scale
    comes in: 256 x 15 x |x| stays finite in f32 for |x| < 2^116."""
    m = 40
    packed, zeros = np.full((m, (n + 1) // 2), 0xFF, np.uint8), np.zeros((m, -(-n // group)), np.uint8)
    scales = R.bits(np.full(zeros.shape, 2.0 ** -20), "bf16")
    top = 2.0 ** 116 * (1 - 2.0 ** -8)
    x = np.stack([np.full(n, top), np.full(n, -top)])
    got = gemv(handle, "bf16", 1, m, n, group, (packed, scales, zeros), x, np.zeros((2, m)), 2)
    # 255 / 256 x 15 x n: below 2^24, exact in f32
    assert same(got, reference("bf16", m, n, group, (packed, scales, zeros), x, None, 2), "bf16")
