"""4-bit weights through the C ABI, against plain 64-bit forms.

Quantised values, scales and zero points must be equal; a value made 16-bit
again is the product rounded once.  Products on whole numbers with scales that
are powers of two are exact in float32, so they are compared bit for bit; on
normal random values an output may be off by
    u |v| + (n + 2) 2^-23 sum|w||x|
(half a step of the 16-bit rounding; a float32 step for each of the n
additions and the two scalings)."""
import numpy as np
import pytest

import expert_ref as R
from test_grouped_gpu import Up, half_of

pytestmark = pytest.mark.gpu


def quantize(h, t, w, group, with_zeros, shift=0):
    m, n = w.shape
    gs = -(-n // group)
    dw = Up(h, R.bits(w, t), shift)
    dp, ds = Up(h, np.zeros((m, (n + 1) // 2), np.uint8), shift // 2), Up(h, np.zeros((m, gs), np.uint16), shift)
    dz = Up(h, np.zeros((m, gs), np.uint8), shift // 2) if with_zeros else None
    h.quantize_w4(m, n, group, dw.buf, dp.buf, ds.buf, dz.buf if dz else None, half=half_of(t))
    h.synchronize()
    return dp.get(), ds.get(), dz.get() if dz else None


def dequantize(h, t, n, group, packed, scales, zeros, shift=0):
    m = packed.shape[0]
    dw = Up(h, np.zeros((m, n), np.uint16), shift)
    dz = Up(h, zeros, shift // 2) if zeros is not None else None
    h.dequantize_w4(m, n, group, Up(h, packed, shift // 2).buf, Up(h, scales, shift).buf, dz.buf if dz else None,
                    dw.buf, half=half_of(t))
    h.synchronize()
    return dw.get()


def same_scales(got, want, t):
    return np.array_equal(np.nan_to_num(R.value(got, t), nan=-1.0), np.nan_to_num(R.value(want, t), nan=-1.0))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("m,n,shift", [(1, 1, 0), (3, 33, 0), (7, 256, 0), (5, 520, 0), (4, 1001, 0), (3, 127, 2), (9, 384, 8)])
def test_quantize_and_back(handle, t, with_zeros, group, m, n, shift):
    rng = np.random.default_rng(m * 1000 + n)
    w = R.value(R.bits(rng.standard_normal((m, n)) * 0.1 + 0.02, t), t)
    packed, scales, zeros = quantize(handle, t, w, group, with_zeros, shift)
    wp, ws, wz = R.quantize(w, group, with_zeros, t)
    assert np.array_equal(scales, ws)
    assert np.array_equal(packed, wp)
    assert wz is None or np.array_equal(zeros, wz)
    back = dequantize(handle, t, n, group, packed, scales, zeros, shift)
    assert np.array_equal(back, R.bits(R.w4_values(packed, scales, zeros, n, group, t), t))
    # what the format promises: half a step of 4 bits, the scale's rounding
    # (eps / 2 of up to 15 steps, which may also clamp), the result's
    s = R.value(scales, t)[:, np.arange(n) // group]
    assert (np.abs(R.value(back, t) - w) <= s * (0.5 + 16 * R.UNIT[t] + (0.5 if with_zeros else 0)) + R.UNIT[t] * np.abs(w) + R.TINY[t]).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("m,n,group,shift", [(3, 4096, 512, 0), (2, 5000, 1024, 0), (5, 2056, 2080, 0), (3, 4096, 512, 2),
                                             (2, 5000, 96, 8), (2, 1001, 320, 0)])
def test_quantize_long_groups(handle, t, with_zeros, m, n, group, shift):
    test_quantize_and_back(handle, t, with_zeros, group, m, n, shift)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
def test_quantize_extremes(handle, t, with_zeros):
    """Groups of zeros, subnormals, the largest values, one sign only, and
    infinities and NaN, which make the group's scale NaN and no other's."""
    import torch

    top, low = torch.finfo(R.HALF[t]).max, torch.finfo(R.HALF[t]).tiny
    sub = low * torch.finfo(R.HALF[t]).eps
    rng = np.random.default_rng(1)
    rows = [np.zeros(64), np.full(64, sub), rng.integers(-20, 21, 64) * sub, np.where(np.arange(64) % 2, top, -top),
            np.full(64, top), np.full(64, -top), np.full(64, 1.0), -np.arange(64.0), np.arange(64.0),
            np.r_[np.inf, np.ones(63)], np.r_[np.ones(63), -np.inf], np.r_[np.ones(31), np.nan, np.ones(32)]]
    w = np.stack([np.r_[r, np.arange(32.0)] for r in rows])
    w = R.value(R.bits(w, t), t)
    packed, scales, zeros = quantize(handle, t, w, 32, with_zeros)
    with np.errstate(invalid="ignore", over="ignore"):
        wp, ws, wz = R.quantize(w, 32, with_zeros, t)
    assert same_scales(scales, ws, t) and np.array_equal(packed, wp)
    assert wz is None or np.array_equal(zeros, wz)
    assert np.isnan(R.value(scales, t)).sum() == 3
    back = R.value(dequantize(handle, t, 96, 32, packed, scales, zeros), t)
    want = np.clip(R.w4_values(packed, scales, zeros, 96, 32, t), -top, top)
    want = R.value(R.bits(want, t), t)
    assert np.array_equal(np.isnan(back), np.isnan(want)) and np.array_equal(back[~np.isnan(want)], want[~np.isnan(want)])
    assert np.isfinite(back[:9]).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("n", [96, 97])
def test_quantize_ties_go_to_even(handle, t, with_zeros, n):
    """Values halfway between two steps, at scales that are not powers of two."""
    rows = []
    for s in (1.0, 1.25, 0.6875, 2.0 ** -9, 3 * 2.0 ** 8):
        for z in (0, 3, 7, 12):
            steps = np.arange(-2 * z, 31 - 2 * z) / 2 if with_zeros else np.arange(-14, 15) / 2
            r = np.zeros(n)
            r[:len(steps)] = steps * s
            r[32:32 + len(steps)] = -steps * s
            r[64:64 + len(steps)] = np.roll(steps, 5) * s
            rows.append(r)
    w = R.value(R.bits(np.stack(rows), t), t)
    for group in (32, 96):
        packed, scales, zeros = quantize(handle, t, w, group, with_zeros)
        wp, ws, wz = R.quantize(w, group, with_zeros, t)
        assert np.array_equal(scales, ws) and np.array_equal(packed, wp)
        assert wz is None or np.array_equal(zeros, wz)


def make(rng, t, matrices, m, n, group, with_zeros, exact=True):
    gs = -(-n // group)
    packed = rng.integers(0, 256, (matrices * m, (n + 1) // 2)).astype(np.uint8)
    s = 2.0 ** rng.integers(-2, 2, (matrices * m, gs)) if exact else rng.standard_normal((matrices * m, gs)) * 0.01
    # the high four bits of a zero point have no meaning
    zeros = rng.integers(0, 256, (matrices * m, gs)).astype(np.uint8) if with_zeros else None
    return packed, R.bits(s, t), zeros


def gemv(h, t, matrices, m, n, group, w, x, y, count, index=None, fan=1, alpha=1.0, beta=0.0, shift=0):
    packed, scales, zeros = w
    dp, ds, dx, dy = Up(h, packed, shift // 2), Up(h, scales, shift), Up(h, R.bits(x, t), shift), Up(h, R.bits(y, t), shift)
    dz = Up(h, zeros, shift // 2) if zeros is not None else None
    z = dz.buf if dz else None
    if index is None:
        h.hgemv_w4(m, n, group, alpha, dp.buf, ds.buf, z, dx.buf, beta, dy.buf, count=count, half=half_of(t))
    else:
        h.hgemv_w4_grouped(matrices, m, n, group, alpha, dp.buf, ds.buf, z, dx.buf, Up(h, index).buf, beta, dy.buf,
                           count=count, fan=fan, half=half_of(t))
    h.synchronize()
    return dy.get()


def reference(t, m, n, group, w, x, y, count, index=None, fan=1, alpha=1.0, beta=0.0, absolute=False):
    v = R.w4_values(*w, n, group, t)
    if absolute:
        v, x, y = np.abs(v), np.abs(x), np.abs(y)
    out = np.zeros((count, m))
    matrices = v.shape[0] // m
    for i in range(count):
        e = 0 if index is None else index[i]
        p = v[e * m:(e + 1) * m] @ x[i // fan] if 0 <= e < matrices else np.zeros(m)
        out[i] = alpha * p + (beta * y[i] if beta else 0)
    return out


def check(h, t, m, n, group, with_zeros, count, seed=0, alpha=1.0, beta=0.0, shift=0):
    rng = np.random.default_rng(seed)
    w = make(rng, t, 1, m, n, group, with_zeros)
    x = rng.integers(-3, 4, (count, n)).astype(np.float64)
    y = rng.integers(-3, 4, (count, m)).astype(np.float64) if beta else np.full((count, m), np.nan)
    got = gemv(h, t, 1, m, n, group, w, x, y, count, alpha=alpha, beta=beta, shift=shift)
    assert np.array_equal(got, R.bits(reference(t, m, n, group, w, x, y, count, alpha=alpha, beta=beta), t))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 512])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 32), (16, 64), (17, 96), (70, 512), (33, 1000), (5, 1033), (130, 2080)])
def test_gemv_is_exact_on_whole_numbers(handle, t, with_zeros, group, m, n):
    check(handle, t, m, n, group, with_zeros, 1)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("count", [2, 3, 7, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("m,n,group,with_zeros", [(40, 320, 32, True), (100, 1000, 128, False), (19, 65, 64, True)])
def test_gemv_of_several_vectors(handle, t, count, m, n, group, with_zeros):
    check(handle, t, m, n, group, with_zeros, count)


@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (-0.5, 2.0), (0.0, 1.0)])
@pytest.mark.parametrize("count", [1, 5])
def test_gemv_alpha_beta(handle, alpha, beta, count):
    check(handle, "f16", 50, 256, 64, True, count, alpha=alpha, beta=beta)


@pytest.mark.parametrize("shift", [2, 4, 8, 16])
@pytest.mark.parametrize("n", [512, 520, 513])
def test_gemv_unaligned_operands(handle, shift, n):
    check(handle, "bf16", 33, n, 64, True, 3, shift=shift)


@pytest.mark.parametrize("m,n,count", [(2048, 4096, 1), (4096, 1024, 8), (300, 16384, 2), (16384, 64, 1)])
@pytest.mark.parametrize("group", [32, 128])
def test_gemv_larger(handle, m, n, count, group):
    check(handle, "f16", m, n, group, True, count)
    check(handle, "bf16", m, n, group, False, count)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("group", [32, 128])
def test_gemv_random_values(handle, t, with_zeros, group):
    rng = np.random.default_rng(3)
    m, n, count = 200, 2100, 3
    w = make(rng, t, 1, m, n, group, with_zeros, exact=False)
    x = R.value(R.bits(rng.standard_normal((count, n)), t), t)
    y = R.value(R.bits(rng.standard_normal((count, m)), t), t)
    got = R.value(gemv(handle, t, 1, m, n, group, w, x, y, count, alpha=0.75, beta=0.5), t)
    args = (t, m, n, group, w, x, y, count)
    want, size = reference(*args, alpha=0.75, beta=0.5), reference(*args, alpha=0.75, beta=0.5, absolute=True)
    assert (np.abs(got - want) <= R.UNIT[t] * np.abs(want) * 1.001 + R.TINY[t] + (n + 2) * 2 * R.U32 * size).all()


@pytest.mark.parametrize("n", [49152, 163840, 327680])
def test_gemv_of_wide_rows(handle, n):
    check(handle, "f16", 37, n, 128, False, 9 if n < 163840 else 3)


def test_gemv_refuses_rows_that_are_too_wide(handle):
    import b2blas

    with pytest.raises(b2blas.CublasError) as e:
        check(handle, "f16", 2, 327681, 128, False, 1)
    assert e.value.status == 5 and "327680" in str(e.value)  # B2B_ERR_NOT_SUPPORTED


def test_gemv_nan_scale_stays_in_its_row(handle):
    rng = np.random.default_rng(4)
    m, n = 40, 256
    packed, scales, _ = make(rng, "f16", 1, m, n, 64, False)
    scales[7, 2] = 0x7E00
    x = np.ones((2, n))
    got = R.value(gemv(handle, "f16", 1, m, n, 64, (packed, scales, None), x, np.zeros((2, m)), 2), "f16")
    assert np.isnan(got[:, 7]).all() and np.isfinite(np.delete(got, 7, 1)).all()


def check_grouped(h, t, experts, m, n, group, with_zeros, index, fan, alpha=1.0, beta=0.0, shift=0, seed=0):
    rng = np.random.default_rng(seed)
    count = len(index)
    w = make(rng, t, experts, m, n, group, with_zeros)
    x = rng.integers(-3, 4, (-(-count // fan), n)).astype(np.float64)
    y = rng.integers(-3, 4, (count, m)).astype(np.float64) if beta else np.full((count, m), np.nan)
    index = np.array(index, np.int32)
    got = gemv(h, t, experts, m, n, group, w, x, y, count, index, fan, alpha, beta, shift)
    want = reference(t, m, n, group, w, x, y, count, index, fan, alpha, beta)
    assert np.array_equal(got, R.bits(want, t))


INDEX = {
    "one": [0], "none": [-1], "beyond": [5, 2 ** 31 - 1, -2 ** 31, 4], "same": [3] * 20, "pairs": [0, 4, 4, 1, 2, 0],
    "dropped": [1, -1, 1, -1, 0, 3, -1], "odd": [2, 2, 1, 0, 3],
}


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("fan", [1, 2, 3])
@pytest.mark.parametrize("case", sorted(INDEX))
def test_grouped_gemv_is_exact_on_whole_numbers(handle, t, with_zeros, fan, case):
    check_grouped(handle, t, 5, 70, 320, 64, with_zeros, INDEX[case], fan)


@pytest.mark.parametrize("m,n", [(1, 1), (33, 65), (20, 1000), (513, 512)])
@pytest.mark.parametrize("count", [1, 9, 300, 700])
def test_grouped_gemv_sizes(handle, m, n, count):
    rng = np.random.default_rng(count)
    check_grouped(handle, "f16", 7, m, n, 32, True, rng.integers(-1, 7, count), 1)


@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (-0.5, 2.0), (0.0, 1.0)])
def test_grouped_gemv_alpha_beta(handle, alpha, beta):
    check_grouped(handle, "bf16", 3, 50, 256, 64, True, [1, -1, 0, 1], 2, alpha, beta)


def test_empty_product_is_zero_whatever_alpha_is(handle):
    w = make(np.random.default_rng(0), "f16", 3, 50, 256, 64, False)
    y = np.full((2, 50), 3.0)
    index = np.array([-1, 9], np.int32)
    got = gemv(handle, "f16", 3, 50, 256, 64, w, np.ones((2, 256)), y, 2, index, 1, float("inf"), 1.0)
    assert np.array_equal(got, R.bits(y, "f16"))


@pytest.mark.parametrize("shift", [2, 8, 16])
def test_grouped_gemv_unaligned_operands(handle, shift):
    check_grouped(handle, "f16", 3, 33, 512, 64, True, [2, 0, 2, 1], 2, shift=shift)


def test_packed_bytes_past_32_bits(handle):
    """More than 2^32 packed bytes and 2^33 values: the last expert's rows."""
    import torch

    import b2blas

    h = handle
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    e, m, n = 3, 65536, 65536
    packed = torch.randint(0, 256, (e, m, n // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = torch.ones(e, m, n // 128, device="cuda").half()
    x = torch.randint(-1, 2, (1, n), generator=gen, device="cuda").half()
    y = torch.zeros(2, m, device="cuda").half()
    index = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    view = lambda t, d=np.uint16: b2blas.DeviceBuffer.from_ptr(h, t.data_ptr(), t.numel(), d, t)  # noqa: E731
    torch.cuda.synchronize()
    h.hgemv_w4_grouped(e, m, n, 128, 2.0 ** -6, view(packed, np.uint8), view(scales), None, view(x), view(index, np.int32),
                       0.0, view(y), count=2, fan=2)
    h.synchronize()
    for i, ex in ((0, 2), (1, 0)):
        for r0 in (0, m - 256):
            p = packed[ex, r0:r0 + 256]
            q = torch.stack((p & 15, p >> 4), -1).reshape(256, n).double() - 8
            assert torch.equal(y[i, r0:r0 + 256], (q @ x[0].double() / 64).half())
    del packed, scales
    torch.cuda.empty_cache()


def test_graph_and_other_stream():
    import torch

    import b2blas

    h = b2blas.Handle(0)
    s = torch.cuda.Stream()
    try:
        h.set_stream(s.cuda_stream)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(5)
        view = lambda t, d=np.uint16: b2blas.DeviceBuffer.from_ptr(h, t.data_ptr(), t.numel(), d, t)  # noqa: E731
        e, m, n, group = 4, 512, 1024, 128
        w = torch.randn(e * m, n, generator=gen, device="cuda").half()
        packed = torch.zeros(e * m, n // 2, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(e * m, n // group, device="cuda").half()
        x = torch.randn(3, n, generator=gen, device="cuda").half()
        index = torch.tensor([0, 3, 3, 1, -1, 2], dtype=torch.int32, device="cuda")
        y, z = torch.zeros(6, m, device="cuda").half(), torch.zeros(3, m, device="cuda").half()
        torch.cuda.synchronize()

        def step():
            h.quantize_w4(e * m, n, group, view(w), view(packed, np.uint8), view(scales))
            h.hgemv_w4_grouped(e, m, n, group, 1.0, view(packed, np.uint8), view(scales), None, view(x),
                               view(index, np.int32), 0.0, view(y), count=6, fan=2)
            h.hgemv_w4(m, n, group, 1.0, view(packed, np.uint8), view(scales), None, view(x), 0.0, view(z), count=3)

        step()
        h.synchronize()
        eager = (y.clone(), z.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
        # new contents of the same buffers: a replay reads them
        index.copy_(torch.tensor([3, 0, 1, 3, 2, -1], dtype=torch.int32))
        x.copy_(x.flip(0))
        packed.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        assert torch.equal(z, eager[1].flip(0))
        step()
        h.synchronize()
        graph_y = y.clone()
        with torch.cuda.stream(s):
            g.replay()
        s.synchronize()
        assert torch.equal(y, graph_y) and not torch.equal(y, eager[0]) and (y[5] == 0).all()
        del g
    finally:
        h.set_stream(None)
        h.close()


@pytest.mark.parametrize("e,m,n,group,count,t,with_zeros", [
    (1, 16384, 16384, 128, 1, "f16", False), (1, 8192, 16384, 32, 8, "bf16", True), (5, 4096, 2048, 64, 40, "f16", True),
    (1, 4096, 4104, 64, 3, "f16", True), (2, 20000, 20480, 256, 3, "bf16", False),
    # vectors that several SMs share: many joins, and rounds of every size
    (1, 18944, 16384, 128, 8, "f16", True), (1, 30000, 40960, 64, 8, "bf16", False), (1, 40, 200000, 128, 2, "f16", False),
    (8, 2048, 16384, 128, 32, "f16", True), (3, 6000, 8200, 64, 21, "bf16", True), (1, 64, 8192, 128, 1, "bf16", False),
    # rounds whose warps are not all needed, in many sets
    (2, 2500, 256, 64, 36, "f16", True), (3, 20000, 768, 32, 70, "bf16", False), (5, 9000, 1000, 128, 60, "f16", True),
    (1, 12000, 1500, 96, 33, "bf16", True), (40, 700, 300, 128, 300, "f16", False),
    # rows that begin at any byte
    (1, 5000, 16388, 128, 1, "f16", False), (1, 3000, 4099, 64, 9, "bf16", True), (4, 2001, 2046, 32, 17, "f16", True)])
def test_gemv_gives_the_same_exact_bits_each_time(handle, e, m, n, group, count, t, with_zeros):
    """Many rounds of every warp's buffers, 20 times over, against exact sums
    of whole numbers."""
    import torch

    import b2blas

    h, dt = handle, R.HALF[t]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    gs, pitch = -(-n // group), (n + 1) // 2
    rand = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=gen, device="cuda")  # noqa: E731
    packed, zeros = rand(0, 256, e * m, pitch).to(torch.uint8), rand(0, 16, e * m, gs).to(torch.uint8) if with_zeros else None
    scales, x = torch.ones(e * m, gs, device="cuda").to(dt), rand(-1, 2, count, n).to(dt)
    index = rand(0, e, count).to(torch.int32)
    want = torch.zeros(count, m, device="cuda").to(dt)
    for i in range(e):
        q = torch.stack((packed[i * m:(i + 1) * m] & 15, packed[i * m:(i + 1) * m] >> 4), -1).flatten(1)[:, :n].float()
        q -= 8 if zeros is None else zeros[i * m:(i + 1) * m].float().repeat_interleave(group, 1)[:, :n]
        want[index == i] = (x[index == i].double() @ q.double().t() / 64).to(dt)
        del q
    view = lambda v, d=np.uint16: None if v is None else b2blas.DeviceBuffer.from_ptr(h, v.data_ptr(), v.numel(), d, v)  # noqa: E731
    for _ in range(20):
        y = torch.full_like(want, float("nan"))
        torch.cuda.synchronize()
        args = (view(packed, np.uint8), view(scales), view(zeros, np.uint8), view(x))
        if e == 1:
            h.hgemv_w4(m, n, group, 2.0 ** -6, *args, 0.0, view(y), count=count, half=half_of(t))
        else:
            h.hgemv_w4_grouped(e, m, n, group, 2.0 ** -6, *args, view(index, np.int32), 0.0, view(y), count=count, half=half_of(t))
        h.synchronize()
        assert torch.equal(y, want)
    del packed, want
    torch.cuda.empty_cache()
