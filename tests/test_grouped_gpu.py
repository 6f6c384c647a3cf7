"""Grouped HGEMM and its gradients through the C ABI, against plain 64-bit
forms.

Most tests use small whole numbers: every product and partial sum is then a
whole number below 2^24, which float32 holds exactly in any order, so the
16-bit result must be the exact value rounded once and is compared bit for
bit.  The tests on normal random values allow
    u |v| + K 2^-23 sum|a||b|
per output: half a step of the 16-bit rounding, and for each of the K
additions one float32 step of the running magnitude (a tensor core may cut a
sum's low bits instead of rounding them: a whole step, 2^-23)."""
import numpy as np
import pytest

import expert_ref as R

pytestmark = pytest.mark.gpu


def half_of(t):
    import b2blas

    return b2blas.Half.F16 if t == "f16" else b2blas.Half.BF16


def whole(rng, shape, top=3):
    return rng.integers(-top, top + 1, shape).astype(np.float64)


class Up:
    """Uploads a host array at a byte offset inside a larger allocation."""

    def __init__(self, h, arr, shift=0):
        import b2blas

        arr = np.ascontiguousarray(arr)
        raw = np.zeros(arr.nbytes + shift + 64, np.uint8)
        raw[shift:shift + arr.nbytes] = arr.reshape(-1).view(np.uint8)
        raw[shift + arr.nbytes:] = 0xA5
        raw[:shift] = 0xA5
        self.h, self.base, self.shift, self.arr = h, h.upload(raw), shift, arr
        self.buf = b2blas.DeviceBuffer.from_ptr(h, self.base.ptr + shift, arr.size, arr.dtype, self.base)

    def get(self):
        raw = self.h.download(self.base)
        end = self.shift + self.arr.nbytes
        assert (raw[:self.shift] == 0xA5).all() and (raw[end:] == 0xA5).all(), "bytes around the buffer changed"
        return raw[self.shift:end].view(self.arr.dtype).reshape(self.arr.shape)


def run_forward(h, t, a, b, off, c, trans, alpha=1.0, beta=0.0, shift=0):
    import b2blas

    groups = len(off) - 1
    n, k = c.shape[1], a.shape[1]
    da, db, dc = Up(h, R.bits(a, t), shift), Up(h, R.bits(b, t), shift), Up(h, R.bits(c, t), shift)
    h.hgemm_grouped(b2blas.GemmConfig(a.shape[0], n, k, alpha, beta), groups, da.buf, db.buf, Up(h, off).buf, dc.buf,
                    trans_b=trans, half=half_of(t))
    h.synchronize()
    return dc.get()


def check_forward(h, t, counts, n, k, trans, first=0, pad=0, alpha=1.0, beta=0.0, shift=0, seed=0):
    rng = np.random.default_rng(seed)
    off = R.offsets_of(counts, first)
    rows = int(off[-1]) + pad
    a = whole(rng, (rows, k))
    b = whole(rng, (len(counts), n, k) if trans else (len(counts), k, n))
    c = whole(rng, (rows, n))
    if first:
        a[:first] = np.nan
    if pad:
        a[rows - pad:] = np.inf
        c[rows - pad:] = np.nan
    if beta == 0:
        c[off[0]:off[-1]] = np.nan  # not read
    with np.errstate(invalid="ignore"):
        want = R.grouped(a, b, off, c, alpha, beta, trans)
    got = run_forward(h, t, a, b, off, c, trans, alpha, beta, shift)
    assert np.array_equal(got, R.bits(want, t))


COUNTS = [[1], [0], [128], [3, 0, 5], [129, 1], [0, 257, 0, 64, 0], [17, 300, 2, 40, 128, 127]]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("n,k", [(1, 1), (8, 8), (64, 16), (72, 200), (256, 64), (264, 72), (520, 136)])
def test_forward_is_exact_on_whole_numbers(handle, t, trans, counts, n, k):
    check_forward(handle, t, counts, n, k, trans)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("n,k", [(1, 8), (7, 5), (63, 65), (65, 63), (257, 129), (515, 1001 // 7)])
def test_forward_odd_sizes(handle, t, trans, n, k):
    check_forward(handle, t, [5, 0, 140, 1], n, k, trans, first=2, pad=3)


@pytest.mark.parametrize("shift", [2, 4, 8, 14])
@pytest.mark.parametrize("trans", [False, True])
def test_forward_unaligned_operands(handle, shift, trans):
    check_forward(handle, "f16", [33, 0, 200], 136, 72, trans, shift=shift)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("n,k", [(264, 72), (65, 63)])
def test_forward_leaves_rows_of_no_group(handle, t, n, k):
    check_forward(handle, t, [40, 0, 130], n, k, False, first=11, pad=150)
    check_forward(handle, t, [0, 0], n, k, False, first=5, pad=5)


@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (2.0, -1.0), (-0.5, 0.5), (0.0, 2.0)])
@pytest.mark.parametrize("n,k", [(136, 72), (65, 63)])
def test_forward_alpha_beta(handle, alpha, beta, n, k):
    # halves of whole numbers stay exact in float32
    check_forward(handle, "f16", [129, 0, 50], n, k, False, pad=2, alpha=alpha, beta=beta)
    check_forward(handle, "bf16", [129, 0, 50], n, k, True, pad=2, alpha=alpha, beta=beta)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("trans", [False, True])
def test_forward_long_groups(handle, t, trans):
    check_forward(handle, t, [1000, 700, 0, 1300], 776, 520, trans, pad=9)


@pytest.mark.parametrize("counts,n,k", [([700, 1300], 2056, 64), ([3] * 40, 1032, 264), ([1] * 1024, 8, 16)])
def test_forward_many_tiles(handle, counts, n, k):
    check_forward(handle, "bf16", counts, n, k, False)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("trans", [False, True])
def test_forward_odd_sizes_of_many_tiles(handle, t, trans):
    check_forward(handle, t, [1400, 0, 900, 1], 1001, 131, trans, first=1, pad=3)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("counts", [[70, 0, 200, 1], [1, 33, 64, 129]])
def test_wgrad_odd_sizes_of_many_tiles(handle, t, f32, counts):
    check_wgrad(handle, t, f32, counts, 1001, 1003, first=1, pad=3)


@pytest.mark.parametrize("t,alpha,beta", [("f16", 1.0, 0.0), ("bf16", -0.5, 2.0)])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts", [[1], [2, 0, 5], [130, 1], [0, 0]])
@pytest.mark.parametrize("n,k", [(8, 4096), (300, 2051), (264, 1032), (1000, 1096)])
def test_forward_few_tiles_of_long_sums(handle, t, alpha, beta, trans, counts, n, k):
    """Few enough tiles that several SMs share the sum of each."""
    check_forward(handle, t, counts, n, k, trans, first=1, pad=2, alpha=alpha, beta=beta)


@pytest.mark.parametrize("t,alpha,beta", [("f16", 1.0, 0.0), ("bf16", -0.5, 2.0)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("counts", [[3000], [700, 0, 1501], [1, 2000], [0, 4096, 0, 7]])
@pytest.mark.parametrize("m,n", [(8, 8), (136, 264), (65, 63), (129, 200)])
def test_wgrad_few_tiles_of_long_sums(handle, t, alpha, beta, f32, counts, m, n):
    check_wgrad(handle, t, f32, counts, m, n, first=1, pad=2, alpha=alpha, beta=beta)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("trans", [False, True])
def test_forward_random_values(handle, t, trans):
    rng = np.random.default_rng(5)
    counts, n, k = [150, 0, 260, 33], 320, 1096
    off = R.offsets_of(counts)
    a = R.value(R.bits(rng.standard_normal((off[-1], k)), t), t)
    b = R.value(R.bits(rng.standard_normal((4, n, k) if trans else (4, k, n)) * k ** -0.5, t), t)
    c = R.value(R.bits(rng.standard_normal((off[-1], n)), t), t)
    got = R.value(run_forward(handle, t, a, b, off, c, trans, 0.75, 0.5), t)
    want = R.grouped(a, b, off, c, 0.75, 0.5, trans)
    size = R.grouped(np.abs(a), np.abs(b), off, np.abs(c), 0.75, 0.5, trans)
    assert (np.abs(got - want) <= R.UNIT[t] * np.abs(want) * 1.001 + R.TINY[t] + (k + 2) * 2 * R.U32 * size).all()


def test_forward_infinities_stay_in_their_rows(handle):
    rng = np.random.default_rng(6)
    off = R.offsets_of([60, 80])
    a, b = whole(rng, (140, 72)), whole(rng, (2, 72, 136)) * 2 + 1  # odd: no zeros
    a[59, 3], a[60, 7], a[139, 71] = np.inf, np.nan, -np.inf
    got = R.value(run_forward(handle, "f16", a, b, off, np.zeros((140, 136)), False), "f16")
    assert np.isinf(got[59]).all() and np.isnan(got[60]).all() and np.isinf(got[139]).all()
    rest = np.delete(np.arange(140), [59, 60, 139])
    assert np.isfinite(got[rest]).all()


def run_wgrad(h, t, f32, a, b, off, c, alpha=1.0, beta=0.0, shift=0):
    import b2blas

    groups, m, n = c.shape
    host = c.astype(np.float32) if f32 else R.bits(c, t)
    da, db, dc = Up(h, R.bits(a, t), shift), Up(h, R.bits(b, t), shift), Up(h, host, 2 * shift if f32 else shift)
    h.hgemm_grouped_wgrad(b2blas.GemmConfig(m, n, a.shape[0], alpha, beta), groups, da.buf, db.buf, Up(h, off).buf,
                          dc.buf, half=half_of(t))
    h.synchronize()
    return dc.get()


def check_wgrad(h, t, f32, counts, m, n, first=0, pad=0, alpha=1.0, beta=0.0, shift=0, seed=0):
    rng = np.random.default_rng(seed)
    off = R.offsets_of(counts, first)
    rows = int(off[-1]) + pad
    a, b, c = whole(rng, (rows, m)), whole(rng, (rows, n)), whole(rng, (len(counts), m, n))
    for x in (a, b):
        x[:first] = np.nan
        x[rows - pad:] = np.nan if pad else 0
    if beta == 0:
        c[:] = np.nan
    want = R.wgrad(a, b, off, c, alpha, beta)
    got = run_wgrad(h, t, f32, a, b, off, c, alpha, beta, shift)
    assert np.array_equal(got, want.astype(np.float32) if f32 else R.bits(want, t))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("m,n", [(1, 1), (8, 8), (64, 72), (136, 264), (264, 520)])
def test_wgrad_is_exact_on_whole_numbers(handle, t, f32, counts, m, n):
    check_wgrad(handle, t, f32, counts, m, n)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("m,n", [(8, 1), (7, 5), (63, 65), (65, 63), (257, 129)])
def test_wgrad_odd_sizes(handle, t, f32, m, n):
    check_wgrad(handle, t, f32, [5, 0, 140, 1], m, n, first=2, pad=3)


@pytest.mark.parametrize("shift", [2, 4, 8, 14])
def test_wgrad_unaligned_operands(handle, shift):
    check_wgrad(handle, "f16", False, [33, 0, 200], 136, 72, shift=shift)
    check_wgrad(handle, "bf16", True, [33, 0, 200], 136, 72, shift=shift)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (-0.5, 0.5), (0.0, 2.0)])
@pytest.mark.parametrize("m,n", [(136, 72), (65, 63)])
def test_wgrad_alpha_beta(handle, f32, alpha, beta, m, n):
    check_wgrad(handle, "bf16", f32, [129, 0, 50], m, n, pad=2, alpha=alpha, beta=beta)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("m,n", [(136, 72), (264, 520), (65, 63)])
def test_wgrad_long_groups(handle, t, f32, m, n):
    check_wgrad(handle, t, f32, [513, 512, 0, 1500, 64], m, n, pad=7)
    check_wgrad(handle, t, f32, [1027, 1, 600], m, n, alpha=-0.5, beta=2.0)


@pytest.mark.parametrize("m,n", [(264, 264), (64, 72)])
def test_wgrad_f32_keeps_f32_sums(handle, m, n):
    """An addition in the accumulators may drop up to 2^-23 of the running sum;
    sums are taken in pieces of 512 terms, 32 additions of 16.  On random terms
    the running sum after i of 32 is about sqrt(i / 32) of the last, so the
    pieces, and with them C, are off by at most 2^-23 * sum_i sqrt(i / 32) =
    21.7 * 2^-23 of their size; the rounded additions of the pieces and inside
    a step add a few 2^-24."""
    rng = np.random.default_rng(12)
    off = R.offsets_of([4096, 2000])
    a, b = (R.value(R.bits(rng.standard_normal((off[-1], w)), "bf16"), "bf16") for w in (m, n))
    c = np.zeros((2, m, n))
    got, want = run_wgrad(handle, "bf16", True, a, b, off, c), R.wgrad(a, b, off, c)
    assert np.linalg.norm(got - want) <= 25 * 2.0 ** -23 * np.linalg.norm(want)


@pytest.mark.parametrize("m,n", [(72, 72), (72, 65), (136, 136), (264, 264), (1025, 1027)])
def test_wgrad_neighbours_nan_stays_out(handle, m, n):
    """Every count from 1 to 40 next to a group of NaN: the last k step of a
    group ends inside a block that holds the next group's rows."""
    rng = np.random.default_rng(8)
    counts = [x for i in range(1, 41) for x in (i, 1)]
    off = R.offsets_of(counts)
    a, b = whole(rng, (off[-1], m)), whole(rng, (off[-1], n))
    for g in range(1, len(counts), 2):
        a[off[g]], b[off[g]] = np.nan, np.inf
    c = np.zeros((len(counts), m, n))
    got = run_wgrad(handle, "f16", False, a, b, off, c)
    with np.errstate(invalid="ignore"):
        want = R.bits(R.wgrad(a, b, off, c), "f16")
    assert np.array_equal(got[0::2], want[0::2])


@pytest.mark.parametrize("f32", [False, True])
def test_wgrad_without_rows(handle, f32):
    import b2blas

    c = np.full((2, 24, 40), 3.0)
    for alpha, beta, want in ((1.0, 0.0, 0.0), (1.0, 0.5, 1.5), (np.inf, 0.5, 1.5)):
        got = run_wgrad(handle, "f16", f32, np.zeros((0, 24)), np.zeros((0, 40)), np.zeros(3, np.int32), c, alpha, beta)
        assert np.array_equal(got, np.full(c.shape, want, np.float32) if f32 else R.bits(np.full(c.shape, want), "f16"))


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_wgrad_random_values(handle, t):
    rng = np.random.default_rng(9)
    counts, m, n = [150, 0, 1060, 33], 200, 320
    off = R.offsets_of(counts)
    a = R.value(R.bits(rng.standard_normal((off[-1], m)), t), t)
    b = R.value(R.bits(rng.standard_normal((off[-1], n)), t), t)
    c = rng.standard_normal((4, m, n)).astype(np.float32).astype(np.float64)
    size = R.wgrad(np.abs(a), np.abs(b), off, np.abs(c), 0.75, 0.5)
    want = R.wgrad(a, b, off, c, 0.75, 0.5)
    got = run_wgrad(handle, t, True, a, b, off, c, 0.75, 0.5)
    sums = (1060 + 2) * 2 * R.U32 * size
    assert (np.abs(got - want) <= sums).all()
    c16 = R.value(R.bits(c, t), t)
    got = R.value(run_wgrad(handle, t, False, a, b, off, c16, 0.75, 0.5), t)
    want = R.wgrad(a, b, off, c16, 0.75, 0.5)
    assert (np.abs(got - want) <= R.UNIT[t] * np.abs(want) * 1.001 + R.TINY[t] + sums).all()


@pytest.mark.parametrize("n,k", [(40, 24), (33, 17)])
def test_gradients_against_differences(handle, n, k):
    """The product is bilinear, so a difference in one operand is exact:
    <G, C(A + E, B) - C(A, B)> = <dA, E>, and the same for B, with whole
    numbers small enough that f16 holds every C and gradient."""
    rng = np.random.default_rng(10)
    t, counts = "f16", [9, 0, 30, 1]
    off = R.offsets_of(counts)
    rows = int(off[-1])
    a, b, g = whole(rng, (rows, k), 2), whole(rng, (4, k, n), 2), whole(rng, (rows, n), 2)
    e, f = whole(rng, (rows, k), 1), whole(rng, (4, k, n), 1)
    c = np.zeros((rows, n))

    def product(a, b):
        return R.value(run_forward(handle, t, a, b, off, c, False), t)

    da = R.value(run_forward(handle, t, g, b, off, np.zeros((rows, k)), True), t)
    db = run_wgrad(handle, t, True, a, g, off, np.zeros((4, k, n))).astype(np.float64)
    base = product(a, b)
    assert (g * (product(a + e, b) - base)).sum() == (da * e).sum()
    assert (g * (product(a, b + f) - base)).sum() == (db * f).sum()


@pytest.mark.parametrize("n", [136, 65])
@pytest.mark.parametrize("off", [[0, 5, 3, 10], [0, 5, 8, 41], [-1, 5, 8, 10], [0, 2 ** 31 - 1, 3, 10]])
def test_refused_offsets_write_nothing(handle, n, off):
    import b2blas

    rng = np.random.default_rng(11)
    rows, k = 40, 72
    off = np.array(off, np.int32)
    a, b = whole(rng, (rows, k)), whole(rng, (3, k, n))
    dc, dw = Up(handle, np.full((rows, n), 7, np.uint16)), Up(handle, np.full((3, k, n), 7, np.float32))
    da, db, do = Up(handle, R.bits(a, "f16")), Up(handle, R.bits(b, "f16")), Up(handle, off)
    dg = Up(handle, np.zeros((rows, n), np.uint16))
    for call in (lambda: handle.hgemm_grouped(b2blas.GemmConfig(rows, n, k), 3, da.buf, db.buf, do.buf, dc.buf),
                 lambda: handle.hgemm_grouped_wgrad(b2blas.GemmConfig(k, n, rows), 3, da.buf, dg.buf, do.buf, dw.buf)):
        call()
        with pytest.raises(b2blas.CublasError) as err:
            handle.synchronize()
        assert err.value.kind == "InvalidArgument" and "offsets" in str(err.value)
        handle.synchronize()  # reported once
    assert (dc.get() == 7).all() and (dw.get() == 7).all()
    check_forward(handle, "f16", [10, 30], n, k, False)


def test_offsets_past_32_bits(handle):
    """C and B of more than 2^31 elements."""
    import torch

    import b2blas

    h = handle
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    small = lambda *s: torch.randint(-3, 4, s, generator=gen, device="cuda").to(torch.float16)  # noqa: E731
    view = lambda t, d=np.uint16: b2blas.DeviceBuffer.from_ptr(h, t.data_ptr(), t.numel(), d, t)  # noqa: E731
    rows, n, k = 70000, 32768, 8
    a, b, c = small(rows, k), small(2, k, n), torch.zeros(rows, n, dtype=torch.float16, device="cuda")
    off = torch.tensor([0, 66000, rows], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    h.hgemm_grouped(b2blas.GemmConfig(rows, n, k), 2, view(a), view(b), view(off, np.int32), view(c))
    h.synchronize()
    for r in (0, 65535, 65536, 65999, 66000, 69999):
        assert torch.equal(c[r].float(), a[r].float() @ b[int(r >= 66000)].float())
    del a, b, c
    k, n = 32768, 32776
    a, b, c = small(6, k), small(3, k, n), torch.zeros(6, n, dtype=torch.float16, device="cuda")
    off = torch.tensor([0, 1, 3, 6], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    h.hgemm_grouped(b2blas.GemmConfig(6, n, k), 3, view(a), view(b), view(off, np.int32), view(c))
    h.synchronize()
    for r, g in ((0, 0), (2, 1), (3, 2), (5, 2)):
        assert torch.equal(c[r].double(), (a[r].double() @ b[g].double()).to(torch.float16).double())
    del a, b, c
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,k", [(900, 256), (130, 4096), (6000, 64)])
def test_two_graphs_of_one_handle_replay_at_once(rows, k):
    """Captured calls keep no state in the handle: two graphs captured through
    it replay on two streams at once and give the eager bits."""
    import torch

    import b2blas

    h = b2blas.Handle(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        gen = torch.Generator(device="cuda")
        gen.manual_seed(4)
        view = lambda t, d=np.uint16: b2blas.DeviceBuffer.from_ptr(h, t.data_ptr(), t.numel(), d, t)  # noqa: E731
        jobs = []
        for n in (520, 515):
            a = torch.randn(rows, k, generator=gen, device="cuda").half()
            b = torch.randn(3, k, n, generator=gen, device="cuda").half()
            c, w = torch.zeros(rows, n, device="cuda").half(), torch.zeros(3, k, n, device="cuda")
            off = torch.tensor([0, 100, 100, rows], dtype=torch.int32, device="cuda")

            def step(a=a, b=b, c=c, w=w, off=off, rows=rows, k=k, n=n):
                h.hgemm_grouped(b2blas.GemmConfig(rows, n, k), 3, view(a), view(b), view(off, np.int32), view(c))
                h.hgemm_grouped_wgrad(b2blas.GemmConfig(k, n, rows), 3, view(a), view(c), view(off, np.int32),
                                      view(w, np.float32))

            jobs.append((step, c, w))
        torch.cuda.synchronize()
        eager, graphs = [], []
        for s, (step, c, w) in zip(streams, jobs):
            h.set_stream(s.cuda_stream)
            step()
            h.synchronize()
            eager.append((c.clone(), w.clone()))
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                step()
            graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(5):
            for _, c, w in jobs:
                c.zero_(), w.zero_()
            torch.cuda.synchronize()
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            for (_, c, w), (ce, we) in zip(jobs, eager):
                assert torch.equal(c, ce) and torch.equal(w, we)
        del graphs
    finally:
        h.set_stream(None)
        h.close()
