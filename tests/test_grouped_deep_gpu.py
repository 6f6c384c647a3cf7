"""Grouped products whose sums are long, in 16-bit C.

The tensor core's f32 additions cut low bits, always toward zero: a step of 16
terms aligns its products and the running sum and loses less than one f32 step
of the running sum, 2^-23 of it, for each of the 17.  A sum of one sign that
stays in the accumulator has lost 1.5e-3 of itself after 2^18 terms (measured
for f16, 2.4 of the 17 a step), three times the rounding to f16 (2^-11).  Sums
are therefore taken in pieces of 4096 terms that are added up with rounding.
In terms of similar size the running sum is on average half the last one, so a
result of T terms is off by at most, of its size,
    256 steps x 17 x 2^-23 / 2 = 2.6e-4   within the pieces
    (T / 4096 + 1) x 2^-24                adding up the pieces, and times alpha
before it is rounded to 16 bits.  Rounding keeps order, so the result lies
between the roundings of the exact value less and plus that."""
import numpy as np
import pytest

import expert_ref as R
from test_grouped_gpu import half_of

pytestmark = pytest.mark.gpu

# (groups' rows or, forward, depth; sizes): the tile that takes them
WGRAD = [
    ([262144], 1160, 1160),                    # CTA pairs
    ([262144] + [1] * 80, 120, 248),           # one CTA, 256 columns or 128
    ([262144] + [1] * 150, 64, 56),            # one CTA, 64 columns
    ([262144], 136, 136),                      # a cluster shares each sum
    ([262144], 1161, 1163),                    # loaded by warps, pairs
    ([262144] + [1] * 150, 65, 63),            # loaded by warps
    ([262144], 65, 63),                        # loaded by warps, shared
    ([1048576], 136, 136),
    ([1048576], 65, 63),
]
FORWARD = [
    ([1100], 1160, 131072),                    # pairs
    ([60, 70], 9480, 65536),                   # one CTA
    ([20] * 40, 248, 65536),                   # one CTA
    ([130], 72, 131072),                       # a cluster shares each sum
    ([1100], 1163, 65537),                     # loaded by warps
    ([60, 70], 4801, 65537),
    ([130], 71, 131073),                       # loaded by warps, shared
    ([60, 70], 4808, 262144),
    ([130], 72, 1048576),
    ([130], 71, 1048577),
]


def view(h, t, kind=np.uint16):
    import b2blas

    return b2blas.DeviceBuffer.from_ptr(h, t.data_ptr(), t.numel(), kind, t)


def offsets(counts):
    import torch

    return torch.tensor(R.offsets_of(counts), device="cuda")


def run(h, t, counts, n, k, a, b, c, alpha, beta, trans=None):
    """trans None: the gradient, C_g = A_g^T B_g, with k columns of A."""
    import torch

    import b2blas

    torch.cuda.synchronize()
    if trans is None:
        h.hgemm_grouped_wgrad(b2blas.GemmConfig(k, n, a.shape[0], alpha, beta), len(counts), view(h, a), view(h, b),
                              view(h, offsets(counts), np.int32), view(h, c), half=half_of(t))
    else:
        h.hgemm_grouped(b2blas.GemmConfig(a.shape[0], n, k, alpha, beta), len(counts), view(h, a), view(h, b),
                        view(h, offsets(counts), np.int32), view(h, c), trans_b=trans, half=half_of(t))
    h.synchronize()


def exact(counts, a, b, trans=None):
    """64-bit products, group by group: rows of C, or for the gradient matrices."""
    import torch

    off, out = R.offsets_of(counts), []
    for g in range(len(counts)):
        x = a[off[g]:off[g + 1]]
        if trans is None:
            v = torch.zeros(a.shape[1], b.shape[1], dtype=torch.float64, device="cuda")
            for r in range(0, x.shape[0], 65536):  # whole matrices in 64 bits would take four times their room
                v += x[r:r + 65536].double().t() @ b[off[g] + r:min(off[g] + r + 65536, off[g + 1])].double()
        else:
            v = torch.zeros(x.shape[0], b.shape[1] if trans else b.shape[2], dtype=torch.float64, device="cuda")
            for j in range(0, x.shape[1], 16384):
                y = b[g][:, j:j + 16384].double().t() if trans else b[g][j:j + 16384].double()
                v += x[:, j:j + 16384].double() @ y
        out.append(v)
    return torch.stack(out) if trans is None else torch.cat(out)


def inputs(t, counts, n, k, trans, make, depth=None):
    """A, B and C of a product: `make(shape)` for the operands."""
    import torch

    rows = sum(counts)
    a = make((rows, k))
    b = make((rows, n) if trans is None else (len(counts), n, k) if trans else (len(counts), k, n))
    c = torch.randint(-3, 4, (len(counts), k, n) if trans is None else (rows, n), device="cuda").to(R.HALF[t])
    return a, b, c


def check_one_sign(h, t, counts, n, k, depth, trans=None):
    import torch

    gen = torch.Generator(device="cuda")
    gen.manual_seed(depth + n)
    a, b, c = inputs(t, counts, n, k, trans, lambda s: (torch.rand(s, generator=gen, device="cuda") + 0.5).to(R.HALF[t]))
    run(h, t, counts, n, k, a, b, c, 1.0 / depth, 0.0, trans)
    want = exact(counts, a, b, trans) / depth
    if trans is None:
        c, want = c[0], want[0]  # the long group's
    sums = 256 * 17 / 2 * 2.0 ** -23 * 1.01 + (depth / 4096 + 1) * 2.0 ** -24
    least, most = ((want * (1 + d)).to(R.HALF[t]) for d in (-sums, sums))
    assert ((c >= least) & (c <= most)).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("counts,m,n", WGRAD)
def test_wgrad_of_one_sign(handle, t, counts, m, n):
    check_one_sign(handle, t, counts, n, m, counts[0])


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts,n,k", FORWARD)
def test_forward_of_one_sign(handle, t, trans, counts, n, k):
    check_one_sign(handle, t, counts, n, k, k, trans)


def check_whole(h, t, counts, n, k, trans, alpha, beta):
    """Values -1, 0 and 1: every partial sum is a whole number below 2^24."""
    import torch

    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    a, b, c = inputs(t, counts, n, k, trans, lambda s: torch.randint(-1, 2, s, generator=gen, device="cuda").to(R.HALF[t]))
    # below 2^13 terms' sums a 64-bit product times alpha, plus whole numbers, is exact in f32
    want = (alpha * exact(counts, a, b, trans) + (beta * c.double() if beta else 0)).float().to(R.HALF[t])
    if not beta:
        c.fill_(float("nan"))
    run(h, t, counts, n, k, a, b, c, alpha, beta, trans)
    assert torch.equal(c, want)


# depths around the pieces' borders, a short sum next to a long one, sizes off
# the tiles' edges
@pytest.mark.parametrize("t,alpha,beta", [("f16", 1.0, 0.0), ("bf16", -0.5, 2.0)])
@pytest.mark.parametrize("m,n", [(1160, 1096), (120, 248), (64, 56), (1161, 1163), (65, 63)])
@pytest.mark.parametrize("counts", [[4096, 4097, 0, 12300, 5], [8192, 8193, 1, 40000], [5000] + [70] * 150, [100000]])
def test_long_wgrad_is_exact_on_whole_numbers(handle, t, alpha, beta, counts, m, n):
    if len(counts) > 100 and m > 1000:
        counts = counts[:8]
    check_whole(handle, t, counts, n, m, None, alpha, beta)


@pytest.mark.parametrize("t,alpha,beta", [("f16", 1.0, 0.0), ("bf16", -0.5, 2.0)])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts,n", [([1100, 0, 300], 1160), ([60, 1, 70], 4808), ([20] * 40, 248), ([130], 72),
                                      ([1400, 3], 1163), ([60, 70], 4801), ([3], 71)])
@pytest.mark.parametrize("k", [4096, 4104, 8192, 12345, 20488])
def test_long_forward_is_exact_on_whole_numbers(handle, t, alpha, beta, trans, counts, n, k):
    check_whole(handle, t, counts, n, k, trans, alpha, beta)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("counts,m,n", [
    ([65536], 1160, 1160),                     # CTA pairs
    ([65536] + [1] * 149, 120, 248),           # one CTA, 256 columns
    ([65536] + [1] * 79, 120, 248),            # 128 columns
    ([65536] + [1] * 149, 64, 56),             # 64 columns
    ([65536], 1161, 1163),                     # loaded by warps
    ([65536] + [1] * 149, 65, 63),
    ([524288], 136, 136),                      # a cluster shares each sum
    ([524288], 65, 63)])
def test_f32_wgrad_of_one_sign(handle, t, counts, m, n):
    """f32 C in pieces of 512: at most 32 steps x 17 x 2^-23 / 2 within them,
    3.2e-5, and one rounding, 2^-24, for each that is added up.  One piece of
    65536 terms loses ten times as much (3.8e-4 measured for f16, 2.4 of the 17
    a step), and so would the eighth of a shared sum of 524288.  The f32 tests
    on whole numbers cannot see that, and the one on random terms has so few
    tiles that clusters share its sums, in parts not much longer than a piece."""
    import torch

    import b2blas

    gen = torch.Generator(device="cuda")
    gen.manual_seed(m)
    depth = counts[0]
    a, b, _ = inputs(t, counts, n, m, None, lambda s: (torch.rand(s, generator=gen, device="cuda") + 0.5).to(R.HALF[t]))
    c = torch.zeros(len(counts), m, n, device="cuda")
    torch.cuda.synchronize()
    handle.hgemm_grouped_wgrad(b2blas.GemmConfig(m, n, sum(counts), 1.0 / depth, 0.0), len(counts), view(handle, a),
                               view(handle, b), view(handle, offsets(counts), np.int32), view(handle, c, np.float32),
                               half=half_of(t))
    handle.synchronize()
    want = exact(counts[:1], a, b)[0] / depth
    off = float(((c[0].double() - want) / want).abs().max())
    assert off <= 32 * 17 / 2 * 2.0 ** -23 * 1.01 + (depth / 512 + 2) * 2.0 ** -24
