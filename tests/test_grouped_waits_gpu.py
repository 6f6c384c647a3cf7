"""Bounded waits of the grouped products under a short limit: none is for more
than what one tile, or the tiles that a warp passed over, may take."""
import numpy as np
import pytest

import expert_ref as R
from test_grouped_deep_gpu import exact, offsets, view

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("m,n,groups", [(128, 64, 150), (512, 264, 80), (512, 260, 80)])
def test_a_long_group_of_whole_blocks_before_a_ragged_one(monkeypatch, f32, m, n, groups):
    """The warp that wipes what follows a group's last row has nothing to do in
    a group of a multiple of 64 rows, and waits for the next one from the
    start: through all 2^21 rows here, 11 ms, under a limit of 1 ms a wait."""
    import torch

    import b2blas

    monkeypatch.setenv("B2B_WAIT_LIMIT_MS", "1")
    counts = [1 << 21] + [0, 3, 64, 1, 130] * 40
    counts = counts[:groups]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)
    small = lambda w: torch.randint(-1, 2, (sum(counts), w), generator=gen, device="cuda").half()  # noqa: E731
    a, b = small(m), small(n)
    c = torch.full((groups, m, n), float("nan"), device="cuda", dtype=torch.float32 if f32 else torch.float16)
    torch.cuda.synchronize()
    with b2blas.Handle(0) as h:
        h.hgemm_grouped_wgrad(b2blas.GemmConfig(m, n, sum(counts)), groups, view(h, a), view(h, b),
                              view(h, offsets(counts), np.int32), view(h, c, np.float32 if f32 else np.uint16))
        h.synchronize()  # raises for a wait that gave up
    assert torch.equal(c.double(), exact(counts, a, b).to(c.dtype).double())
