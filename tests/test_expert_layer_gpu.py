"""The grouped and 4-bit-weight operators together, as an expert layer uses
them: a training step in 16 bits, and serving from 4-bit weights.

Every product is compared with the 64-bit product of the operands that the
kernels themselves produced, within
    u |v| + K 2^-23 sum|a||b|
(half a step of the 16-bit rounding, a float32 step for each addition)."""
import numpy as np
import pytest

import expert_ref as R

pytestmark = pytest.mark.gpu


def near(got, want, size, k, t):
    unit, tiny = (R.UNIT[t], R.TINY[t]) if t else (0.0, 0.0)
    bound = unit * want.abs() * 1.001 + tiny + (k + 2) * 2 * R.U32 * size
    return bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hidden,inner", [(256, 384), (200, 136), (129, 255)])
def test_training_step(t, hidden, inner):
    """y = relu(x W1) W2 for tokens sorted by expert, and the gradients of a
    linear loss, with the weights' added to f32 sums that hold a step before."""
    import torch

    import b2blas

    h = b2blas.Handle(0)
    try:
        h.set_stream(torch.cuda.current_stream().cuda_stream)
        dt, half = R.HALF[t], b2blas.Half.F16 if t == "f16" else b2blas.Half.BF16
        gen = torch.Generator(device="cuda")
        gen.manual_seed(1)
        rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
        view = lambda v, d=np.uint16: b2blas.DeviceBuffer.from_ptr(h, v.data_ptr(), v.numel(), d, v)  # noqa: E731
        experts, tokens, spare = 6, 500, 12
        chosen = torch.randint(0, experts - 1, (tokens,), generator=gen, device="cuda")  # the last one gets none
        order = torch.argsort(chosen, stable=True)
        off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        off[1:] = torch.bincount(chosen, minlength=experts).cumsum(0)
        rows = tokens + spare  # a padded batch
        x = torch.full((rows, hidden), float("nan"), device="cuda").to(dt)
        x[:tokens] = rand(tokens, hidden).to(dt)[order]
        w1, w2 = ((rand(experts, a, b) * a ** -0.5).to(dt) for a, b in ((hidden, inner), (inner, hidden)))
        dy = torch.full((rows, hidden), float("inf"), device="cuda").to(dt)
        dy[:tokens] = rand(tokens, hidden).to(dt)

        def product(a, b, n, k, trans=False):
            c = torch.full((rows, n), 7.0, device="cuda").to(dt)
            h.hgemm_grouped(b2blas.GemmConfig(rows, n, k), experts, view(a), view(b), view(off, np.int32), view(c), trans_b=trans, half=half)
            bounds = off.tolist()
            for g in range(experts):
                r = slice(bounds[g], bounds[g + 1])
                m = (b[g].t() if trans else b[g]).double()
                assert near(c[r], a[r].double() @ m, a[r].double().abs() @ m.abs(), k, t)
            assert (c[tokens:] == 7).all()
            return c

        def weight_gradient(a, b, m, n):
            held = rand(experts, m, n)
            c = held.clone()
            h.hgemm_grouped_wgrad(b2blas.GemmConfig(m, n, rows, 0.5, 1.0), experts, view(a), view(b), view(off, np.int32),
                                  view(c, np.float32), half=half)
            bounds = off.tolist()
            for g in range(experts):
                r = slice(bounds[g], bounds[g + 1])
                want = 0.5 * (a[r].double().t() @ b[r].double()) + held[g].double()
                size = a[r].double().abs().t() @ b[r].double().abs() + held[g].double().abs()
                assert near(c[g], want, size, tokens, None)
            assert torch.equal(c[experts - 1], held[experts - 1])

        u = product(x, w1, inner, hidden)
        a = torch.relu(u)
        product(a, w2, hidden, inner)
        da = product(dy, w2, inner, hidden, trans=True)
        du = torch.where(u > 0, da, torch.zeros_like(da))
        product(du, w1, hidden, inner, trans=True)
        weight_gradient(x, du, hidden, inner)
        weight_gradient(a, dy, inner, hidden)
        h.synchronize()
    finally:
        h.set_stream(None)
        h.close()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("n,m,group", [(256, 384, 128), (520, 130, 32), (131, 77, 64)])
def test_serving(t, with_zeros, n, m, group):
    """Weights made 4-bit once; a prompt takes them back in 16 bits through the
    grouped product, single tokens take them as they are: both are products
    with the same quantised weights."""
    import torch

    import b2blas

    h = b2blas.Handle(0)
    try:
        h.set_stream(torch.cuda.current_stream().cuda_stream)
        dt, half = R.HALF[t], b2blas.Half.F16 if t == "f16" else b2blas.Half.BF16
        gen = torch.Generator(device="cuda")
        gen.manual_seed(2)
        rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
        view = lambda v, d=np.uint16: b2blas.DeviceBuffer.from_ptr(h, v.data_ptr(), v.numel(), d, v)  # noqa: E731
        experts, fan, tokens = 4, 2, 7
        gs, pitch = -(-n // group), (n + 1) // 2
        w = (rand(experts, m, n) * n ** -0.5).to(dt)
        packed = torch.zeros(experts, m, pitch, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(experts, m, gs, device="cuda").to(dt)
        zeros = torch.zeros(experts, m, gs, dtype=torch.uint8, device="cuda") if with_zeros else None
        z = view(zeros, np.uint8) if with_zeros else None
        h.quantize_w4(experts * m, n, group, view(w), view(packed, np.uint8), view(scales), z, half=half)
        w16 = torch.zeros_like(w)
        h.dequantize_w4(experts * m, n, group, view(packed, np.uint8), view(scales), z, view(w16), half=half)
        h.synchronize()
        # half a step (and half a zero point's) and the roundings of scale and result
        step = scales.double().repeat_interleave(group, 2)[..., :n]
        bound = step * (0.5 + 16 * R.UNIT[t] + (0.5 if with_zeros else 0)) + R.UNIT[t] * w.double().abs() + R.TINY[t]
        assert ((w16.double() - w.double()).abs() <= bound).all()

        x = rand(tokens, n).to(dt)
        index = torch.randint(0, experts, (tokens * fan,), generator=gen, device="cuda").to(torch.int32)
        y = torch.zeros(tokens * fan, m, device="cuda").to(dt)
        h.hgemv_w4_grouped(experts, m, n, group, 1.0, view(packed, np.uint8), view(scales), z, view(x), view(index, np.int32),
                           0.0, view(y), count=tokens * fan, fan=fan, half=half)
        # the same products as a prompt's: rows sorted by expert, W as the n x k operand
        order = torch.argsort(index, stable=True)
        off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
        off[1:] = torch.bincount(index, minlength=experts).cumsum(0)
        rows = x[order // fan].contiguous()
        c = torch.zeros(tokens * fan, m, device="cuda").to(dt)
        h.hgemm_grouped(b2blas.GemmConfig(tokens * fan, m, n), experts, view(rows), view(w16), view(off, np.int32), view(c),
                        trans_b=True, half=half)
        h.synchronize()
        q = torch.stack((packed & 15, packed >> 4), -1).flatten(2)[..., :n].double()
        exact = step * (q - (8 if zeros is None else zeros.double().repeat_interleave(group, 2)[..., :n]))
        for i, e in enumerate(index.tolist()):
            v = x[i // fan].double()
            assert near(y[i], exact[e] @ v, exact[e].abs() @ v.abs(), n, t)
        for i, j in enumerate(order.tolist()):
            m16, v = w16[index[j].item()].double(), x[j // fan].double()
            assert near(c[i], m16 @ v, m16.abs() @ v.abs(), n, t)
    finally:
        h.set_stream(None)
        h.close()


def test_two_handles_on_two_streams():
    """Two handles, each on a stream of its own, work at once and give what
    each gives alone."""
    import torch

    import b2blas

    handles = [b2blas.Handle(0), b2blas.Handle(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    try:
        gen = torch.Generator(device="cuda")
        gen.manual_seed(3)
        jobs = []
        for h, s, n in zip(handles, streams, (1024, 1000)):
            h.set_stream(s.cuda_stream)
            view = lambda v, d=np.uint16, h=h: b2blas.DeviceBuffer.from_ptr(h, v.data_ptr(), v.numel(), d, v)  # noqa: E731
            rows, k, experts = 700, 512, 4
            a = torch.randn(rows, k, generator=gen, device="cuda").half()
            b = torch.randn(experts, k, n, generator=gen, device="cuda").half()
            off = torch.tensor([0, 1, 300, 300, 690], dtype=torch.int32, device="cuda")
            index = torch.randint(-1, experts, (40,), generator=gen, device="cuda").to(torch.int32)
            packed = torch.randint(0, 256, (experts * n, k // 2), generator=gen, device="cuda").to(torch.uint8)
            scales = torch.rand(experts * n, k // 64, generator=gen, device="cuda").half()
            c, w = torch.zeros(rows, n, device="cuda").half(), torch.zeros(experts, k, n, device="cuda")
            y = torch.zeros(40, n, device="cuda").half()

            def step(h=h, view=view, a=a, b=b, off=off, index=index, packed=packed, scales=scales, c=c, w=w, y=y, n=n, rows=rows, k=k, experts=experts):
                h.hgemm_grouped(b2blas.GemmConfig(rows, n, k), experts, view(a), view(b), view(off, np.int32), view(c))
                h.hgemm_grouped_wgrad(b2blas.GemmConfig(k, n, rows), experts, view(a), view(c), view(off, np.int32), view(w, np.float32))
                h.hgemv_w4_grouped(experts, n, k, 64, 1.0, view(packed, np.uint8), view(scales), None, view(a), view(index, np.int32),
                                   0.0, view(y), count=40)

            jobs.append((step, (c, w, y)))
        torch.cuda.synchronize()
        alone = []
        for h, (step, out) in zip(handles, jobs):
            step()
            h.synchronize()
            alone.append([v.clone() for v in out])
        torch.cuda.synchronize()
        for _ in range(5):
            for _, out in jobs:
                for v in out:
                    v.zero_()
            torch.cuda.synchronize()
            for _ in range(3):
                for step, _ in jobs:
                    step()
            for h in handles:
                h.synchronize()
            for (_, out), want in zip(jobs, alone):
                assert all(torch.equal(v, u) for v, u in zip(out, want))
    finally:
        for h in handles:
            h.set_stream(None)
            h.close()
