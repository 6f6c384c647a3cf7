"""The cases on which the products of an expert layer are measured.

Five operators, all on row-major operands in binary16 or bfloat16:

  grouped   C[r] = A[r] B_g for the rows r of group g, rows sorted by group; B_g is k x n, or
            n x k where "trans" is true (the gradient with respect to A)
  wgrad     C_g = A[rows of g]^T B[rows of g], in the operands' type or in float32
  w4        a matrix to 4-bit values with one scale (and zero point) per group of columns, and back
  gemv4     y_i = W x_i for 4-bit W and one or a few vectors
  gemv4g    y_i = W_e(i) x_{i / fan}: each product with the 4-bit weights of the expert that its
            index names; -1 names none and gives zeros

`own` chooses between the plain form in torch and the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

HALF = {"f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"

# ------------------------------------------------------------------ cases


def listed():
    return [
        # an expert layer's first product in training or prefill: long skewed groups
        dict(name="grouped_16384x4096x4096_g8", op="grouped", type="f16", groups=8, active=8, rows=16384, pad=0, n=4096, k=4096, trans=False),
        # the same layer's gradient of the activations: many ragged groups, some empty, a padded batch
        dict(name="grouped_t_8192x2048x1024_g64", op="grouped", type="bf16", groups=64, active=59, rows=8192, pad=77, n=2048, k=1024, trans=True),
        # one decoding step of a small batch: two or three rows for each active expert
        dict(name="grouped_32x4096x2048_g16", op="grouped", type="bf16", groups=16, active=12, rows=32, pad=0, n=4096, k=2048, trans=False),
        # odd sizes: rows of A, B and C start at every 2-byte boundary
        dict(name="grouped_1000x515x1001_g5", op="grouped", type="f16", groups=5, active=4, rows=1000, pad=3, n=515, k=1001, trans=False),
        # the gradient of the weights, kept in float32 for the optimizer
        dict(name="wgrad_16384_2048x4096_g8", op="wgrad", type="bf16", out="f32", groups=8, active=8, rows=16384, pad=0, m=2048, n=4096),
        # many small experts, a few of which got no token
        dict(name="wgrad_4096_1024x1024_g32", op="wgrad", type="f16", out="half", groups=32, active=29, rows=4096, pad=50, m=1024, n=1024),
        # weights made 4-bit once at load, and made 16-bit again for a long prompt
        dict(name="w4_4096x4096_g128", op="w4", type="f16", m=4096, n=4096, group=128, zeros=False),
        # a short last group and rows that end inside a byte, with zero points
        dict(name="w4_1000x2049_g64", op="w4", type="bf16", m=1000, n=2049, group=64, zeros=True),
        # one token through a large projection
        dict(name="gemv4_16384x16384_g128_1", op="gemv4", type="f16", m=16384, n=16384, group=128, zeros=False, count=1),
        # eight sequences decoded together, small groups with zero points
        dict(name="gemv4_4096x4096_g32_8", op="gemv4", type="bf16", m=4096, n=4096, group=32, zeros=True, count=8),
        # one token through the two experts that a router gave it: latency
        dict(name="gemv4g_1024x512_e8_2", op="gemv4g", type="f16", groups=8, m=1024, n=512, group=64, zeros=False, count=2, fan=2, drop=False),
        # sixteen tokens, two experts each, some pairs dropped
        dict(name="gemv4g_4096x2048_e32_32", op="gemv4g", type="bf16", groups=32, m=4096, n=2048, group=128, zeros=True, count=32, fan=2, drop=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]: whole multiples of 64 or 8, or any number."""
    v = _log(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return min(hi, max(lo, v // step * step))


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(("grouped", "grouped", "wgrad", "w4", "gemv4", "gemv4g"))
        half = rng.choice(("f16", "bf16"))
        if op in ("grouped", "wgrad"):
            groups = _log(rng, 1, 64)
            rows = _log(rng, 1, 16384)
            active = max(1, min(rows, groups - rng.choice((0, 0, groups // 4))))
            case = dict(op=op, type=half, groups=groups, active=active, rows=rows, pad=rng.choice((0, 0, 5, 130)))
            if op == "grouped":
                case.update(n=_size(rng, 16, 4096), k=_size(rng, 16, 4096), trans=rng.random() < 0.5)
            else:
                case.update(m=_size(rng, 16, 4096), n=_size(rng, 16, 4096), out=rng.choice(("half", "f32")))
                if groups * case["m"] * case["n"] > 2 ** 28:
                    continue
        else:
            case = dict(op=op, type=half, group=rng.choice((32, 64, 128, 256)), zeros=rng.random() < 0.5)
            if op == "gemv4g":
                fan = rng.choice((1, 2, 4))
                case.update(groups=_log(rng, 2, 64), m=_size(rng, 16, 4096), n=_size(rng, 16, 4096), count=fan * _log(rng, 1, 32), fan=fan,
                            drop=rng.random() < 0.3)
                if case["count"] * case["m"] * case["n"] > 2 ** 30 or case["groups"] * case["m"] * case["n"] > 2 ** 29:
                    continue
            else:
                case.update(m=_size(rng, 16, 16384), n=_size(rng, 16, 16384))
                if op == "gemv4":
                    case["count"] = rng.choice((1, 1, 2, 3, 4, 8, 11, 16))
                elif case["m"] * case["n"] > 2 ** 26:
                    continue
        if work(case)["flops"] <= most:
            return case


# ------------------------------------------------------------------ inputs


def _counts(case, seed):
    """Rows of each group: `active` of them get at least one, the rest of the rows fall unevenly."""
    r = np.random.RandomState(seed % (2 ** 31))
    share = np.zeros(case["groups"])
    chosen = r.permutation(case["groups"])[:case["active"]]
    share[chosen] = r.gamma(3.0, 1.0, case["active"])
    counts = r.multinomial(case["rows"] - case["active"], share / share.sum())
    counts[chosen] += 1
    return counts


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _quantise(w, group, with_zeros):
    """4-bit values (uint8, 0..15), scales in w's type and zero points (uint8) of each row's groups of columns."""
    m, n = w.shape
    gs = -(-n // group)
    v = torch.zeros(m, gs * group, dtype=torch.float32, device=w.device)
    v[:, :n] = w.float()
    v = v.view(m, gs, group)
    if with_zeros:
        lo, hi = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
        scale = ((hi * 0.5 - lo * 0.5) / 7.5).to(w.dtype)
        s = scale.double()
        zero = torch.where(s > 0, (-lo.double() / s).round().clamp(0, 15), torch.zeros_like(s))
    else:
        scale = (v.abs().amax(2) / 7).to(w.dtype)
        s = scale.double()
        zero = torch.full_like(s, 8)
    q = torch.where(s[:, :, None] > 0, (v.double() / s[:, :, None]).round() + zero[:, :, None], zero[:, :, None])
    return q.clamp(0, 15).to(torch.uint8).view(m, -1)[:, :n], scale, zero.to(torch.uint8)


def _pack(q):
    """Two values to a byte, the even column in the low four bits; a row of odd length ends with four zero bits."""
    q = torch.nn.functional.pad(q, (0, q.shape[1] % 2))
    return q[:, 0::2] | (q[:, 1::2] << 4)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    t = HALF[case["type"]]
    s = dict(case=case)
    if case["op"] in ("grouped", "wgrad"):
        counts = _counts(case, seed)
        total = case["rows"] + case["pad"]
        s["most"] = int(counts.max())
        s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEV)
        if case["op"] == "grouped":
            k, n = case["k"], case["n"]
            s["a"] = _normal(gen, (total, k), t)
            s["b"] = _normal(gen, (case["groups"], n, k) if case["trans"] else (case["groups"], k, n), t, k ** -0.5)
            s["c"] = torch.zeros(total, n, dtype=t, device=DEV)
        else:
            s["a"] = _normal(gen, (total, case["m"]), t)
            s["b"] = _normal(gen, (total, case["n"]), t, 0.05)
            s["c"] = torch.zeros(case["groups"], case["m"], case["n"], dtype=torch.float32 if case["out"] == "f32" else t, device=DEV)
        return s
    m, n, group = case["m"], case["n"], case["group"]
    gs = -(-n // group)
    if case["op"] == "w4":
        s["w"] = _normal(gen, (m, n), t, n ** -0.5)
        s["packed"] = torch.zeros(m, -(-n // 2), dtype=torch.uint8, device=DEV)
        s["scales"] = torch.zeros(m, gs, dtype=t, device=DEV)
        s["zeros"] = torch.zeros(m, gs, dtype=torch.uint8, device=DEV) if case["zeros"] else None
        s["back"] = torch.zeros(m, n, dtype=t, device=DEV)
        return s
    experts = case.get("groups", 1)
    q, s["scales"], zero = _quantise(_normal(gen, (experts * m, n), t, n ** -0.5), group, case["zeros"])
    s["packed"], s["zeros"] = _pack(q), zero if case["zeros"] else None
    fan = case.get("fan", 1)
    s["x"] = _normal(gen, (case["count"] // fan, n), t)
    s["y"] = torch.zeros(case["count"], m, dtype=t, device=DEV)
    if case["op"] == "gemv4g":
        # a router gives a token `fan` experts; distinct ones where there are enough
        r = np.random.RandomState(seed % (2 ** 31))
        index = np.concatenate([r.choice(experts, fan, replace=fan > experts) for _ in range(case["count"] // fan)])
        if case["drop"]:
            index[r.random_sample(case["count"]) < 0.1] = -1
        s["index"] = torch.tensor(index, dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms


def _groups_of(s):
    """Row numbers [groups, most] of each group, and which of them the group has."""
    at = torch.arange(s["most"], device=DEV)
    first, last = s["offsets"][:-1, None].long(), s["offsets"][1:, None].long()
    has = first + at < last
    return torch.where(has, first + at, torch.zeros_like(first + at)), has


def _plain_grouped(s):
    rows, has = _groups_of(s)
    b = s["b"].float()
    product = torch.matmul(s["a"].float()[rows], b.transpose(1, 2) if s["case"]["trans"] else b)
    s["c"][rows[has]] = product[has].to(s["c"].dtype)
    return s["c"]


def _plain_wgrad(s):
    rows, has = _groups_of(s)
    a = torch.where(has[:, :, None], s["a"].float()[rows], torch.zeros((), device=DEV))
    b = torch.where(has[:, :, None], s["b"].float()[rows], torch.zeros((), device=DEV))
    return torch.matmul(a.transpose(1, 2), b).to(s["c"].dtype)


def _plain_values(packed, scales, zeros, n, group):
    """The float32 values of 4-bit rows [..., n]."""
    q = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)[..., :n].float()
    col = torch.arange(n, device=DEV) // group
    zero = 8.0 if zeros is None else zeros.float()[..., col]
    return (q - zero) * scales.float()[..., col]


def _plain_w4(s):
    case = s["case"]
    q, scales, zeros = _quantise(s["w"], case["group"], case["zeros"])
    s["packed"].copy_(_pack(q))
    top = torch.finfo(s["w"].dtype).max
    back = _plain_values(s["packed"], scales, zeros if case["zeros"] else None, case["n"], case["group"]).clamp(-top, top).to(s["w"].dtype)
    return [back, scales] + ([zeros] if case["zeros"] else [])


def _plain_gemv4(s):
    case = s["case"]
    w = _plain_values(s["packed"], s["scales"], s["zeros"], case["n"], case["group"])
    return torch.matmul(s["x"].float(), w.t()).to(s["x"].dtype)


def _plain_gemv4g(s):
    case = s["case"]
    at = s["index"].long().clamp(min=0)
    m = case["m"]
    of = lambda v: None if v is None else v.view(case["groups"], m, -1)[at]  # noqa: E731
    w = _plain_values(of(s["packed"]), of(s["scales"]), of(s["zeros"]), case["n"], case["group"])
    x = s["x"].float().repeat_interleave(case["fan"], 0)
    y = torch.matmul(w, x[:, :, None])[:, :, 0]
    return torch.where(s["index"][:, None] >= 0, y, torch.zeros((), device=DEV)).to(s["x"].dtype)


# ------------------------------------------------------------------ the framework's calls

_kept = {}


def _handle():
    """The program's handle of the current device, on the current stream."""
    if "m" not in _kept:
        import os
        import sys
        sys.path.insert(1, os.path.join(os.getcwd(), "cublas-rs_b200"))
        import b2blas
        _kept["m"] = b2blas
    device = torch.cuda.current_device()
    stream = torch._C._cuda_getCurrentRawStream(device)  # torch.cuda.current_stream() takes 3 us to make its object
    if device not in _kept:
        _kept[device] = [_kept["m"].Handle(device), None]
    kept = _kept[device]
    if kept[1] != stream:
        kept[0].set_stream(stream)
        kept[1] = stream
    return _kept["m"], kept[0]


_KIND = {torch.float16: np.uint16, torch.bfloat16: np.uint16, torch.float32: np.float32, torch.int32: np.int32, torch.uint8: np.uint8}


def _own(s):
    b2, h = _handle()
    case = s["case"]
    half = b2.Half.F16 if case["type"] == "f16" else b2.Half.BF16
    buf = lambda t: None if t is None else b2.DeviceBuffer.from_ptr(h, t.data_ptr(), t.numel(), _KIND[t.dtype], t)  # noqa: E731
    if case["op"] == "grouped":
        h.hgemm_grouped(b2.GemmConfig(s["a"].shape[0], case["n"], case["k"]), case["groups"], buf(s["a"]), buf(s["b"]), buf(s["offsets"]), buf(s["c"]),
                        trans_b=case["trans"], half=half)
        return s["c"]
    if case["op"] == "wgrad":
        h.hgemm_grouped_wgrad(b2.GemmConfig(case["m"], case["n"], s["a"].shape[0]), case["groups"], buf(s["a"]), buf(s["b"]), buf(s["offsets"]), buf(s["c"]),
                              half=half)
        return s["c"]
    m, n, group = case["m"], case["n"], case["group"]
    if case["op"] == "w4":
        packed, scales, zeros = buf(s["packed"]), buf(s["scales"]), buf(s["zeros"])
        h.quantize_w4(m, n, group, buf(s["w"]), packed, scales, zeros, half=half)
        h.dequantize_w4(m, n, group, packed, scales, zeros, buf(s["back"]), half=half)
        return [s["back"], s["scales"]] + ([s["zeros"]] if case["zeros"] else [])
    if case["op"] == "gemv4":
        h.hgemv_w4(m, n, group, 1.0, buf(s["packed"]), buf(s["scales"]), buf(s["zeros"]), buf(s["x"]), 0.0, buf(s["y"]), count=case["count"], half=half)
        return s["y"]
    h.hgemv_w4_grouped(case["groups"], m, n, group, 1.0, buf(s["packed"]), buf(s["scales"]), buf(s["zeros"]), buf(s["x"]), buf(s["index"]), 0.0, buf(s["y"]),
                       count=case["count"], fan=case["fan"], half=half)
    return s["y"]


def run(state):
    if own:
        return _own(state)
    return {"grouped": _plain_grouped, "wgrad": _plain_wgrad, "w4": _plain_w4, "gemv4": _plain_gemv4, "gemv4g": _plain_gemv4g}[state["case"]["op"]](state)


# ------------------------------------------------------------------ work and exact values


def work(case):
    op = case["op"]
    if op == "grouped":
        r, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": 2 * (r * k + case["active"] * k * n + r * n), "flops": 2 * r * n * k}
    if op == "wgrad":
        r, m, n = case["rows"], case["m"], case["n"]
        return {"bytes": 2 * r * (m + n) + case["groups"] * m * n * (4 if case["out"] == "f32" else 2), "flops": 2 * r * m * n}
    m, n = case["m"], case["n"]
    gs = -(-n // case["group"])
    held = m * (-(-n // 2)) + m * gs * (3 if case["zeros"] else 2)  # packed values, scales, zero points
    if op == "w4":
        return {"bytes": 2 * m * n + 2 * held + 2 * m * n, "flops": 4 * m * n}
    count = case["count"]
    # products that name one expert share its weights: the expected number of experts named
    e = case.get("groups", 1)
    fan = min(case.get("fan", 1), e)
    experts = e * (1 - (1 - fan / e) ** (count // case.get("fan", 1)))
    return {"bytes": int(experts * held) + 2 * (count // case.get("fan", 1)) * n + 2 * count * m, "flops": 2 * count * m * n}


def exact(case, seed):
    """The definition in float64, one group, matrix or product at a time."""
    s = prepare(case, seed)
    if case["op"] == "grouped":
        c = torch.zeros(s["c"].shape, dtype=torch.float64, device=DEV)
        bounds = s["offsets"].tolist()
        for g in range(case["groups"]):
            if bounds[g] < bounds[g + 1]:
                b = s["b"][g].double()
                c[bounds[g]:bounds[g + 1]] = s["a"][bounds[g]:bounds[g + 1]].double() @ (b.t() if case["trans"] else b)
        return c
    if case["op"] == "wgrad":
        c = torch.zeros(s["c"].shape, dtype=torch.float64, device=DEV)
        bounds = s["offsets"].tolist()
        for g in range(case["groups"]):
            rows = slice(bounds[g], bounds[g + 1])
            c[g] = s["a"][rows].double().t() @ s["b"][rows].double()
        return c
    m, n, group = case["m"], case["n"], case["group"]
    if case["op"] == "w4":
        w = s["w"].double()
        back = torch.zeros_like(w)
        scales, zeros = [], []
        for c0 in range(0, n, group):
            v = w[:, c0:c0 + group]
            if case["zeros"]:
                lo, hi = torch.minimum(v.min(1).values, v.new_zeros(())), torch.maximum(v.max(1).values, v.new_zeros(()))
                d = ((hi - lo) / 15).to(s["w"].dtype).double()
                z = torch.round(-lo / d).clamp(0, 15)
                q = (torch.round(v / d[:, None]) + z[:, None]).clamp(0, 15) - z[:, None]
                zeros.append(z)
            else:
                d = (v.abs().max(1).values / 7).to(s["w"].dtype).double()
                q = torch.round(v / d[:, None]).clamp(-8, 7)
            back[:, c0:c0 + group] = q * d[:, None]
            scales.append(d)
        return [back, torch.stack(scales, 1)] + ([torch.stack(zeros, 1).to(torch.uint8)] if case["zeros"] else [])
    low = (s["packed"] & 15).double()
    high = torch.div(s["packed"], 16, rounding_mode="floor").double()

    def matrix(e):
        q = torch.zeros(m, low.shape[1] * 2, dtype=torch.float64, device=DEV)
        rows = slice(e * m, (e + 1) * m)
        q[:, 0::2], q[:, 1::2] = low[rows], high[rows]
        q = q[:, :n].clone()
        for j in range(0, -(-n // group)):
            part = q[:, j * group:(j + 1) * group]
            part -= 8 if s["zeros"] is None else s["zeros"][rows, j:j + 1].double()
            part *= s["scales"][rows, j:j + 1].double()
        return q

    y = torch.zeros(s["y"].shape, dtype=torch.float64, device=DEV)
    if case["op"] == "gemv4":
        return s["x"].double() @ matrix(0).t()
    for i, e in enumerate(s["index"].tolist()):
        if e >= 0:
            y[i] = matrix(e) @ s["x"][i // case["fan"]].double()
    return y
