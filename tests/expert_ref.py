"""Plain 64-bit forms of the grouped and 4-bit-weight operators, and the
16-bit conversions their tests use (numpy and torch on the CPU)."""
import numpy as np
import torch

HALF = {"f16": torch.float16, "bf16": torch.bfloat16}
# A rounding to 16 bits is off by at most half a step: eps / 2 of the value,
# or half the least subnormal.
UNIT = {t: torch.finfo(HALF[t]).eps / 2 for t in HALF}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}
U32 = 2.0 ** -24


def bits(v, t):
    """float array -> uint16 bit patterns, rounded to nearest even.  float64
    goes through float32; the tests that compare bits pass values that float32
    holds exactly."""
    return torch.from_numpy(np.ascontiguousarray(v, np.float32)).to(HALF[t]).view(torch.int16).numpy().view(np.uint16)


def value(b, t):
    """uint16 bit patterns -> float64."""
    return torch.from_numpy(np.ascontiguousarray(b).view(np.int16)).view(HALF[t]).double().numpy()


def offsets_of(counts, first=0):
    return np.concatenate([[first], first + np.cumsum(counts)]).astype(np.int32)


def grouped(a, b, off, c, alpha=1.0, beta=0.0, trans_b=False):
    """C[r] = alpha A[r] op(B_g) + beta C[r]; other rows of c are returned as they are."""
    out = c.copy()
    for g in range(len(off) - 1):
        r = slice(off[g], off[g + 1])
        v = alpha * (a[r] @ (b[g].T if trans_b else b[g]))
        out[r] = v if beta == 0 else v + beta * c[r]
    return out


def wgrad(a, b, off, c, alpha=1.0, beta=0.0):
    out = np.empty_like(c)
    for g in range(len(off) - 1):
        r = slice(off[g], off[g + 1])
        v = alpha * (a[r].T @ b[r])
        out[g] = v if beta == 0 else v + beta * c[g]
    return out


def quantize(w, group, with_zeros, t):
    """float64 matrix of 16-bit values -> (packed, scales as bits, zeros or None)."""
    m, n = w.shape
    gs = -(-n // group)
    q = np.zeros((m, n + n % 2), np.uint8)
    scales, zeros = np.zeros((m, gs), np.uint16), np.zeros((m, gs), np.uint8)
    for i in range(m):
        for j in range(gs):
            v = w[i, j * group:(j + 1) * group]
            lo, hi = min(v.min(), 0.0), max(v.max(), 0.0)
            s = (hi - lo) / 15 if with_zeros else max(hi, -lo) / 7
            s16 = bits(np.array([s if np.isfinite(v).all() else np.nan], np.float32), t)
            s = value(s16, t)[0]
            z = (min(np.rint(-lo / s), 15) if s > 0 else 0) if with_zeros else 8
            scales[i, j], zeros[i, j] = s16[0], z
            q[i, j * group:j * group + len(v)] = np.clip(np.rint(v / s) + z, 0, 15) if s > 0 else z
    return q[:, 0::2] | q[:, 1::2] << 4, scales, zeros if with_zeros else None


def w4_values(packed, scales, zeros, n, group, t):
    """float64 values of packed rows."""
    q = np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)[:, :n].astype(np.float64)
    col = np.arange(n) // group
    z = 8.0 if zeros is None else (zeros & 15).astype(np.float64)[:, col]
    return (q - z) * value(scales, t)[:, col]
