"""Plain 64-bit forms of the 8-bit block-scaled format and its products (CPU, float64): what tests/test_fp8_gpu.py and
tests/test_embed_gpu.py compare with."""
import math

import numpy as np


def quantise(v, rows=1):
    """v [M, K] float64 -> (values of the codes [M, K], scale exponents [ceil(M / rows), ceil(K / 128)]): blocks of rows x 128, the smallest
    power of two 2^e >= -127 with amax <= 448 2^e, codes rounded to e4m3 (nearest, ties to even); infinities and NaN become NaN and do
    not enter the scale"""
    v = np.asarray(v, dtype=np.float64)
    M, K = v.shape
    out = np.empty_like(v)
    exps = np.empty((-(-M // rows), -(-K // 128)), dtype=np.int64)
    for i in range(exps.shape[0]):
        for j in range(exps.shape[1]):
            b = v[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128]
            fin = b[np.isfinite(b)]
            amax = float(np.abs(fin).max()) if fin.size else 0.0
            e = -127
            if amax > 0:
                m, x = math.frexp(amax)              # amax = m 2^x, 0.5 <= m < 1;  448 = 0.875 * 2^9
                e = max(-127, x - 9 + (1 if m > 0.875 else 0))
            exps[i, j] = e
            with np.errstate(invalid="ignore"):
                t = np.where(np.isfinite(b), b, np.nan) * 2.0 ** -e
                _, x = np.frexp(np.maximum(np.abs(np.nan_to_num(t)), 2.0 ** -6))   # |t| in [2^(x-1), 2^x): step 2^(x-4)
                step = 2.0 ** (x - 4)
                out[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128] = np.rint(t / step) * step * 2.0 ** e
    return out, exps


def gelu_tanh(a):
    return 0.5 * a * (1.0 + np.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a ** 3)))


ACTS = {0: lambda v: v, 1: lambda v: v / (1.0 + np.exp(-v)), 3: lambda v: np.maximum(v, 0.0),
        4: lambda v: 0.5 * v * (1.0 + np.vectorize(math.erf)(v / math.sqrt(2.0))), 5: gelu_tanh}


def half_step(dtype_name):
    """a rounding is off by at most half a step, eps / 2 relative to the value"""
    return {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}[dtype_name]


def sum_bound(K):
    """relative to the sum of the terms' magnitudes: K fp32 additions in any order, each off by at most one unit in the last place
    (2^-23: the matrix unit may truncate where a rounded addition would be off by half of that)"""
    return K * 2.0 ** -23


def pipe_bound(x, w):
    """what the 8-bit matrix pipe may drop of x w^T: it adds the products of eight consecutive contraction steps aligned to the largest of
    them and drops bits below 2^-13 of its exponent: eight products, each off by less than that unit, so 2^-10 of the group's largest
    product, itself at most the product of the two largest magnitudes"""
    g = lambda t: np.abs(np.pad(t, ((0, 0), (0, -t.shape[1] % 8)))).reshape(t.shape[0], -1, 8).max(2)
    return 2.0 ** -10 * (g(x) @ g(w).T)
