"""The stages of one block of the 8-bit T5 encoder, each against the 64-bit form of that stage on the stage's OWN recorded input, under bounds
of its own rounding (nothing compounds).  A record is a dict of float64 arrays: h_in, n1, q, k, v, o, h1, n2, f, h_out; codes (n1, n2 and the
gated f) are pairs (values, scale exponents)."""
import numpy as np

from tests import fp8_ref as R

HALF = R.half_step("bf16")


def norm(h, w, eps):
    return h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w


def _codes_excess(got, ref, e):
    """how far codes lie outside what `ref`, known to within `e`, may become: a scale that fits an amax within it, half a step of e4m3 (2^-4
    relative, 2^-10 scales below its normal range)"""
    values, exps = got
    M, K = ref.shape
    kb = -(-K // 128)
    blocks = lambda t: np.pad(t, ((0, 0), (0, kb * 128 - K))).reshape(M, kb, 128).max(2)
    sc = 2.0 ** exps.astype(np.float64)
    least, most = blocks(np.maximum(np.abs(ref) - e, 0.0)), blocks(np.abs(ref) + e)
    if (least > 448.0 * sc).any() or ((most <= 224.0 * sc) & (exps > -127)).any():
        return np.inf
    full = np.repeat(sc, 128, 1)[:, :K]
    t = values / full                                                # e4m3 numbers: multiples of 2^(p - 3) in [2^p, 2^(p + 1)), p >= -6
    if (np.abs(t) > 448.0).any() or np.mod(t / 2.0 ** (np.frexp(np.maximum(np.abs(t), 2.0 ** -6))[1] - 4.0), 1.0).any():
        return np.inf
    return float((np.abs(values - ref) - np.maximum(2.0 ** -4 * (np.abs(ref) + e), 2.0 ** -10 * full) - e).max())


def _product_excess(got, x, w, add=0.0, relu=False):
    """of a bf16 result x w^T + add: fp32 sums, the 8-bit pipe's groups, one rounding"""
    ref = x @ w.T
    e = R.sum_bound(x.shape[1] + 4) * (np.abs(x) @ np.abs(w).T + np.abs(add)) + R.pipe_bound(x, w)
    ref = ref + add
    if relu:
        ref = np.maximum(ref, 0.0)
    return float((np.abs(got - ref) - e - HALF * (np.abs(ref) + e)).max())


def attention(q, k, v, bias, kb, shape):
    """shape (B, S, H, d): softmax(q k^T + bias + kb) v, its weighted sum of |v|, and the largest error that fp32 scores may have"""
    B, S, H, d = shape
    t = lambda m: m.reshape(B, S, H, d).transpose(0, 2, 1, 3)
    q, k, v = t(q), t(k), t(v)
    s = q @ k.transpose(0, 1, 3, 2) + bias[None]
    off = (d + 8) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).transpose(0, 1, 3, 2) + np.abs(bias)[None]).max(-1, keepdims=True)
    s = s + kb[:, None, None, :]
    p = np.exp(s - s.max(-1, keepdims=True))
    p = p / p.sum(-1, keepdims=True)
    back = lambda m: m.transpose(0, 2, 1, 3).reshape(B * S, H * d)
    return back(p @ v), back(p @ np.abs(v)), back(np.broadcast_to(off, (B, H, S, d)))


def excess(rec, w, cfg, bias, kb, shape):
    """stage -> how far it lies outside its bounds (right: at most 0).  w: the block's parameters, float64; cfg: eps, gated"""
    w8 = {m: R.quantise(w[m], 128)[0] for m in w if w[m].ndim == 2}
    eps, out = cfg["eps"], {}

    def norm_excess(codes, h, g):
        ref = norm(h, g, eps)
        return _codes_excess(codes, ref, (h.shape[1] + 8) * 2.0 ** -24 * np.abs(ref))   # K squares added, root, quotient, two products

    out["n1"] = norm_excess(rec["n1"], rec["h_in"], w["norm1"])
    for m in "qkv":
        out[m] = _product_excess(rec[m], rec["n1"][0], w8[m])
    o, mag, off = attention(rec["q"], rec["k"], rec["v"], bias, kb, shape)
    # weights off by twice the scores' error, exp and quotient by 2^-18, S additions
    e = (2.0 * off + 2.0 ** -18 + (shape[1] + 8) * 2.0 ** -24) * mag
    out["o"] = float((np.abs(rec["o"] - o) - e - HALF * (np.abs(o) + e)).max())
    out["h1"] = _product_excess(rec["h1"], R.quantise(rec["o"])[0], w8["o"], rec["h_in"])
    out["n2"] = norm_excess(rec["n2"], rec["h1"], w["norm2"])
    n2 = rec["n2"][0]
    if cfg["gated"]:
        a, b = n2 @ w8["wi_0"].T, n2 @ w8["wi_1"].T
        ea, eb = (R.sum_bound(n2.shape[1]) * (np.abs(n2) @ np.abs(w8[m]).T) + R.pipe_bound(n2, w8[m]) for m in ("wi_0", "wi_1"))
        g = R.gelu_tanh(a)
        # (the slope of the GELU, 1.13, and its fast form, 2e-6)
        out["f"] = _codes_excess(rec["f"], g * b, 1.2 * ea * (np.abs(b) + eb) + (np.abs(g) + 2e-6) * eb + 2e-6 * (1 + np.abs(a)) * np.abs(b))
        f = rec["f"][0]
    else:
        out["f"] = _product_excess(rec["f"], n2, w8["wi"], relu=True)
        f = R.quantise(rec["f"])[0]
    out["h_out"] = _product_excess(rec["h_out"], f, w8["wo"], rec["h1"])
    return out
