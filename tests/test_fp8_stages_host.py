"""CPU: the stage bounds of tests/fp8_stages.py accept the 64-bit block that rounds where the encoder rounds, and see every planted mistake."""
import numpy as np
import pytest
import torch

from tests import fp8_ref as R
from tests import fp8_stages as S

SHAPE = (2, 24, 4, 16)
D, F = 64, 160


def _bf(v):
    return torch.from_numpy(np.ascontiguousarray(v)).float().to(torch.bfloat16).double().numpy()


def _parts(gated):
    r = np.random.RandomState(3)
    n = SHAPE[2] * SHAPE[3]
    w = {m: r.randn(n, D) * D ** -0.5 for m in "qkv"}
    w.update(o=r.randn(D, n) * n ** -0.5, wo=r.randn(D, F) * F ** -0.5, norm1=1 + 0.2 * r.randn(D), norm2=1 + 0.2 * r.randn(D))
    w.update({m: r.randn(F, D) * D ** -0.5 for m in (("wi_0", "wi_1") if gated else ("wi",))})
    bias = r.randn(SHAPE[2], SHAPE[1], SHAPE[1])
    kb = np.where(np.arange(SHAPE[1])[None] < np.array([[9], [24]]), 0.0, float(torch.finfo(torch.float32).min))
    return w, dict(eps=1e-6, gated=gated), bias, kb, _bf(r.randn(SHAPE[0] * SHAPE[1], D))


def _block(w, cfg, bias, kb, h, plant=None):
    """the block in 64 bits, rounded where the encoder rounds; plant: one thing done differently"""
    eps = 1e-2 if plant == "eps" else cfg["eps"]
    raw = lambda v: (v, R.quantise(v)[1])
    q8 = lambda v, name: raw(v) if plant == f"{name} unquantised" else R.quantise(v)
    w8 = lambda m: w[m] if plant == f"{m} weight unquantised" else R.quantise(w[m], 128)[0]
    r = dict(h_in=h, n1=q8(S.norm(h, w["norm1"], eps), "n1"))
    for m in "qkv":
        r[m] = _bf(r["n1"][0] @ w8(m).T)
    if plant == "q and k exchanged":
        r["q"], r["k"] = r["k"], r["q"]
    o = S.attention(r["q"], r["k"], r["v"], 0 * bias if plant == "no bias" else bias, 0 * kb if plant == "no mask" else kb, SHAPE)[0]
    r["o"] = _bf(o * SHAPE[3] ** -0.5 if plant == "scaled scores" else o)
    r["h1"] = _bf(q8(r["o"], "o")[0] @ w8("o").T + (0 if plant == "no residual" else h))
    r["n2"] = q8(S.norm(h if plant == "second norm of the input" else r["h1"], w["norm2"], eps), "n2")
    n2 = r["n2"][0]
    if cfg["gated"]:
        a, b = n2 @ w8("wi_0").T, n2 @ w8("wi_1").T
        if plant == "gate exchanged":
            a, b = b, a
        r["f"] = q8(R.gelu_tanh(a) * b, "f")
        f = r["f"][0]
    else:
        r["f"] = _bf(np.maximum(n2 @ w8("wi").T, 0.0))
        f = q8(r["f"], "f")[0]
    r["h_out"] = _bf(f @ w8("wo").T + (h if plant == "residual of the input" else r["h1"]))
    return r


BOTH = ["eps", "n1 unquantised", "n2 unquantised", "o unquantised", "f unquantised", "q weight unquantised", "v weight unquantised", "o weight unquantised",
        "wo weight unquantised", "q and k exchanged", "no bias", "no mask", "scaled scores", "no residual", "second norm of the input", "residual of the input"]
PLANTS = [(True, p) for p in BOTH + ["wi_0 weight unquantised", "wi_1 weight unquantised", "gate exchanged"]] + [(False, p) for p in BOTH + ["wi weight unquantised"]]


@pytest.mark.parametrize("gated", [True, False])
def test_the_blocks_own_rounding_is_within_the_bounds(gated):
    w, cfg, bias, kb, h = _parts(gated)
    out = S.excess(_block(w, cfg, bias, kb, h), w, cfg, bias, kb, SHAPE)
    assert all(v <= 0 for v in out.values()), out


@pytest.mark.parametrize("gated,plant", PLANTS)
def test_a_planted_mistake_is_seen(gated, plant):
    w, cfg, bias, kb, h = _parts(gated)
    out = S.excess(_block(w, cfg, bias, kb, h, plant), w, cfg, bias, kb, SHAPE)
    assert max(out.values()) > 0, out
