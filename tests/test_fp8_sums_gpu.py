"""How the 8-bit products are summed, on operands chosen for it: a group of eight products whose large ones cancel, blocks at the lower end of
the scales.  fp32 results: fp32 products and sums.  bf16 results and the gated product: the 8-bit matrix pipe, which drops what lies
2^-13 below the largest of eight consecutive products."""
import numpy as np
import pytest
import torch

from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _ops():
    from flash_diffusion_amd import ops
    return ops


def _np(t):
    return t.detach().double().cpu().numpy()


def _cancelling(M, K, seed):
    """rows whose groups of eight hold +L and -L at random places and values of up to L 2^-6 beside them; e4m3 values, scale 1"""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, K // 8, 8, generator=g)).clamp(-3.5, 3.5)
    L = 2.0 ** torch.randint(5, 9, (M, K // 8, 1), generator=g)
    place = torch.rand(M, K // 8, 8, generator=g).argsort(-1)
    x = torch.where(place == 0, L, torch.where(place == 1, -L, x)).reshape(M, K)
    x[:, ::128] = 448.0
    return x.to(torch.float8_e4m3fn).float()


# a fused product, a streamed one, tiles
@pytest.mark.parametrize("M", [1, 40, 400])
@pytest.mark.parametrize("N,K", [(64, 128), (300, 640), (512, 4096)])
def test_large_products_that_cancel(M, N, K):
    ops = _ops()
    x = _cancelling(M, K, M + K)
    w = torch.ones(N, K)
    w[:, 5::16] = torch.randint(1, 8, (N, len(range(5, K, 16))), generator=torch.Generator().manual_seed(N)).float()
    W = ops.pack_weight_fp8(w.cuda())
    xv, wv = _np(x), _np(w)                        # (their own codes)
    assert np.array_equal(R.quantise(xv)[0], xv) and np.array_equal(_np(W.values()), wv)
    ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    exact = R.sum_bound(K + 4) * mag
    f32 = _np(ops.gemm_fp8(x.cuda(), W, out_f32=True))
    assert (np.abs(f32 - ref) <= exact + 2.0 ** -24 * (np.abs(ref) + exact)).all()
    e = exact + R.pipe_bound(xv, wv)
    got = _np(ops.gemm_fp8(x.cuda(), W))
    assert (np.abs(got - ref) <= e + 2.0 ** -8 * (np.abs(ref) + e)).all()


@pytest.mark.parametrize("M", [1, 40, 400])
def test_what_the_8_bit_pipe_keeps_of_a_group(M):
    """448 - 448 + s: s from 448's 2^-13 on is kept whole by both, a smaller one by the fp32 result"""
    ops = _ops()
    w = torch.ones(40, 256)
    W = ops.pack_weight_fp8(w.cuda())
    for e in range(-9, 9):
        x = torch.zeros(M, 256)
        x[:, 9], x[:, 12], x[:, 15] = 448.0, 2.0 ** e, -448.0        # one group
        assert bool((ops.gemm_fp8(x.cuda(), W, out_f32=True) == 2.0 ** e).all())
        got = ops.gemm_fp8(x.cuda(), W).float()
        assert bool(((got - 2.0 ** e).abs() <= 2.0 ** -10 * 448.0).all())
        if e >= 8 - 13 + 1:
            assert bool((got == 2.0 ** e).all())
        x[:, 12], x[:, 100] = 0.0, 2.0 ** e                          # two groups: fp32 sums between them
        assert bool((ops.gemm_fp8(x.cuda(), W).float() == 2.0 ** e).all())


@pytest.mark.parametrize("M", [3, 60, 300])
@pytest.mark.parametrize("small,large", [(1e-35, 1e3), (1e-36, 1.0), (1e-37, 1e30), (1e-38, 1e20), (1e-40, 1e30), (1e-42, 1e30)])
def test_fp32_results_of_the_smallest_scales(M, small, large):
    """an fp32 result widens the codes to bf16 with their scale: exactly from 2^-124 on, below that to multiples of 2^-133, the step of bf16's
    subnormal numbers (half of it: 2^-134)"""
    ops = _ops()
    N, K = 200, 640
    g = torch.Generator().manual_seed(M)
    a, b = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    for xs, ws in ((small, large), (large, small)):
        x, w = (a.double() * xs).float(), (b.double() * ws).float()
        q, W = ops.quant_fp8(x.cuda()), ops.pack_weight_fp8(w.cuda())
        xv, xe = R.quantise(_np(x))
        wv, we = R.quantise(_np(w), 128)
        ref, mag = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
        lost = lambda v, e, rows: 2.0 ** -134 * (np.repeat(np.repeat(e, 128, 1)[:, :K], rows, 0)[:v.shape[0]] < -124)
        dx, dw = lost(xv, xe, 1), lost(wv, we, 128)
        e = R.sum_bound(K + 4) * mag + dx @ np.abs(wv).T + np.abs(xv) @ dw.T + K * 2.0 ** -149
        got = _np(ops.gemm_fp8(q, W, out_f32=True))
        assert (np.abs(got - ref) <= e + 2.0 ** -24 * (np.abs(ref) + e)).all(), float((np.abs(got - ref) / mag).max())
        pipe = R.sum_bound(K + 4) * mag + R.pipe_bound(xv, wv) + 2.0 ** -133          # (the 8-bit pipe takes every scale as it is)
        assert (np.abs(_np(ops.gemm_fp8(q, W)) - ref) <= pipe + 2.0 ** -8 * (np.abs(ref) + pipe)).all()


@pytest.mark.parametrize("M", [1, 130])
def test_the_gated_product_of_large_products_that_cancel(M):
    ops = _ops()
    K, N = 640, 256
    x = _cancelling(M, K, 3) / 64.0
    w0, w1 = torch.ones(N, K) / 16.0, torch.ones(N, K) / 16.0
    w0[:, 5::16] = torch.randint(1, 8, (N, K // 16), generator=torch.Generator().manual_seed(1)) / 16.0
    w1[:, 3::16] = torch.randint(1, 8, (N, K // 16), generator=torch.Generator().manual_seed(2)) / 16.0
    xv, v0, v1 = _np(x), _np(w0), _np(w1)
    a, b = xv @ v0.T, xv @ v1.T
    ref = R.gelu_tanh(a) * b
    # (the errors as for any gated product: both products', the slope of the GELU (1.13) and its fast form (2e-6), half a step of the codes)
    ea = R.sum_bound(K) * (np.abs(xv) @ np.abs(v0).T) + R.pipe_bound(xv, v0)
    eb = R.sum_bound(K) * (np.abs(xv) @ np.abs(v1).T) + R.pipe_bound(xv, v1)
    e = 1.2 * ea * (np.abs(b) + eb) + (np.abs(R.gelu_tanh(a)) + 2e-6) * eb + 2e-6 * (1 + np.abs(a)) * np.abs(b)
    h = ops.gated_fp8(x.cuda(), ops.pack_weight_fp8(w0.cuda()), ops.pack_weight_fp8(w1.cuda()))
    full = np.repeat(2.0 ** (h.parts()[1].view(torch.uint8).cpu().numpy().astype(np.float64) - 127), 128, 1)[:, :N]
    tol = np.maximum(2.0 ** -4 * (np.abs(ref) + e), 2.0 ** -10 * full) + e
    assert (np.abs(_np(h.values()) - ref) <= tol).all()
