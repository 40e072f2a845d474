"""The 8-bit block-scaled products (csrc/fp8.hip) against 64-bit plain forms: the quantiser's codes and scales exactly, the products within
the rounding of fp32 sums and of the output type, over sizes that divide by nothing, strides, infinities, empty and single rows."""
import numpy as np
import pytest
import torch

from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAMES = {BF16: "bf16", F32: "f32"}


def _ops():
    from flash_diffusion_amd import ops
    return ops


def _rand(*shape, seed=0, dtype=F32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread != 1.0:
        x = x * torch.exp(spread * torch.randn(shape[-1], generator=g))
    return x.to(dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


def _exps(q, *a):
    """the exponents of an operand's scales"""
    return q.parts(*a)[1].view(torch.uint8).cpu().numpy().astype(np.int64) - 127


def ops_untile(codes, rows, K):
    return _ops()._untile(codes, rows, K).view(torch.uint8)


# ---- the format --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (2, 127), (3, 129), (5, 512), (4, 513), (17, 1155), (64, 4096), (2, 10240)])
def test_quantised_rows_are_the_formats(M, K, dtype):
    x = _rand(M, K, seed=M * K, dtype=dtype, spread=2.0)
    q = _ops().quant_fp8(x.cuda())
    want, exps = R.quantise(_np(x))
    assert np.array_equal(_np(q.values(F32)), want)
    assert np.array_equal(_exps(q), exps)
    pad = -(-K // 128) * 128
    assert not ops_untile(q.codes, M, pad)[:, K:].any()                     # padding: zero codes


def test_quantiser_at_the_borders_of_a_scale_and_of_a_code():
    rows = [[448.0] + [0.0] * 127, [449.0] + [1.0] * 127, [447.0] * 128, [0.0] * 128, [2.0 ** -126] * 128, [1e-40] * 128, [3e38] * 128,
            [float(2 ** k) for k in range(-64, 64)], [17.0, 18.0, 19.0, 20.0, 21.0, 22.0, 23.0, 25.0] * 15 + [448.0] * 8,
            [2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 2.0 ** -11, 0.0, -0.0, -2.0 ** -10] * 15 + [448.0] * 8]
    x = torch.tensor(rows, dtype=torch.float32)
    q = _ops().quant_fp8(x.cuda())
    want, exps = R.quantise(_np(x))
    # (values below 2^-126 are compared through codes and scale bytes: torch's own products of subnormals are not what is tested here)
    codes = _np(q.parts()[0].float())
    assert np.array_equal(codes * 2.0 ** np.repeat(exps, 128, 1).astype(np.float64), want)
    assert np.array_equal(_exps(q), exps)


def test_all_256_codes_are_their_own_rounding_and_midpoints_go_to_even():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    vals = codes[torch.isfinite(codes)].sort().values.unique()
    mids = (vals[1:] + vals[:-1]) / 2
    x = torch.cat([vals, mids])
    x = torch.cat([x, torch.zeros(-x.numel() % 127)]).view(-1, 127)
    x = torch.cat([x, torch.full((x.shape[0], 1), 448.0)], 1)               # (448 in every block: scale 2^0)
    q = _ops().quant_fp8(x.cuda())
    want, exps = R.quantise(_np(x))
    assert not exps.any() and np.array_equal(_np(q.values(F32)), want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinities_and_nan_become_nan_and_leave_the_scale_alone(dtype):
    """(the product of three rows quantises them inside, that of forty does not)"""
    x = _rand(3, 256, dtype=dtype)
    x[0, 5], x[0, 6], x[1, 200] = float("inf"), float("nan"), float("-inf")
    x[2, :128] = float("nan")
    q = _ops().quant_fp8(x.cuda())
    want, _ = R.quantise(_np(x))
    got = _np(q.values(F32))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    w = _ops().pack_weight_fp8(_rand(70, 256, seed=3).cuda())
    for rep in (1, 14):
        y = _ops().gemm_fp8(x.cuda().repeat(rep, 1), w, out_f32=True)
        assert bool(torch.isnan(y).all())                                   # every row holds one
    x[1] = 1.0                                                              # ... and one that holds none is not touched
    y = _ops().gemm_fp8(x.cuda(), w, out_f32=True)
    assert bool(torch.isfinite(y[1]).all()) and bool(torch.isnan(y[0]).all())


@pytest.mark.parametrize("M,K", [(1, 8), (2, 64), (3, 1000), (5, 4096), (2, 8200), (33, 1155)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_then_quantise(M, K, dtype):
    x, w, eps = _rand(M, K, seed=K, dtype=dtype, spread=0.5), 1.0 + 0.2 * _rand(K, seed=1), 1e-6
    q = _ops().rmsnorm_fp8(x.cuda(), w.cuda(), eps)
    v = _np(x)
    ref = v / np.sqrt((v * v).mean(1, keepdims=True) + eps) * _np(w)
    _near_codes(q, ref, (K + 8) * 2.0 ** -24)       # K fp32 additions of squares, square root, quotient and two products


def _near_codes(q, ref, rel):
    """the quantised rows hold `ref` computed with a relative error up to `rel`: scales as the format says for an amax within it, codes off
    by at most half a step of e4m3 (2^-4 relative, 2^-10 scales below the normal range) and that error"""
    M, K = ref.shape
    kb = -(-K // 128)
    s = _exps(q)
    pad = np.pad(np.abs(ref), ((0, 0), (0, kb * 128 - K))).reshape(M, kb, 128)
    amax = pad.max(2)
    sc = 2.0 ** s.astype(np.float64)
    slack = 1.0 + 2.0 * rel
    assert (amax <= 448.0 * sc * slack).all() and ((amax * slack >= 224.0 * sc) | (s == -127)).all()
    got = _np(q.values(F32))
    full = np.repeat(sc, 128, 1)[:, :K]
    tol = np.maximum(2.0 ** -4 * np.abs(ref), 2.0 ** -10 * full) * (1 + 2 * rel) + 2 * rel * np.abs(ref)
    assert (np.abs(got - ref) <= tol).all(), float((np.abs(got - ref) - tol).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (129, 127), (300, 1155), (640, 257)])
def test_packed_weight_and_its_transpose(N, K, dtype):
    w = _rand(N, K, seed=N + K, dtype=dtype, spread=1.0)
    p = _ops().pack_weight_fp8(w.cuda(), transposed=True)
    want, exps = R.quantise(_np(w), rows=128)
    assert np.array_equal(_np(p.values(F32)), want)
    assert np.array_equal(_exps(p), exps) and np.array_equal(_exps(p, True), exps.T)
    assert torch.equal(p.parts(True)[0].view(torch.uint8), p.parts()[0].view(torch.uint8).t())
    up = lambda n, to: -(-n // to) * to                                  # padding: zero codes
    for c, n, k in ((p.codes, N, K), (p.codes_t, K, N)):
        t = ops_untile(c, up(n, 256), up(k, 128))
        assert not t[:, k:].any() and not t[n:].any()


# ---- products ----------------------------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (16, 100, 4096), (16, 100, 4100), (9, 260, 8192), (1, 50, 65536), (2, 33, 65537), (1, 129, 127), (1, 4096, 4096), (3, 64, 128), (8, 96, 640), (16, 200, 1000), (17, 130, 257), (33, 1000, 640), (65, 1, 512),
         (64, 300, 640), (77, 768, 768), (129, 257, 385), (300, 65, 1152), (255, 513, 130), (700, 520, 200), (1000, 1030, 129)]


def _check(got, ref, xv, wv, dtype, add=0.0, extra=0.0, slope=1.0):
    """ref float64 of xv wv^T (+ terms of magnitude `add`): fp32 sums, what the 8-bit pipe drops where the result is bf16, and one rounding
    to dtype; slope: of what is applied to the sum"""
    e = R.sum_bound(xv.shape[1] + 4) * (np.abs(xv) @ np.abs(wv).T + add) * slope + extra
    if dtype == BF16:
        e = e + slope * R.pipe_bound(xv, wv)
    tol = e + R.half_step(NAMES[dtype]) * (np.abs(ref) + e)
    d = np.abs(_np(got) - ref)
    assert got.dtype == dtype and (d <= tol).all(), (float((d - tol).max()), float(d.max()))


@pytest.mark.parametrize("xt,yt", [(BF16, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, xt, yt):
    ops = _ops()
    x, w = _rand(M, K, seed=1, dtype=xt, spread=1.0), _rand(N, K, seed=2) * K ** -0.5
    b, r = _rand(N, seed=3), _rand(M, N, seed=4, dtype=yt)
    W = ops.pack_weight_fp8(w.cuda())
    xv, wv = R.quantise(_np(x))[0], R.quantise(_np(w), 128)[0]
    ref = xv @ wv.T
    X = x.cuda()
    y = ops.gemm_fp8(X, W, out_f32=yt == F32)
    _check(y, ref, xv, wv, yt)
    if M <= 16:                                                       # quantised inside the product: the same codes
        assert torch.equal(y, ops.gemm_fp8(ops.quant_fp8(X), W, out_f32=yt == F32))
    _check(ops.gemm_fp8(ops.quant_fp8(X), W, bias=b.cuda(), residual=r.cuda(), out_f32=yt == F32), ref + _np(b) + _np(r), xv, wv, yt,
           add=np.abs(_np(b)) + np.abs(_np(r)))


@pytest.mark.parametrize("M", [5, 150])
@pytest.mark.parametrize("act", [1, 3, 4, 5])
def test_activations_in_the_epilogue(M, act):
    ops = _ops()
    N, K = 140, 300
    x, w, b = _rand(M, K, seed=1), _rand(N, K, seed=2) * K ** -0.5, _rand(N, seed=3)
    xv, wv = R.quantise(_np(x))[0], R.quantise(_np(w), 128)[0]
    pre = xv @ wv.T + _np(b)
    # the activations' slope is at most 1.13 (both GELUs; SiLU 1.10); the erf / exp / reciprocal forms are good to 2e-6 absolute
    # for |v| of a few units
    _check(ops.gemm_fp8(x.cuda(), ops.pack_weight_fp8(w.cuda()), bias=b.cuda(), act=act, out_f32=True), R.ACTS[act](pre), xv, wv, F32,
           add=np.abs(_np(b)), extra=2e-6 * (1 + np.abs(pre)), slope=1.2)


@pytest.mark.parametrize("M,N,K", [(1, 130, 200), (16, 64, 256), (50, 300, 130), (200, 257, 520)])
def test_strides_offsets_and_preallocated_results(M, N, K):
    ops = _ops()
    wide = _rand(M, K + 9, seed=5, dtype=BF16).cuda()
    x = wide[:, 3:3 + K]                                              # rows that start at odd addresses
    w = _rand(N + 2, K + 5, seed=6).cuda()[1:N + 1, 2:2 + K] * K ** -0.5
    big = torch.full((M + 2, N + 7), 7.0, dtype=BF16, device="cuda")
    res = _rand(M, 2 * N, seed=7, dtype=BF16).cuda()[:, N - 1:2 * N - 1]
    out = big[1:M + 1, 3:3 + N]
    got = ops.gemm_fp8(x, ops.pack_weight_fp8(w), residual=res, out=out)
    assert got is out
    xv, wv = R.quantise(_np(x))[0], R.quantise(_np(w), 128)[0]
    _check(out, xv @ wv.T + _np(res), xv, wv, BF16, add=np.abs(_np(res)))
    mask = torch.ones_like(big, dtype=torch.bool)
    mask[1:M + 1, 3:3 + N] = False
    assert bool((big[mask] == 7.0).all())                             # nothing beside the result is written


def test_an_empty_product():
    ops = _ops()
    W = ops.pack_weight_fp8(_rand(40, 130).cuda(), transposed=True)
    assert ops.gemm_fp8(torch.empty(0, 130, device="cuda"), W).shape == (0, 40)
    assert ops.gemm_fp8(ops.quant_fp8(torch.empty(0, 130, device="cuda")), W, out_f32=True).shape == (0, 40)
    assert ops.gemm_fp8_dgrad(torch.empty(0, 40, device="cuda"), W).shape == (0, 130)
    assert ops.gated_fp8(torch.empty(0, 130, device="cuda"), W, W).values().shape == (0, 40)


@pytest.mark.parametrize("dt,xt", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (2, 129, 127), (16, 640, 300), (50, 257, 260), (231, 770, 385), (600, 300, 520)])
def test_input_gradient(M, N, K, dt, xt):
    ops = _ops()
    dy, w = 1e-3 * _rand(M, N, seed=1, spread=1.0).to(dt), _rand(N, K, seed=2) * K ** -0.5
    dy = dy.to(dt)
    W = ops.pack_weight_fp8(w.cuda(), transposed=True)
    dv, wv = R.quantise(_np(dy))[0], R.quantise(_np(w), 128)[0]
    _check(ops.gemm_fp8_dgrad(dy.cuda(), W, out_f32=xt == F32), dv @ wv, dv, wv.T, xt)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 256, 300), (5, 128, 128), (16, 320, 520), (33, 129, 127), (64, 200, 640), (70, 384, 256),
                                   (130, 300, 257), (260, 640, 512)])
def test_gated_product(M, N, K):
    ops = _ops()
    x, w0, w1 = _rand(M, K, seed=1, dtype=BF16), _rand(N, K, seed=2) * K ** -0.5, _rand(N, K, seed=3) * K ** -0.5
    h = ops.gated_fp8(x.cuda(), ops.pack_weight_fp8(w0.cuda()), ops.pack_weight_fp8(w1.cuda()))
    xv, v0, v1 = R.quantise(_np(x))[0], R.quantise(_np(w0), 128)[0], R.quantise(_np(w1), 128)[0]
    a, b = xv @ v0.T, xv @ v1.T
    ma, mb = np.abs(xv) @ np.abs(v0).T, np.abs(xv) @ np.abs(v1).T
    ref = R.gelu_tanh(a) * b
    # the absolute errors of both products (fp32 sums, what the 8-bit pipe drops), the slope of the GELU (1.13) and its fast form (2e-6)
    ea, eb = R.sum_bound(K) * ma + R.pipe_bound(xv, v0), R.sum_bound(K) * mb + R.pipe_bound(xv, v1)
    e = 1.2 * ea * (np.abs(b) + eb) + (np.abs(R.gelu_tanh(a)) + 2e-6) * eb + 2e-6 * (1 + np.abs(a)) * np.abs(b)
    nb = -(-N // 128)
    s = _exps(h)
    pad = lambda t: np.pad(t, ((0, 0), (0, nb * 128 - N))).reshape(M, nb, 128).max(2)
    sc = 2.0 ** s.astype(np.float64)
    assert (pad(np.maximum(np.abs(ref) - e, 0)) <= 448.0 * sc).all()
    assert ((pad(np.abs(ref) + e) > 224.0 * sc) | (s == -127)).all()
    full = np.repeat(sc, 128, 1)[:, :N]
    got = _np(h.values(F32))
    tol = np.maximum(2.0 ** -4 * (np.abs(ref) + e), 2.0 ** -10 * full) + e
    assert (np.abs(got - ref) <= tol).all(), float((np.abs(got - ref) - tol).max())
    assert not ops_untile(h.codes, M, nb * 128)[:, N:].any()


def test_the_gated_feed_forward_as_a_whole():
    """norm -> gated product -> product with the residual, against the 64-bit plain form with its own quantisations.  A code whose value lies
    within the products' error (1e-4 of it) of a rounding border goes the other way, by one step (2^-3): about one in a thousand.  The
    bound below is for one in a hundred: sqrt(1e-2) * 2^-4 of the feed-forward's share in the 2-norm, and the bf16 rounding"""
    ops = _ops()
    M, D, Fh = 70, 520, 1100
    x, g = _rand(M, D, seed=1, dtype=BF16), 1 + 0.2 * _rand(D, seed=2)
    w0, w1, wo = _rand(Fh, D, seed=3) * D ** -0.5, _rand(Fh, D, seed=4) * D ** -0.5, _rand(D, Fh, seed=5) * Fh ** -0.5
    P = lambda w: ops.pack_weight_fp8(w.cuda())
    X = x.cuda()
    y = ops.gemm_fp8(ops.gated_fp8(ops.rmsnorm_fp8(X, g.cuda(), 1e-6), P(w0), P(w1)), P(wo), residual=X)
    v = _np(x)
    n = R.quantise(v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6) * _np(g))[0]
    q = lambda w: R.quantise(_np(w), 128)[0]
    h = R.quantise(R.gelu_tanh(n @ q(w0).T) * (n @ q(w1).T))[0]
    f = h @ q(wo).T
    off = np.linalg.norm(_np(y) - (f + v))
    assert off <= 0.1 * 2.0 ** -4 * np.linalg.norm(f) + 2.0 ** -8 * np.linalg.norm(f + v)


# ---- large products: tiles of every size, several of them per workgroup, contractions in segments, rows in two launches ----------------------
def _pipe64(x, w):
    """R.pipe_bound on the GPU"""
    g = lambda t: torch.nn.functional.pad(t, (0, -t.shape[1] % 8)).abs().reshape(t.shape[0], -1, 8).amax(2)
    return 2.0 ** -10 * (g(x) @ g(w).t().contiguous())


def _operands64(M, N, K, seed):
    ops = _ops()
    x, w = _rand(M, K, seed=seed, dtype=BF16, spread=1.0).cuda(), (_rand(N, K, seed=seed + 1) * K ** -0.5).cuda()
    q, W = ops.quant_fp8(x), ops.pack_weight_fp8(w)                    # (compared with the plain format above)
    return q, W, q.values(F32).double(), W.values(F32).double()


LARGE = [(1920, 4096, 520), (1930, 2568, 6300), (4096, 4096, 6272), (2048, 2051, 1300), (3500, 5120, 2048), (5000, 1800, 1030), (700, 6152, 385),
         (4360, 2176, 200)]


@pytest.mark.parametrize("yt", [BF16, F32])
@pytest.mark.parametrize("M,N,K", LARGE)
def test_large_product(M, N, K, yt):
    ops = _ops()
    q, W, xv, wv = _operands64(M, N, K, M + N)
    b, r = _rand(N, seed=3).cuda(), _rand(M, N, seed=4, dtype=yt).cuda()
    ref, mag = xv @ wv.t().contiguous(), xv.abs() @ wv.abs().t().contiguous()
    pipe = _pipe64(xv, wv) if yt == BF16 else 0.0
    for bias, res in ((None, None), (b, r)):
        want = ref if bias is None else ref + b.double() + r.double()
        add = 0.0 if bias is None else b.double().abs() + r.double().abs()
        e = R.sum_bound(K + 4) * (mag + add) + pipe                   # (as in _check)
        tol = e + R.half_step(NAMES[yt]) * (want.abs() + e)
        d = (ops.gemm_fp8(q, W, bias=bias, residual=res, out_f32=yt == F32).double() - want).abs()
        assert bool((d <= tol).all()), (float((d - tol).max()), float(d.max()))
    out = r.clone()                                                   # the result over its own residual
    assert torch.equal(ops.gemm_fp8(q, W, bias=b, residual=out, out=out), ops.gemm_fp8(q, W, bias=b, residual=r, out_f32=yt == F32))


@pytest.mark.parametrize("M,N,K", [(3500, 2560, 2048), (2048, 4096, 384), (1100, 2600, 300), (1920, 1300, 6272)])
def test_large_gated_product(M, N, K):
    ops = _ops()
    q, W0, xv, v0 = _operands64(M, N, K, 5)
    W1 = ops.pack_weight_fp8((_rand(N, K, seed=9) * K ** -0.5).cuda())
    v1 = W1.values(F32).double()
    h = ops.gated_fp8(q, W0, W1)
    t = lambda w: w.t().contiguous()
    a, b, ax = xv @ t(v0), xv @ t(v1), xv.abs()
    gelu = torch.nn.functional.gelu(a, approximate="tanh")
    ref = gelu * b
    # (as in test_gated_product)
    ea, eb = R.sum_bound(K) * (ax @ t(v0.abs())) + _pipe64(xv, v0), R.sum_bound(K) * (ax @ t(v1.abs())) + _pipe64(xv, v1)
    e = 1.2 * ea * (b.abs() + eb) + (gelu.abs() + 2e-6) * eb + 2e-6 * (1 + a.abs()) * b.abs()
    nb = -(-N // 128)
    s = torch.from_numpy(_exps(h)).cuda()
    pad = lambda u: torch.nn.functional.pad(u, (0, nb * 128 - N)).reshape(M, nb, 128).amax(2)
    sc = torch.pow(2.0, s.double())
    assert bool((pad((ref.abs() - e).clamp_min(0)) <= 448.0 * sc).all())
    assert bool(((pad(ref.abs() + e) > 224.0 * sc) | (s == -127)).all())
    full = sc.repeat_interleave(128, 1)[:, :N]
    d = (h.values(F32).double() - ref).abs()
    tol = torch.maximum(2.0 ** -4 * (ref.abs() + e), 2.0 ** -10 * full) + e
    assert bool((d <= tol).all()), float((d - tol).max())


def test_two_runs_are_bit_identical_and_a_graph_replays_them():
    ops = _ops()
    M, N, K = 200, 300, 520
    x = _rand(M, K, seed=1, dtype=BF16).cuda()
    W = ops.pack_weight_fp8((_rand(N, K, seed=2) * K ** -0.5).cuda(), transposed=True)
    W2 = ops.pack_weight_fp8((_rand(N, K, seed=3) * K ** -0.5).cuda())

    def step():
        y = ops.gemm_fp8(x, W)
        h = ops.gated_fp8(ops.rmsnorm_fp8(x, None, 0.0), W, W2)
        return y, h.values(), ops.gemm_fp8_dgrad(y, W), ops.gemm_fp8(x[:3], W)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 7, 8, 9):
        x.copy_(_rand(M, K, seed=seed, dtype=BF16))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_results_over_operands():
    """out over A is refused, out over the residual is the same rows or refused, other columns of one buffer are fine"""
    ops = _ops()
    W = ops.pack_weight_fp8(_rand(64, 64, seed=1).cuda())
    for M in (3, 40):
        x, big = _rand(M, 64, seed=2, dtype=BF16).cuda(), torch.zeros(M, 160, dtype=BF16, device="cuda")
        with pytest.raises(ValueError, match="share"):
            ops.gemm_fp8(x, W, out=x)
        with pytest.raises(ValueError, match="share"):
            ops.gemm_fp8(big[:, :64], W, out=big[:, 63:127])
        with pytest.raises(ValueError, match="residual"):
            ops.gemm_fp8(x, W, residual=big[:, :64], out=big[:, 8:72])
        want, r = ops.gemm_fp8(x, W), _rand(M, 64, seed=3, dtype=BF16).cuda()
        big[:, :64], big[:, 128:] = x, 5.0
        assert torch.equal(ops.gemm_fp8(big[:, :64], W, out=big[:, 64:128]), want)
        assert torch.equal(big[:, :64], x) and bool((big[:, 128:] == 5.0).all())
        both = ops.gemm_fp8(x, W, residual=r)
        assert torch.equal(ops.gemm_fp8(x, W, residual=r, out=r), both) and torch.equal(r, both)


def test_rows_beyond_two_to_the_32_bytes():
    ops = _ops()
    M, reps, N, K = 1000, 1070, 72, 4096                               # 1070000 rows: 8.8e9 bytes of bf16, 4.4e9 of codes
    x, w = _rand(M, K, seed=1, dtype=BF16).cuda(), ops.pack_weight_fp8((_rand(N, K, seed=2) * K ** -0.5).cuda())
    X = x.repeat(reps, 1)
    y = ops.gemm_fp8(X, w)
    assert torch.equal(y.view(reps, M, N), y[:M].expand(reps, M, N))    # the same rows, whatever their place
    xv, wv = ops.quant_fp8(x).values(F32).double(), w.values(F32).double()
    _check(y[-M:], _np(xv) @ _np(wv).T, _np(xv), _np(wv), BF16)
    h = ops.gated_fp8(X, w, w).values().view(reps, M, N)
    assert torch.equal(h, h[:1].expand(reps, M, N)) and torch.equal(h[0], ops.gated_fp8(X[:64000], w, w).values()[:M])


@pytest.mark.parametrize("N,K", [(8, 64), (40, 100)])
def test_many_short_rows(N, K):
    """more row tiles than the second dimension of a grid holds"""
    ops = _ops()
    M, reps = 2 ** 10 + 16, 2100
    x, w = _rand(M, K, seed=1, dtype=BF16).cuda(), ops.pack_weight_fp8((_rand(N, K, seed=2) * K ** -0.5).cuda())
    for f32 in (False, True):
        y = ops.gemm_fp8(x.repeat(reps, 1), w, out_f32=f32).view(reps, M, N)
        xv, wv = _np(ops.quant_fp8(x).values(F32)), _np(w.values(F32))
        _check(y[-1], xv @ wv.T, xv, wv, F32 if f32 else BF16)
        assert torch.equal(y, y[:1].expand(reps, M, N))


def test_refusals_on_the_gpu():
    ops = _ops()
    W = ops.pack_weight_fp8(_rand(64, 130).cuda())
    x = _rand(4, 130, dtype=BF16).cuda()
    bad = [lambda: ops.gemm_fp8(x.cpu(), W), lambda: ops.gemm_fp8(x[:, :129], W), lambda: ops.gemm_fp8(x.half(), W),
           lambda: ops.gemm_fp8(x.t(), W), lambda: ops.gemm_fp8(x[:1].expand(4, 130), W), lambda: ops.gemm_fp8(x[0], W),
           lambda: ops.gemm_fp8(x, W, bias=torch.zeros(64, dtype=BF16, device="cuda")), lambda: ops.gemm_fp8(x, W, bias=torch.zeros(63, device="cuda")),
           lambda: ops.gemm_fp8(x, W, residual=torch.zeros(4, 64, device="cuda")),                   # bf16 result, fp32 residual
           lambda: ops.gemm_fp8(x, W, residual=torch.zeros(4, 64, dtype=BF16, device="cuda"), act=ops.ACT_RELU),
           lambda: ops.gemm_fp8(x, W, act=ops.ACT_GEGLU), lambda: ops.gemm_fp8(x, W, act=17), lambda: ops.gemm_fp8(x, W, out=torch.empty(4, 63, device="cuda")),
           lambda: ops.gemm_fp8_dgrad(_rand(4, 64).cuda(), W), lambda: ops.gated_fp8(x, W, ops.pack_weight_fp8(_rand(65, 130).cuda())),
           lambda: ops.pack_weight_fp8(torch.empty(0, 4, device="cuda")), lambda: ops.quant_fp8(torch.empty(3, 0, device="cuda")),
           lambda: ops.rmsnorm_fp8(x, torch.ones(129, device="cuda"), 1e-6), lambda: ops.gemm_fp8(ops.quant_fp8(x[:, :100]), W)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"case {i} was accepted")
