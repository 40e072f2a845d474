"""Rows, tokens and tables of more than one launch's threads (2^32 along a grid): the kernels of the 8-bit products and of the embedding."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _ops():
    from flash_diffusion_amd import ops
    return ops


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


PART, REPS = 1 << 16, 1025                    # 2^26 + 2^16 rows


def test_rows_quantised_in_several_launches():
    ops = _ops()
    x, norm = _rand(PART, 3, dtype=BF16).cuda(), (1 + 0.1 * _rand(3, seed=1)).cuda()
    for f in (ops.quant_fp8, lambda t: ops.rmsnorm_fp8(t, norm, 1e-6)):
        one, all_ = f(x), f(x.repeat(REPS, 1))
        assert torch.equal(all_.codes.view(REPS, -1), one.codes.expand(REPS, -1))
        assert torch.equal(all_.scales.view(REPS, -1), one.scales.expand(REPS, -1))
        del one, all_


@pytest.mark.parametrize("out_f32", [False, True])
def test_a_product_of_more_rows_than_a_launch_of_short_tiles_holds(out_f32):
    ops = _ops()
    x, w = _rand(PART, 64, dtype=BF16).cuda(), ops.pack_weight_fp8(_rand(8, 64, seed=1).cuda())
    want = ops.gemm_fp8(x, w, out_f32=out_f32)
    y = ops.gemm_fp8(x.repeat(REPS, 1), w, out_f32=out_f32).view(REPS, PART, 8)
    # (another kernel may run here than for the part: fp32 sums of 64 terms in another order, the 8-bit pipe's bits, one rounding)
    xv, wv = ops.quant_fp8(x).values().double(), w.values().double()
    mag = xv.abs() @ wv.abs().t().contiguous()
    tol = 2 * mag * (2.0 ** -16 if out_f32 else 2.0 ** -10) + (0 if out_f32 else 2.0 ** -7) * want.double().abs()
    assert bool(((y[-1].double() - want.double()).abs() <= tol).all()) and torch.equal(y, y[:1].expand(REPS, PART, 8))


def test_tokens_looked_up_in_several_launches():
    ops = _ops()
    B, S, D = 900000, 77, 2                   # 69.3 million tokens; no slice of 2^25 is a multiple of 77
    table, pos = _rand(300, D).cuda(), _rand(S, D, seed=1).cuda()
    ids = torch.randint(0, 300, (B, S), generator=torch.Generator().manual_seed(2)).cuda()
    assert torch.equal(ops.embed_fwd(table, ids, pos=pos, dtype=F32), table[ids] + pos)


@pytest.mark.parametrize("n", [0, 5, 3000])
def test_the_gradient_of_a_table_whose_zeros_take_two_launches(n):
    ops = _ops()
    V, D = (1 << 28) + 1000, 2
    ids = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(1))
    if n:
        ids[:4] = torch.tensor([0, V - 1, (1 << 28) - 17, (1 << 28) - 1])
    ids = ids.cuda()
    dy = torch.ones(n, D, device="cuda")
    full = torch.full((V, D), float("nan"), device="cuda")             # (the allocator hands its memory to the gradient)
    del full
    g = ops.embed_bwd(dy, ids, V)
    rows, count = torch.unique(ids, return_counts=True)
    assert torch.equal(g[rows], count.float()[:, None].expand(-1, D))
    g[rows] = 0.0
    assert not bool(torch.isnan(g.view(-1).max())) and int(torch.count_nonzero(g)) == 0
