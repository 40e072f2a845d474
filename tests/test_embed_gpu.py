"""The token-embedding lookup and its table's gradient (csrc/embed.hip) against 64-bit plain forms."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _ops():
    from flash_diffusion_amd import ops
    return ops


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("tt,ot,it", [(F32, BF16, torch.int64), (F32, F32, torch.int32), (BF16, BF16, torch.int32), (BF16, F32, torch.int64)])
@pytest.mark.parametrize("B,S,V,D", [(1, 1, 1, 1), (2, 77, 500, 768), (3, 5, 40, 7), (1, 130, 1000, 65), (4, 16, 33, 130), (2, 9, 90, 1028)])
def test_lookup(B, S, V, D, tt, ot, it):
    ops = _ops()
    g = torch.Generator().manual_seed(B * S + D)
    table, ids, pos = _rand(V, D, seed=1, dtype=tt), torch.randint(0, V, (B, S), generator=g).to(it), _rand(S + 3, D, seed=2)
    for scale, p in ((1.0, None), (0.5, pos), (D ** 0.5, None), (-3.0, pos)):
        got = ops.embed_fwd(table.cuda(), ids.cuda(), scale=scale, pos=None if p is None else p.cuda(), dtype=ot)
        # (the scale travels as fp32)
        ref = _np(table)[ids.numpy()] * float(np.float32(scale)) + (0.0 if p is None else _np(p)[None, :S])
        assert got.shape == (B, S, D) and got.dtype == ot
        # one fused multiply-add in fp32 and one rounding to the result's type (fp32: the first is the last)
        e = np.abs(ref) * (HALF[ot] + (2.0 ** -24 if ot == BF16 else 0.0)) * (1 + 2.0 ** -8)
        assert (np.abs(_np(got) - ref) <= e).all()


def test_lookup_of_one_unscaled_row_is_a_copy_and_of_a_strided_table_too():
    ops = _ops()
    wide = _rand(20, 50, seed=3).cuda()
    ids = torch.tensor([3, 0, 19, 3], device="cuda")
    assert torch.equal(ops.embed_fwd(wide[:, 5:38], ids, dtype=F32), wide[:, 5:38][ids])
    assert torch.equal(ops.embed_fwd(wide[::2, 1:34], ids[:2], dtype=BF16), wide[::2, 1:34][ids[:2]].to(BF16))
    assert ops.embed_fwd(wide, torch.empty(2, 0, dtype=torch.int64, device="cuda")).shape == (2, 0, 50)
    assert torch.equal(ops.embed_fwd(wide, torch.tensor(4, device="cuda"), dtype=F32), wide[4])


def test_an_id_outside_the_table_reads_as_nan_and_gets_no_gradient():
    ops = _ops()
    table = _rand(10, 24).cuda()
    ids = torch.tensor([[1, 10, -1], [9, 2 ** 40, 0]], device="cuda")
    y = ops.embed_fwd(table, ids, dtype=F32)
    bad = torch.tensor([[False, True, True], [False, True, False]], device="cuda")
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], table[ids[~bad]])
    g = ops.embed_bwd(torch.ones(2, 3, 24, device="cuda"), ids, 10)
    want = torch.zeros(10, 24, device="cuda")
    want[[0, 1, 9]] = 1.0
    assert torch.equal(g, want)


def _ids_of(kind, n, V, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((n,), V // 2)
    if kind == "all":
        return torch.randperm(max(n, V), generator=g)[:n] % V
    if kind == "runs":            # runs of 1, 2, 3, ... positions that end inside, at and behind a chunk's edge, shuffled
        ids = torch.cat([torch.full((k,), k % V) for k in range(1, 2 + int((2 * n) ** 0.5))])[:n]
        return torch.cat([ids, torch.zeros(n - ids.numel(), dtype=torch.long)])[torch.randperm(n, generator=g)]
    ids = torch.randint(0, V, (n,), generator=g)          # "padded": two thirds are id 0
    return torch.where(torch.rand(n, generator=g) < 0.67, torch.zeros_like(ids), ids)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("kind", ["one", "all", "runs", "padded"])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (31, 7, 3), (32, 50, 64), (33, 50, 65), (64, 300, 130), (257, 100, 257), (1232, 2000, 96), (4096, 900, 12),
                                   (4097, 900, 12), (5000, 700, 40), (20000, 3000, 5)])
def test_gradient(n, V, D, kind, dt):
    ops = _ops()
    ids = _ids_of(kind, n, V, n + V)
    dy = _rand(n, D, seed=n, dtype=dt)
    got = ops.embed_bwd(dy.cuda(), ids.cuda(), V, scale=0.75)
    v = _np(dy)
    ref, mag, cnt = np.zeros((V, D)), np.zeros((V, D)), np.zeros((V, 1))
    np.add.at(ref, ids.numpy(), v)
    np.add.at(mag, ids.numpy(), np.abs(v))
    np.add.at(cnt, ids.numpy(), 1.0)
    # count - 1 rounded additions of partial sums that never exceed mag, and the scale's product
    assert (np.abs(_np(got) - 0.75 * ref) <= 0.75 * (cnt + 1) * 2.0 ** -24 * mag).all()
    again = ops.embed_bwd(dy.cuda(), ids.cuda().to(torch.int32), V, scale=0.75)
    assert torch.equal(got, again)                                     # a fixed order: the same bits


# in the sorted list: runs that begin and end on, before and behind the edges of 16 and 64 positions, over one edge and over many
RUNS = {"edges": [16, 48, 64, 1, 63, 65, 128, 15, 17, 31, 33, 2, 62, 64, 63, 1, 127, 129], "long": [7, 1100, 2, 1024, 64, 1089, 1, 4000, 63],
        "whole": [64, 64, 64], "short": [1] * 200, "tail": [64, 1], "one more": [65]}


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("D", [5, 72, 520])
@pytest.mark.parametrize("runs", list(RUNS))
def test_gradient_of_runs_in_the_sorted_list(runs, D, dt):
    ops = _ops()
    lengths = RUNS[runs]
    V = 2 * len(lengths) + 35                                          # every other row of the table has no token
    ids = torch.cat([torch.full((k,), 2 * i + 1) for i, k in enumerate(lengths)])
    g = torch.Generator().manual_seed(len(ids) + D)
    ids = ids[torch.randperm(len(ids), generator=g)]
    dy = _rand(len(ids), D, seed=7, dtype=dt)
    v = _np(dy)
    ref, mag, cnt = np.zeros((V, D)), np.zeros((V, D)), np.zeros((V, 1))
    np.add.at(ref, ids.numpy(), v)
    np.add.at(mag, ids.numpy(), np.abs(v))
    np.add.at(cnt, ids.numpy(), 1.0)
    full = torch.full((V, D), float("nan"), device="cuda")             # (the allocator hands its memory to the gradient)
    del full
    got = _np(ops.embed_bwd(dy.cuda(), ids.cuda(), V, scale=0.75))
    assert (np.abs(got - 0.75 * ref) <= 0.75 * (cnt + 1) * 2.0 ** -24 * mag).all()      # (as above)
    start = _rand(V, D, seed=8)
    out = _np(ops.embed_bwd(dy.cuda(), ids.cuda(), V, scale=0.75, out=start.cuda()))
    s = _np(start)
    assert (np.abs(out - (s + 0.75 * ref)) <= (cnt + 2) * 2.0 ** -24 * (0.75 * mag + np.abs(s))).all()


@pytest.mark.parametrize("n", [63, 64, 65, 2047, 2048, 2049, 2304])
def test_gradient_where_the_order_is_found_another_way(n):
    ops = _ops()
    V, D = 150, 8
    ids, dy = _ids_of("padded", n, V, n), _rand(n, D, seed=n).round()  # (integers: sums are exact)
    ref = torch.zeros(V, D).index_add_(0, ids, dy)
    assert torch.equal(ops.embed_bwd(dy.cuda(), ids.cuda(), V).cpu(), ref)


@pytest.mark.parametrize("kind", ["one", "all", "runs", "padded"])
@pytest.mark.parametrize("n,D", [(128, 8), (129, 70), (192, 1), (255, 520), (256, 9), (257, 9)])
def test_gradient_of_short_lists(n, D, kind):
    ops = _ops()
    V = 40
    ids = _ids_of(kind, n, V, n)
    ids[::37] = torch.tensor([-1, V, 2 ** 31, -(2 ** 40)])[torch.arange(len(ids[::37])) % 4]     # (some outside the table)
    dy = torch.randint(-3, 4, (n, D), generator=torch.Generator().manual_seed(n))
    ok = (ids >= 0) & (ids < V)
    ref = torch.zeros(V, D, dtype=torch.int64).index_add_(0, ids[ok], dy[ok]).float()
    for dt in (F32, BF16):                                             # (small integers: sums are exact)
        full = torch.full((V, D), float("nan"), device="cuda")
        del full
        assert torch.equal(ops.embed_bwd(dy.to(dt).cuda(), ids.cuda(), V).cpu(), ref)
        out = torch.ones(V, D, device="cuda")
        assert torch.equal(ops.embed_bwd(dy.to(dt).cuda(), ids.cuda(), V, out=out).cpu(), ref + 1)


@pytest.mark.parametrize("n,it", [(131073, torch.int32), (300000, torch.int64)])
def test_gradient_of_long_lists(n, it):
    ops = _ops()
    V, D = 700, 12
    ids, dy = _ids_of("padded", n, V, n), torch.randint(-3, 4, (n, D), generator=torch.Generator().manual_seed(n))
    ref = torch.zeros(V, D, dtype=torch.int64).index_add_(0, ids, dy).float()
    for dt in (F32, BF16):                                             # (integers below 2^24: sums are exact)
        assert torch.equal(ops.embed_bwd(dy.to(dt).cuda(), ids.to(it).cuda(), V).cpu(), ref)
        out = torch.ones(V, D, device="cuda")
        assert torch.equal(ops.embed_bwd(dy.to(dt).cuda(), ids.to(it).cuda(), V, out=out).cpu(), ref + 1)


def test_tables_beyond_two_to_the_31_elements():
    ops = _ops()
    V, D = 540000, 4096
    ids = torch.tensor([[0, V - 1, V - 2], [524287, 524288, 524289]], device="cuda")
    table = torch.zeros(V, D, dtype=BF16, device="cuda")
    rows = _rand(6, D, dtype=BF16).cuda()
    table[ids.view(-1)] = rows
    assert torch.equal(ops.embed_fwd(table, ids).view(6, D), rows)
    del table
    g = ops.embed_bwd(rows.view(2, 3, D), ids, V)
    assert torch.equal(g[ids.view(-1)], rows.float())
    g[ids.view(-1)] = 0.0
    assert not g.any()


def test_gradient_accumulates_into_strided_rows_and_leaves_the_others():
    ops = _ops()
    n, V, D = 200, 64, 70
    ids = _ids_of("padded", n, V // 2, 3)
    dy = _rand(4, n // 4, D + 6, seed=1).cuda()[..., 3:3 + D]
    big = _rand(V, D + 5, seed=2).cuda()
    out = big[:, 2:2 + D]
    before = big.clone()
    assert ops.embed_bwd(dy, ids.view(4, -1).cuda(), V, out=out) is out
    ref, mag = np.zeros((V, D)), np.zeros((V, D))
    np.add.at(ref, ids.numpy(), _np(dy).reshape(n, D))
    np.add.at(mag, ids.numpy(), np.abs(_np(dy).reshape(n, D)))
    b = _np(before)[:, 2:2 + D]
    cnt = np.bincount(ids.numpy(), minlength=V)[:, None]
    assert (np.abs(_np(out) - (b + ref)) <= (cnt + 2) * 2.0 ** -24 * (mag + np.abs(b))).all()
    hit = torch.tensor(np.bincount(ids.numpy(), minlength=V) > 0, device="cuda")
    assert torch.equal(out[~hit], before[:, 2:2 + D][~hit])
    assert torch.equal(big[:, :2], before[:, :2]) and torch.equal(big[:, 2 + D:], before[:, 2 + D:])


def test_gradient_of_no_tokens_is_zero():
    ops = _ops()
    e = torch.empty(0, dtype=torch.int64, device="cuda")
    assert not ops.embed_bwd(torch.empty(0, 9, device="cuda"), e, 5).any()
    out = torch.ones(5, 9, device="cuda")
    assert bool((ops.embed_bwd(torch.empty(0, 9, device="cuda"), e, 5, out=out) == 1).all())


def test_a_graph_replays_lookup_and_gradient():
    ops = _ops()
    V, D, B, S = 90, 72, 3, 50
    table, dy = _rand(V, D).cuda(), _rand(B, S, D, seed=1).cuda()
    ids = _ids_of("padded", B * S, V, 1).view(B, S).cuda()

    def step():
        return ops.embed_fwd(table, ids), ops.embed_bwd(dy, ids, V)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (2, 3, 4):
        ids.copy_(_ids_of("padded", B * S, V, seed).view(B, S))
        dy.copy_(_rand(B, S, D, seed=seed))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_refusals_on_the_gpu():
    ops = _ops()
    t, ids = _rand(10, 8).cuda(), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    bad = [lambda: ops.embed_fwd(t.cpu(), ids), lambda: ops.embed_fwd(t, ids.cpu()), lambda: ops.embed_fwd(t, ids.float()),
           lambda: ops.embed_fwd(t.t(), ids), lambda: ops.embed_fwd(t.half(), ids), lambda: ops.embed_fwd(t, ids, pos=t[:2]),
           lambda: ops.embed_fwd(t, ids, pos=t[:, :7]), lambda: ops.embed_fwd(t, ids, pos=t.bfloat16()), lambda: ops.embed_fwd(t, ids, dtype=torch.float16),
           lambda: ops.embed_fwd(t[:0], ids), lambda: ops.embed_bwd(t, ids, 10), lambda: ops.embed_bwd(torch.zeros(2, 3, 8, device="cuda").half(), ids, 10),
           lambda: ops.embed_bwd(torch.zeros(2, 3, 8, device="cuda"), ids, 10, out=torch.zeros(9, 8, device="cuda")),
           lambda: ops.embed_bwd(torch.zeros(2, 3, 8, device="cuda"), ids, 10, out=torch.zeros(10, 8, dtype=BF16, device="cuda")),
           lambda: ops.embed_bwd(torch.zeros(2, 3, 8, device="cuda"), ids, 0)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"case {i} was accepted")
