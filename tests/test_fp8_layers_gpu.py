"""The layers over the 8-bit products and the lookup (flash_diffusion_amd/fp8.py) and the text encoder that runs on them."""
import copy

import numpy as np
import pytest
import torch

from tests import fp8_ref as R
from tests.golden_util import rel_err
from tests.test_t5_gpu import CASES, _hf

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _np(t):
    return t.detach().double().cpu().numpy()


# ---- the encoder ---------------------------------------------------------------------------------------------------------------------
def _bf(v):
    return _np(torch.from_numpy(np.ascontiguousarray(v)).float().to(BF16))


def _emulated(hf, kw, ids, mask, jitter=0.0):
    """the fp8 encoder in 64 bits, rounding where it rounds: codes of norms, attention output and gated product, bf16 stream, q / k / v.
    jitter: every product is off by that much of its root mean square, at random"""
    rng = np.random.RandomState(7)

    def mm(x, w):
        y = x @ w.T
        return y + jitter * np.sqrt((y * y).mean()) * rng.randn(*y.shape) if jitter else y

    from flash_diffusion_amd.t5 import relative_position_bucket
    p = {k: _np(v) for k, v in hf.state_dict().items()}
    q8 = lambda v: R.quantise(v)[0]
    w8 = lambda name: R.quantise(p[name], 128)[0]
    B, S = ids.shape
    H, dk, eps = kw["num_heads"], kw["d_kv"], 1e-6
    norm = lambda h, w: h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w
    pos = torch.arange(S)
    bucket = relative_position_bucket(pos[None] - pos[:, None], kw.get("relative_attention_num_buckets", 32),
                                      kw.get("relative_attention_max_distance", 128)).numpy()
    bias = p["encoder.block.0.layer.0.SelfAttention.relative_attention_bias.weight"][bucket].transpose(2, 0, 1)
    kb = np.where(mask.numpy() > 0, 0.0, float(torch.finfo(F32).min))
    h = _bf(p["shared.weight"][ids.numpy().reshape(-1)])
    for i in range(kw["num_layers"]):
        a, f = f"encoder.block.{i}.layer.0.", f"encoder.block.{i}.layer.1."
        n = q8(norm(h, p[a + "layer_norm.weight"]))
        q, k, v = (_bf(mm(n, w8(a + f"SelfAttention.{m}.weight"))).reshape(B, S, H, dk).transpose(0, 2, 1, 3) for m in "qkv")
        s = q @ k.transpose(0, 1, 3, 2) + bias[None] + kb[:, None, None, :]
        s = np.exp(s - s.max(-1, keepdims=True))
        o = _bf(((s / s.sum(-1, keepdims=True)) @ v).transpose(0, 2, 1, 3).reshape(B * S, H * dk))
        h = _bf(mm(q8(o), w8(a + "SelfAttention.o.weight")) + h)
        n = q8(norm(h, p[f + "layer_norm.weight"]))
        if kw["feed_forward_proj"] == "gated-gelu":
            g = q8(R.gelu_tanh(mm(n, w8(f + "DenseReluDense.wi_0.weight"))) * mm(n, w8(f + "DenseReluDense.wi_1.weight")))
        else:
            g = q8(_bf(np.maximum(mm(n, w8(f + "DenseReluDense.wi.weight")), 0.0)))
        h = _bf(mm(g, w8(f + "DenseReluDense.wo.weight")) + h)
    return norm(h, p["encoder.final_layer_norm.weight"]).reshape(B, S, -1)


@pytest.mark.parametrize("layers", [1, None])
@pytest.mark.parametrize("name", list(CASES))
def test_the_fp8_encoder_is_its_64_bit_emulation(name, layers):
    """Both sides round at the same places, but the chain of quantisers magnifies what lies before it: an error e of a product turns about
    e / 2^-4 of the next codes by a step of up to 2^-3, and unscaled attention scores magnify those.  The bar is therefore the definition's
    own answer to errors of the size that the products may have: every product of the emulation off by 2^-13 of its root mean square (the
    unit below which the 8-bit pipe drops bits, relative to the largest of eight products), twice that answer in the 2-norm.
    (The first form of this test had 2e-2 for a bar, from one branch's codes alone, without the magnification: the emulation itself moves by
    3.0e-2 on the tiny cases when its products are off by 1e-5.)"""
    from flash_diffusion_amd.t5 import MiT5EncoderModel
    kw = dict(CASES[name], num_layers=layers or CASES[name]["num_layers"])
    hf = _hf(kw)
    mi = MiT5EncoderModel(**kw, precision="fp8")
    mi.load_state_dict(hf.state_dict(), strict=True)
    mi = mi.cuda()
    mi.freeze()
    g = torch.Generator().manual_seed(1)
    B, S = 2, 60
    ids = torch.randint(2, kw["vocab_size"], (B, S), generator=g)
    mask = torch.ones(B, S, dtype=torch.long)
    ids[0, 20:], mask[0, 20:] = 0, 0
    out = mi(ids.cuda(), attention_mask=mask.cuda(), output_hidden_states=True)
    assert len(out.hidden_states) == kw["num_layers"] + 1
    want = _emulated(hf, kw, ids, mask)
    bar = 2.0 * np.linalg.norm(_emulated(hf, kw, ids, mask, jitter=2.0 ** -13) - want) / np.linalg.norm(want)
    err = rel_err(out.last_hidden_state, torch.from_numpy(want))
    print(f"{name} x {kw['num_layers']}: {err:.2e}, bar {bar:.2e}")
    assert err <= bar
    again = mi(ids.cuda(), attention_mask=mask.cuda()).last_hidden_state
    assert torch.equal(again, out.last_hidden_state)


def test_a_weight_is_packed_again_when_it_changes_and_copies_pack_their_own():
    from flash_diffusion_amd.t5 import _W
    from flash_diffusion_amd import ops
    m = _W(70, 40).cuda()
    for p in m.parameters():
        p.requires_grad_(False)
    first = m.operand8(m.weight)
    assert m.operand8(m.weight) is first
    before = first.values().clone()
    m.weight.mul_(2.0)                                       # in place
    second = m.operand8(m.weight)
    assert second is not first and torch.equal(second.values(), 2.0 * before)
    m.weight = torch.nn.Parameter(torch.ones(70, 40, device="cuda"), requires_grad=False)
    assert bool((m.operand8(m.weight).values() == 1.0).all())
    m.weight.data = torch.full((70, 40), 3.0, device="cuda")  # what .to() does
    assert bool((m.operand8(m.weight).values() == 3.0).all())
    c = copy.deepcopy(m)
    c.weight.fill_(5.0)
    assert bool((c.operand8(c.weight).values() == 5.0).all()) and bool((m.operand8(m.weight).values() == 3.0).all())
    # another stream waits for the packing: the product there is the one of this stream
    x = _rand(33, 40, seed=1, dtype=BF16).cuda()
    want = ops.gemm_fp8(x, ops.pack_weight_fp8(_rand(70, 40, seed=2).cuda()))
    torch.cuda.synchronize()
    m.weight.copy_(_rand(70, 40, seed=2))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    a.wait_stream(torch.cuda.current_stream())
    b.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(a):
        m.operand8(m.weight)
    with torch.cuda.stream(b):
        got = ops.gemm_fp8(x, m.operand8(m.weight))
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_packing_under_capture_is_refused():
    from flash_diffusion_amd.fp8 import PackedFp8
    w = _rand(20, 30).cuda()
    p, q = PackedFp8(), PackedFp8()
    q(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before a graph"):
            p(w)
        assert q(w) is not None
        w + 1


def test_a_captured_graph_sees_a_weight_that_is_packed_again():
    from flash_diffusion_amd import ops
    from flash_diffusion_amd.fp8 import PackedFp8
    w, x, p = _rand(70, 260).cuda(), _rand(40, 260, seed=1).cuda(), PackedFp8()
    p(w)
    ops.gemm_fp8(x, p(w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.gemm_fp8(x, p(w))
    for seed in (2, 3):
        w.copy_(_rand(70, 260, seed=seed))
        want = ops.gemm_fp8(x, p(w))                         # packs again
        noise = [torch.full((70000,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]   # (memory that had been freed)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and len(noise) == 8
    q = p(w)
    w = _rand(71, 260).cuda()                                # another shape: its own memory
    assert p(w).N == 71 and q.N == 70
    with pytest.raises(ValueError, match="into"):
        ops.pack_weight_fp8(w, into=q)
    with pytest.raises(ValueError, match="into"):
        ops.pack_weight_fp8(w, True, into=p(w))


def test_layers_under_a_captured_backward():
    """forward and backward of lookup and 8-bit layer in one graph, replayed with new inputs between eager work"""
    from flash_diffusion_amd.fp8 import Fp8Linear, TokenEmbedding, _LookupFn
    emb, lin = TokenEmbedding(50, 136).cuda(), Fp8Linear(_rand(40, 136, seed=1).cuda(), _rand(40, seed=2).cuda())
    ids, dy = torch.randint(0, 50, (3, 30)).cuda(), _rand(3, 30, 40, seed=3, dtype=BF16).cuda()

    def step():
        w = emb.weight.detach().requires_grad_()             # (a leaf of this graph alone)
        out = lin(_LookupFn.apply(w, None, ids, 0.5, BF16))
        return out.detach(), torch.autograd.grad(out, w, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (4, 5, 6):
        ids.copy_(torch.randint(0, 50, (3, 30), generator=torch.Generator().manual_seed(seed)))
        dy.copy_(_rand(3, 30, 40, seed=seed))
        emb.weight.data.copy_(_rand(50, 136, seed=seed))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_second_derivatives_are_refused():
    from flash_diffusion_amd.fp8 import Fp8Linear, TokenEmbedding
    lin, emb = Fp8Linear(_rand(40, 136, seed=1).cuda()), TokenEmbedding(9, 8).cuda()
    x = _rand(5, 136).cuda().requires_grad_()
    for leaf, y in ((x, lin(x)), (emb.weight, emb(torch.tensor([1, 2], device="cuda"), dtype=F32))):
        (g,) = torch.autograd.grad((y * y).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


# ---- the trained table in front of frozen 8-bit layers ---------------------------------------------------------------------------------
def test_a_token_table_learns_through_frozen_8_bit_layers():
    """lookup -> two linear maps -> a weighted sum: the table's gradient against the formula in 64 bits on the values that the layers hold"""
    from flash_diffusion_amd.fp8 import Fp8Linear, TokenEmbedding
    V, D, E, F, B, S = 50, 72, 130, 40, 3, 20
    emb = TokenEmbedding(V, D).cuda()
    l1 = Fp8Linear(_rand(E, D, seed=1).cuda() * D ** -0.5, _rand(E, seed=2).cuda())
    l2 = Fp8Linear(_rand(F, E, seed=3).cuda() * E ** -0.5)
    ids = torch.randint(0, V // 2, (B, S), generator=torch.Generator().manual_seed(4)).cuda()
    c = _rand(B, S, F, seed=5).cuda()
    y = l2(l1(emb(ids, scale=0.5, dtype=F32)))
    assert y.shape == (B, S, F) and y.dtype == F32
    (y * c).sum().backward()
    w1, w2 = _np(l1.packed().values()), _np(l2.packed().values())
    v = R.quantise(0.5 * _np(emb.weight)[ids.cpu().numpy()].reshape(-1, D))[0] @ w1.T + _np(l1.bias)
    assert np.allclose(_np(y).reshape(-1, F), R.quantise(v)[0] @ w2.T, atol=2.0 ** -3 * 0.2)      # (a code that went the other way)
    g2 = R.quantise(_np(c).reshape(-1, F))[0] @ w2                            # what flows into the second layer's input
    d1 = R.quantise(g2)[0] @ w1
    want, mag = np.zeros((V, D)), np.zeros((V, D))
    np.add.at(want, ids.cpu().numpy().reshape(-1), 0.5 * d1)
    # g2 is exact to fp32 sums; a code of it may go the other way by one step (2^-3) where it lies that near a border: one in 2^14 or
    # fewer; the bar allows one in a hundred
    assert np.linalg.norm(_np(emb.weight.grad) - want) <= 0.1 * 2.0 ** -4 * np.linalg.norm(want)
    assert not emb.weight.grad[V // 2:].any()


def test_the_layers_input_gradient_against_differences():
    """y is a step function of x; over a step d as large as x the difference of <c, y> is <c W^T, d> up to the two quantisations' errors, whose
    sizes are known here"""
    from flash_diffusion_amd.fp8 import Fp8Linear
    lin = Fp8Linear(_rand(60, 200, seed=1).cuda() * 200 ** -0.5)
    x, d, c = _rand(30, 200, seed=2), _rand(30, 200, seed=3), _rand(30, 60, seed=4)
    X = x.cuda().requires_grad_(True)
    y = lin(X)
    (y * c.cuda()).sum().backward()
    diff = float(((lin((x + d).cuda()) - y).double() * c.cuda().double()).sum())
    w = _np(lin.packed().values())
    slope = _np(c) @ w
    e = lambda t: np.abs(R.quantise(_np(t))[0] - _np(t))
    slack = (np.abs(slope) * (e(x) + e(x + d))).sum() + (np.abs(e(c) @ np.abs(w)) * np.abs(_np(d))).sum() + 1e-5 * np.abs(slope).sum()
    assert abs(diff - float((X.grad.double().cpu() * d.double()).sum())) <= slack


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_fp8_linear_shapes_types_and_moves(dtype):
    from flash_diffusion_amd.fp8 import Fp8Linear
    src = torch.nn.Linear(100, 60).cuda()
    lin = Fp8Linear.from_linear(src)
    assert not list(lin.parameters()) and set(lin.state_dict()) == {"codes", "scales", "codes_t", "scales_t", "bias"}
    x = _rand(2, 5, 100, seed=1, dtype=dtype).cuda().requires_grad_(True)
    y = lin(x)
    assert y.shape == (2, 5, 60) and y.dtype == dtype
    y.sum().backward()                                        # (an expanded gradient: stride 0)
    assert x.grad.shape == x.shape and x.grad.dtype == dtype and bool(torch.isfinite(x.grad).all())
    other = Fp8Linear(torch.zeros(60, 100, device="cuda"), torch.zeros(60))
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other(x), y) and torch.equal(copy.deepcopy(lin)(x), y)
    assert lin(x[:0]).shape == (0, 5, 60)
    z = lin(x.transpose(0, 1))                                # not contiguous
    assert torch.equal(z, y.transpose(0, 1))


# ---- the lookup's gradients ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [1.0, 0.3])
def test_token_embedding_gradients_of_table_and_positions(scale):
    from flash_diffusion_amd.fp8 import TokenEmbedding
    V, D, B, S = 40, 24, 4, 9
    emb = TokenEmbedding(V, D).cuda()
    ref = torch.nn.Embedding(V, D).double().cuda()
    ref.weight.data.copy_(emb.weight.data)
    pos = _rand(S + 2, D, seed=1).cuda().requires_grad_(True)
    pr = pos.detach().double().requires_grad_(True)
    ids = torch.randint(0, V, (B, S), generator=torch.Generator().manual_seed(2)).cuda()
    c = _rand(B, S, D, seed=3).cuda()
    (emb(ids, scale=scale, pos=pos, dtype=F32) * c).sum().backward()
    ((ref(ids) * scale + pr[:S]) * c.double()).sum().backward()
    cnt = B * S
    assert (emb.weight.grad.double() - ref.weight.grad).abs().max() <= (cnt + 2) * 2.0 ** -24 * c.abs().double().sum(0).sum(0).max()
    assert (pos.grad.double() - pr.grad).abs().max() <= (B + 1) * 2.0 ** -24 * c.abs().double().sum(0).max()
    # against differences: the lookup is linear, so one entry's difference is its gradient up to fp32 rounding of the sums
    with torch.no_grad():
        f = lambda: float((emb(ids, scale=scale, pos=pos, dtype=F32).double() * c.double()).sum())
        t = int(ids[1, 3])
        a = f()
        emb.weight[t, 5] += 1.0
        b = f()
    assert abs((b - a) - float(emb.weight.grad[t, 5])) <= 1e-4


def test_the_encoders_lookup_is_the_gather_it_replaces():
    from flash_diffusion_amd import ops
    w, pos = _rand(300, 64, seed=1).cuda(), _rand(77, 64, seed=2).cuda()
    ids = torch.randint(0, 300, (3, 50), generator=torch.Generator().manual_seed(3)).cuda()
    assert torch.equal(ops.embed_fwd(w, ids, dtype=F32), w[ids]) and torch.equal(ops.embed_fwd(w, ids), w[ids].to(BF16))
    assert torch.equal(ops.embed_fwd(w, ids, pos=pos, dtype=F32), w[ids] + pos[:50]) and torch.equal(ops.embed_fwd(w, ids, pos=pos), (w[ids] + pos[:50]).to(BF16))


def test_the_encoders_embeddings_stay_torchs_and_negative_ids_count_from_the_end():
    from flash_diffusion_amd import ops
    from flash_diffusion_amd.clip import MiCLIPTextModel
    from flash_diffusion_amd.t5 import MiT5EncoderModel
    torch.manual_seed(0)
    t5 = MiT5EncoderModel(vocab_size=20, d_model=16, d_kv=8, d_ff=24, num_layers=1, num_heads=2).cuda()
    clip = MiCLIPTextModel(vocab_size=20, hidden_size=16, intermediate_size=24, num_hidden_layers=1, num_attention_heads=2).cuda()
    ids = torch.tensor([[3, 19, 0, 18], [1, 2, 19, 5]], device="cuda")
    back = torch.where(ids > 10, ids - 20, ids)
    for table in (t5.shared, clip.text_model.embeddings.token_embedding):      # called by itself: fp32, differentiable
        assert table(ids).dtype == F32 and torch.equal(table(ids), table.weight[ids]) and table(ids).requires_grad
        assert torch.equal(ops.embed_fwd(table.weight, back, dtype=F32, wrap=True), table.weight[ids])
        assert bool(torch.isnan(ops.embed_fwd(table.weight, torch.tensor([-21, 20], device="cuda"), wrap=True)).all())
    assert torch.equal(t5(back.int()).last_hidden_state, t5(ids).last_hidden_state)
    # (CLIP's pooled row is taken by the largest id, which the negative form changes)
    assert torch.equal(clip(back).last_hidden_state, clip(ids).last_hidden_state)


def _mixed_step(ops, s):
    n = ops.rmsnorm_fp8(s["x"], None, 1e-6)
    h = ops.gated_fp8(n, s["w0"], s["w1"])
    y = ops.gemm_fp8(h, s["wo"], residual=s["x"])
    return y, ops.gemm_fp8_dgrad(y, s["wo"], out_f32=True), ops.embed_fwd(s["table"], s["ids"]), ops.embed_bwd(y, s["ids"], 300, scale=0.5)


def _mixed_state(ops, seed, rows):
    P = lambda n, k, t=False: ops.pack_weight_fp8((_rand(n, k, seed=seed + n) * k ** -0.5).cuda(), transposed=t)
    ids = torch.randint(0, 300, (rows,), generator=torch.Generator().manual_seed(seed)).cuda()
    return dict(x=_rand(rows, 264, seed=seed, dtype=BF16).cuda(), w0=P(520, 264), w1=P(520, 264), wo=P(264, 520, True),
                table=_rand(300, 264, seed=seed + 1).cuda(), ids=ids)


def test_two_streams_at_once():
    from flash_diffusion_amd import ops
    states = [_mixed_state(ops, seed, rows) for seed, rows in ((1, 700), (2, 90), (3, 3000))]
    want = [_mixed_step(ops, s) for s in states]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in states], [[] for _ in states]
    for _ in range(10):
        for i, (st, s) in enumerate(zip(streams, states)):
            with torch.cuda.stream(st):
                got[i].append(_mixed_step(ops, s))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(w, r))


def test_two_graphs_of_one_pool_replayed_in_turns():
    """their scratch lies in one pool: each replay recomputes what it reads"""
    from flash_diffusion_amd import ops
    a, b = _mixed_state(ops, 4, 400), _mixed_state(ops, 5, 1500)
    for s in (a, b):
        _mixed_step(ops, s)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        ya = _mixed_step(ops, a)
    with torch.cuda.graph(gb, pool=ga.pool()):
        yb = _mixed_step(ops, b)
    for seed in (6, 7, 8):
        a["x"].copy_(_rand(400, 264, seed=seed))
        b["x"].copy_(_rand(1500, 264, seed=seed + 9))
        for g, y, s in ((ga, ya, a), (gb, yb, b), (ga, ya, a)):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(y, _mixed_step(ops, s)))
