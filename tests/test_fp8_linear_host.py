"""CPU: what fp8.Fp8Linear and fp8.TokenEmbedding hand to the products and the lookup, on plain stand-ins of those that keep their checks."""
import pytest
import torch

from flash_diffusion_amd import fp8, ops

F32 = torch.float32


class _Weight:
    """a weight in the place of ops.Fp8Weight, and as the buffers that Fp8Linear keeps: its values, and those of its transpose"""

    def __init__(self, w):
        self.N, self.K = w.shape
        self.codes = self.scales = self.scales_t = w.detach().clone()
        self.codes_t = w.detach().t().clone()


@pytest.fixture
def linear(monkeypatch):
    """a Fp8Linear over plain fp32 products (the checks of their operands are the entry points' own)"""
    monkeypatch.setattr(ops, "_here", lambda t, what: t)
    monkeypatch.setattr(ops, "pack_weight_fp8", lambda w, transposed=False: _Weight(w))

    def product(A, W, bias=None, out_f32=False):
        ops._rows(A, "A")
        y = A.float() @ W.codes.t()
        return (y if bias is None else y + bias).to(F32 if out_f32 else torch.bfloat16)

    def dgrad(dY, W, out_f32=False):
        ops._rows(dY, "dY")
        return (dY.float() @ W.codes_t.t()).to(F32 if out_f32 else torch.bfloat16)

    monkeypatch.setattr(ops, "gemm_fp8", product)
    monkeypatch.setattr(ops, "gemm_fp8_dgrad", dgrad)
    return fp8.Fp8Linear(torch.randn(6, 5, generator=torch.Generator().manual_seed(0)), torch.arange(6.0))


INPUTS = {"transposed": lambda x: x.t(), "one row for all": lambda x: x[:, :1].t().expand(7, 5), "one row in a batch": lambda x: x[:, 0].expand(2, 3, 5),
          "overlapping rows": lambda x: x.reshape(-1).as_strided((8, 5), (2, 1)), "a vector": lambda x: x[:, 2], "every second column": lambda x: x.reshape(-1, 10)[:, ::2],
          "batch moved": lambda x: x.t().reshape(2, 2, 5).transpose(0, 1), "no rows": lambda x: x.t()[:0], "rows apart": lambda x: x.reshape(-1, 10)[:, :5]}


@pytest.mark.parametrize("kind", list(INPUTS))
def test_linear_takes_inputs_of_any_layout(linear, kind):
    base = torch.randn(5, 4, generator=torch.Generator().manual_seed(1)).requires_grad_()
    x = INPUTS[kind](base)
    w, b = linear.codes, linear.bias
    y = linear(x)
    want = torch.nn.functional.linear(x, w, b)
    assert y.shape == want.shape and torch.allclose(y, want, atol=1e-5)
    (got,) = torch.autograd.grad(y.sum(), base)
    assert torch.allclose(got, torch.autograd.grad(want.sum(), base)[0], atol=1e-5)


def test_a_backward_behind_a_weight_that_was_overwritten_is_refused(linear):
    """as torch's own layers do: the gradient would be that of another weight than the forward's"""
    x = torch.randn(3, 5).requires_grad_()
    y = linear(x)
    other = {k: v * 2.0 for k, v in linear.state_dict().items()}
    linear.load_state_dict(other)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    linear(x).sum().backward()
    assert torch.allclose(x.grad, linear.codes.sum(0).expand(3, 5), atol=1e-5)


@pytest.fixture
def embedding(monkeypatch):
    """a TokenEmbedding over plain fp32 sums (the gradient's own check of shapes)"""
    monkeypatch.setattr(ops, "embed_fwd", lambda w, ids, scale=1.0, pos=None, dtype=F32:
                        (w[ids] * scale + (0.0 if pos is None else pos[:ids.shape[-1] if ids.dim() else 1].view(*ids.shape[-1:], 4))).to(dtype))

    def grad(dy, ids, V, scale=1.0):
        assert dy.shape[:-1] == ids.shape and ids.is_contiguous()
        return torch.zeros(V, dy.shape[-1]).index_add_(0, ids.reshape(-1).long(), scale * dy.reshape(ids.numel(), dy.shape[-1]))

    monkeypatch.setattr(ops, "embed_bwd", grad)
    return fp8.TokenEmbedding(9, 4)


@pytest.mark.parametrize("shape", [(), (1,), (3,), (2, 3), (2, 0), (2, 1, 3)])
def test_gradients_of_table_and_positions_for_ids_of_any_shape(embedding, shape):
    ids = torch.randint(0, 9, shape, generator=torch.Generator().manual_seed(1))
    pos = torch.randn(5, 4, generator=torch.Generator().manual_seed(2)).requires_grad_()
    c = torch.randn(*shape, 4, generator=torch.Generator().manual_seed(3))
    (embedding(ids, scale=0.5, pos=pos, dtype=F32) * c).sum().backward()
    w, q = embedding.weight.detach().clone().requires_grad_(), pos.detach().clone().requires_grad_()
    t = torch.arange(shape[-1]) if shape else torch.tensor(0)
    ((w[ids] * 0.5 + q[t]) * c).sum().backward()
    assert torch.allclose(embedding.weight.grad, w.grad, atol=1e-6) and torch.allclose(pos.grad, q.grad, atol=1e-6)


def test_backwards_that_a_frozen_weight_allows(linear):
    """a second backward needs nothing that the first one frees, and a layer made in inference mode passes gradients on"""
    x = torch.randn(3, 5).requires_grad_()
    y = linear(x).sum()
    y.backward()
    with torch.inference_mode():
        made = fp8.Fp8Linear(torch.ones(6, 5))
    z = torch.randn(3, 5).requires_grad_()
    made(z).sum().backward()
    assert torch.equal(z.grad, torch.full((3, 5), 6.0))
    first = linear(x)
    g = torch.ones_like(first)
    a, b = torch.autograd.grad(first, x, g)[0], torch.autograd.grad(first, x, g)[0]
    assert torch.equal(a, b)
