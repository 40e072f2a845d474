"""fp8.Fp8Linear and fp8.TokenEmbedding on inputs as a program has them: any layout, weights that are loaded between forward and backward."""
import pytest
import torch

from tests.test_fp8_linear_host import INPUTS

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", list(INPUTS))
def test_a_layout_gives_what_its_copy_gives(kind, dtype):
    from flash_diffusion_amd.fp8 import Fp8Linear
    lin = Fp8Linear(_rand(60, 5, seed=1).cuda(), _rand(60, seed=2).cuda())
    a = _rand(5, 4, dtype=dtype).cuda().requires_grad_()
    b = a.detach().clone().requires_grad_()
    x, c = INPUTS[kind](a), INPUTS[kind](b).contiguous()
    y, z = lin(x), lin(c)
    assert y.shape == (*x.shape[:-1], 60) and y.dtype == dtype and torch.equal(y, z)
    y.sum().backward()
    z.sum().backward()
    assert torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("shape", [(), (1,), (2, 0), (2, 1, 30)])
def test_gradients_of_table_and_positions_for_ids_of_any_shape(shape):
    from flash_diffusion_amd.fp8 import TokenEmbedding
    emb = TokenEmbedding(40, 24).cuda()
    ids = torch.randint(0, 40, shape, generator=torch.Generator().manual_seed(1)).cuda()
    pos = _rand(33, 24, seed=2).cuda().requires_grad_()
    c = _rand(*shape, 24, seed=3).round().cuda()                # (integers: sums are exact)
    (emb(ids, pos=pos, dtype=F32) * c).sum().backward()
    w, q = emb.weight.detach().clone().requires_grad_(), pos.detach().clone().requires_grad_()
    t = torch.arange(shape[-1] if shape else 1, device="cuda")
    ((w[ids] + q[t].view(*ids.shape[-1:], 24)) * c).sum().backward()
    assert torch.equal(emb.weight.grad, w.grad) and torch.equal(pos.grad, q.grad)
