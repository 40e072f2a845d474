"""CPU: which results over operands the 8-bit products accept, on a stand-in of the library that launches nothing."""
import pytest
import torch

from flash_diffusion_amd import ops

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture
def W(monkeypatch):
    class Lib:
        def fdmi_gemm_fp8(self, d, stream):
            return 0

        def fdmi_fp8_scratch_bytes(self, M, K):
            return 0

    monkeypatch.setattr(ops, "_here", lambda t, what: t)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    monkeypatch.setattr(ops, "lib", Lib)
    monkeypatch.setattr(ops, "check", lambda rc: None)
    return ops.Fp8Weight(8, 16, "cpu", True)


def test_one_row_may_be_the_residual_whatever_its_stride(W):
    """(the stride of a single row says nothing)"""
    x, big = torch.zeros(1, 16, dtype=BF16), torch.zeros(4, 20, dtype=BF16)
    row = big[2, 3:11]
    for res, out in ((row.view(1, 8), big[2:3, 3:11]), (big[2:3, 3:11], row.view(1, 8)), (row.view(1, 8), row.view(1, 8))):
        assert ops.gemm_fp8(x, W, residual=res, out=out) is out
    with pytest.raises(ValueError, match="residual"):
        ops.gemm_fp8(x, W, residual=big[2:3, 4:12], out=row.view(1, 8))
    with pytest.raises(ValueError, match="residual"):
        ops.gemm_fp8(torch.zeros(2, 16, dtype=BF16), W, residual=big[:2, :8], out=big.view(-1)[:16].view(2, 8))


def test_a_result_over_the_bias_is_refused(W):
    """(workgroups read it while others already write)"""
    x, out = torch.zeros(3, 16), torch.zeros(3, 8)
    with pytest.raises(ValueError, match="bias"):
        ops.gemm_fp8(x, W, bias=out[1], out=out)
    assert ops.gemm_fp8(x, W, bias=torch.zeros(8), out=out) is out
