"""CPU: sizes beyond what one launch holds are refused by name, before anything is launched."""
import ctypes as C

import pytest

from tests.test_fp8_host import GATED, P, _desc, _lib


@pytest.mark.parametrize("kw", [dict(M=1 << 30, N=64, K=64, ldc=64), dict(M=1 << 30, N=64, K=64, ldc=64, out_f32=1), dict(M=1 << 30, N=1, K=128, ldc=1),
                                {**GATED, "M": 1 << 30, "N": 1 << 17, "K": 64}, {**GATED, "M": 1 << 30, "N": 1 << 17, "K": 4096}])
def test_a_product_of_too_many_tiles(kw):
    L = _lib().lib()
    assert L.fdmi_gemm_fp8(C.byref(_desc(**kw)), None) != 0 and b"too many tiles" in L.fdmi_last_error()


@pytest.mark.parametrize("n,D,f32", [(0, 65535 * 256 + 1, 1), (3, 1 << 25, 0), (1 << 17, 1 << 21, 1), (1 << 30, (1 << 21) + 1, 1)])
def test_a_gradient_of_too_many_columns(n, D, f32):
    L = _lib().lib()
    assert L.fdmi_embed_bwd(P, f32, D, P, 1, n, 10, D, 1.0, 0, P, D, P, None) != 0 and b"too many columns" in L.fdmi_last_error()
