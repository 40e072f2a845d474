"""CPU: what the 8-bit product and embedding entry points refuse before anything is launched, and the wrappers' checks of host tensors."""
import ctypes as C

import pytest
import torch

P = 1 << 20          # an address that is aligned and never read: every call below is refused by its arguments


def _lib():
    from flash_diffusion_amd import _lib
    return _lib


def _desc(**kw):
    d = _lib().Fp8Desc()
    base = dict(M=4, N=64, K=130, X=P, sx=P, W=P, sw=P, C=P, ldc=64)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


GATED = dict(W2=P, sw2=P, C=None, H=P, sh=P)


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(N=0), dict(K=0), dict(X=None), dict(X=P + 8), dict(sx=None), dict(sx=P + 2), dict(W=None), dict(W=P + 4), dict(sw=None),
    dict(sw=P + 1), dict(C=None), dict(ldc=63), dict(act=2), dict(act=6), dict(act=-1), dict(act=3, residual=P, ldr=64),
    dict(residual=P, ldr=63), dict(x=P, ldxr=129), dict(H=P), dict(sh=P), dict(K=(1 << 17) + 1),
    {**GATED, "C": P}, {**GATED, "sw2": None}, {**GATED, "W2": P + 8}, {**GATED, "H": None}, {**GATED, "H": P + 4}, {**GATED, "sh": None},
    {**GATED, "bias": P}, {**GATED, "act": 5}, {**GATED, "residual": P, "ldr": 64}])
def test_gemm_fp8_refuses(kw):
    L = _lib().lib()
    d = _desc(**kw)
    assert L.fdmi_gemm_fp8(C.byref(d), None) != 0
    assert b"gemm_fp8" in L.fdmi_last_error()


@pytest.mark.parametrize("kw", [dict(M=(1 << 30) + 1), dict(N=(1 << 17) + 1, ldc=1 << 18), {**GATED, "N": (1 << 17) + 1}])
def test_gemm_fp8_refuses_sizes_beyond_its_indexes(kw):
    L = _lib().lib()
    assert L.fdmi_gemm_fp8(C.byref(_desc(**kw)), None) != 0 and b"gemm_fp8" in L.fdmi_last_error()
    assert L.fdmi_quant_fp8(P, 0, 130, None, 0.0, P, P, (1 << 30) + 1, 130, None) != 0 and b"quant_fp8" in L.fdmi_last_error()


def test_shared_memory_of_rows_is_seen():
    """(what a product refuses of out: the check itself, on host tensors)"""
    from flash_diffusion_amd.ops import _overlap
    b = torch.zeros(10, 40)
    assert _overlap(b, b) and _overlap(b[:, :20], b[:, 19:]) and _overlap(b[2:5], b[4:8]) and _overlap(b[:, 5:9], b[3:4, 8:30])
    assert not _overlap(b[:, :20], b[:, 20:]) and not _overlap(b[:, 20:], b[:, :20]) and not _overlap(b[:5], b[5:]) and not _overlap(b, torch.zeros(10, 40))
    assert not _overlap(b[2:, 3:7], b[:-2, 7:20]) and not _overlap(b[:0], b) and _overlap(b[1:9:2, :20], b[1:9, :10])
    assert _overlap(b[:9, 30:40], b.view(-1)[35:35 + 9 * 40].view(9, 40)[:, :10])          # runs over the end of a row


def test_empty_calls_are_accepted_without_a_gpu():
    L = _lib().lib()
    assert L.fdmi_gemm_fp8(C.byref(_desc(M=0)), None) == 0
    assert L.fdmi_quant_fp8(None, 0, 130, None, 0.0, None, None, 0, 130, None) == 0
    assert L.fdmi_embed_fwd(None, 1, 10, 8, 8, None, 1, 0, 1.0, None, 0, 0, None, 0, None) == 0
    assert L.fdmi_embed_bwd_ws_bytes(0, 8) == 0 and L.fdmi_embed_bwd_ws_bytes(33, 8) >= 33 * 8 + 2 * 2 * 8 * 4


@pytest.mark.parametrize("args", [
    (None, 0, 130, None, 0.0, P, P, 3, 130), (P, 0, 129, None, 0.0, P, P, 3, 130), (P, 0, 130, None, 0.0, P + 1, P, 3, 130),
    (P, 0, 130, None, 0.0, None, P, 3, 130), (P, 0, 130, None, 0.0, P, P + 2, 3, 130), (P, 0, 130, None, 0.0, P, P, -3, 130),
    (P, 0, 130, None, 0.0, P, P, 3, 0)])
def test_quant_fp8_refuses(args):
    L = _lib().lib()
    assert L.fdmi_quant_fp8(*args, None) != 0 and b"quant_fp8" in L.fdmi_last_error()


@pytest.mark.parametrize("args", [
    (P, 1, 130, 0, 130, P, P, None, None), (None, 1, 130, 64, 130, P, P, None, None), (P, 1, 100, 64, 130, P, P, None, None),
    (P, 1, 130, 64, 130, P + 4, P, None, None), (P, 1, 130, 64, 130, P, None, None, None), (P, 1, 130, 64, 130, P, P, P + 8, P),
    (P, 1, 130, 64, 130, P, P, P, None)])
def test_pack_fp8_refuses(args):
    L = _lib().lib()
    assert L.fdmi_pack_fp8(*args, None) != 0 and b"pack_fp8" in L.fdmi_last_error()


def test_embed_refuses():
    L = _lib().lib()
    for a in ((P, 1, 0, 8, 8, P, 1, 3, 1.0, None, 0, 0, P, 0), (P, 1, 10, 0, 8, P, 1, 3, 1.0, None, 0, 0, P, 0), (P, 1, 10, 8, 7, P, 1, 3, 1.0, None, 0, 0, P, 0),
              (P, 1, 10, 8, 8, None, 1, 3, 1.0, None, 0, 0, P, 0), (P, 1, 10, 8, 8, P, 1, 3, 1.0, P, 0, 8, P, 0), (P, 1, 10, 8, 8, P, 1, 3, 1.0, P, 3, 7, P, 0),
              (P, 1, 10, 8, 8, P, 1, -1, 1.0, None, 0, 0, P, 0), (P, 1, 10, 8, 8, P, 1, 3, 1.0, None, 0, 0, None, 0), (P, 1, 1 << 31, 8, 8, P, 1, 3, 1.0, None, 0, 0, P, 0)):
        assert L.fdmi_embed_fwd(*a, None) != 0 and b"embed_fwd" in L.fdmi_last_error()
    for a in ((P, 1, 8, P, 1, 3, 0, 8, 1.0, 0, P, 8, P), (P, 1, 7, P, 1, 3, 10, 8, 1.0, 0, P, 8, P), (P, 1, 8, P, 1, 3, 10, 8, 1.0, 0, P, 7, P), (P, 1, 8, P, 1, 3, 10, 8, 1.0, 0, None, 8, P),
              (P, 1, 8, P, 1, 3, 10, 8, 1.0, 0, P, 8, None), (P, 1, 8, P, 1, 3, 10, 8, 1.0, 0, P, 8, P + 4), (P, 1, 8, P, 1, 1 << 31, 10, 8, 1.0, 0, P, 8, P)):
        assert L.fdmi_embed_bwd(*a, None) != 0 and b"embed_bwd" in L.fdmi_last_error()


def test_wrappers_refuse_host_tensors():
    from flash_diffusion_amd import ops
    x = torch.zeros(4, 130)
    for f in (lambda: ops.quant_fp8(x), lambda: ops.rmsnorm_fp8(x, torch.ones(130), 1e-6), lambda: ops.pack_weight_fp8(x),
              lambda: ops.embed_fwd(x, torch.zeros(3, dtype=torch.int64)), lambda: ops.embed_bwd(x, torch.zeros(4, dtype=torch.int64), 9)):
        with pytest.raises(ValueError, match="current GPU"):
            f()


def test_the_reference_quantiser_agrees_with_torchs_cast():
    """the 64-bit form the GPU tests compare with, against torch's own e4m3 rounding of the scaled values (CPU)"""
    import numpy as np
    from tests import fp8_ref as R
    g = torch.Generator().manual_seed(0)
    x = torch.randn(9, 700, generator=g) * torch.exp(3 * torch.randn(700, generator=g))
    got, exps = R.quantise(x.numpy())
    s = torch.from_numpy(2.0 ** np.repeat(exps, 128, 1)[:, :700].astype(np.float64))
    want = (x.double() / s).float().to(torch.float8_e4m3fn).double() * s
    assert np.array_equal(got, want.numpy())
    m = np.abs(np.pad(x.numpy(), ((0, 0), (0, 68))).reshape(9, 6, 128)).max(2)
    sc = 2.0 ** exps.astype(np.float64)
    assert (m <= 448 * sc).all() and (m > 224 * sc).all()


def test_layers_refuse_what_they_do_not_implement_and_caches_copy_empty():
    import copy
    import pickle
    from flash_diffusion_amd.fp8 import PackedFp8, TokenEmbedding
    for kw in (dict(padding_idx=0), dict(max_norm=1.0), dict(scale_grad_by_freq=True), dict(sparse=True)):
        with pytest.raises(NotImplementedError):
            TokenEmbedding(10, 4, **kw)
    assert set(TokenEmbedding(10, 4).state_dict()) == {"weight"}
    p = PackedFp8(transposed=True)
    p._of = object()
    for c in (copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert c.transposed and c._of is None


def test_t5_and_clip_keep_their_state_dict_names_and_modes():
    from flash_diffusion_amd.clip import MiCLIPTextModel
    from flash_diffusion_amd.t5 import MiT5EncoderModel
    kw = dict(vocab_size=20, d_model=16, d_kv=8, d_ff=24, num_layers=1, num_heads=2)
    for precision in ("bf16", "fp32", "fp8"):
        sd = MiT5EncoderModel(**kw, precision=precision).state_dict()
        assert {"shared.weight", "encoder.embed_tokens.weight", "encoder.block.0.layer.1.DenseReluDense.wi_1.weight"} <= set(sd)
        assert not any("operand8" in k for k in sd)
    with pytest.raises(AssertionError):
        MiT5EncoderModel(**kw, precision="int8")
    assert "text_model.embeddings.token_embedding.weight" in MiCLIPTextModel(vocab_size=20, hidden_size=16, intermediate_size=24, num_hidden_layers=1, num_attention_heads=2).state_dict()
