"""The text encoder in 8 bits (MiT5EncoderModel(precision="fp8")): every stage of every block against its 64-bit form on that stage's own input
(tests/fp8_stages.py), and the encoder's distance from the unquantised one."""
import numpy as np
import pytest
import torch

from tests import fp8_stages as S
from tests.golden_util import parity_log, rel_err
from tests.test_fp8_layers_gpu import _emulated
from tests.test_t5_gpu import CASES, _hf

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _np(t):
    return t.detach().double().cpu().numpy()


def _encoder(kw):
    from flash_diffusion_amd.t5 import MiT5EncoderModel
    hf = _hf(kw)
    mi = MiT5EncoderModel(**kw, precision="fp8")
    mi.load_state_dict(hf.state_dict(), strict=True)
    mi = mi.cuda()
    mi.freeze()
    return hf, mi


def _prompts(kw, B, S_):
    g = torch.Generator().manual_seed(1)
    ids, mask = torch.randint(2, kw["vocab_size"], (B, S_), generator=g), torch.ones(B, S_, dtype=torch.long)
    ids[0, S_ // 3:], mask[0, S_ // 3:] = 0, 0
    return ids, mask


@pytest.mark.parametrize("name", list(CASES))
def test_every_stage_is_its_64_bit_form(name, monkeypatch):
    from flash_diffusion_amd import ops
    from flash_diffusion_amd.t5 import relative_position_bucket
    kw = CASES[name]
    hf, mi = _encoder(kw)
    seen = []

    def record(f):
        plain = getattr(ops, f)

        def call(*a, **k):
            r = plain(*a, **k)
            seen.append((f, a, k, r))
            return r

        monkeypatch.setattr(ops, f, call)

    for f in ("rmsnorm_fp8", "gemm_fp8", "gated_fp8", "attn_bias_fwd", "rmsnorm"):
        record(f)
    B, T, H, d = 2, 40, kw["num_heads"], kw["d_kv"]
    ids, mask = _prompts(kw, B, T)
    out = mi(ids.cuda(), attention_mask=mask.cuda())
    gated = kw["feed_forward_proj"] == "gated-gelu"
    order = ["rmsnorm_fp8", "gemm_fp8", "gemm_fp8", "gemm_fp8", "attn_bias_fwd", "gemm_fp8", "rmsnorm_fp8", "gated_fp8" if gated else "gemm_fp8", "gemm_fp8"]
    L = kw["num_layers"]
    assert [s[0] for s in seen] == order * L + ["rmsnorm"]

    def codes(q):
        c, e = q.parts()
        e = e.view(torch.uint8).cpu().numpy().astype(np.int64) - 127
        return _np(c.float()) * np.repeat(2.0 ** e.astype(np.float64), 128, 1)[:, :q.K], e

    rows = lambda t: _np(t).reshape(B * T, -1)
    p = {k: _np(v) for k, v in hf.state_dict().items()}
    pos = torch.arange(T)
    bucket = relative_position_bucket(pos[None] - pos[:, None], kw.get("relative_attention_num_buckets", 32),
                                      kw.get("relative_attention_max_distance", 128)).numpy()
    bias = p["encoder.block.0.layer.0.SelfAttention.relative_attention_bias.weight"][bucket].transpose(2, 0, 1)
    kb = np.where(mask.numpy() > 0, 0.0, float(torch.finfo(F32).min))
    for i in range(L):
        n1, q, k, v, o, h1, n2, f, h2 = (s[3] for s in seen[9 * i:9 * i + 9])
        a, b = f"encoder.block.{i}.layer.0.", f"encoder.block.{i}.layer.1."
        w = {m: p[a + f"SelfAttention.{m}.weight"] for m in "qkvo"}
        w.update({m: p[b + f"DenseReluDense.{m}.weight"] for m in (("wi_0", "wi_1", "wo") if gated else ("wi", "wo"))})
        w.update(norm1=p[a + "layer_norm.weight"], norm2=p[b + "layer_norm.weight"])
        rec = dict(h_in=rows(seen[9 * i][1][0]), n1=codes(n1), q=rows(q), k=rows(k), v=rows(v), o=rows(o), h1=rows(h1), n2=codes(n2),
                   f=codes(f) if gated else rows(f), h_out=rows(h2))
        out_of = S.excess(rec, w, dict(eps=1e-6, gated=gated), bias, kb, (B, T, H, d))
        print(name, i, {m: f"{x:.1e}" for m, x in out_of.items()})
        assert all(x <= 0 for x in out_of.values()), (i, out_of)
        # a block begins with what the one before left, the first with the table's rows
        assert np.array_equal(rec["h_in"], rows(seen[9 * i - 1][3]) if i else rows(torch.from_numpy(p["shared.weight"][ids.numpy()]).to(BF16)))
    last = seen[-1]
    assert np.array_equal(rows(last[1][0]), rows(seen[-2][3])) and torch.equal(last[3].float().view_as(out.last_hidden_state), out.last_hidden_state)


@pytest.mark.parametrize("layers", [1, None])
@pytest.mark.parametrize("name", list(CASES))
def test_the_distance_from_the_unquantised_encoder(name, layers):
    """what the format costs: in the 2-norm over last_hidden_state, the definition's own distance from transformers' fp32 encoder (its 64-bit
    emulation) and what products off by 2^-13 of their root mean square may add to it (the emulation's answer, twice)"""
    kw = dict(CASES[name], num_layers=layers or CASES[name]["num_layers"])
    hf, mi = _encoder(kw)
    ids, mask = _prompts(kw, 2, 60)
    with torch.no_grad():
        want = _np(hf(input_ids=ids, attention_mask=mask).last_hidden_state)
    own = _emulated(hf, kw, ids, mask)
    dist = lambda a, b: np.linalg.norm(a - b) / np.linalg.norm(want)
    bar = dist(own, want) + 2.0 * dist(_emulated(hf, kw, ids, mask, jitter=2.0 ** -13), own)
    err = rel_err(mi(ids.cuda(), attention_mask=mask.cuda()).last_hidden_state, torch.from_numpy(want))
    msg = f"t5 fp8 {name} x {kw['num_layers']}: {err:.2e} from transformers fp32; its 64-bit emulation {dist(own, want):.2e}, bar {bar:.2e}"
    parity_log(msg, "nets_parity.txt")
    assert err <= bar
