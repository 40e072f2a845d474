"""The text encoders' lookups: position rows by position_ids, tables of the types and layouts that indexing takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _clip(precision="fp32", **kw):
    from flash_diffusion_amd.clip import MiCLIPTextModel
    torch.manual_seed(0)
    m = MiCLIPTextModel(vocab_size=50, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=2, max_position_embeddings=20,
                        precision=precision, **kw).cuda()
    m.freeze()
    return m


def _t5(precision="fp32"):
    from flash_diffusion_amd.t5 import MiT5EncoderModel
    torch.manual_seed(0)
    m = MiT5EncoderModel(vocab_size=50, d_model=32, d_kv=16, d_ff=64, num_layers=2, num_heads=2, precision=precision).cuda()
    m.freeze()
    return m


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
def test_clips_position_rows_are_those_of_position_ids(precision):
    """a caller's own positions: as position rows in that order"""
    a, b = _clip(precision), _clip(precision)
    ids = torch.randint(0, 50, (3, 11), generator=torch.Generator().manual_seed(1)).cuda()
    order = torch.randperm(20, generator=torch.Generator().manual_seed(2)).cuda()
    plain = a(ids).last_hidden_state
    a.text_model.embeddings.position_ids = order[None]
    pos = b.text_model.embeddings.position_embedding
    pos.weight = torch.nn.Parameter(pos.weight[order], requires_grad=False)
    got, want = (m(ids, output_hidden_states=True) for m in (a, b))
    assert torch.equal(got.hidden_states[0], want.hidden_states[0]) and torch.equal(got.last_hidden_state, want.last_hidden_state)
    assert torch.equal(a(ids).last_hidden_state, want.last_hidden_state) and not torch.equal(plain, want.last_hidden_state)
    with pytest.raises((ValueError, RuntimeError)):
        a(torch.zeros(1, 21, dtype=torch.long, device="cuda"))


KINDS = {"half": lambda w: w.half(), "double": lambda w: w.double(), "bf16": lambda w: w.to(BF16), "transposed": lambda w: w.t().contiguous().t()}


@pytest.mark.parametrize("kind", list(KINDS))
def test_tables_of_other_types_and_layouts(kind):
    ids = torch.randint(0, 50, (3, 11), generator=torch.Generator().manual_seed(1)).cuda()

    def outputs(build, tables, change):
        m = build()
        for t in tables(m):
            t.weight = torch.nn.Parameter(change(t.weight.data), requires_grad=False)
        o = m(ids, output_hidden_states=True)
        return torch.stack([o.last_hidden_state, *(h.float() for h in o.hidden_states)])

    values = lambda w: KINDS[kind](w).float().contiguous()               # the same values in fp32
    for build, tables in ((_t5, lambda m: [m.shared]), (_clip, lambda m: [m.text_model.embeddings.token_embedding]),
                          (_clip, lambda m: [m.text_model.embeddings.position_embedding])):
        assert torch.equal(outputs(build, tables, KINDS[kind]), outputs(build, tables, values))
