"""The operators around the frozen text encoders that are timed and checked: the 8-bit matrix product with a scale for each block of
128 (forward, the gated feed-forward built from it, the gradient of its input) and the token-embedding lookup with its gradient.

The 8-bit format: along the contraction every 128 values of a row of activations share one power-of-two scale, every 128 x 128 values
of a weight share one; 2^e is the smallest power with amax <= 448 2^e, a code is the value / 2^e rounded to e4m3 (to nearest, ties to
even).  Products of codes are summed in 32 bits or more, the result is rounded once.

`own` False: elementary torch operations in fp32; `own` True: the framework's entry points."""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GELU_C = math.sqrt(2.0 / math.pi)
EPS = 1e-6          # T5LayerNorm


def listed():
    return [
        # the text encoders' products.  An empty prompt is one token: a matrix-vector product that streams the weight once
        dict(name="linear 1 token 4096x4096", op="linear", rows=1, k=4096, n=4096, x="bf16", y="bf16", bias=False, residual=True),
        # two SD3 prompts (77 + 256 tokens) and sizes that divide by nothing
        dict(name="linear 666 1155x1537", op="linear", rows=666, k=1155, n=1537, x="f32", y="f32", bias=True, residual=False),
        # 16 prompts of 120 tokens (PixArt) through T5-XXL's o projection with the residual
        dict(name="linear 1920 4096x4096", op="linear", rows=1920, k=4096, n=4096, x="bf16", y="bf16", bias=False, residual=True),
        # 64 prompts of 256 tokens (SD3) through wi of T5-XXL: the largest product
        dict(name="linear 16384 4096x10240", op="linear", rows=16384, k=4096, n=10240, x="bf16", y="bf16", bias=False, residual=False),
        # the gated feed-forward block of a quarter-width T5 on one prompt, and of T5-XXL on 16 prompts
        dict(name="feed-forward 120 1024x2560", op="feed_forward", rows=120, d=1024, f=2560),
        dict(name="feed-forward 1920 4096x10240", op="feed_forward", rows=1920, d=4096, f=10240),
        # what a learned token table in front of frozen 8-bit layers needs: the input gradient of a product
        dict(name="input gradient 231 1155x770", op="input_gradient", rows=231, k=1155, n=770, dy="f32", dx="f32"),
        dict(name="input gradient 1920 4096x10240", op="input_gradient", rows=1920, k=4096, n=10240, dy="bf16", dx="bf16"),
        # CLIP's lookup of 2 prompts with position rows; 64 T5 prompts of 512 tokens
        dict(name="embedding 2x77 768", op="embedding", batch=2, length=77, vocab=49408, d=768, scale=1.0, pos=True),
        dict(name="embedding 64x512 4096", op="embedding", batch=64, length=512, vocab=32128, d=4096, scale=0.5, pos=False),
        # the gradients of the two tables: CLIP's for 16 prompts, T5's for 32 (most tokens of a batch are padding)
        dict(name="embedding gradient 16x77 768", op="embedding_gradient", batch=16, length=77, vocab=49408, d=768, scale=1.0, dy="f32"),
        dict(name="embedding gradient 32x512 4096", op="embedding_gradient", batch=32, length=512, vocab=32128, d=4096, scale=0.5,
             dy="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "feed_forward", "input_gradient", "embedding", "embedding_gradient"])
    if op in ("linear", "input_gradient"):
        while True:
            rows, k, n = _log(rng, 1, 16384), _log(rng, 64, 10240), _log(rng, 64, 12288)
            if rng.random() < 0.5:
                k, n = -(-k // 128) * 128, -(-n // 64) * 64
            if rows * k * n <= 16384 * 4096 * 10240:
                break
        a, b = rng.choice(["bf16", "f32"]), rng.choice(["bf16", "f32"])
        if op == "linear":
            return dict(op=op, rows=rows, k=k, n=n, x=a, y=b, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
        return dict(op=op, rows=rows, k=k, n=n, dy=a, dx=b)
    if op == "feed_forward":
        return dict(op=op, rows=_log(rng, 1, 4096), d=8 * _log(rng, 8, 512), f=8 * _log(rng, 8, 1280))
    batch, length = _log(rng, 1, 64), _log(rng, 1, 512)
    vocab, d = _log(rng, 300, 49408), _log(rng, 64, 2048)
    scale = rng.choice([1.0, 0.5, math.sqrt(d)])
    if op == "embedding":
        return dict(op=op, batch=batch, length=length, vocab=vocab, d=d, scale=scale, pos=rng.random() < 0.5)
    return dict(op=op, batch=batch, length=length, vocab=vocab, d=d, scale=scale, dy=rng.choice(["bf16", "f32"]))


# ---- inputs ----------------------------------------------------------------------------------------------------------------------
def _activations(g, rows, width, dtype):
    """hidden states of a text encoder: normal values, channels of unequal size, a few of them far larger than the others"""
    size = torch.exp(0.5 * torch.randn(width, generator=g, device="cuda"))
    size = torch.where(torch.rand(width, generator=g, device="cuda") < 0.01, 20.0 * size, size)
    return (torch.randn(rows, width, generator=g, device="cuda") * size).to(dtype)


def _matrix(g, n, k):
    return torch.randn(n, k, generator=g, device="cuda") * k ** -0.5


def _tokens(g, batch, length, vocab):
    """prompts of unequal length, frequent words more often than rare ones, id 0 behind each prompt's end"""
    u = torch.rand(batch, length, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.exp(u * math.log(vocab)).long().clamp(1, vocab) - 1
    ends = torch.randint(1, length + 1, (batch, 1), generator=g, device="cuda")
    return torch.where(torch.arange(length, device="cuda")[None] < ends, ids, torch.zeros_like(ids))


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "linear":
        s = dict(x=_activations(g, case["rows"], case["k"], TYPES[case["x"]]), w=_matrix(g, case["n"], case["k"]))
        s["bias"] = torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
        s["residual"] = torch.randn(case["rows"], case["n"], generator=g, device="cuda").to(TYPES[case["y"]]) if case["residual"] else None
        return s
    if op == "feed_forward":
        d, f = case["d"], case["f"]
        return dict(x=_activations(g, case["rows"], d, torch.bfloat16), norm=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"),
                    wi_0=_matrix(g, f, d), wi_1=_matrix(g, f, d), wo=_matrix(g, d, f))
    if op == "input_gradient":
        return dict(dy=1e-3 * _activations(g, case["rows"], case["n"], TYPES[case["dy"]]).float(), w=_matrix(g, case["n"], case["k"]))
    if op == "embedding":
        s = dict(table=torch.randn(case["vocab"], case["d"], generator=g, device="cuda"),
                 ids=_tokens(g, case["batch"], case["length"], case["vocab"]))
        s["pos"] = torch.randn(case["length"], case["d"], generator=g, device="cuda") if case["pos"] else None
        return s
    ids = _tokens(g, case["batch"], case["length"], case["vocab"])
    return dict(ids=ids, dy=torch.randn(case["batch"], case["length"], case["d"], generator=g, device="cuda").to(TYPES[case["dy"]]))


_WEIGHTS = ("w", "wi_0", "wi_1", "wo")


def prepare(case, seed):
    """The inputs, and the weights in the 8-bit form that a program keeps of them: codes and scales here, the framework's handle there
    (an input gradient's handle holds the transposed codes as well)."""
    s = _inputs(case, seed)
    if case["op"] == "input_gradient":
        s["dy"] = s["dy"].to(TYPES[case["dy"]])
    for name in _WEIGHTS:
        if name in s:
            if own:
                from flash_diffusion_amd import ops
                s[name] = ops.pack_weight_fp8(s[name], transposed=case["op"] == "input_gradient")
            else:
                s[name] = _codes(s[name], 128)
    return dict(case=case, **s)


# ---- the plain form --------------------------------------------------------------------------------------------------------------
def _codes(v, rows):
    """(e4m3 codes, power-of-two scales) of v [M, K] fp32 by blocks of `rows` x 128; the codes in whole blocks, zeros behind v's edge"""
    m, k = v.shape
    mb, kb = -(-m // rows), -(-k // 128)
    p = torch.nn.functional.pad(v, (0, kb * 128 - k, 0, mb * rows - m)).view(mb, rows, kb, 128)
    amax = p.abs().amax(dim=(1, 3))
    mant, ex = torch.frexp(amax)                                     # amax = mant 2^ex, mant in [0.5, 1);  448 = 0.875 * 2^9
    e = torch.where(amax > 0, ex - 9 + (mant > 0.875).int(), torch.full_like(ex, -127)).clamp(-127, 127)
    up = ((127 - e) << 23).view(torch.float32)                       # 2^-e, exact
    codes = (p * up[:, None, :, None]).to(F8)
    return codes.view(mb * rows, kb * 128)[:m], 1.0 / up


def _values(codes, scales, rows):
    m = codes.shape[0]
    mb, kb = scales.shape
    s = scales.repeat_interleave(rows, 0)[:m]
    return (codes.float().view(m, kb, 128) * s[:, :, None]).view(m, kb * 128)


def _rounded(v):
    return _values(*_codes(v.float(), 1), 1)


def _gelu(a):
    return 0.5 * a * (1.0 + torch.tanh(GELU_C * (a + 0.044715 * a * a * a)))


def _plain(s, op):
    case = s["case"]
    if op == "linear":
        y = _rounded(s["x"]) @ _values(*s["w"], 128).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(TYPES[case["y"]])
    if op == "feed_forward":
        x = s["x"].float()
        n = _rounded(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["norm"])
        h = _rounded(_gelu(n @ _values(*s["wi_0"], 128).t()) * (n @ _values(*s["wi_1"], 128).t()))
        return (h @ _values(*s["wo"], 128).t() + x).to(torch.bfloat16)
    if op == "input_gradient":
        w = _values(*s["w"], 128)[:, :case["k"]]
        return (_rounded(s["dy"])[:, :case["n"]] @ w).to(TYPES[case["dx"]])
    if op == "embedding":
        h = s["table"][s["ids"]] * case["scale"]
        if s["pos"] is not None:
            h = h + s["pos"]
        return h.to(torch.bfloat16)
    grad = torch.zeros(case["vocab"], case["d"], device="cuda")
    return grad.index_add_(0, s["ids"].reshape(-1), s["dy"].reshape(-1, case["d"]).float() * case["scale"])


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return _plain(state, op)
    from flash_diffusion_amd import ops
    if op == "linear":
        return ops.gemm_fp8(state["x"], state["w"], bias=state["bias"], residual=state["residual"], out_f32=case["y"] == "f32")
    if op == "feed_forward":      # the layer as MiT5EncoderModel(precision="fp8") runs it
        n = ops.rmsnorm_fp8(state["x"], state["norm"], EPS)
        h = ops.gated_fp8(n, state["wi_0"], state["wi_1"])
        return ops.gemm_fp8(h, state["wo"], residual=state["x"])
    if op == "input_gradient":
        return ops.gemm_fp8_dgrad(state["dy"], state["w"], out_f32=case["dx"] == "f32")
    if op == "embedding":
        return ops.embed_fwd(state["table"], state["ids"], scale=case["scale"], pos=state["pos"])
    return ops.embed_bwd(state["dy"], state["ids"], case["vocab"], scale=case["scale"])


def work(case):
    size = {"bf16": 2, "f32": 4}
    op = case["op"]
    if op in ("linear", "input_gradient"):
        m, k, n = case["rows"], case["k"], case["n"]
        w = n * k + -(-n // 128) * -(-k // 128)
        if op == "linear":
            out = (1 + case["residual"]) * m * n * size[case["y"]]
            return dict(bytes=m * k * size[case["x"]] + w + out + 4 * n * case["bias"], flops=2 * m * n * k)
        return dict(bytes=m * n * size[case["dy"]] + w + m * k * size[case["dx"]], flops=2 * m * n * k)
    if op == "feed_forward":
        m, d, f = case["rows"], case["d"], case["f"]
        return dict(bytes=2 * m * d * 2 + 3 * d * f + 4 * d, flops=6 * m * d * f)
    tokens, d = case["batch"] * case["length"], case["d"]
    if op == "embedding":
        return dict(bytes=tokens * (8 + d * 6) + case["pos"] * case["length"] * d * 4, flops=2 * tokens * d)
    return dict(bytes=tokens * (8 + d * size[case["dy"]]) + case["vocab"] * d * 4, flops=2 * tokens * d)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e in float64 from the bits of its exponent: pow() may be an ulp off, which breaks ties the wrong way"""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _near(v, block):
    """v [M, K] float64 -> the values its 8-bit form stands for; block (rows, 128).  A code is the nearest multiple of 2^(p - 3) for
    |code| in [2^p, 2^(p + 1)), p >= -6 (the subnormal step below)."""
    out = torch.empty_like(v)
    for c in range(0, v.shape[1], 128):
        part = v[:, c:c + 128]
        if block == 1:
            amax = part.abs().amax(1, keepdim=True)
        else:
            amax = torch.cat([part[r:r + block].abs().max().expand(part[r:r + block].shape[0], 1) for r in range(0, v.shape[0], block)])
        e = (torch.frexp(amax)[1] - 9).clamp(-127, 126)                # 256 2^e <= amax < 512 2^e
        e = torch.where(amax > 448.0 * _pow2(e), e + 1, e)
        t = part * _pow2(-e)
        step = _pow2(torch.frexp(t.abs().clamp(min=2.0 ** -6))[1] - 4)
        out[:, c:c + 128] = torch.round(t / step) * step * _pow2(e)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "linear":
        y = _near(s["x"].double(), 1) @ _near(s["w"].double(), 128).t()
        if case["bias"]:
            y += s["bias"].double()
        if case["residual"]:
            y += s["residual"].double()
        return y
    if op == "feed_forward":
        x = s["x"].double()
        n = _near(x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * s["norm"].double(), 1)
        a, b = n @ _near(s["wi_0"].double(), 128).t(), n @ _near(s["wi_1"].double(), 128).t()
        h = a * torch.sigmoid(2.0 * GELU_C * (a + 0.044715 * a ** 3)) * b         # (1 + tanh u) / 2 = sigmoid(2 u)
        return _near(h, 1) @ _near(s["wo"].double(), 128).t() + x
    if op == "input_gradient":
        return _near(s["dy"].to(TYPES[case["dy"]]).double(), 1) @ _near(s["w"].double(), 128)
    if op == "embedding":
        h = torch.nn.functional.embedding(s["ids"], s["table"].double()) * case["scale"]
        return h if s["pos"] is None else h + s["pos"].double()
    ids, perm = torch.sort(s["ids"].reshape(-1), stable=True)
    rows = s["dy"].double().reshape(-1, case["d"])[perm]
    sums = torch.zeros(case["vocab"], case["d"], dtype=torch.float64, device="cuda")
    found, count = torch.unique_consecutive(ids, return_counts=True)
    ends = torch.cumsum(count, 0)
    if rows.shape[1] * rows.shape[0] > 1 << 28:
        return None
    total = torch.cat([torch.zeros(1, case["d"], dtype=torch.float64, device="cuda"), torch.cumsum(rows, 0)])
    sums[found] = (total[ends] - total[ends - count]) * case["scale"]
    return sums
