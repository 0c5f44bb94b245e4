"""Performance cases of the operators of layers in 8-bit integers: the norms around a block, the rows' quantisers and the product.

A layer whose weights and activations are both 8-bit integers passes through four operators: `norm_block` (what a block adds is normed, gated,
scaled and added to the residual stream, and the stream normed for the next block, in bf16 or in 8 bits with a scale for each token),
`quant_rows_int8` and `act_mul_int8` (rows, or activations of a feed-forward's gate and up halves, in 8 bits with a scale for each token) and `gemm_int8`
(the product of such rows with weights in 8 bits and a scale for each output channel).  A case is one `norm_block`, one linear layer (quantiser
and product), or one feed-forward (norms, product, activation, product).

With `own` false the operators are computed from elementary torch operations, with `own` true by the framework's kernels.
"""

import math
import random

import torch

own = False

STREAM_LIMIT = 4001 * 8192              # numbers in the residual stream of the largest norm
WEIGHT_LIMIT = 28672 * 4096             # numbers in the largest weight matrix
PRODUCT_LIMIT = 4001 * 28672 * 4096
FFN_LIMIT = 2048 * 3 * 14336 * 4096


def _norm(tokens, width, post=True, gate="none", scale=1.0, layernorm=False, **more):
    return dict(op="norm", tokens=tokens, width=width, post=post, gate=gate, scale=scale, layernorm=layernorm, **more)


def _linear(tokens, inputs, outputs, bias=False, padded=False, **more):
    return dict(op="linear", tokens=tokens, inputs=inputs, outputs=outputs, bias=bias, padded=padded, **more)


def _ffn(tokens, width, features, act="silu", post=False, scale=1.0, **more):
    return dict(op="ffn", tokens=tokens, width=width, features=features, act=act, post=post, scale=scale, **more)


def listed():
    return [
        # a lone user's next token: norms on both sides of a block, latency alone
        _norm(1, 4096, name="norms_1"),
        # a decode batch of a cross-attention layer: a gate that is zero for tokens without an image, no norm behind the block
        _norm(259, 4096, post=False, gate="token", name="norms_gated_259"),
        # a prefill step with a gate for each channel, layer norms with biases, and an odd width
        _norm(1500, 2049, gate="channel", layernorm=True, name="norms_layer_odd"),
        # a long prefill of a wide model, residual multiplier
        _norm(4001, 8192, scale=0.22, name="norms_4001"),
        # the query, key and value projection of a lone user's next token
        _linear(1, 4096, 6144, name="linear_1"),
        # the same for an odd batch, with sizes that fill no tile and no 16 bytes
        _linear(137, 1021, 2050, bias=True, padded=True, name="linear_odd"),
        # the down projection of a full decode batch
        _linear(256, 14336, 4096, name="linear_256"),
        # the gate and up projection of a long prefill
        _linear(4001, 4096, 28672, name="linear_4001"),
        # a feed-forward for one token
        _ffn(1, 4096, 14336, name="ffn_1"),
        # the same for a decode batch, with norms on both sides of the attention in front
        _ffn(48, 4096, 14336, act="gelu_tanh", post=True, name="ffn_48"),
        # a prefill step
        _ffn(2048, 4096, 14336, scale=0.22, name="ffn_2048"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "ffn"])
    if op == "norm":
        tokens, width = _log(rng, 1, 8192), _log(rng, 64, 8192)
        width = max(64, min(width, STREAM_LIMIT // tokens))
        width = rng.choice([width, width // 8 * 8, width // 8 * 8])
        return _norm(tokens, width, rng.choice([True, True, False]), rng.choice(["none", "channel", "token", "one"]), rng.choice([1.0, 1.0, 0.22]),
                     rng.choice([False, False, True]))
    tokens = _log(rng, 1, 4001 if op == "linear" else 2048)
    a = _log(rng, 64, 14336)
    a = rng.choice([a, a // 16 * 16, a // 16 * 16])
    most = min(28672, WEIGHT_LIMIT // a, PRODUCT_LIMIT // (a * tokens)) if op == "linear" else min(14336, FFN_LIMIT // (3 * a * tokens), WEIGHT_LIMIT // (2 * a))
    b = _log(rng, 64, max(64, most))
    if op == "linear":
        return _linear(tokens, a, b, rng.choice([False, True]), rng.choice([False, True]))
    return _ffn(tokens, a, b, rng.choice(["silu", "silu", "gelu_tanh", "relu"]), rng.choice([False, True]), rng.choice([1.0, 0.22]))


# ------------------------------------------------------------------------------------------------ preparing

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + what) % (1 << 62))


def _rand(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(std)


def _rows(gen, tokens, width):
    """Activations: rows of different size, some channels that stand out."""
    channel = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    size = torch.exp(0.5 * torch.randn(tokens, 1, generator=gen, device="cuda"))
    return (torch.randn(tokens, width, generator=gen, device="cuda") * channel * size).to(torch.bfloat16)


def _weight(gen, outputs, inputs, std):
    """A matrix in 8 bits with a scale for each output channel, as a checkpoint or the quantiser of a model's weights lays it out: rows 16 bytes apart or a
    multiple of that."""
    q = torch.zeros(outputs, (inputs + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :inputs]
    scale = torch.empty(outputs, device="cuda")
    for a in range(0, outputs, 4096):
        w = torch.randn(min(4096, outputs - a), inputs, generator=gen, device="cuda") * std
        scale[a:a + 4096] = w.abs().amax(1) / 127
        q[a:a + 4096] = torch.round(w / scale[a:a + 4096, None]).clamp(-127, 127).to(torch.int8)
    return q, scale


def prepare(case, seed):
    g, T = _gen(seed, 3), case["tokens"]
    if case["op"] == "linear":
        K, N = case["inputs"], case["outputs"]
        wide = (K + 63) // 64 * 64 if case["padded"] else K      # rows of a wider buffer
        x = _rows(g, T, wide)[:, :K]
        w, ws = _weight(g, N, K, K ** -0.5)
        return dict(op="linear", x=x, w=w, ws=ws, bias=_rand(g, N) if case["bias"] else None)
    H = case["width"]
    near = lambda std: (1 + _rand(g, H, std=std, dtype=torch.float32)).to(torch.bfloat16)
    s = dict(op=case["op"], y=_rows(g, T, H), residual=_rand(g, T, H, std=4.0), weight=near(0.2), post=near(0.2) if case["post"] else None, scale=case["scale"],
             eps=1e-6, residual_out=torch.empty(T, H, dtype=torch.bfloat16, device="cuda"))
    if case["op"] == "norm":
        gates = dict(none=lambda: None, one=lambda: _rand(g, 1), channel=lambda: _rand(g, H, std=0.3),
                     token=lambda: (torch.rand(T, 1, generator=g, device="cuda") < 0.7).to(torch.bfloat16))
        s.update(gate=gates[case["gate"]](), layernorm=case["layernorm"], bias=_rand(g, H, std=0.1) if case["layernorm"] else None,
                 post_bias=_rand(g, H, std=0.1) if case["layernorm"] and case["post"] else None)
        return s
    I = case["features"]
    up, up_scale = _weight(g, 2 * I, H, H ** -0.5)
    down, down_scale = _weight(g, H, I, I ** -0.5)
    s.update(up=up, up_scale=up_scale, down=down, down_scale=down_scale, features=I, act=case["act"])
    return s


# ------------------------------------------------------------------------------------------------ running

def run(state):
    with torch.inference_mode():
        if own:
            return _run_own(state)
        return dict(norm=_plain_norm, linear=_plain_linear, ffn=_plain_ffn)[state["op"]](state)


_ops = None


def _run_own(s):
    global _ops
    if _ops is None:
        from lorax_b200.ops import get_ops
        _ops = get_ops("cuda")
    if s["op"] == "norm":
        x = _ops.norm_block(s["y"], s["residual"], s["weight"], s["eps"], post_weight=s["post"], gate=s["gate"], scale=s["scale"], bias=s["bias"],
                            post_bias=s["post_bias"], layernorm=s["layernorm"], residual_out=s["residual_out"])
        return dict(residual=s["residual_out"], x=x)
    if s["op"] == "linear":
        return _ops.gemm_int8(_ops.quant_rows_int8(s["x"]), s["w"], s["ws"], bias=s["bias"])
    x = _ops.norm_block(s["y"], s["residual"], s["weight"], s["eps"], post_weight=s["post"], scale=s["scale"], residual_out=s["residual_out"], int8=True)
    h = _ops.gemm_int8(x, s["up"], s["up_scale"])
    y = _ops.gemm_int8(_ops.act_mul_int8(h, s["features"], s["act"]), s["down"], s["down_scale"])
    return dict(residual=s["residual_out"], y=y)


def _normed(x, weight, bias, eps, layernorm):
    if layernorm:
        x = x - x.mean(1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + eps) * weight.float()
    return x if bias is None else x + bias.float()


def _add_and_norm(s, gate=None, bias=None, post_bias=None, layernorm=False):
    """The stream with the block's part, in its own type, and that stream normed, in 32 bits."""
    y = s["y"].float()
    if s["post"] is not None:
        y = _normed(y, s["post"], post_bias, s["eps"], layernorm)
    y = y * s["scale"]
    if gate is not None:
        y = y * gate.float()
    residual = (s["residual"].float() + y).to(s["residual"].dtype)
    return residual, _normed(residual.float(), s["weight"], bias, s["eps"], layernorm)


def _quantised(x):
    """Rows in 8 bits and their scales.  The quotients in 64 bits: a value's step is decided at a border."""
    scale = x.abs().amax(1) / 127
    return torch.round(x.double() / torch.where(scale > 0, scale, 1)[:, None].double()).clamp(-127, 127), scale


def _product(x, scale, w, w_scale, bias=None):
    """Sums of thousands of products of whole numbers pass 2^24: 64 bits."""
    y = (x @ w.double().t()).float() * scale[:, None] * w_scale
    return (y if bias is None else y + bias.float()).to(torch.bfloat16)


def _act(x, act):
    if act == "relu":
        return x.clamp_min(0)
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x / (1 + torch.exp(-x))


def _plain_norm(s):
    residual, x = _add_and_norm(s, s["gate"], s["bias"], s["post_bias"], s["layernorm"])
    return dict(residual=residual, x=x.to(torch.bfloat16))


def _plain_linear(s):
    return _product(*_quantised(s["x"].float()), s["w"], s["ws"], s["bias"])


def _plain_ffn(s):
    residual, x = _add_and_norm(s)
    h, I = _product(*_quantised(x), s["up"], s["up_scale"]).float(), s["features"]
    return dict(residual=residual, y=_product(*_quantised(_act(h[:, :I], s["act"]) * h[:, I:]), s["down"], s["down_scale"]))


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    with torch.inference_mode():
        s = prepare(case, seed)
        if s["op"] == "linear":
            return _exact_product(s["x"].double(), s["w"], s["ws"], s["bias"])
        d, H = (lambda t: None if t is None else t.double()), s["y"].shape[1]
        if s.get("layernorm"):
            norm = lambda x, w, b: torch.nn.functional.layer_norm(x, (H,), d(w), d(b), s["eps"])
        else:
            norm = lambda x, w, b: torch.nn.functional.rms_norm(x, (H,), d(w), s["eps"])
        y = d(s["y"]) if s["post"] is None else norm(d(s["y"]), s["post"], s.get("post_bias"))
        gate = 1.0 if s.get("gate") is None else d(s["gate"])
        residual = torch.addcmul(d(s["residual"]), y, torch.as_tensor(gate, dtype=torch.float64, device="cuda"), value=s["scale"])
        x = norm(residual.to(torch.bfloat16).double(), s["weight"], s.get("bias"))      # (the next block reads the stream as it is stored)
        if s["op"] == "norm":
            return dict(residual=residual, x=x)
        h = _exact_product(x, s["up"], s["up_scale"], None).to(torch.bfloat16).double()
        gate, up = h.split(s["features"], dim=1)
        f = torch.nn.functional
        gate = dict(silu=f.silu, relu=f.relu, gelu_tanh=lambda t: f.gelu(t, approximate="tanh"))[s["act"]](gate)
        return dict(residual=residual, y=_exact_product(gate * up, s["down"], s["down_scale"], None))


def _exact_product(x, w, w_scale, bias):
    parts = []
    for rows in x.split(1024):
        step = (rows.abs().max(dim=1, keepdim=True).values / 127).float().double()      # (scales are held in 32 bits)
        whole = torch.nan_to_num(rows / step).round()
        y = torch.cat([torch.einsum("tk,nk->tn", whole, part.double()) for part in w.split(8192)], 1) * (step * w_scale.double())
        parts.append(y if bias is None else y + bias.double())
    return torch.cat(parts)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    T = case["tokens"]
    if case["op"] == "linear":
        K, N = case["inputs"], case["outputs"]
        return dict(bytes=2 * T * K + N * K + 4 * N + 2 * T * N + (2 * N if case["bias"] else 0), flops=2.0 * T * N * K)
    H = case["width"]
    stream = 8 * T * H + 2 * H * (2 if case["post"] else 1)
    if case["op"] == "norm":
        H2 = 2 * H * (2 if case["post"] else 1) if case["layernorm"] else 0
        return dict(bytes=stream + H2 + 2 * dict(none=0, one=1, channel=H, token=T)[case["gate"]], flops=16.0 * T * H)
    I = case["features"]
    return dict(bytes=stream + 3 * H * I + 4 * (2 * I + H), flops=6.0 * T * H * I)
