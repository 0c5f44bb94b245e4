"""Operators of layers in 8-bit integers on the GPU, against their definitions in 64 bits.

Tolerances.  A result in bf16 is rounded once: 2^-8 of it.  What is computed in 32 bits loses some 2^-24 a step; the steps are counted beside each bound."""
import pytest
import torch

from lorax_b200.ops import native, native_int8  # noqa: F401  (the bindings of every operator first)
from lorax_b200.ops import reference as ref
from lorax_b200.ops.reference import Int8Rows

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HALF, E = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from lorax_b200.ops import native
    native.load()
    yield native
    native.workspace().check_status()


def _gen(*seed):
    return torch.Generator(device="cuda").manual_seed(hash(seed) % (1 << 40))


def _randn(g, *shape, dtype=BF, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _int8(g, rows, K, at=0):
    """Random bytes; `at`: rows of a wider buffer that begin `at` bytes into it."""
    wide = (K + at + 15) // 16 * 16
    return torch.randint(-127, 128, (rows, wide), generator=g, device="cuda", dtype=torch.int8)[:, at:at + K]


# ------------------------------------------------------------------------------------------------ rows
def _check_rows(r, v, steps):
    """`v`: the values in 64 bits, of which the kernel's differ by `steps` of 2^-24 of the row's largest at most."""
    top = v.abs().amax(1)
    assert ((r.scale.double() - top / 127).abs() <= top / 127 * (steps + 2) * E).all()
    off = (r.q.double() * r.scale.double()[:, None] - v).abs()
    assert (off <= r.scale.double()[:, None] * 0.5 * (1 + 4 * E) + top[:, None] * steps * E).all()
    assert ((r.q.int().abs().amax(1) == 127) | (top == 0)).all()


@pytest.mark.parametrize("T", [1, 3, 150, 1027])
@pytest.mark.parametrize("K", [1, 7, 8, 64, 1021, 2048, 4096, 8200, 14336])
def test_rows_equal_the_plain_form(ops, T, K):
    x = _randn(_gen(T, K), T, K, std=3.0)
    x[:, 0] = 127 * 2.0 ** -3                       # with scales of 2^-3 and quotients at halves in many rows
    x[:, K // 2] = 2.5 * 2.0 ** -3
    r, want = ops.quant_rows_int8(x), ref.quant_rows_int8(x.cpu())
    assert torch.equal(r.scale.cpu(), want.scale) and torch.equal(r.q.cpu(), want.q)


@pytest.mark.parametrize("T,K", [(2, 16392), (1, 40000), (149, 20001)])
def test_rows_longer_than_a_block_holds(ops, T, K):
    x = _randn(_gen(T, K), T, K)
    r, want = ops.quant_rows_int8(x), ref.quant_rows_int8(x.cpu())
    assert torch.equal(r.scale.cpu(), want.scale) and torch.equal(r.q.cpu(), want.q)


@pytest.mark.parametrize("at,wide", [(0, 80), (1, 80), (8, 80), (3, 75)])
def test_rows_of_a_wider_buffer(ops, at, wide):
    x = _randn(_gen(at, wide), 40, wide)[:, at:at + 64]
    r, want = ops.quant_rows_int8(x), ref.quant_rows_int8(x.cpu())
    assert torch.equal(r.scale.cpu(), want.scale) and torch.equal(r.q.cpu(), want.q)


@pytest.mark.parametrize("K", [1, 5, 9, 16, 23, 1000, 1001, 4099])
@pytest.mark.parametrize("at", [0, 1, 2, 3, 5, 8])
def test_rows_that_begin_anywhere(ops, K, at):
    x = _randn(_gen(K, at), 11, 2 * K + 11)
    r, want = ops.quant_rows_int8(x[:, at:at + K]), ref.quant_rows_int8(x[:, at:at + K].cpu())
    assert torch.equal(r.scale.cpu(), want.scale) and torch.equal(r.q.cpu(), want.q)
    v = x[:, at:at + 2 * K]
    out = torch.full((11, K + 1), 3.0, device="cuda", dtype=BF)
    r = ops.act_mul_int8(v, K, "relu", out=out[:, 1:])
    v = v[:, :K].double().clamp_min(0) * v[:, K:].double()
    # (one rounding of the product)
    _check_rows(r, v, 1)
    assert ((out[:, 1:].double() - v).abs() <= HALF * v.abs() + 2 * E * v.abs()).all() and (out[:, 0] == 3).all()


@pytest.mark.parametrize("K", [24, 25])
def test_rows_without_a_scale(ops, K):
    x = _randn(_gen(K), 9, K)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 6] = float("-inf")
    x[3, K - 1] = float("nan")
    x[4] = 0
    x[4, 3] = 2.0 ** -133                           # the least bf16
    x[5] *= 2.0 ** -126
    x[6] = torch.finfo(BF).max
    x[7, 0] = torch.finfo(BF).min
    r, want = ops.quant_rows_int8(x), ref.quant_rows_int8(x.cpu())
    assert r.scale[1:4].isnan().all() and torch.equal(r.q.cpu(), want.q)
    keep = [0, 4, 5, 6, 7, 8]
    assert torch.equal(r.scale.cpu()[keep], want.scale[keep])
    w, ws = ref.quantize_weight_int8(_randn(_gen(1), 33, K, dtype=torch.float32))
    y = ops.gemm_int8(r, w, ws)
    # (rows of the largest bf16 pass it where the sum of their products does, and nowhere else)
    want = (r.q.double() @ w.double().t()) * r.scale.double()[:, None] * ws.double()
    assert (y[0] == 0).all() and y[1:4].isnan().all() and torch.equal(y[keep].isfinite(), want[keep].to(BF).isfinite())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "relu2"])
@pytest.mark.parametrize("T,I,gated", [(1, 14336, True), (5, 33, True), (200, 1000, True), (3, 17, False), (150, 512, False), (2, 20000, True)])
def test_activations(ops, act, T, I, gated):
    x = _randn(_gen(T, I), T, 2 * I if gated else I, std=2.0)
    out = torch.full((T, I), 7.0, device="cuda", dtype=BF)
    r = ops.act_mul_int8(x, I, act, gated, out=out)
    v = ref._act(x[:, :I].double(), act)
    if gated:
        v = v * x[:, I:].double()
    # of a value: exp within 2^-21 of itself for |x| below 10 or so, tanh and erf within some 2^-22 of 1, four roundings: 24 steps of the largest value
    _check_rows(r, v, 24)
    top = v.abs().amax(1, keepdim=True)
    assert ((out.double() - v).abs() <= HALF * v.abs() + 24 * E * top).all()
    assert torch.equal(ops.act_mul_int8(x, I, act, gated).q, r.q)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("n", [8, 100])
def test_rows_whose_gates_are_all_shut_keep_their_digits(ops, act, n):
    """The largest value of such a row is tiny, and its scale goes by it: what counts is a value's own relative error."""
    x = (-4 - 8 * torch.rand(60, n, generator=_gen(n), device="cuda")).to(BF)
    z = x.double()
    if act == "gelu":
        v = 0.5 * z * torch.special.erfc(-z * 0.5 ** 0.5)
        steps = (z * z).amax(1) + 16           # an argument's rounding moves erfc by 2 z^2 = x^2 of its own; erfc's last places, two products
    else:
        u = z if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)
        v = z * torch.sigmoid(u)
        steps = 8 * u.abs().amax(1) + 16       # the exponent's roundings (five in the polynomial, two in front of exp2) move the exponential by as much
    r = ops.act_mul_int8(x, n, act, gated=False)
    top = v.abs().amax(1)
    assert ((r.scale.double() - top / 127).abs() <= top / 127 * (steps + 2) * E).all()
    off = (r.q.double() * r.scale.double()[:, None] - v).abs()
    assert (off <= r.scale.double()[:, None] * (0.5 + 2.0 ** -20) + (top * steps * E)[:, None]).all()


@pytest.mark.parametrize("T,n", [(1, 8), (5, 64), (700, 256), (1300, 1000), (601, 4096), (300, 8192), (301, 14336), (200, 16384)])
@pytest.mark.parametrize("act,gated", [(None, False), ("silu", True), ("relu2", False)])
def test_both_forms_of_quantisers(ops, T, n, act, gated):
    """A block per row, and blocks that stay: the same bits, since a row's maximum and quotients depend on no order."""
    x = _randn(_gen(T, n), T, 2 * n if gated else n, std=2.0)
    x[T // 2] = 0
    x[T // 3, 5] = float("nan")
    outs = [torch.full((T, n), 7.0, device="cuda", dtype=BF) for _ in range(2)]
    a, b = (native_int8._on(x, native_int8._rows, x, x.stride(0), T, n, native._ACTS[act] if act else -1, gated, o, ring) for ring, o in enumerate(outs))
    assert torch.equal(a.q, b.q) and torch.equal(a.scale.view(torch.int32), b.scale.view(torch.int32)) and torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
    if act is None:
        want = ref.quant_rows_int8(x.cpu())
        assert torch.equal(b.q.cpu(), want.q) and (outs[1] == x)[x == x].all()


def test_activations_keep_what_is_not_a_number(ops):
    x = _randn(_gen(3), 4, 64)
    x[1, 3] = float("nan")
    x[2, 40] = float("inf")
    for act in ("silu", "gelu", "gelu_tanh", "relu", "relu2"):
        r = ops.act_mul_int8(x, 32, act)
        assert r.scale.isfinite().tolist()[0::3] == [True, True] and r.scale[1].isnan(), act


# ------------------------------------------------------------------------------------------------ norms
def _norm64(v, w, b, eps, offset, layernorm):
    if layernorm:
        v = v - v.mean(1, keepdim=True)
    r = (v * v).mean(1, keepdim=True).add(eps).rsqrt()
    y = v * r * (w.double() + offset)
    # 32-bit sums of a row's squares and values, a reciprocal root, three products: 64 steps of the largest normed value, and of the offset's mean
    slack = 64 * E * ((v * r).abs().amax(1, keepdim=True) * (w.double().abs() + abs(offset)))
    if b is not None:
        y = y + b.double()
        slack = slack + 2 * E * b.double().abs()
    return y, slack


def _norm_by(ring, y, res, w, eps, post_weight=None, gate=None, scale=1.0, bias=None, post_bias=None, weight_offset=0.0, layernorm=False, residual_out=None, out=None,
             int8=False):
    checked = ref.check_norm_block(y, res, w, post_weight, gate, scale, bias, post_bias, residual_out, out, int8)
    return native_int8._on(res, native_int8._norm_block, checked, eps, scale, weight_offset, layernorm, out, int8, ring)


def _check_norm(ops, T, H, post, gate, scale, layernorm, int8, bias=True, offset=0.0, eps=1e-5, at=0, ring=-1):
    def call(y, res, w, eps, post_weight=None, gate=None, scale=1.0, bias=None, post_bias=None, weight_offset=0.0, layernorm=False, residual_out=None, out=None, int8=False):
        if ring < 0:
            return ops.norm_block(y, res, w, eps, post_weight, gate, scale, bias, post_bias, weight_offset, layernorm, residual_out, out, int8)
        return _norm_by(ring, y, res, w, eps, post_weight, gate, scale, bias, post_bias, weight_offset, layernorm, residual_out, out, int8)
    g = _gen(T, H, post, scale, layernorm)
    wide = H + at
    y, res = _randn(g, T, wide)[:, at:], _randn(g, T, wide, std=3.0)[:, at:]
    w, pw = 1 + _randn(g, H, std=0.2), 1 + _randn(g, H, std=0.2)
    b, pb = (_randn(g, H, std=0.3), _randn(g, H, std=0.3)) if bias else (None, None)
    gates = dict(none=None, one=_randn(g, 1), zero=torch.tensor(0.0, device="cuda", dtype=BF), channel=_randn(g, H), token=_randn(g, T, 1), all=_randn(g, T, H))
    gate = gates[gate]
    h = torch.full((T, wide), 5.0, device="cuda", dtype=BF)[:, at:]
    keep = res.clone()
    kw = dict(post_weight=pw if post else None, gate=gate, scale=scale, bias=b, post_bias=pb if post else None, weight_offset=offset, layernorm=layernorm)
    out = torch.full((T, H), 5.0, device="cuda", dtype=BF) if int8 == "both" else None
    x = call(y, res, w, eps, residual_out=h, out=out, int8=bool(int8), **kw)
    assert torch.equal(res, keep)
    part, slack = (y.double(), 0.0) if not post else _norm64(y.double(), pw, kw["post_bias"], eps, offset, layernorm)
    f = scale * (1.0 if gate is None else gate.double())
    want = res.double() + f * part
    assert ((h.double() - want).abs() <= HALF * want.abs() + torch.as_tensor(f, device="cuda").abs() * (slack + 4 * E * part.abs()) + 2 * E * want.abs()).all()
    want, slack = _norm64(h.double(), w, b, eps, offset, layernorm)
    if int8:
        top = want.abs().amax(1)
        assert ((x.scale.double() - top / 127).abs() <= slack.amax(1) / 127 + 4 * E * top / 127).all()
        assert ((x.q.double() * x.scale.double()[:, None] - want).abs() <= x.scale.double()[:, None] * (0.5 + 2.0 ** -18) + 2 * slack.amax(1, keepdim=True)).all()
    value = out if int8 == "both" else None if int8 else x
    if value is not None:
        assert ((value.double() - want).abs() <= HALF * want.abs() + slack * (1 + HALF)).all()
    # in place, the same bits
    again = call(y, res, w, eps, int8=bool(int8), **kw)
    assert torch.equal(res, h) and (torch.equal(again.q, x.q) and torch.equal(again.scale, x.scale) if int8 else torch.equal(again, x))


@pytest.mark.parametrize("T,H", [(1, 4096), (1, 1), (2, 7), (5, 8), (148, 1000), (149, 1000), (300, 2049), (3, 8192), (150, 8192), (2, 16384), (151, 16384), (2, 16383)])
@pytest.mark.parametrize("layernorm", [False, True])
@pytest.mark.parametrize("int8", [False, True])
def test_norms(ops, T, H, layernorm, int8):
    _check_norm(ops, T, H, True, "none", 1.0, layernorm, int8)


@pytest.mark.parametrize("gate", ["none", "one", "zero", "channel", "token", "all"])
@pytest.mark.parametrize("post,int8", [(True, "both"), (False, False)])
@pytest.mark.parametrize("H", [512, 333])
def test_gates(ops, gate, post, int8, H):
    _check_norm(ops, 37, H, post, gate, 0.22, False, int8, bias=False, offset=1.0)


@pytest.mark.parametrize("gate", ["none", "one", "channel", "token", "all"])
@pytest.mark.parametrize("T,H", [(1, 8), (3, 256), (700, 64), (1300, 1000), (700, 4096), (301, 8192), (300, 16384)])
@pytest.mark.parametrize("layernorm", [False, True])
def test_both_forms_of_norms(ops, gate, T, H, layernorm):
    """A block per row, and blocks that stay."""
    for ring in (0, 1):
        _check_norm(ops, T, H, gate != "one", gate, 0.5, layernorm, "both" if gate in ("token", "all") else gate == "none", ring=ring, bias=layernorm)


@pytest.mark.parametrize("T,H", [(1, 512), (700, 512), (33, 511), (1500, 4096)])
@pytest.mark.parametrize("layernorm", [False, True])
def test_a_norm_without_a_block_in_front_by_both_forms(ops, T, H, layernorm):
    g = _gen(9, T, H)
    res, w, b = _randn(g, T, H), _randn(g, H), _randn(g, H)
    keep = res.clone()
    want, slack = _norm64(res.double(), w, b, 1e-5, 0.0, layernorm)
    for x in (*(_norm_by(ring, None, res, w, 1e-5, bias=b, layernorm=layernorm) for ring in (0, 1)), ops.norm_block(None, res, w, 1e-5, bias=b, layernorm=layernorm)):
        assert ((x.double() - want).abs() <= HALF * want.abs() + slack * (1 + HALF)).all()
    out = torch.empty_like(res)
    r = ops.norm_block(None, res, w, 1e-5, bias=b, layernorm=layernorm, int8=True, out=out)
    assert torch.equal(out, x) and torch.equal(res, keep)
    off = (r.q.double() * r.scale.double()[:, None] - want).abs()
    assert (off <= r.scale.double()[:, None] * (0.5 + 2.0 ** -18) + 2 * slack.amax(1, keepdim=True)).all()
    assert ops.norm_block(None, res, w, 1e-5, bias=b, layernorm=layernorm, out=res) is res and torch.equal(res, out)      # over the residual itself


@pytest.mark.parametrize("T,H", [(2, 100), (700, 2048), (50, 333)])
def test_results_over_the_inputs(ops, T, H):
    """Every place that a result may take: over y, over the residual, each over the other's."""
    g = _gen(4, T, H)
    y, res, w = _randn(g, T, H), _randn(g, T, H), 1 + _randn(g, H, std=0.1)
    h, x = torch.empty_like(res), torch.empty_like(res)
    ops.norm_block(y, res, w, 1e-5, post_weight=w, residual_out=h, out=x)
    for to, out in (("y", "residual"), ("residual", "y"), ("y", None), (None, "y"), ("residual", None), (None, "residual")):
        at = dict(y=y.clone(), residual=res.clone())
        if to != "residual" and out == "residual" and to is None:
            at["h"] = torch.empty_like(res)
            to = "h"
        got = ops.norm_block(at["y"], at["residual"], w, 1e-5, post_weight=w, residual_out=at.get(to), out=at.get(out))
        assert torch.equal(got, x) and torch.equal(at[to or "residual"], h) and (out is None or got is at[out])


@pytest.mark.parametrize("H", [1, 2, 6, 7, 9, 15, 17, 257, 1001, 2049, 4095, 8190, 16377])
@pytest.mark.parametrize("layernorm,int8", [(False, "both"), (True, False), (True, True)])
def test_rows_of_any_width_in_tensors_without_gaps(ops, H, layernorm, int8):
    """Every distance of a row from 16 bytes, the same in all tensors, and rows of which each tensor's begin elsewhere."""
    _check_norm(ops, 17, H, True, "channel", 0.5, layernorm, int8)
    g = _gen(H)
    y, res, w = _randn(g, 17, H + 3)[:, 1:H + 1], _randn(g, 17, H), 1 + _randn(g, H, std=0.1)
    out = torch.full((17, H + 5), 5.0, device="cuda", dtype=BF)
    h = torch.empty_like(res)
    ops.norm_block(y, res, w, 1e-5, residual_out=h, out=out[:, 2:H + 2], layernorm=layernorm)
    want = res.double() + y.double()
    assert ((h.double() - want).abs() <= HALF * want.abs() + 2 * E * want.abs()).all() and (out[:, :2] == 5).all() and (out[:, H + 2:] == 5).all()
    want, slack = _norm64(h.double(), w, None, 1e-5, 0.0, layernorm)
    assert ((out[:, 2:H + 2].double() - want).abs() <= HALF * want.abs() + slack * (1 + HALF)).all()


@pytest.mark.parametrize("T,H", [(1, 3), (7, 9), (8, 1), (9, 255), (23, 65), (1500, 65), (700, 1021), (600, 2050), (1300, 2049), (310, 4097), (20, 4601)])
@pytest.mark.parametrize("layernorm,gate,int8", [(False, "none", False), (False, "token", True), (True, "channel", "both"), (True, "all", False)])
def test_rows_of_any_width_by_blocks_that_stay(ops, T, H, layernorm, gate, int8):
    """Blocks on rows of one distance from 16 bytes; fewer rows than blocks, more, and the library's own choice."""
    for ring in (1, -1):
        _check_norm(ops, T, H, gate != "all", gate, 0.5, layernorm, int8, bias=layernorm, ring=ring)


@pytest.mark.parametrize("H", [15, 2049])
def test_blocks_that_stay_on_rows_that_are_not_finite(ops, H):
    """... keep what is not a number in its row, the neighbours' first and last bytes among what a row loads."""
    g, T = _gen(H), 1600
    y, res, w = _randn(g, T, H), _randn(g, T, H), 1 + _randn(g, H, std=0.1)
    at = torch.arange(3, T, 7, device="cuda")
    y[at[0::4], H - 1], y[at[1::4], 0], res[at[2::4], 0], res[at[3::4], H - 1] = float("nan"), float("inf"), float("-inf"), float("nan")
    h = torch.empty_like(res)
    r = _norm_by(1, y, res, w, 1e-5, post_weight=w, residual_out=h, int8=True)
    bad = torch.zeros(T, dtype=torch.bool, device="cuda")
    bad[at] = True
    assert torch.equal(r.scale.isnan(), bad) and (r.q[bad] == 0).all()
    y, res = y.where(~bad[:, None], 0), res.where(~bad[:, None], 0)
    good = _norm_by(1, y, res, w, 1e-5, post_weight=w, residual_out=h.clone(), int8=True)
    assert torch.equal(r.q[~bad], good.q[~bad]) and torch.equal(r.scale[~bad], good.scale[~bad])


@pytest.mark.parametrize("H", [5, 64, 1001, 2048])
@pytest.mark.parametrize("at", [1, 4, 8])
def test_vectors_that_begin_anywhere(ops, H, at):
    """Weights, biases and gates inside a larger buffer."""
    g = _gen(H, at)
    buf = 1 + _randn(g, 5 * (H + 16), std=0.2)
    w, pw, b, pb, gate = (buf[i * (H + 16) + at:i * (H + 16) + at + H] for i in range(5))
    y, res = _randn(g, 33, H), _randn(g, 33, H)
    for layernorm in (False, True):
        for vectors in ((w, pw, b, pb, gate), (w.clone(), pw, b, pb.clone(), gate.clone()), (w.clone(), pw.clone(), b.clone(), pb.clone(), gate)):
            h = torch.empty_like(res)
            x = ops.norm_block(y, res, vectors[0], 1e-5, post_weight=vectors[1], gate=vectors[4], bias=vectors[2], post_bias=vectors[3], layernorm=layernorm, residual_out=h)
            part, slack = _norm64(y.double(), pw, pb, 1e-5, 0.0, layernorm)
            want = res.double() + gate.double() * part
            assert ((h.double() - want).abs() <= HALF * want.abs() + gate.double().abs() * (slack + 4 * E * part.abs()) + 2 * E * want.abs()).all()
            want, slack = _norm64(h.double(), w, b, 1e-5, 0.0, layernorm)
            assert ((x.double() - want).abs() <= HALF * want.abs() + slack * (1 + HALF)).all()


@pytest.mark.parametrize("at", [1, 8])
def test_norms_of_rows_that_begin_inside_a_buffer(ops, at):
    _check_norm(ops, 200, 256, True, "channel", 1.0, True, True, at=at)


@pytest.mark.parametrize("H", [64, 65])
def test_rows_of_zeros_and_numbers_that_are_not_finite_stay_in_their_rows(ops, H):
    g = _gen(H)
    y, res, w = _randn(g, 6, H), _randn(g, 6, H), _randn(g, H)
    y[0] = 0
    res[0] = 0
    y[2, 3] = float("nan")
    res[3, 4] = float("inf")
    y[4, 5] = float("inf")
    h = torch.empty_like(res)
    for int8 in (False, True):
        x = ops.norm_block(y, res, w, 1e-6, residual_out=h, int8=int8)
        bad = x.scale.isnan() if int8 else x.isnan().any(1)
        assert bad.tolist() == [False, False, True, True, True, False]
        assert ((x.q if int8 else x)[0] == 0).all()
    assert torch.equal(h.isfinite().all(1), torch.tensor([True, True, False, False, False, True], device="cuda"))
    # a gate of zero leaves a row as it is, unless what it shuts out is not finite
    gate = torch.zeros(6, 1, device="cuda", dtype=BF)
    ops.norm_block(y, res, w, 1e-6, gate=gate, residual_out=h)
    assert torch.equal(h[[0, 1, 3, 5]], res[[0, 1, 3, 5]]) and h[2, 3].isnan() and h[4, 5].isnan()


def test_large_means_do_not_cost_a_layer_norm_its_precision(ops):
    """Squares are taken of what the mean leaves: 1000 +- 4 in bf16 is 1000 and its neighbours."""
    res = 1000 + _randn(_gen(1), 4, 2048, dtype=torch.float32, std=8.0)
    res = res.to(BF)
    w = torch.ones(2048, device="cuda", dtype=BF)
    x = ops.norm_block(None, res, w, 1e-5, layernorm=True)
    want = torch.nn.functional.layer_norm(res.double(), (2048,), eps=1e-5)
    # the mean is off by 32 steps of 1000 at most, the values have a deviation of 8
    assert ((x.double() - want).abs() <= HALF * want.abs() + 64 * E * 1000 / 8).all()


# ------------------------------------------------------------------------------------------------ products
def _check_product(ops, T, N, K, bias=True, at=0, out=None, plan=None):
    g = _gen(T, N, K)
    q, w = _int8(g, T, K, at), _int8(g, N, K, at)
    xs, ws = torch.rand(T, generator=g, device="cuda") * 0.1, torch.rand(N, generator=g, device="cuda") * 0.01
    b = _randn(g, N) if bias else None
    if plan is None:
        y = ops.gemm_int8(Int8Rows(q, xs), w, ws, bias=b, out=out)
    else:
        x = Int8Rows(q, xs)
        y = native_int8._on(w, native_int8._gemm_int8, x, w, ws, b, out, ref.check_gemm_int8(x, w, ws, b, out, BF), False, plan)
    s = (q.double() @ w.double().t()) * (xs.double()[:, None] * ws.double())
    want = s + (0 if b is None else b.double())
    # the sum to 32 bits, two products, the bias: four roundings; then one to bf16
    assert y.shape == (T, N) and y.dtype == BF
    assert ((y.double() - want).abs() <= HALF * want.abs() + 5 * E * (s.abs() + want.abs())).all()
    return y


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 128, 137, 200, 256, 257, 300, 513])
@pytest.mark.parametrize("N,K", [(256, 512), (130, 1021)])
def test_products(ops, T, N, K):
    _check_product(ops, T, N, K)


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 127, 128, 129, 131, 255, 1000, 4099])
@pytest.mark.parametrize("T,K", [(1, 256), (20, 300)])
def test_products_of_any_number_of_channels(ops, N, T, K):
    _check_product(ops, T, N, K, bias=N % 2 == 0)


@pytest.mark.parametrize("K", [1, 15, 16, 17, 127, 128, 129, 255, 384, 511, 640, 900, 1100, 2048, 2300, 4096, 8192, 14336])
@pytest.mark.parametrize("T", [1, 48, 260])
def test_products_of_any_depth(ops, K, T):
    """K in one part or shared by up to eight CTAs."""
    _check_product(ops, T, 192, K, bias=False)


@pytest.mark.parametrize("T,N,K", [(1, 6144, 4096), (1, 28672, 4096), (7, 4096, 14336), (64, 28672, 4096), (256, 4096, 14336), (1500, 4096, 4096), (2048, 6144, 1024),
                                   (700, 11008, 2048), (4001, 2050, 520)])
def test_large_products(ops, T, N, K):
    _check_product(ops, T, N, K)


@pytest.mark.parametrize("pairs,bn,parts", [(False, 16, 1), (False, 48, 8), (False, 128, 3), (False, 256, 5), (True, 32, 1), (True, 96, 1), (True, 256, 1), (True, 64, 2),
                                            (True, 256, 3), (True, 160, 4)])
@pytest.mark.parametrize("T,N,K", [(1, 300, 1100), (33, 129, 1024), (520, 1000, 1030), (300, 2050, 2048)])
def test_every_plan(ops, pairs, bn, parts, T, N, K):
    """Single CTAs and pairs, every share of K, tiles that end behind the last token and channel."""
    _check_product(ops, T, N, K, plan=(pairs, bn, parts))


def test_plans_that_do_not_exist_are_refused(ops):
    for plan in ((False, 8, 1), (False, 272, 1), (False, 24, 1), (True, 48, 1), (True, 64, 5), (False, 64, 9), (False, 64, 0), (False, 64, 3)):
        with pytest.raises(ops.NativeError):
            _check_product(ops, 3, 64, 256, plan=plan)


@pytest.mark.parametrize("T", [3, 400])
def test_rows_and_results_in_wider_buffers(ops, T):
    buf = torch.full((T, 400), 3.0, device="cuda", dtype=BF)
    for a, n in ((0, 333), (1, 332), (4, 336), (8, 200)):
        buf.fill_(3.0)
        _check_product(ops, T, n, 320, at=16, out=buf[:, a:a + n])
        assert (buf[:, :a] == 3).all() and (buf[:, a + n:] == 3).all()


def test_the_longest_sums_are_whole(ops):
    K = ref.INT8_MAX_K
    q = torch.full((2, K + 1), -127, device="cuda", dtype=torch.int8)[:, :K]
    q[1] = -128
    w = torch.full((3, K + 1), -128, device="cuda", dtype=torch.int8)[:, :K]
    w[1] = 127
    y = ops.gemm_int8(Int8Rows(q, torch.full((2,), 2.0 ** -31, device="cuda")), w, torch.ones(3, device="cuda"))
    want = (q.double() @ w.double().t() * 2.0 ** -31).to(BF)
    assert torch.equal(y, want)


def test_rows_behind_the_last_one_are_left_alone(ops):
    for T in (1, 5, 130, 300):
        buf = torch.full((T + 3, 256), 9.0, device="cuda", dtype=BF)
        _check_product(ops, T, 256, 256, out=buf[:T])
        assert (buf[T:] == 9).all()


def test_offsets_past_32_bits(ops):
    """Tensors of more than 2^31 numbers: the first and the last rows."""
    T, K = 140000, 16384
    x = torch.zeros(T, K, device="cuda", dtype=BF)
    g = _gen(11)
    ends = torch.tensor([0, 1, T // 2, T - 2, T - 1], device="cuda")
    x[ends] = _randn(g, 5, K)
    r = ops.quant_rows_int8(x)
    want = ref.quant_rows_int8(x[ends].cpu())
    assert torch.equal(r.q[ends].cpu(), want.q) and torch.equal(r.scale[ends].cpu(), want.scale) and not r.scale[2:T // 2].any()
    w = 1 + _randn(g, K, std=0.1)
    before = x[ends]
    small = ops.norm_block(before.clone(), before.clone(), w, 1e-5)
    big = ops.norm_block(x, x, w, 1e-5)             # (y and the residual are one tensor, which the sum replaces)
    assert torch.equal(x[ends], 2 * before) and ((big[ends].double() - small.double()).abs() <= 2 * HALF * small.double().abs()).all()
    del big, x
    wq, ws = ref.quantize_weight_int8(_randn(g, 16384, 64, dtype=torch.float32))
    rows = Int8Rows(r.q[:, :64], r.scale)
    y = ops.gemm_int8(rows, wq, ws)
    part = ops.gemm_int8(Int8Rows(r.q[ends, :64].contiguous(), r.scale[ends]), wq, ws)
    assert torch.equal(y[ends], part)


def test_the_same_tensor_twice(ops):
    """y as the residual, one weight for both norms, a gate that is the weight, rows that are both operands of a product."""
    x, w = _randn(_gen(2), 40, 256), 1 + _randn(_gen(3), 256, std=0.1)
    h = torch.empty_like(x)
    a = ops.norm_block(x, x, w, 1e-5, post_weight=w, gate=w, residual_out=h)
    b = ops.norm_block(x.clone(), x.clone(), w.clone(), 1e-5, post_weight=w.clone(), gate=w.clone())
    assert torch.equal(a, b)
    keep = x.clone()
    ops.norm_block(x, x, w, 1e-5, post_weight=w, gate=w)
    assert torch.equal(x, h)
    r = ops.quant_rows_int8(keep)
    y = ops.gemm_int8(r, r.q, r.scale)
    want = (r.q.double() @ r.q.double().t()) * r.scale.double()[:, None] * r.scale.double()
    assert ((y.double() - want).abs() <= (HALF + 6 * E) * want.abs()).all()


def test_calls_on_another_stream_than_the_default(ops):
    y, res, w, up, down, I = _state(65, 512, 640)
    want = _feed_forward(ops, y, res.clone(), w, up, down, I)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [_feed_forward(ops, y, res.clone(), w, up, down, I) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


# ------------------------------------------------------------------------------------------------ together
def _feed_forward(ops, y, res, w, up, down, I):
    x = ops.norm_block(y, res, w, 1e-5, post_weight=w, int8=True)
    h = ops.gemm_int8(x, *up)
    return h, ops.gemm_int8(ops.act_mul_int8(h, I, "silu"), *down)


def _state(T, H, I, seed=0):
    g = _gen(T, H, I, seed)
    up = ref.quantize_weight_int8(_randn(g, 2 * I, H, dtype=torch.float32, std=H ** -0.5))
    down = ref.quantize_weight_int8(_randn(g, H, I, dtype=torch.float32, std=I ** -0.5))
    return _randn(g, T, H), _randn(g, T, H), 1 + _randn(g, H, std=0.1), up, down, I


@pytest.mark.parametrize("T,H,I", [(1, 1024, 2816), (48, 512, 1000), (333, 1032, 520)])
def test_a_feed_forward(ops, T, H, I):
    """Norms, product, activation, product: each step against its definition on what the step before it gave, and the whole against the same in bf16 weights."""
    y, res, w, up, down, I = _state(T, H, I)
    h0 = res.clone()
    h, out = _feed_forward(ops, y, h0, w, up, down, I)
    a = torch.nn.functional.silu(h[:, :I].double()) * h[:, I:].double()
    whole = a @ (down[0].double() * down[1].double()[:, None]).t()
    # the rows' rounding: half a step of max / 127, of random sign, over I products of weights of the size I^-0.5; six deviations, and the result's own rounding
    sd = (a.abs().amax(1) / 127 / 12 ** 0.5)[:, None] * (down[0].double() * down[1].double()[:, None]).square().sum(1).sqrt()
    assert ((out.double() - whole).abs() <= 6 * sd + HALF * whole.abs()).all()


def test_captured_graphs_and_streams(ops):
    """Two captured passes replayed at the same time on two streams, while a third runs eagerly: none has scratch that another one uses."""
    states = [_state(T, 1024, 1536, T) for T in (1, 17, 300)]
    want = [_feed_forward(ops, y, res.clone(), *rest) for y, res, *rest in states]
    graphs = []
    for y, res, *rest in states[:2]:
        r, work = res.clone(), torch.empty_like(res)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            work.copy_(r)
            _feed_forward(ops, y, work, *rest)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                work.copy_(r)
                out = _feed_forward(ops, y, work, *rest)
        graphs.append((g, s, out, r, work))          # (a graph keeps no tensor alive that was made outside)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s, *_ in graphs:
            with torch.cuda.stream(s):
                g.replay()
        y, res, *rest = states[2]
        eager = _feed_forward(ops, y, res.clone(), *rest)
    torch.cuda.synchronize()
    for got, w in zip([graphs[0][2], graphs[1][2], eager], want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_results_do_not_depend_on_other_rows(ops):
    """A row's sums are whole numbers and its norms its own: alone, and among any number of others, the same bits."""
    y, res, w, up, down, I = _state(300, 512, 768)
    h, out = _feed_forward(ops, y, res.clone(), w, up, down, I)
    for a, b in ((0, 1), (5, 22), (100, 300)):
        h1, out1 = _feed_forward(ops, y[a:b], res[a:b].clone(), w, up, down, I)
        assert torch.equal(h1, h[a:b]) and torch.equal(out1, out[a:b])


def test_empty_calls_launch_nothing(ops):
    w, ws = ref.quantize_weight_int8(torch.randn(5, 16, device="cuda"))
    n = ops.launch_count
    r = ops.quant_rows_int8(torch.empty(0, 16, device="cuda", dtype=BF))
    assert ops.gemm_int8(r, w, ws).shape == (0, 5) and ops.launch_count == n
    assert ops.norm_block(None, torch.empty(0, 16, device="cuda", dtype=BF), torch.ones(16, device="cuda", dtype=BF), 1e-6).shape == (0, 16)
    assert ops.launch_count == n


# ------------------------------------------------------------------------------------------------ models
TARGETS = ["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"]


def _model(device, dtype, config=None):
    from lorax_b200.config import tiny_llama
    from lorax_b200.models.decoder import DecoderModel, Int8Weight
    cfg = config or tiny_llama()
    model = DecoderModel.random_init(cfg, device, dtype, seed=0, std=0.05)
    model.quantize("w8a8")
    assert isinstance(model.layers[0].gate_up_w, Int8Weight)
    return cfg, model


def _adapters(cfg, model):
    from lorax_b200.adapters.lora import random_adapter
    from lorax_b200.adapters.manager import AdapterManager
    mgr = AdapterManager(model, arena_bytes=64 << 20, host_bytes=128 << 20)
    for i in range(3):
        c, mm = random_adapter(cfg, r=[8, 16, 32][i], alpha=16, target_modules=TARGETS, seed=10 + i, std_a=0.05, std_b=0.05)
        mgr.register(f"a{i}", c, mm)
        assert mgr.load(i + 1, f"a{i}")
    return mgr


@pytest.mark.parametrize("adapters", [False, True])
def test_a_model_in_8_bit_integers_matches_the_plain_operators(ops, adapters):
    from lorax_b200.runtime.kv_cache import KVCache
    from lorax_b200.runtime.runner import ModelRunner, PrefillItem
    g = torch.Generator().manual_seed(3)
    outs = []
    for device, dtype in (("cuda", BF), ("cpu", torch.float32)):
        cfg, m = _model(device, dtype)
        if adapters:
            _adapters(cfg, m)
        if device == "cuda":
            prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (17, 64, 90)]
        kv = KVCache(cfg.num_hidden_layers, 32, m.nkv, m.d, m.dtype, m.device)
        r = ModelRunner(m, kv, max_batch=4, max_seq_tokens=256, max_prefill_tokens=512, use_graphs=False)
        items = [PrefillItem(p, 0, [1 + 3 * i, 2 + 3 * i, 3 + 3 * i], adapter_index=i if adapters else 0) for i, p in enumerate(prompts)]
        outs.append(r.prefill(items)[2].float().cpu())
    # bf16 activations and weights (rounded before they are quantised) against 32 bits: what the same model in bf16 weights is allowed (0.03), and the steps of a
    # 127th that fall to the other side on the way, as far off as the rounding to 8 bits itself
    assert (outs[0] - outs[1]).norm() / outs[1].norm() < 0.06


@pytest.mark.parametrize("kind", ["gemma2", "granite", "gpt_neox", "cohere", "mixtral"])
def test_models_of_other_shapes_match_the_plain_operators(ops, kind):
    """Norms on both sides, a residual multiplier, parallel blocks with two norms or one, experts that stay in bf16."""
    from lorax_b200.config import ModelConfig
    from lorax_b200.runtime.kv_cache import KVCache
    from lorax_b200.runtime.runner import ModelRunner, PrefillItem
    more = dict(gemma2=dict(norm_weight_offset=1.0, tie_word_embeddings=True, hidden_act="gelu_pytorch_tanh"), granite=dict(residual_multiplier=0.22),
                gpt_neox=dict(parallel_residual=True, norm_type="layernorm", hidden_act="gelu"), cohere=dict(parallel_residual=True, norm_type="layernorm_nobias"),
                mixtral=dict(num_local_experts=4, num_experts_per_tok=2))[kind]
    c = ModelConfig(model_type=kind, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, intermediate_size=512, vocab_size=256, head_dim=64,
                    max_position_embeddings=256, **more)
    prompts = [torch.randint(0, 256, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (5, 70)]
    outs = []
    for device, dtype in (("cuda", BF), ("cpu", torch.float32)):
        m = _model(device, dtype, c)[1] if kind != "mixtral" else _model_of(c, device, dtype)
        kv = KVCache(c.num_hidden_layers, 16, m.nkv, m.d, m.dtype, m.device)
        r = ModelRunner(m, kv, max_batch=4, max_seq_tokens=128, max_prefill_tokens=256, use_graphs=False)
        outs.append(r.prefill([PrefillItem(p, 0, [1 + 3 * i, 2 + 3 * i, 3 + 3 * i], adapter_index=0) for i, p in enumerate(prompts)])[2].float().cpu())
    assert (outs[0] - outs[1]).norm() / outs[1].norm() < 0.06      # (as for the model above)


def _model_of(c, device, dtype):
    from lorax_b200.models.decoder import DecoderModel
    m = DecoderModel.random_init(c, device, dtype, seed=0, std=0.05)
    m.quantize("w8a8")
    return m


def test_generation_with_graphs_is_that_without(ops):
    """Captured decode steps, adapters among them, give the tokens of eager ones: no operator's result depends on the rows beside it."""
    from lorax_b200.config import EngineConfig
    from lorax_b200.runtime.engine import Engine
    cfg, m = _model("cuda", BF)
    _adapters(cfg, m)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, cfg.vocab_size, (30 + i,), generator=g).tolist() for i in range(6)]
    a, b = (Engine(m, EngineConfig(max_total_tokens=256, max_batch_prefill_tokens=1024), num_blocks=128, max_batch=8, use_graphs=graphs).generate(
        prompts, max_new_tokens=16, adapter_indices=[0, 1, 2, 3, 1, 0]) for graphs in (True, False))
    assert a == b and all(len(x) == 16 for x in a)
