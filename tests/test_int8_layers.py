"""Operators of layers in 8-bit integers on the CPU: what they compute, and what they refuse in front of any launch."""
import pytest
import torch

from lorax_b200.ops import reference as ref
from lorax_b200.ops.reference import Int8Rows

BF = torch.bfloat16


def _ops():
    """The plain forms and the bindings: both check their arguments in the same way (the bindings raise before they look for a device)."""
    from lorax_b200.ops import native
    return (ref, native)


def test_rows_are_rounded_to_the_nearest_step():
    x = torch.randn(17, 259, generator=torch.Generator().manual_seed(1)) * 3
    r = ref.quant_rows_int8(x)
    assert r.q.dtype == torch.int8 and r.q.stride(0) == 272 and r.scale.dtype == torch.float32
    top = x.abs().amax(1)
    assert torch.equal(r.scale, top / torch.full_like(top, 127.0))
    back = r.q.double() * r.scale.double()[:, None]
    assert ((back - x.double()).abs() <= 0.5 * r.scale.double()[:, None] * (1 + 2 ** -20)).all()
    assert (r.q.int().abs().amax(1) == 127).all()


def test_ties_go_to_the_even_integer_and_neighbours_of_ties_do_not():
    """A row whose scale is 1: halves are ties, and the numbers beside them are not."""
    up = torch.nextafter(torch.tensor(2.5), torch.tensor(9.0))
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, up.item(), 126.5, -126.5]])
    assert ref.quant_rows_int8(x).q.tolist() == [[127, 0, 2, 2, 0, -2, -2, 3, 126, -126]]


def test_rows_without_a_scale():
    x = torch.tensor([[0.0, -0.0, 0.0], [1.0, float("inf"), 2.0], [float("nan"), 1.0, 2.0], [3.0, 1.0, -3.0], [2.0 ** -149, 0.0, 0.0]])
    r = ref.quant_rows_int8(x)
    assert r.scale[0] == 0 and r.scale[1].isnan() and r.scale[2].isnan() and r.scale[4] == 0
    assert r.q.tolist() == [[0, 0, 0], [0, 0, 0], [0, 0, 0], [127, 42, -127], [0, 0, 0]]
    w, ws = ref.quantize_weight_int8(torch.randn(5, 3))
    y = ref.gemm_int8(r, w, ws, bias=torch.ones(5), dtype=torch.float32)
    assert (y[0] == 1).all() and y[1:3].isnan().all() and y[3:].isfinite().all()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "relu2"])
@pytest.mark.parametrize("gated", [True, False])
def test_activations(act, gated):
    x = torch.randn(6, 2 * 33 if gated else 33, generator=torch.Generator().manual_seed(2))
    out = torch.empty(6, 33)
    r = ref.act_mul_int8(x, 33, act, gated, out=out)
    assert torch.equal(out, ref.act_mul(x, 33, act, gated=gated))
    s = ref.quant_rows_int8(out)
    assert torch.equal(r.q, s.q) and torch.equal(r.scale, s.scale)


@pytest.mark.parametrize("layernorm", [False, True])
def test_a_norm_without_extras_is_norm_residual(layernorm):
    g = torch.Generator().manual_seed(3)
    y, res, w, b = torch.randn(4, 40, generator=g), torch.randn(4, 40, generator=g), torch.randn(40, generator=g), torch.randn(40, generator=g)
    r0, r1 = res.clone(), res.clone()
    a = ref.norm_residual(y, r0, w, 1e-5, bias=b, weight_offset=1.0, x_scale=0.22, layernorm=layernorm)
    c = ref.norm_block(y, r1, w, 1e-5, bias=b, weight_offset=1.0, scale=0.22, layernorm=layernorm)
    torch.testing.assert_close(c, a, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(r1, r0, rtol=1e-6, atol=1e-6)
    assert torch.equal(ref.norm_block(None, res, w, 1e-5, layernorm=layernorm), ref.norm_residual(res, None, w, 1e-5, layernorm=layernorm)) or layernorm


def test_gates_of_every_shape():
    g = torch.Generator().manual_seed(4)
    y, res, w, pw = torch.randn(5, 24, generator=g), torch.randn(5, 24, generator=g), torch.randn(24, generator=g), torch.randn(24, generator=g)
    for gate in (torch.tensor(0.5), torch.tensor([0.5]), torch.randn(24, generator=g), torch.tensor([[1.0], [0.0], [1.0], [0.0], [0.0]]), torch.randn(5, 24, generator=g)):
        h = torch.empty_like(res)
        x = ref.norm_block(y, res, w, 1e-6, post_weight=pw, gate=gate, scale=0.5, residual_out=h)
        n = y * torch.rsqrt((y * y).mean(1, keepdim=True) + 1e-6) * pw
        torch.testing.assert_close(h, res + 0.5 * gate * n, rtol=1e-6, atol=1e-6)
        torch.testing.assert_close(x, h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * w, rtol=1e-6, atol=1e-6)
        if gate.dim() == 2 and gate.shape[1] == 1:
            assert torch.equal(h[1], res[1])           # a token whose gate is shut keeps its stream
    r = ref.norm_block(y, res.clone(), w, 1e-6, int8=True)
    assert isinstance(r, Int8Rows) and torch.equal(r.q, ref.quant_rows_int8(ref.norm_block(y, res.clone(), w, 1e-6)).q)


def test_products_are_whole():
    g = torch.Generator().manual_seed(5)
    q, w = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8) for s in ((3, 1 << 12), (7, 1 << 12)))
    one = lambda n: torch.ones(n)
    y = ref.gemm_int8(Int8Rows(q, one(3)), w, one(7), dtype=torch.float32)
    assert torch.equal(y, (q.long() @ w.long().t()).float())


def test_weights_in_pieces_are_those_in_one(monkeypatch):
    w = torch.randn(300, 400, generator=torch.Generator().manual_seed(6))
    whole = ref.quantize_weight_int8(w)
    real = torch.Tensor.split
    monkeypatch.setattr(torch.Tensor, "split", lambda t, n, dim=0: real(t, min(n, 77), dim))
    parts = ref.quantize_weight_int8(w)
    assert all(torch.equal(a, b) for a, b in zip(whole, parts)) and parts[0].stride() == whole[0].stride()


def test_empty_calls():
    w, ws = ref.quantize_weight_int8(torch.randn(5, 8))
    r = ref.quant_rows_int8(torch.empty(0, 8))
    assert ref.gemm_int8(r, w, ws).shape == (0, 5)
    assert ref.norm_block(torch.empty(0, 8), torch.empty(0, 8), torch.ones(8), 1e-6).shape == (0, 8)
    assert ref.act_mul_int8(torch.empty(0, 8), 4).q.shape == (0, 4)


def _rows(T, K):
    return ref.empty_int8_rows(T, K, torch.empty(0))


NORM = dict(y=torch.zeros(3, 16, dtype=BF), residual=torch.zeros(3, 16, dtype=BF), weight=torch.ones(16, dtype=BF), eps=1e-6)
_BUF = torch.zeros(3, 64, dtype=BF)


@pytest.mark.parametrize("change", [
    dict(y=torch.zeros(2, 16, dtype=BF)), dict(y=torch.zeros(3, 16)), dict(residual=torch.zeros(16, dtype=BF)), dict(y=torch.zeros(16, 3, dtype=BF).t()),
    dict(weight=torch.ones(8, dtype=BF)), dict(weight=torch.ones(16)), dict(weight=torch.ones(32, dtype=BF)[::2]), dict(weight=None),
    dict(post_bias=torch.zeros(16, dtype=BF)), dict(post_weight=torch.ones(1, dtype=BF)), dict(gate=torch.ones(3, dtype=BF)), dict(gate=torch.ones(16)),
    dict(gate=torch.ones(3, 32, dtype=BF)[:, ::2]), dict(gate=0.5), dict(y=1.0), dict(gate=torch.ones(1, 1, 16, dtype=BF)), dict(y=None, scale=0.5), dict(y=None, gate=torch.ones(1, dtype=BF)),
    dict(y=None, post_weight=torch.ones(16, dtype=BF)), dict(y=None, residual_out=torch.zeros(3, 16, dtype=BF)),
    dict(y=_BUF[:, :16], residual=_BUF[:, 8:24]), dict(y=_BUF[:, :16], residual_out=_BUF[:, 8:24]), dict(residual_out=torch.zeros(3, 16)),
    dict(residual=torch.zeros(2, 16385, dtype=BF), y=torch.zeros(2, 16385, dtype=BF), weight=torch.zeros(16385, dtype=BF)), dict(out=torch.zeros(3, 17, dtype=BF))])
def test_norms_that_are_refused(change):
    for ops in _ops():
        with pytest.raises(ValueError, match="norm_block"):
            ops.norm_block(**{**NORM, **change})


def test_results_on_top_of_inputs():
    """y and the residual may be written over, value by value; anything else may not, and rows of one buffer may take turns."""
    buf = torch.zeros(3, 32, dtype=BF)
    ok = [dict(residual_out=NORM["residual"]), dict(y=NORM["residual"]), dict(out=NORM["y"]), dict(residual_out=NORM["y"]), dict(y=buf[:, :16], residual=buf[:, 16:]), dict(y=buf[:, :16], residual=buf[:, 16:], out=buf[:, :16])]
    for change in ok:
        ref.norm_block(**{**NORM, **change})
    vec = torch.ones(48, dtype=BF)
    bad = [dict(out=NORM["residual"]), dict(residual_out=vec.view(3, 16), weight=vec[:16]), dict(out=vec.view(3, 16), gate=vec[16:32]),
           dict(out=vec[:48].view(3, 16), residual_out=vec[:48].view(3, 16)), dict(out=buf[:, :16], residual_out=buf[:, 8:24])]
    for change in bad:
        for ops in _ops():
            with pytest.raises(ValueError, match="norm_block"):
                ops.norm_block(**{**NORM, **change})


GEMM = dict(x=_rows(3, 32), w=torch.zeros(5, 32, dtype=torch.int8), w_scale=torch.ones(5))


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(3, 32, dtype=torch.int8)), dict(x=_rows(3, 48)), dict(x=Int8Rows(torch.zeros(3, 32), torch.ones(3))), dict(x=Int8Rows(_rows(3, 32).q, torch.ones(4))),
    dict(x=Int8Rows(torch.zeros(3, 40, dtype=torch.int8)[:, :32], torch.ones(3))), dict(x=Int8Rows(torch.zeros(3, 48, dtype=torch.int8)[:, 8:40], torch.ones(3))),
    dict(x=Int8Rows(_rows(3, 32).q, torch.ones(3, dtype=torch.float64))), dict(w=torch.zeros(5, 32)), dict(w=torch.zeros(32, 5, dtype=torch.int8).t()),
    dict(w_scale=torch.ones(5, 1)), dict(w_scale=0.5), dict(w=None), dict(w_scale=torch.ones(10)[::2]), dict(bias=torch.ones(5)), dict(bias=torch.ones(4, dtype=BF)),
    dict(out=torch.zeros(3, 6, dtype=BF)), dict(out=torch.zeros(3, 5)), dict(out=torch.zeros(5, 3, dtype=BF).t()), dict(x=_rows(3, 0), w=torch.zeros(5, 0, dtype=torch.int8)),
    dict(x=_rows(1, 1 << 17), w=torch.zeros(1, 1 << 17, dtype=torch.int8), w_scale=torch.ones(1))])
def test_products_that_are_refused(change):
    for ops in _ops():
        with pytest.raises(ValueError, match="gemm_int8"):
            ops.gemm_int8(**{**GEMM, **change})


def test_a_product_on_top_of_its_scales_is_refused():
    x = Int8Rows(_rows(4, 32).q, torch.ones(4))
    out = x.scale.view(BF)[:4].view(4, 1)
    for ops in _ops():
        with pytest.raises(ValueError, match="apart"):
            ops.gemm_int8(x, torch.zeros(1, 32, dtype=torch.int8), torch.ones(1), out=out)


@pytest.mark.parametrize("x", [torch.zeros(3, dtype=BF), torch.zeros(3, 0, dtype=BF), torch.zeros(8, 3, dtype=BF).t(), torch.zeros(1, 4, dtype=BF).expand(3, 4),
                               torch.zeros(3, 4, dtype=torch.int32)])
def test_rows_that_are_refused(x):
    for ops in _ops():
        with pytest.raises(ValueError, match="quant_rows_int8"):
            ops.quant_rows_int8(x)


def test_activations_that_are_refused():
    x = torch.zeros(3, 16, dtype=BF)
    for ops in _ops():
        for args, kw in (((x, 7), {}), ((x, 8, "tanh"), {}), ((x, 0), {}), ((x, 8, "silu", False), {}), ((x[0], 8), {}), ((x, 8), dict(out=x[:, :8])),
                         ((x, 8), dict(out=torch.zeros(3, 8))), ((x, 8), dict(out=torch.zeros(3, 9, dtype=BF)))):
            with pytest.raises(ValueError, match="act_mul_int8"):
                ops.act_mul_int8(*args, **kw)


def test_the_bindings_take_bf16_on_a_gpu():
    from lorax_b200.ops import native
    for call in (lambda: native.quant_rows_int8(torch.zeros(3, 16)), lambda: native.act_mul_int8(torch.zeros(3, 16), 8),
                 lambda: native.norm_block(torch.zeros(3, 16), torch.zeros(3, 16), torch.ones(16), 1e-6),
                 lambda: native.gemm_int8(_rows(3, 32), torch.zeros(5, 32, dtype=torch.int8), torch.ones(5), dtype=torch.float32)):
        with pytest.raises(ValueError, match="bf16"):
            call()
    for call in (lambda: native.quant_rows_int8(torch.zeros(3, 16, dtype=BF)), lambda: native.norm_block(**NORM), lambda: native.gemm_int8(**GEMM)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_limits_of_the_library_and_of_python_agree(monkeypatch):
    from lorax_b200.ops import native, native_int8
    native_int8.check_limits(native.load())
    for name, value in (("NORM_BLOCK_MAX_WIDTH", ref.NORM_BLOCK_MAX_WIDTH + 1), ("INT8_MAX_K", ref.INT8_MAX_K + 1), ("_NORM", native_int8._GEMM), ("_ROWS", native_int8._GEMM),
                        ("_GEMM", native_int8._ROWS)):
        monkeypatch.setattr(native_int8, name, value)
        with pytest.raises(native.NativeError, match="C\\+\\+ says"):
            native_int8.check_limits(native.load())
        monkeypatch.undo()


@pytest.mark.parametrize("rows", [(1 << 31) - 1, (1 << 31) - (1 << 16) + 1, 1 << 31, 1 << 40])
def test_the_library_refuses_rows_whose_numbers_pass_31_bits(rows):
    """Tiles and rows in flight behind the last one are counted in 32 bits.  (The library says no in front of its first use of a device or of an address.)"""
    from lorax_b200.ops import native, native_int8
    lib = native.load()
    assert lib.lx_norm_block(native_int8._NORM.pack(*([0] * 18), rows, 8, 0, 0, 148, 1, 0, 1e-6, 0.0, 1.0)) < 0
    assert lib.lx_rows_int8(native_int8._ROWS.pack(*([0] * 7), rows, 8, -1, 0, 0, 148, 1, 0)) < 0
    for T, N in ((rows, 1), (1, rows)):
        assert lib.lx_gemm_int8(native_int8._GEMM.pack(0, 16, 0, 0, 16, 0, 0, 0, 8, T, N, 16, 0, 0, 148, 0, 0)) < 0
        if rows < 1 << 31:
            assert lib.lx_gemm_int8_plan(T, N, 16, 148, (native_int8.I * 4)(74, 33, 22, 15), (native_int8.I * 4)()) < 0


def _plan(T, N, K, sms=148, clusters=(74, 33, 22, 15)):
    import ctypes

    from lorax_b200.ops import native
    out = (ctypes.c_int * 4)()
    assert native.load().lx_gemm_int8_plan(T, N, K, sms, (ctypes.c_int * 4)(*clusters), out) == 0
    return tuple(out)


@pytest.mark.parametrize("sms,clusters", [(148, (74, 33, 22, 15)), (148, (0, 0, 0, 0)), (20, (10, 4, 2, 1)), (1, (0, 0, 0, 0))])
def test_plans_stay_within_what_tiles_and_clusters_allow(sms, clusters):
    rng = __import__("random").Random(7)
    sizes = [(1, 1, 1), (1 << 20, 1, 1), (1, 1 << 20, 128), (4001, 28672, 4096), (300, 100, (1 << 17) - 1)]
    sizes += [tuple(int(2 ** rng.uniform(0, top)) for top in (13, 15, 15)) for _ in range(400)]
    for T, N, K in sizes:
        pairs, bn, parts, stages = _plan(T, N, K, sms, clusters)
        blocks = -(-K // 128)
        assert 1 <= parts <= blocks and 16 <= bn <= 256
        if pairs:
            assert bn % 32 == 0 and parts <= 4 and clusters[parts - 1] > 0 and T > 32
            assert parts == 1 or -(-N // 256) * -(-T // bn) <= clusters[parts - 1]      # a cluster has one tile, and all run at the same time
        else:
            # the ring holds a tile's sums, and fits beside scales and barriers
            assert bn % 16 == 0 and parts <= 8 and 4 <= stages <= 16 and stages * (128 + bn) * 128 >= bn * 512 and stages * (128 + bn) * 128 <= 216 * 1024


@pytest.mark.parametrize("size,pairs,parts", [
    ((1, 28672, 4096), False, 1),       # 20.2 us; shared by two CTAs 25.6
    ((1, 4096, 14336), False, 8),       # 12.1; by four 14.7, alone 34.5
    ((48, 6144, 4096), False, 4),       # 9.0; alone 14
    ((256, 4096, 14336), False, 4),     # 21.2; pairs sharing by three 21.6
    ((512, 4096, 14336), True, 2),      # 27.3; single CTAs 30.3, pairs alone 42
    ((256, 28672, 4096), True, 1),      # 32.4; single CTAs 42.2
    ((4001, 28672, 4096), True, 1)])
def test_plans_that_measured_quickest(size, pairs, parts):
    got = _plan(*size)
    assert (got[0] > 0, got[2]) == (pairs, parts)


# ------------------------------------------------------------------------------------------------ models
def _step(model, T=9):
    from lorax_b200.models.decoder import StepInputs
    c = model.config
    kv = [torch.zeros(2, model.nkv, 2, 32, model.d, dtype=model.dtype) for _ in range(c.num_hidden_layers)]
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    seq, q0 = ref.prefill_tiles([T])
    inp = StepInputs(input_ids=torch.arange(3, 3 + T, dtype=torch.int32), positions=torch.arange(T, dtype=torch.int32), slots=torch.arange(32, 32 + T, dtype=torch.int32),
                     is_prefill=True, block_tables=i32(1).view(1, 1), cu_q=i32(0, T), cache_lens=i32(0), tile_seq=torch.as_tensor(seq, dtype=torch.int32),
                     tile_q0=torch.as_tensor(q0, dtype=torch.int32))
    return model.forward(inp, kv)


@pytest.mark.parametrize("kind", ["llama", "gemma2", "granite", "gpt_neox", "cohere", "gpt2", "mixtral"])
def test_a_model_in_8_bit_integers_is_near_the_same_in_32_bits(kind):
    """Norms on both sides (gemma2), residual multiplier (granite), parallel blocks with one norm or two (cohere, gpt_neox), layer norms and biases (gpt2), experts."""
    from lorax_b200.config import ModelConfig
    from lorax_b200.models.decoder import DecoderModel, Int8Weight
    more = dict(gemma2=dict(norm_weight_offset=1.0, tie_word_embeddings=True, hidden_act="gelu_pytorch_tanh"), granite=dict(residual_multiplier=0.22),
                gpt_neox=dict(parallel_residual=True, norm_type="layernorm", hidden_act="gelu"), cohere=dict(parallel_residual=True, norm_type="layernorm_nobias"),
                gpt2=dict(norm_type="layernorm", learned_positions=True, mlp_bias=True, attention_bias=True, hidden_act="gelu_new"),
                mixtral=dict(num_local_experts=4, num_experts_per_tok=2)).get(kind, {})
    c = ModelConfig(model_type=kind, hidden_size=64, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=4 if kind == "gpt2" else 2, intermediate_size=96, vocab_size=128,
                    head_dim=16, max_position_embeddings=64, **more)
    dense = DecoderModel.random_init(c, "cpu", torch.float32, seed=3, std=0.1)
    small = DecoderModel.random_init(c, "cpu", torch.float32, seed=3, std=0.1)
    small.quantize("w8a8")
    assert small.quantized == "w8a8" and all(isinstance(lw.qkv_w, Int8Weight) and isinstance(lw.o_w, Int8Weight) for lw in small.layers)
    a, b = _step(dense), _step(small)
    assert torch.isfinite(b).all()
    # twelve products, each off by two roundings of a 127th of a row's largest value (some 3 deviations), 0.29 / 127 * 3 = 0.7 % of a result twice, of random
    # sign: 0.01 * sqrt(12) = 3.4 %; twice that for what attention and norms make of it
    assert (a - b).norm() / a.norm() < 0.07
    again = DecoderModel.random_init(c, "cpu", torch.float32, seed=3, std=0.1)
    again.quantize("w8a8")
    assert torch.equal(_step(again), b)


def test_layer_by_layer_designs_are_not_quantised():
    from lorax_b200.models.decoder import DecoderModel
    m = DecoderModel.__new__(DecoderModel)
    m.mixed, m.config = True, type("C", (), dict(model_type="x"))()
    with pytest.raises(ValueError, match="not supported"):
        m.quantize("w8a8")


def test_w8a8_is_a_name_of_the_shard_s_quantize_flag():
    from lorax_b200.server.cli import QUANTIZE_CHOICES
    assert "w8a8" in QUANTIZE_CHOICES


# ------------------------------------------------------------------------------------------------ devices
def test_operators_run_on_their_tensors_device_whichever_is_current(monkeypatch):
    """Tensors of a second device while the first is current: launches, with the second device's stream, while it is the current one."""
    from lorax_b200.ops import native, native_int8
    current, launches = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        def __getattr__(self, name):
            at = dict(lx_norm_block=(native_int8._NORM, 24), lx_rows_int8=(native_int8._ROWS, 14), lx_gemm_int8=(native_int8._GEMM, 16))[name]
            return lambda block: (launches.append((name, current[0], at[0].unpack(block)[at[1]])), 0)[1]

    class Space:
        status, num_sms = torch.zeros(1, dtype=torch.int32), 148
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    monkeypatch.setattr(native_int8, "_devices", {})
    monkeypatch.setattr(native_int8.nv, "load", Library)
    monkeypatch.setattr(native_int8.nv, "workspace", lambda d: Space())
    x = torch.zeros(3, 32, dtype=BF)
    native.quant_rows_int8(x)
    native.act_mul_int8(x, inter=16)
    native.norm_block(None, residual=x, weight=x[0], eps=1e-6)
    native.gemm_int8(**GEMM)
    assert launches == [(n, 1, 101) for n in ("lx_rows_int8", "lx_rows_int8", "lx_norm_block", "lx_gemm_int8")] and current == [0]
    current[0] = 1
    native.quant_rows_int8(x)
    assert launches[-1] == ("lx_rows_int8", 1, 101) and current == [1]


def test_what_a_launch_gets(monkeypatch):
    """The packed blocks, field by field: addresses, distances (a single row's own says nothing), sizes and flags."""
    from lorax_b200.ops import native, native_int8
    got = {}

    class Library:
        def __getattr__(self, name):
            return lambda block: (got.update({name: block}), 0)[1]
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 7, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(native_int8, "_devices", {0: (148, 5)})
    monkeypatch.setattr(native_int8.nv, "load", Library)
    y, res, w, pw, b, pb = (torch.zeros(*s, dtype=BF) for s in ((3, 40), (3, 24), (24,), (24,), (24,), (24,)))
    gate, h, out = torch.zeros(3, 1, dtype=BF), torch.zeros(3, 24, dtype=BF), torch.zeros(3, 32, dtype=BF)
    r = native.norm_block(y[:, 8:32], res, w, 1e-5, post_weight=pw, gate=gate, scale=0.5, bias=b, post_bias=pb, weight_offset=1.0, layernorm=True, residual_out=h, out=out[:, :24],
                          int8=True)
    f = native_int8._NORM.unpack(got["lx_norm_block"])
    assert f[:25] == (y.data_ptr() + 16, 40, res.data_ptr(), 24, h.data_ptr(), 24, pw.data_ptr(), pb.data_ptr(), w.data_ptr(), b.data_ptr(), gate.data_ptr(), 1, 0, out.data_ptr(), 32,
                      r.q.data_ptr(), 32, r.scale.data_ptr(), 3, 24, 1, 5, 148, -1, 7) and f[25:] == (1e-5, 1.0, 0.5)
    x = native.norm_block(None, res[:1], w, 1e-5)
    f = native_int8._NORM.unpack(got["lx_norm_block"])
    assert f[:6] == (0, 0, res.data_ptr(), 32, 0, 0) and f[13:18] == (x.data_ptr(), 24, 0, 32, 0) and x.shape == (1, 24)
    native.norm_block(y[:, 8:32], res, w, 1e-5)
    assert native_int8._NORM.unpack(got["lx_norm_block"])[4:6] == (res.data_ptr(), 24)          # in place
    v = native.act_mul_int8(y, 20, "relu2", out=out[:, 1:21])
    assert native_int8._ROWS.unpack(got["lx_rows_int8"]) == (y.data_ptr(), 40, v.q.data_ptr(), 32, v.scale.data_ptr(), out.data_ptr() + 2, 32, 3, 20, 4, 1, 5, 148, -1, 7)
    wq, ws = ref.quantize_weight_int8(torch.randn(5, 20))
    z = native.gemm_int8(v, wq, ws, bias=b[:5], w_const=True)
    assert z.shape == (3, 5) and z.stride() == (8, 1)
    assert native_int8._GEMM.unpack(got["lx_gemm_int8"]) == (v.q.data_ptr(), 32, v.scale.data_ptr(), wq.data_ptr(), 32, ws.data_ptr(), b.data_ptr(), z.data_ptr(), 8, 3, 5, 20, 1, 5, 148, 0, 7)


def test_a_checkpoint_is_served_in_8_bit_integers(tmp_path):
    """`--quantize w8a8` of the shard: the dense checkpoint's projections are quantised on load, and a prompt runs through them."""
    import json

    from safetensors.torch import save_file
    from tokenizers import Tokenizer, models, pre_tokenizers

    from lorax_b200.config import EngineConfig, tiny_llama
    from lorax_b200.models.decoder import DecoderModel, Int8Weight
    from lorax_b200.models.loading import export_hf_state_dict
    from lorax_b200.server.runtime import build_runtime
    cfg = tiny_llama()
    dense = DecoderModel.random_init(cfg, "cpu", torch.float32, seed=1)
    save_file(export_hf_state_dict(dense), str(tmp_path / "model.safetensors"))
    (tmp_path / "config.json").write_text(json.dumps({
        "model_type": "llama", "vocab_size": cfg.vocab_size, "hidden_size": cfg.hidden_size, "intermediate_size": cfg.intermediate_size,
        "num_hidden_layers": cfg.num_hidden_layers, "num_attention_heads": cfg.num_attention_heads, "num_key_value_heads": cfg.num_key_value_heads,
        "rms_norm_eps": cfg.rms_norm_eps, "rope_theta": cfg.rope_theta, "max_position_embeddings": 2048, "torch_dtype": "float32"}))
    tok = Tokenizer(models.WordLevel({f"w{i}": i for i in range(cfg.vocab_size)}, unk_token="w0"))
    tok.pre_tokenizer = pre_tokenizers.Whitespace()
    tok.save(str(tmp_path / "tokenizer.json"))
    (tmp_path / "tokenizer_config.json").write_text(json.dumps({"tokenizer_class": "PreTrainedTokenizerFast", "unk_token": "w0", "eos_token": "w2"}))
    rt = build_runtime(str(tmp_path), EngineConfig(max_input_length=40, max_total_tokens=64), device="cpu", source="local", quantize="w8a8", num_blocks=32, max_batch=4)
    model = rt.runner.model if hasattr(rt, "runner") else rt.model
    assert model.quantized == "w8a8" and isinstance(model.layers[-1].down_w, Int8Weight)
    want = DecoderModel.random_init(cfg, "cpu", torch.float32, seed=1)
    want.quantize("w8a8")
    assert torch.equal(model.layers[0].qkv_w.q, want.layers[0].qkv_w.q) and torch.equal(_step(model), _step(want))
