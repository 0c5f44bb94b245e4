"""Calls of the operators of short ragged steps that are easily answered wrongly, on the CPU: what they refuse, and what the plain forms say."""
import random

import pytest
import torch

from lorax_b200.ops import native, reference
from tests.test_step_operators import BF16, _moe_args, _refused, _tables_args, ints


# ------------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("over", [dict(tiles=((64, 2 ** 31 - 1),)), dict(tiles=((64, 1), (64, 2 ** 30 + 1))), dict(lora_tiles=2 ** 31 - 1),
                                  dict(lora_tiles=2 ** 30, lead=torch.zeros(1, 4, dtype=torch.int32))])
def test_tables_refuse_lists_whose_blocks_would_count_past_32_bits(over):
    _refused("step_tables", **_tables_args(**over))


def _tables_by_hand(n, cached, adapter, held, pages, tokens, M, page, window, tiles, lora_tiles, lora_rows, row_offset):
    """Sequence by sequence, token by token."""
    n, cached, held = ([max(v, 0) for v in row] for row in (n, cached, held))
    B, at, cu, tables, rows, lora = len(n), 0, [0], [], [], []
    for b in range(B):
        entry = [pages[at + j] if at + j < len(pages) else 0 for j in range(held[b])]
        at += held[b]
        turns = 0 < held[b] < M and window > 0 and held[b] * page >= window + page
        tables.append([entry[j % held[b]] if turns else entry[j] if j < held[b] else 0 for j in range(M)])
        for p in range(cached[b], cached[b] + n[b]):
            rows.append((p, tables[b][min(p // page, M - 1)] * page + p % page, adapter[b]))
        if adapter[b] >= 0:
            lora += [(adapter[b], row_offset + cu[b] + r, min(lora_rows, n[b] - r), 0) for r in range(0, n[b], lora_rows)]
        cu.append(cu[-1] + n[b])
    fill = lambda got, want, blank: (got + [blank] * want)[:want]
    rows, lora = fill(rows, tokens, (0, -1, -1)), fill(lora, lora_tiles, (-1, 0, 0, 0))
    lists = [fill([(b, q) for b in range(B) for q in range(0, n[b], h)], count, (-1, 0)) for h, count in tiles]
    return cu, [list(c) for c in zip(*rows)] if rows else [[], [], []], tables, lists, [list(r) for r in lora]


def test_tables_of_any_lengths_without_a_word_from_the_host(monkeypatch):
    """Lengths below zero, page lists that end early, counts beyond and below what the lengths make; the arrays of any number of sequences are made whole."""
    rng, tolist = random.Random(9), torch.Tensor.tolist
    for case in range(300):
        B = rng.choice([0, 1, 2, 5, 17])
        n = [rng.choice([-2, 0, 1, rng.randint(1, 150)]) for _ in range(B)]
        cached = [rng.choice([-1, 0, rng.randint(0, 300)]) for _ in range(B)]
        adapter, held = [rng.randint(-2, 3) for _ in range(B)], [rng.choice([-1, 0, 1, 2, 5, 9]) for _ in range(B)]
        pages = [rng.randint(0, 99) for _ in range(max(0, sum(max(v, 0) for v in held) + rng.choice([0, 0, -3, 4])))]
        tokens = max(0, sum(max(v, 0) for v in n) + rng.choice([0, 0, -3, 5]))
        M, page, window = rng.choice([1, 2, 5, 8, 12]), rng.choice([1, 16, 32, 7]), rng.choice([0, 0, 16, 64])
        tiles = tuple((rng.choice([1, 3, 64, 128]), rng.randint(0, 30)) for _ in range(rng.randint(0, 4)))
        lora_tiles, lora_rows, offset = rng.randint(0, 20), rng.choice([1, 8, 32]), rng.randint(0, 9)
        lead = ints([1, 2, 3, 0]) if case % 3 == 0 else None
        with monkeypatch.context() as m:
            m.setattr(torch.Tensor, "tolist", lambda t: pytest.fail("read back"))
            got = reference.step_tables(ints(n, cached, adapter, held).view(4, B), ints(*pages), tokens, M, page, window, tiles, lora_tiles, lora_rows, offset, lead)
        cu, rows, tables, lists, lora = _tables_by_hand(n, cached, adapter, held, pages, tokens, M, page, window, tiles, lora_tiles, lora_rows, offset)
        assert tolist(got.cu_q) == cu and [tolist(x) for x in (got.positions, got.slots, got.tok_slot)] == rows and tolist(got.block_tables) == tables
        assert [list(zip(*map(tolist, pair))) for pair in got.tiles] == lists
        assert tolist(got.lora_tiles) == (tolist(lead) if lead is not None else []) + lora
        assert all(t.dtype == torch.int32 for t in (got.cu_q, got.positions, got.slots, got.tok_slot, got.block_tables, got.lora_tiles))


# ------------------------------------------------------------------------------------------------ experts
def test_experts_refuse_a_result_on_top_of_their_inputs():
    """Tokens are routed by every block of the second kernel too, while others write."""
    a = _moe_args(T=4)
    rows = torch.zeros(8, 64, dtype=BF16)
    for over in (dict(out=a["x"]), dict(out=a["router_w"]), dict(out=a["w13"][1, :4]), dict(out=a["w2"].view(-1)[64:320].view(4, 64)),
                 dict(x=rows[:4], out=rows[3:7]), dict(x=rows[4:], out=rows[1:5]), dict(x=rows[0:8:2], out=rows[0:8:2]),
                 dict(x=torch.zeros(4, 128, dtype=BF16)[:, :64])):
        args = {**a, **over}
        if "out" not in over:
            args["out"] = args["x"].as_strided((4, 64), (128, 1), 32)
        with_out = dict(args)
        _refused("moe_few", **with_out)


def test_experts_into_a_result_between_the_rows_of_their_inputs():
    """Rows that take turns share nothing: such a result is written as any other."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g)
    wr, w13, w2 = r(4, 64), r(4, 64, 64), r(4, 64, 32)
    buf = torch.zeros(4, 128)
    buf[:, :64] = r(4, 64)
    want = reference.moe_few(buf[:, :64].clone(), wr, w13, w2, 2)
    got = reference.moe_few(buf[:, :64], wr, w13, w2, 2, out=buf[:, 64:])
    assert torch.equal(got, want) and torch.equal(buf[:, 64:], want)
    lines = torch.zeros(8, 64)
    lines[::2] = buf[:, :64]
    assert torch.equal(reference.moe_few(lines[::2], wr, w13, w2, 2, out=lines[1::2]), want)


@pytest.mark.parametrize("renorm", [True, False])
def test_a_token_with_a_logit_that_is_no_number_has_no_weights(renorm):
    """Whether or not the expert whose logit it is would be chosen, on the rank that has it and on the others."""
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g)
    x, wr, w13, w2 = r(3, 32), r(6, 32), r(6, 48, 32), r(6, 32, 24)
    bad = wr.clone()
    bad[4, 0] = float("nan")
    assert reference.moe_few(x, bad, w13, w2, 2, renorm=renorm).isnan().all()
    ids = torch.sort(torch.where(torch.arange(6) == 4, float("-inf"), x @ wr.t()), dim=1, descending=True, stable=True).indices[:, :2]
    for e in range(6):
        part = reference.moe_few(x, bad, w13[e:e + 1], w2[e:e + 1], 2, e, renorm=renorm)
        for t in range(3):
            assert part[t].isnan().all() if e in ids[t] else (part[t] == 0).all()
    x[1, 3] = float("nan")                                   # one token's numbers are its own
    clean = reference.moe_few(x[[0, 2]], wr, w13, w2, 2, renorm=renorm)
    got = reference.moe_few(x, wr, w13, w2, 2, renorm=renorm)
    assert got[1].isnan().all() and torch.allclose(got[[0, 2]], clean)


def test_the_narrowest_layers_take_the_operator_for_a_few_tokens_by_their_features_too():
    from lorax_b200.models.moe import few_tokens
    assert few_tokens(1, 2, 8, 512, 14336) and few_tokens(4, 2, 8, 512, 14336) and not few_tokens(8, 2, 8, 512, 14336) and few_tokens(8, 2, 8, 512, 8192)
    assert not few_tokens(1, 9, 9, 512, 10752) and few_tokens(1, 9, 9, 768, 10752) and few_tokens(16, 9, 9, 2048, 10752)
    assert few_tokens(3, 4, 32, 512, 2048) and not few_tokens(4, 4, 32, 512, 2048) and not few_tokens(9, 2, 8, 1024, 64)


def test_the_ring_of_a_few_tokens_experts_has_more_than_one_stage():
    """With one stage its copies and its products take turns: no width, features or number of an expert's tokens may leave just that."""
    lib = native.load()
    for H in (8, 512, 1024, 2048, 2304, 2368, 4096, 4600, 4736, 6144, 7104, 7168, 8192, 9216, 9472, 9480, 16384, 20000):
        for inter in (8, 64, 200, 1024, 1032, 4096, 4104, 8192, 14336, 14344):
            for T in range(1, 17):
                for most in range(1, T + 1):
                    for sms in (148, 132):
                        assert lib.lx_moe_few_down_stages(T, H, inter, most, sms) > 1, (T, H, inter, most, sms)


# ------------------------------------------------------------------------------------------------ scores
def test_the_best_of_rows_without_sorting_them(monkeypatch):
    """As a stable sort of whole rows has them, whatever the ties and masks; no row of the vocabulary is sorted."""
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(4)
    rows = [torch.randn(300, generator=g), torch.randn(300, generator=g).round(), torch.zeros(300), torch.full((300,), -inf), torch.full((300,), nan),
            torch.where(torch.rand(300, generator=g) < 0.95, -inf, torch.randn(300, generator=g)), torch.cat([torch.full((290,), 1.0), torch.arange(10.0)]),
            torch.where(torch.rand(300, generator=g) < 0.5, nan, torch.randn(300, generator=g)), torch.tensor([-0.0, 0.0] * 150)]
    x = torch.stack(rows)
    order = torch.sort(torch.where(x.isnan(), -inf, x), dim=1, descending=True, stable=True).indices
    lengths = []
    sort = torch.sort
    monkeypatch.setattr(torch, "sort", lambda t, *a, **kw: (lengths.append(t.shape[1]), sort(t, *a, **kw))[1])
    for dtype in (torch.float32, BF16):
        for k in (1, 2, 7, 32):
            want = order if dtype == torch.float32 else torch.argsort(torch.where(x.isnan(), -inf, x).to(dtype).float(), dim=1, descending=True, stable=True)
            assert torch.equal(reference.token_scores(x.to(dtype), k=k).top_ids.long(), want[:, :k])
    assert max(lengths) <= 32
    assert reference.token_scores(torch.zeros(0, 8), k=3).top_ids.shape == (0, 3)
    assert reference.token_scores(torch.ones(2, 3), k=3).top_ids.tolist() == [[0, 1, 2]] * 2


def test_scores_without_the_entropy():
    x = torch.randn(3, 50, generator=torch.Generator().manual_seed(5))
    whole, some = (reference.token_scores(x, ints(1, 2, 60), k=4, softcap=3.0, entropy=e) for e in (True, False))
    assert some.entropy is None and whole.entropy.shape == (3,)
    assert torch.equal(some.logprobs[:2], whole.logprobs[:2]) and some.logprobs[2].isnan()
    assert torch.equal(some.top_ids, whole.top_ids) and torch.equal(some.top_logprobs, whole.top_logprobs)


def test_sampling_asks_for_no_entropy(monkeypatch):
    """Rows of a whole vocabulary are not gone over for what nobody reads."""
    from lorax_b200.sampling.chooser import HeterogeneousNextTokenChooser, NextTokenParams
    asked, scores = [], reference.token_scores
    monkeypatch.setattr(reference, "token_scores", lambda *a, **kw: (asked.append(kw), scores(*a, **kw))[1])
    c = HeterogeneousNextTokenChooser([NextTokenParams(return_k_alternatives=2), NextTokenParams()], "cpu", 50)
    c(None, None, torch.randn(2, 50, generator=torch.Generator().manual_seed(6)))
    assert [kw.get("entropy") for kw in asked] == [False]


@pytest.mark.parametrize("k", [1, reference.TOP_MAX, reference.TOP_MAX + 1])
def test_alternatives_of_a_chooser_index_its_scores(k):
    """Token ids as `topk` gave them, of one type however many there are."""
    from lorax_b200.sampling.chooser import HeterogeneousNextTokenChooser, NextTokenParams
    logits = torch.randn(2, 100, generator=torch.Generator().manual_seed(7))
    c = HeterogeneousNextTokenChooser([NextTokenParams(return_k_alternatives=k), NextTokenParams()], "cpu", 100)
    ids, _, (alt, lp) = c(None, None, logits.clone())
    assert alt.dtype == ids.dtype == torch.int64
    assert torch.allclose(torch.log_softmax(logits, -1).gather(1, alt), lp, atol=1e-6)


# ------------------------------------------------------------------------------------------------ devices
def test_operators_run_on_their_tensors_device_whichever_is_current(monkeypatch):
    """Tensors of a second device while the first is current: launches, with the second device's stream, while it is the current one."""
    from lorax_b200.ops import native_steps
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
            return lambda *a: (launches.append((name, current[0], a[-1])), 0)[1]

    class Space:
        status, num_sms = torch.zeros(1, dtype=torch.int32), 148
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    monkeypatch.setattr(native_steps.nv, "load", Library)
    monkeypatch.setattr(native_steps.nv, "workspace", lambda d: Space())
    native.token_scores(torch.zeros(2, 8, dtype=BF16), k=2)
    native.token_scores(logits=torch.zeros(2, 8), targets=ints(1, 2))
    native.moe_few(**_moe_args())
    native.step_tables(ints([3], [0], [-1], [1]), ints(5), 3, 2, 32)
    current[0] = 1
    native.token_scores(torch.zeros(2, 8, dtype=BF16))
    assert launches == [(n, 1, 101) for n in ("lx_token_scores", "lx_token_scores", "lx_moe_few", "lx_step_tables", "lx_token_scores")] and current == [1]


def test_kernels_refuse_tensors_that_are_on_no_device():
    for call in (lambda: native.token_scores(torch.zeros(2, 8)), lambda: native.moe_few(**_moe_args()),
                 lambda: native.step_tables(ints([3], [0], [-1], [1]), ints(5), 3, 2, 32)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


# ------------------------------------------------------------------------------------------------ bindings
@pytest.mark.parametrize("name", ["STEP_SEQS_MAX", "MOE_FEW_TOKENS", "TOP_MAX"])
def test_limits_that_drift_apart_are_found_when_the_library_is_loaded(monkeypatch, name):
    from lorax_b200.ops import native_steps
    lib = native.load()
    native_steps.check_limits(lib)
    monkeypatch.setattr(native_steps, name, getattr(reference, name) + 1)
    with pytest.raises(native.NativeError, match="Python says"):
        native_steps.check_limits(lib)


@pytest.mark.parametrize("made", [2, 3])
def test_the_launches_of_the_experts_are_counted_as_they_were_made(monkeypatch, made):
    from lorax_b200.ops import native_steps

    class Library:
        def lx_moe_few(self, *a):
            return made
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(native_steps.nv, "load", Library)
    monkeypatch.setattr(native_steps.nv, "workspace", lambda d: type("", (), dict(status=torch.zeros(1), num_sms=148)))
    before = native.launch_count
    native.moe_few(**_moe_args())
    assert native.launch_count - before == made
    made = -5
    with pytest.raises(native.NativeError, match="-5"):
        native.moe_few(**_moe_args())
