"""Operators of short ragged steps on the CPU: what they refuse, and the plain statements against the code that built these arrays before."""
import random

import pytest
import torch

from lorax_b200.ops import native, reference

BF16 = torch.bfloat16
INF, NAN = float("inf"), float("nan")


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _refused(call, *a, **kw):
    """By both forms, and by the CUDA one in front of everything that needs a GPU."""
    for ops in (reference, native):
        with pytest.raises(ValueError):
            getattr(ops, call)(*a, **kw)


# ------------------------------------------------------------------------------------------------ tables
def _tables_args(**over):
    a = dict(seqs=ints([3], [0], [-1], [1]), pages=ints(5), tokens=3, max_blocks=2, page=32)
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(seqs=ints([3], [0], [-1], [1]).long()), dict(seqs=ints([3], [0], [-1])), dict(seqs=ints(3, 0, -1, 1)), dict(seqs=torch.zeros(4, 6, dtype=torch.int32)[:, ::2]),
    dict(seqs=torch.zeros(4, reference.STEP_SEQS_MAX + 1, dtype=torch.int32)), dict(pages=ints(5).long()), dict(pages=ints([5])), dict(pages=ints(5, 6, 7, 8)[::2]),
    dict(tokens=-1), dict(max_blocks=0), dict(page=0), dict(window=-1), dict(tiles=((0, 1),)), dict(tiles=((64, -1),)), dict(tiles=((64, 1),) * 5),
    dict(lora_tiles=-1), dict(lora_rows=0), dict(lead=ints(1, 2, 3, 4)), dict(lead=ints([1, 2, 3])), dict(lead=ints([1, 2, 3, 4]).long()),
    dict(lead=torch.zeros(5, 4, dtype=torch.int32).view(-1)[1:17].view(4, 4))])
def test_tables_refuse(over):
    _refused("step_tables", **_tables_args(**over))


@pytest.mark.parametrize("over", [
    dict(tokens=2 ** 31), dict(max_blocks=2 ** 31), dict(page=2 ** 32 + 32), dict(window=2 ** 31), dict(tiles=((2 ** 31, 1),)), dict(tiles=((64, 2 ** 31),)),
    dict(lora_tiles=2 ** 31), dict(lora_rows=2 ** 31), dict(row_offset=-1), dict(row_offset=2 ** 31)])
def test_tables_refuse_what_is_past_32_bits(over):
    _refused("step_tables", **_tables_args(**over))


@pytest.mark.parametrize("window", [0, 64])
def test_tables_are_the_ones_of_the_step_assembly(window):
    """Positions, slots and adapter slots as `prefill_metadata` makes them from cumulative lengths and padded tables; tables, tiles and adapter
    tiles as the runner's lists were."""
    rng = random.Random(window)
    B, M, page = 9, 7, 32
    n = [rng.choice([0, 1, 31, 32, 33, 70, 130]) for _ in range(B)]
    cached = [rng.randint(0, 90) for _ in range(B)]
    slot = [rng.choice([-1, 0, 3]) for _ in range(B)]
    pages = [[rng.randint(1, 99) for _ in range(rng.choice([1, 2, 3, 7, 9]))] for _ in range(B)]

    def row(blocks):
        k = len(blocks)
        if k >= M:
            return blocks[:M]
        if window and k * page >= window + page:
            return [blocks[i % k] for i in range(M)]
        return blocks + [0] * (M - k)
    T = sum(n)
    cu = [sum(n[:b]) for b in range(B + 1)]
    bt = ints(*[row(p) for p in pages])
    want = reference.prefill_metadata(ints(*cu), ints(*cached), ints(*slot), bt, page, T)
    lora = [[slot[b], 5 + cu[b] + a, min(32, n[b] - a), 0] for b in range(B) if slot[b] >= 0 for a in range(0, n[b], 32)]
    t64, t128 = reference.prefill_tiles(n), reference.prefill_tiles(n, 128)
    lead = ints([7, 0, 5, 0])
    got = reference.step_tables(ints(n, cached, slot, [len(p) for p in pages]), ints(*[x for p in pages for x in p]), T, M, page, window=window,
                                tiles=((64, len(t64[0])), (128, len(t128[0]) + 2)), lora_tiles=len(lora) + 1, row_offset=5, lead=lead)
    assert got.cu_q.tolist() == cu and torch.equal(got.block_tables, bt)
    assert torch.equal(got.positions, want[0]) and torch.equal(got.slots, want[1]) and torch.equal(got.tok_slot, want[2])
    assert [x.tolist() for x in got.tiles[0]] == list(t64)
    assert [x.tolist() for x in got.tiles[1]] == [t128[0] + [-1, -1], t128[1] + [0, 0]]
    assert got.lora_tiles.tolist() == [[7, 0, 5, 0]] + lora + [[-1, 0, 0, 0]]


def test_tables_fill_what_the_lengths_do_not_reach_and_leave_out_what_they_pass():
    seqs, pages = ints([3, 2], [31, 0], [4, -1], [2, 1]), ints(9, 8, 7)
    got = reference.step_tables(seqs, pages, 7, 2, 32, tiles=((2, 5),), lora_tiles=2)
    assert got.slots.tolist() == [9 * 32 + 31, 8 * 32, 8 * 32 + 1, 7 * 32, 7 * 32 + 1, -1, -1] and got.tok_slot.tolist() == [4, 4, 4, -1, -1, -1, -1]
    assert got.positions.tolist() == [31, 32, 33, 0, 1, 0, 0] and got.lora_tiles.tolist() == [[4, 0, 3, 0], [-1, 0, 0, 0]]
    assert [x.tolist() for x in got.tiles[0]] == [[0, 0, 1, -1, -1], [0, 2, 0, 0, 0]]
    short = reference.step_tables(seqs, pages, 2, 2, 32, tiles=((2, 1),), lora_tiles=0)
    assert short.slots.tolist() == [9 * 32 + 31, 8 * 32] and short.cu_q.tolist() == [0, 3, 5] and short.lora_tiles.shape == (0, 4)


# ------------------------------------------------------------------------------------------------ experts
def _moe_args(T=2, E=4, k=2, H=64, I=32, **over):
    a = dict(x=torch.zeros(T, H, dtype=BF16), router_w=torch.zeros(E, H, dtype=BF16), w13=torch.zeros(E, 2 * I, H, dtype=BF16),
             w2=torch.zeros(E, H, I, dtype=BF16), k=k)
    a.update(over)
    return a


@pytest.mark.parametrize("over", [
    dict(T=17), dict(k=0), dict(k=5), dict(E=40, k=33), dict(E=257), dict(H=60), dict(I=12), dict(e0=1), dict(e0=-1), dict(act="tanh"),
    dict(x=torch.zeros(2, 64)), dict(x=torch.zeros(64, dtype=BF16)), dict(x=torch.zeros(2, 128, dtype=BF16)[:, ::2]), dict(x=torch.zeros(2, 68, dtype=BF16)[:, :64]),
    dict(x=torch.zeros(130, dtype=BF16)[1:129].view(2, 64)), dict(router_w=torch.zeros(4, 32, dtype=BF16)), dict(router_w=torch.zeros(4, 64)),
    dict(w13=torch.zeros(4, 48, 64, dtype=BF16)), dict(w13=torch.zeros(8, 64, 64, dtype=BF16)[::2]), dict(w2=torch.zeros(4, 32, 64, dtype=BF16).transpose(1, 2)),
    dict(out=torch.zeros(3, 64, dtype=BF16)), dict(out=torch.zeros(2, 64)), dict(out=torch.zeros(64, 2, dtype=BF16).t())])
def test_experts_refuse(over):
    _refused("moe_few", **_moe_args(**over))


@pytest.mark.parametrize("over", [
    dict(x=torch.zeros(1, 64, dtype=BF16).expand(2, -1)), dict(x=torch.zeros(88, dtype=BF16).as_strided((2, 64), (16, 1))),
    dict(router_w=torch.zeros(1, 64, dtype=BF16).expand(4, -1)), dict(out=torch.zeros(1, 64, dtype=BF16).expand(2, -1))])
def test_experts_refuse_rows_on_top_of_one_another(over):
    _refused("moe_few", **_moe_args(**over))


def test_experts_of_the_kernels_are_bf16():
    a = {k: v.float() if isinstance(v, torch.Tensor) else v for k, v in _moe_args().items()}
    reference.moe_few(**a)
    with pytest.raises(ValueError, match="bf16"):
        native.moe_few(**a)


@pytest.mark.parametrize("renorm,e0,e_local", [(True, 0, 6), (False, 0, 6), (True, 2, 3)])
def test_experts_as_a_dense_sum(renorm, e0, e_local):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)
    x, wr, w13, w2 = r(5, 32), r(6, 32), r(e_local, 48, 32) / 6, r(e_local, 32, 24) / 5
    z = (x.double() @ wr.double().t())
    want = torch.zeros(5, 32, dtype=torch.float64)
    for t in range(5):
        best = sorted(range(6), key=lambda e: -z[t, e])[:2]
        p = torch.softmax(z[t, best] if renorm else z[t], 0)
        for j, e in enumerate(best):
            if e0 <= e < e0 + e_local:
                a = w13[e - e0].double() @ x[t].double()
                want[t] += 1.5 * p[j if renorm else e] * (w2[e - e0].double() @ (torch.nn.functional.silu(a[:24]) * a[24:]))
    got = reference.moe_few(x, wr, w13, w2, 2, e0, renorm=renorm, scale=1.5)
    assert torch.allclose(got.double(), want, rtol=1e-4, atol=1e-5)


# ------------------------------------------------------------------------------------------------ scores
@pytest.mark.parametrize("over", [
    dict(logits=torch.zeros(8)), dict(logits=torch.zeros(2, 0)), dict(logits=torch.zeros(2, 16)[:, ::2]), dict(logits=torch.zeros(1, 8).expand(2, 8)),
    dict(k=-1), dict(k=9), dict(logits=torch.zeros(2, 64), k=33), dict(softcap=-1.0), dict(targets=ints(1)), dict(targets=torch.zeros(2)), dict(targets=ints([1], [2]))])
def test_scores_refuse(over):
    _refused("token_scores", **{**dict(logits=torch.zeros(2, 8)), **over})


def test_scores_of_the_kernels_are_bf16_or_fp32():
    with pytest.raises(ValueError, match="float16"):
        native.token_scores(torch.zeros(2, 8, dtype=torch.float16))


def test_scores_of_rows_with_masks():
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[1.0, -inf, 1.0, 0.0], [-inf] * 4, [0.0, nan, 1.0, 2.0], [0.0, inf, 1.0, 2.0], [-inf, 3.0, -inf, -inf]])
    s = reference.token_scores(x, torch.tensor([2, 0, 0, 1, 4]), k=3)
    assert s.top_ids.tolist() == [[0, 2, 3], [0, 1, 2], [3, 2, 0], [1, 3, 2], [1, 0, 2]]
    z = 2 * torch.e + 1
    assert torch.allclose(s.logprobs[0], torch.tensor(1 - torch.log(torch.tensor(z)).item()))
    assert s.entropy[4] == 0 and s.top_logprobs[4].tolist() == [0.0, -inf, -inf]
    assert s.logprobs[1:].isnan().all() and s.entropy[1:4].isnan().all()


# ------------------------------------------------------------------------------------------------ where they are called
def test_which_layers_take_the_operator_for_a_few_tokens():
    from lorax_b200.models.moe import few_tokens
    assert few_tokens(1, 2, 8, 4096) and few_tokens(16, 2, 8, 4096) and not few_tokens(17, 2, 8, 4096) and few_tokens(16, 8, 128, 2048)
    assert few_tokens(8, 8, 128, 1024) and not few_tokens(9, 8, 128, 1024)
    assert few_tokens(3, 4, 32, 512) and not few_tokens(4, 4, 32, 512) and few_tokens(8, 2, 8, 512) and not few_tokens(9, 2, 8, 512)


def _tiny(device, dtype, **over):
    from lorax_b200.config import ModelConfig
    from lorax_b200.models.decoder import DecoderModel
    from lorax_b200.runtime.kv_cache import KVCache
    from lorax_b200.runtime.runner import ModelRunner
    cfg = ModelConfig(**{**dict(model_type="mixtral", vocab_size=512, hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=4,
                                num_key_value_heads=2, head_dim=64, rope_theta=1e4, max_position_embeddings=1024, num_local_experts=4, num_experts_per_tok=2,
                                torch_dtype="bfloat16"), **over})
    m = DecoderModel.random_init(cfg, device, dtype, seed=2, std=0.05)
    return m, ModelRunner(m, KVCache(cfg.num_hidden_layers, 32, m.nkv, m.d, m.dtype, m.device), max_batch=4, max_seq_tokens=512, max_prefill_tokens=512, use_graphs=False)


def test_scores_refuse_caps_that_are_no_fp32_numbers_and_vocabularies_past_30_bits():
    logits = torch.zeros(2, 8)
    for cap in (INF, NAN, -1.0, 1e39, 1e-50):
        _refused("token_scores", logits, softcap=cap)
    _refused("token_scores", torch.empty(1, 1 << 30, device="meta"))


def test_the_runner_refuses_to_score_nothing_and_too_many_alternatives():
    from lorax_b200.runtime.runner import PrefillItem
    m, r = _tiny("cpu", torch.float32)
    before = [t.clone() for layer in r.kv.layers for t in layer]
    for items, k in (([], 0), ([PrefillItem([], 0, [1])], 0), ([PrefillItem([5], 0, [1]), PrefillItem([], 0, [2])], 0), ([PrefillItem([5], 0, [1])], 33),
                     ([PrefillItem([5], 0, [1])], -1)):
        with pytest.raises(ValueError, match="score"):
            r.score(items, k=k)
    assert all(torch.equal(a, b) for a, b in zip(before, (t for layer in r.kv.layers for t in layer)))


@pytest.mark.parametrize("cap", [0.0, 2.0])
def test_scores_of_prompts_by_the_runner(cap):
    """Every token's score is that of the logits which a prefill of the same items returns; the last row of an item has no next token."""
    from lorax_b200.runtime.runner import PrefillItem
    m, r = _tiny("cpu", torch.float32, final_logit_softcapping=cap or None)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (5, 1, 40)]
    items = [PrefillItem(p, 0, [1 + 2 * i, 2 + 2 * i]) for i, p in enumerate(prompts)]
    got = r.score(items, k=3)
    _, _, logits = r.prefill([PrefillItem(p, 0, [1 + 2 * i, 2 + 2 * i], all_logprobs=True) for i, p in enumerate(prompts)])
    lp = torch.log_softmax(logits, -1)
    row = 0
    for p in prompts:
        for i, _ in enumerate(p):
            if i + 1 < len(p):
                assert abs(got.logprobs[row].item() - lp[row, p[i + 1]].item()) < 1e-4
            else:
                assert got.logprobs[row].isnan()
            best = lp[row].topk(3)
            assert torch.allclose(got.top_logprobs[row], best.values, atol=1e-4) and got.top_ids[row].tolist() == best.indices.tolist()
            assert abs(got.entropy[row].item() + (lp[row].exp() * lp[row]).sum().item()) < 1e-3
            row += 1
    assert row == got.entropy.shape[0]
    # a continuation of a cached prompt: the scores behind its tokens are those of the whole prompt
    whole = got.logprobs[6:46]
    rest = r.score([PrefillItem(prompts[2][24:], 24, [5, 6])])
    assert torch.allclose(rest.logprobs[:15], whole[24:39], atol=1e-4) and rest.top_ids.shape == (16, 0)


def test_alternatives_beyond_the_kernels():
    """The chooser answers with any number of alternatives: the operator's up to its most, the sorted row's beyond."""
    from lorax_b200.sampling.chooser import HeterogeneousNextTokenChooser, NextTokenParams
    logits = torch.randn(2, 100, generator=torch.Generator().manual_seed(1))
    lp = torch.log_softmax(logits, -1)
    for k in (1, reference.TOP_MAX, reference.TOP_MAX + 1, 100):
        c = HeterogeneousNextTokenChooser([NextTokenParams(return_k_alternatives=k), NextTokenParams()], "cpu", 100)
        ids, got, (alt, alp) = c(None, None, logits.clone())
        best = lp.topk(k, -1)
        assert ids.tolist() == logits.argmax(-1).tolist() and torch.allclose(got, lp.max(-1).values, atol=1e-6)
        assert alt.tolist() == best.indices.tolist() and torch.allclose(alp, best.values, atol=1e-6)


def test_a_step_of_more_sequences_than_the_kernel_takes():
    from lorax_b200.runtime.runner import PrefillItem
    m, r = _tiny("cpu", torch.float32)
    r.max_prefill_tokens = n = reference.STEP_SEQS_MAX + 5
    inp, _ = r._prefill_inputs([PrefillItem([i % 512], i % 7, [1 + i % 9]) for i in range(n)])
    assert inp.cu_q.tolist() == list(range(n + 1)) and inp.positions.tolist() == [i % 7 for i in range(n)]
    assert inp.slots.tolist() == [(1 + i % 9) * r.page + i % 7 for i in range(n)] and inp.tile_seq.tolist() == list(range(n))
