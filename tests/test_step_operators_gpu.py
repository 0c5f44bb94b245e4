"""Operators of short ragged steps on the GPU against their definitions in 64 bits.

Tolerances, from the arithmetic: half a step of a rounding is 2^-24 of the value in fp32 and 2^-8 in bf16.
  scores   the sum of a row's exponentials: a thread adds V / 512 terms one after the other, then some thirty merges, half a step each; an
           exponential is off by 2^-22 and by the rounding of its argument.  log s is off by as much, absolutely; u / s by as much times E|c - m|,
           which is at most log V + 1.  A cap adds four roundings of a value up to the cap to every logit.
  experts  products of bf16 are exact in fp32; a warp adds K / 128 MMAs of 16 terms one after the other, then eight warps' sums, a step (2^-23)
           each of the sum of magnitudes.  The value and remainder of h leave 2^-17 of it out.  The result is rounded to bf16.
"""
import math
import random

import pytest
import torch

from lorax_b200.ops import reference

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from lorax_b200.ops import native

BF16, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


# ------------------------------------------------------------------------------------------------ tables
def _requests(seed, B, longest, deepest, pages):
    rng = random.Random(seed)
    n = [rng.choice([0, 1, rng.randint(1, longest), rng.randint(1, longest)]) for _ in range(B)]
    return (n, [rng.randint(0, deepest) for _ in range(B)], [rng.randint(-1, 5) for _ in range(B)], [rng.randint(0 if seed % 2 else 1, pages) for _ in range(B)])


@pytest.mark.parametrize("B,longest,deepest,pages,M,page,window", [
    (1, 1, 0, 1, 1, 32, 0), (1, 3000, 0, 94, 95, 32, 0), (7, 200, 500, 22, 22, 32, 0), (33, 5, 4000, 127, 64, 32, 0), (40, 100, 700, 9, 40, 32, 128),
    (257, 70, 300, 12, 13, 16, 0), (4096, 4, 64, 3, 3, 32, 64), (300, 9, 9000, 290, 301, 32, 8192)])
def test_tables(B, longest, deepest, pages, M, page, window):
    n, cached, slot, held = _requests(B, B, longest, deepest, pages)
    flat = random.Random(B + 1).choices(range(1, 100000), k=sum(held))
    seqs, pg = ints(n, cached, slot, held), torch.tensor(flat, dtype=torch.int32)
    up = lambda a, b: (a + b - 1) // b
    kw = dict(window=window, tiles=((64, sum(up(a, 64) for a in n)), (128, sum(up(a, 128) for a in n) + 3), (192, 0), (7, max(0, sum(up(a, 7) for a in n) - 2))),
              lora_tiles=sum(up(a, 32) for a, s in zip(n, slot) if s >= 0) + 1, row_offset=B)
    lead = ints(*[[i, i, 1, 0] for i in range(B)])
    for tokens in (sum(n), sum(n) + 5, max(0, sum(n) - 3)):
        want = reference.step_tables(seqs, pg, tokens, M, page, lead=lead, **kw)
        got = native.step_tables(seqs.cuda(), pg.cuda(), tokens, M, page, lead=lead.cuda(), **kw)
        for name in ("cu_q", "positions", "slots", "tok_slot", "block_tables", "lora_tiles"):
            assert torch.equal(getattr(got, name).cpu(), getattr(want, name)), (name, tokens)
        for a, b in zip(got.tiles, want.tiles):
            assert torch.equal(a[0].cpu(), b[0]) and torch.equal(a[1].cpu(), b[1])


def test_tables_without_sequences_and_with_bad_lengths():
    none = native.step_tables(torch.empty(4, 0, dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 3, 5, 32, tiles=((64, 2),), lora_tiles=1)
    assert none.cu_q.tolist() == [0] and none.slots.tolist() == [-1] * 3 and none.block_tables.shape == (0, 5) and none.tiles[0][0].tolist() == [-1, -1]
    assert none.lora_tiles.tolist() == [[-1, 0, 0, 0]]
    # lengths below zero count as zero, pages past the list as page 0: nothing is read out of bounds
    seqs, pages = ints([-4, 3, 2], [5, -7, 2 ** 31 - 2], [1, 2, -1], [-1, 4, 9]), ints(11, 12)
    got = native.step_tables(seqs.cuda(), pages.cuda(), 5, 4, 32, tiles=((2, 3),), lora_tiles=1)
    assert got.cu_q.tolist() == [0, 0, 3, 5] and got.positions[:3].tolist() == [0, 1, 2] and got.slots[:3].tolist() == [352, 353, 354]
    assert got.block_tables.tolist() == [[0] * 4, [11, 12, 0, 0], [0] * 4] and got.tiles[0][0].tolist() == [1, 1, 2] and got.lora_tiles.tolist() == [[2, 0, 3, 0]]


def test_tables_of_sums_past_32_bits_and_of_high_tiles():
    """Page counts whose sum wraps around read nothing out of range; a tile higher than any sequence is one a sequence."""
    seqs, pages = ints([3, 4, 5, 6], [0, 0, 0, 0], [-1, 1, 1, -1], [2 ** 30, 2 ** 30, 2 ** 30, 2 ** 30 - 1]), ints(4, 5, 6)
    got = native.step_tables(seqs.cuda(), pages.cuda(), 18, 5, 32, tiles=((2 ** 31 - 1, 5),), lora_tiles=3, lora_rows=2 ** 31 - 1)
    want = reference.step_tables(seqs[:, :1], pages, 3, 5, 32)
    assert torch.equal(got.block_tables[:1].cpu(), want.block_tables) and (got.block_tables[1:] == 0).all()
    assert [x.tolist() for x in got.tiles[0]] == [[0, 1, 2, 3, -1], [0, 0, 0, 0, 0]]
    assert got.lora_tiles.tolist() == [[1, 3, 4, 0], [1, 7, 5, 0], [-1, 0, 0, 0]]


# ------------------------------------------------------------------------------------------------ scores
def _scores_oracle(logits, targets, k, cap):
    raw = logits.double()
    x = cap * torch.tanh(raw / cap) if cap else raw
    m = x.max(1, keepdim=True).values
    e = torch.exp(x - m)
    s = e.sum(1, keepdim=True)
    lp = (x - m) - torch.log(s)
    p = e / s
    order = torch.where(raw.isnan(), torch.full_like(raw, -INF), raw)
    ids = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :k]
    ok = (targets >= 0) & (targets < raw.shape[1])
    got = torch.where(ok, lp.gather(1, targets.clamp(0, raw.shape[1] - 1).long()[:, None])[:, 0], torch.full_like(lp[:, 0], NAN))
    return got, -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1), ids, lp.gather(1, ids)


def _close(got, want, atol, rtol=2.0 ** -22):
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    fin = want.isfinite()
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()])
    err = (got - want).abs()[fin] - rtol * want.abs()[fin]
    assert err.numel() == 0 or err.max().item() <= atol, (err.max().item(), atol)


def _check_scores(logits, targets, k, cap=0.0):
    V = logits.shape[1]
    got = native.token_scores(logits, targets, k=k, softcap=cap)
    lp, ent, ids, best = _scores_oracle(logits, targets, k, cap)
    assert torch.equal(got.top_ids.long(), ids)
    off = (V / 512 + 64) * 2.0 ** -24 + 16 * 2.0 ** -24 + 8 * cap * 2.0 ** -24
    _close(got.logprobs, lp, off)
    _close(got.top_logprobs, best, off)
    _close(got.entropy, ent, off * (2 + 2 * math.log(V + 1)))
    return got


def _logits(T, V, dtype, seed, wide=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, V + wide, generator=g, device="cuda") * 3
    x[:, :: max(1, V // 7)] += 6
    return x.to(dtype)[:, :V], torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,V", [(1, 1), (1, 7), (2, 33), (1, 512), (3, 511), (4, 4095), (5, 4096), (2, 4097), (1, 32000), (7, 32003), (2, 128256), (1, 262147), (40, 32000),
                                 (80, 9001), (149, 2048), (300, 1000), (160, 70001)])
def test_scores(T, V, dtype, cap):
    logits, targets = _logits(T, V, dtype, T + V)
    for k in sorted({0, min(1, V), min(5, V), min(20, V), min(32, V)}):
        _check_scores(logits, targets, k, cap)


@pytest.mark.parametrize("T", [100, 140, 200, 256, 300])      # (seven, six, four, three and two CTAs a row)
def test_scores_of_long_rows_in_any_number_of_parts(T):
    logits, targets = _logits(T, 120001, BF16, T)
    _check_scores(logits, targets, 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [1, 5, 8, 9, 15, 16, 17, 23, 4099])
def test_scores_of_rows_at_every_place_of_a_load(dtype, V):
    """Rows that start and end anywhere between two 16-byte boundaries; ties and masks in what lies in front of and behind the wide loads."""
    whole, _ = _logits(12, V + 8, dtype, V)
    for at in range(8):
        x = whole[:, at:at + V].clone() if V == 1 else whole[:, at:at + V]
        targets = torch.arange(12, device="cuda") % V
        for k in {0, min(V, 3), min(V, 32)}:
            _check_scores(x, targets, k)
            _check_scores(torch.zeros_like(whole)[:, at:at + V], targets, k)
            masked = torch.full_like(whole, -INF)[:, at:at + V]
            masked[:, [0, -1]] = 1.0
            _check_scores(masked, targets, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("wide", [1, 3, 64])
def test_scores_of_rows_apart_and_off_their_alignment(dtype, wide):
    for T, V in ((3, 5000), (200, 1111)):
        logits, targets = _logits(T, V, dtype, wide, wide)
        _check_scores(logits, targets, 9)
        _check_scores(logits[:, 1:], targets.clamp(max=V - 2).long(), 9)
        _check_scores(logits[1:2], targets[1:2], 4)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 3, 170])      # (eight CTAs a row, and one)
def test_scores_of_rows_with_masks_ties_and_no_distribution(T, dtype):
    V = 9001
    low = torch.finfo(dtype).min
    base, targets = _logits(T, V, dtype, 5)

    def row(change):
        x = base.clone()
        change(x)
        return x
    keep = torch.zeros(V, dtype=torch.bool, device="cuda")
    keep[[17, 4000, 4001, 8999]] = True
    for change in (lambda x: x.fill_(0.25), lambda x: x.fill_(-INF), lambda x: x.fill_(low), lambda x: x.masked_fill_(~keep, -INF), lambda x: x.masked_fill_(~keep, low),
                   lambda x: x[:, :9000].fill_(-INF), lambda x: x[:, 1:].fill_(low), lambda x: x[:, 4321].fill_(NAN), lambda x: x[:, 7].fill_(INF), lambda x: x[:, 7:9].fill_(INF),
                   lambda x: x.fill_(NAN), lambda x: x.copy_(x.sort(1).values), lambda x: x.copy_(x.sort(1, descending=True).values), lambda x: x.mul_(0).neg_(),
                   lambda x: (x.fill_(-INF), x[:, 0].fill_(NAN)), lambda x: x.copy_(x.round()), lambda x: x.mul_(1000), lambda x: (x.fill_(low), x[:, ::3].fill_(-INF))):
        for k in (0, 1, 6, 32):
            _check_scores(row(change), targets, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2, 170])
def test_scores_under_a_cap_of_rows_with_masks(T, dtype):
    """A cap takes infinities and lowest values to its two ends: all tokens have a probability."""
    V, low = 9001, torch.finfo(dtype).min
    base, targets = _logits(T, V, dtype, 6)
    for value in (-INF, INF, low, NAN):
        for rows in (slice(None), slice(1)):
            for cols in (slice(None), slice(0, V - 1), slice(4000, 4003)):
                x = base.clone()
                x[rows, cols] = value
                for k in (0, 6):
                    _check_scores(x, targets, k, 30.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("by", [700.0, -700.0, 1500.0, 2040.0, -2046.0, 5e4, -1e9, 1e30])
def test_scores_of_logits_far_from_zero(dtype, by):
    for T, V in ((2, 9001), (160, 4007)):
        logits, targets = _logits(T, V, F32, 11)
        x = (logits + by).to(dtype)
        x[-1, : V // 2] = 0                     # (a maximum that leaves the range, or comes back into it, on the way)
        x[0, V // 2:] = 0
        for k in (0, 3):
            _check_scores(x, targets, k)


@pytest.mark.parametrize("around", [-2048.0, 2048.0])
@pytest.mark.parametrize("T", [1, 900])
def test_scores_of_maxima_that_grow_past_the_end_of_a_range(around, T):
    """Half of a row's weight on either side of where the form of the exponents changes, in the order of the row."""
    x = torch.linspace(around - 0.5, around + 0.5, 70001, device="cuda").expand(T, -1).contiguous()
    for k in (0, 2):
        _check_scores(x, torch.arange(T, device="cuda") * 77, k)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_when_more_candidates_than_the_list_holds(dtype):
    """Thirty-one threads whose strided elements are all above the bound that the thirty-second one sets."""
    T, V, k = 160, 512 * 8 * 17 + 5, 32
    vec = 8 if dtype == BF16 else 4
    thread = torch.arange(V, device="cuda") // vec % 512
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(T, V, generator=g, device="cuda") + torch.where(thread < 31, 2.0, torch.where(thread == 31, 0.5, -2.0))
    _check_scores(x.to(dtype), torch.randint(0, V, (T,), generator=g, device="cuda"), k)


def test_scores_of_targets_outside_and_without_rows():
    logits, _ = _logits(4, 100, BF16, 2)
    for wide in (torch.int32, torch.int64):
        got = _check_scores(logits, torch.tensor([-1, 99, 100, 0], device="cuda", dtype=wide), 2)
        assert got.logprobs.isnan().tolist() == [True, False, True, False]
    assert native.token_scores(logits, torch.tensor([2 ** 40 + 1] * 4, device="cuda")).logprobs.isnan().all()
    strided = torch.zeros(4, 2, dtype=torch.int32, device="cuda")[:, 0]
    assert torch.equal(native.token_scores(logits, strided).logprobs, native.token_scores(logits, torch.zeros(4, dtype=torch.int32, device="cuda")).logprobs)
    none = native.token_scores(logits, None, k=3)
    assert none.logprobs is None and none.top_ids.shape == (4, 3)
    empty = native.token_scores(logits[:0], torch.empty(0, dtype=torch.int32, device="cuda"), k=3)
    assert empty.logprobs.shape == (0,) and empty.entropy.shape == (0,) and empty.top_ids.shape == (0, 3)


def test_scores_past_32_bits_of_elements():
    V, T = 262144, 8200                                      # 2^31 elements and more
    x = torch.zeros(T, V, dtype=BF16, device="cuda")
    rows = torch.tensor([0, 4095, 8191, 8192, T - 1])
    x[rows, rows * 31] = 5
    t = torch.arange(T, device="cuda", dtype=torch.int32) * 31
    got = native.token_scores(x, t, k=1)
    at = rows.cuda()
    assert got.top_ids[at, 0].tolist() == (rows * 31).tolist()
    _close(got.logprobs[at], torch.full((5,), 5 - math.log(V - 1 + math.exp(5)), dtype=torch.float64, device="cuda"), (V / 512 + 80) * 2.0 ** -24)


# ------------------------------------------------------------------------------------------------ experts
_ACTS = {"silu": (torch.nn.functional.silu, 1.1), "gelu": (torch.nn.functional.gelu, 1.13), "gelu_tanh": (lambda x: torch.nn.functional.gelu(x, approximate="tanh"), 1.13),
         "relu": (torch.relu, 1.0)}


def _experts_oracle(x, wr, w13, w2, k, e0, act, renorm, scale):
    """-> (result, how far the kernel's may be off), both in 64 bits, and the rows whose choice of experts is clear of the rounding of the logits."""
    f, slope = _ACTS[act]
    x, (T, H), inter, E = x.double(), x.shape, w2.shape[2], wr.shape[0]
    z, zabs = x @ wr.double().t(), x.abs() @ wr.double().abs().t()
    order = torch.sort(z, dim=1, descending=True, stable=True).indices
    ids = order[:, :k]
    gamma = lambda K: (K / 128 + 32) * 2.0 ** -23
    zerr = (gamma(H) * zabs).max().item() if T else 0.0
    clear = torch.ones(T, dtype=torch.bool, device=x.device) if k == E else (z.gather(1, order[:, k - 1:k]) - z.gather(1, order[:, k:k + 1]))[:, 0] > 2 * zerr
    p = (torch.softmax(z.gather(1, ids), 1) if renorm else torch.softmax(z, 1).gather(1, ids)) * scale
    out, off = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T):
        for j, e in enumerate(ids[t].tolist()):
            if not e0 <= e < e0 + w13.shape[0]:
                continue
            W, D = w13[e - e0].double(), w2[e - e0].double()
            a, mag = W @ x[t], W.abs() @ x[t].abs()
            g, u = a[:inter], a[inter:]
            h = f(g) * u
            herr = gamma(H) * (slope * mag[:inter] * u.abs() + (f(g).abs() + slope * gamma(H) * mag[:inter]) * mag[inter:]) + h.abs() * (2.0 ** -16 + 4 * zerr) + 2.0 ** -120
            out[t] += p[t, j] * (D @ h)
            off[t] += p[t, j] * (D.abs() @ (herr + gamma(inter * min(E, T * k)) * h.abs()))
    return out, off + 2.0 ** -8 * (out.abs() + off), clear


def _experts(T, E, k, H, inter, e0=0, e_local=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + T * 31 + E)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(BF16)
    e_local = E if e_local is None else e_local
    return r(T, H), r(E, H, std=2 * H ** -0.5), r(e_local, 2 * inter, H, std=H ** -0.5), r(e_local, H, inter, std=inter ** -0.5)


def _check_experts(a, k, e0=0, act="silu", renorm=True, scale=1.0, **kw):
    got = native.moe_few(*a, k, e0, act, renorm=renorm, scale=scale, **kw)
    want, off, clear = _experts_oracle(*a, k, e0, act, renorm, scale)
    assert clear.float().mean() > 0.6 or clear.numel() < 4
    ratio = ((got.double() - want).abs() / off.clamp_min(1e-300))[clear & ~want.isnan().any(1)]
    assert ratio.numel() == 0 or ratio.max().item() <= 1, ratio.max().item()
    return got


@pytest.mark.parametrize("T,E,k,H,I", [
    (1, 8, 2, 512, 256), (1, 1, 1, 8, 8), (1, 4, 4, 64, 40), (2, 3, 2, 264, 72), (3, 8, 2, 4096, 1024), (5, 16, 4, 1000, 1208), (7, 64, 8, 2048, 104), (8, 8, 1, 256, 128),
    (9, 8, 2, 512, 256), (16, 8, 2, 1024, 768), (16, 128, 8, 520, 264), (16, 256, 32, 128, 16), (11, 256, 5, 2000, 8), (16, 2, 2, 6144, 200), (13, 5, 3, 9480, 24),
    (4, 40, 6, 2368, 512), (6, 8, 2, 20000, 64)])
def test_experts(T, E, k, H, I):
    a = _experts(T, E, k, H, I)
    for act in _ACTS:
        _check_experts(a, k, act=act)
    _check_experts(a, k, renorm=False, scale=2.5)
    native.workspace().check_status()


@pytest.mark.parametrize("e0,e_local", [(0, 3), (2, 4), (5, 3), (7, 1), (3, 0)])
def test_experts_of_this_rank(e0, e_local):
    a = _experts(6, 8, 2, 256, 128, e0, e_local)
    got = _check_experts(a, 2, e0)
    if e_local == 0:
        assert (got == 0).all()


def test_experts_of_rows_apart_into_a_given_result():
    x, wr, w13, w2 = _experts(5, 8, 2, 512, 256)
    wide = torch.full((5, 640), 7.0, dtype=BF16, device="cuda")
    wide[:, 64:576] = x
    wr_wide = torch.cat([wr, wr], 1)[:, :512]
    out = torch.full((5, 523), 3.0, dtype=BF16, device="cuda")
    got = _check_experts((wide[:, 64:576], wr_wide, w13, w2), 2, out=out[:, 5:517])
    assert got.data_ptr() == out[:, 5:].data_ptr() and (out[:, :5] == 3).all() and (out[:, 517:] == 3).all()
    assert torch.equal(got, native.moe_few(x, wr, w13, w2, 2))
    assert native.moe_few(x[:0], wr, w13, w2, 2).shape == (0, 512)


def test_one_token_and_one_expert_of_any_row_stride():
    x, wr, w13, w2 = _experts(1, 1, 1, 128, 64)
    want = native.moe_few(x, wr, w13, w2, 1)
    assert torch.equal(native.moe_few(x[0].expand(1, -1), wr[0].expand(1, -1), w13, w2, 1), want)
    assert torch.equal(native.moe_few(x.as_strided((1, 128), (1, 1)), wr.as_strided((1, 128), (1, 1)), w13, w2, 1), want)


@pytest.mark.parametrize("T,E,k,H,I", [(16, 8, 4, 9480, 1000), (9, 4, 4, 8200, 520), (3, 3, 1, 4744, 584), (16, 16, 16, 7112, 72)])
def test_experts_wider_than_a_round_of_rows_with_rests(T, E, k, H, I):
    _check_experts(_experts(T, E, k, H, I), k)
    native.workspace().check_status()


def test_experts_choose_the_lower_number_on_ties_and_none_twice():
    x, wr, w13, w2 = _experts(4, 8, 3, 256, 64)
    wr[:] = wr[:1]                                           # all logits equal: experts 0, 1, 2, a third each
    got = native.moe_few(x, wr, w13, w2, 3)
    want = sum((torch.nn.functional.silu(x.double() @ w13[e, :64].double().t()) * (x.double() @ w13[e, 64:].double().t())) @ w2[e].double().t() for e in range(3)) / 3
    assert (got.double() - want).norm() / want.norm() < 2.0 ** -8
    x[2] = NAN                                               # one token without numbers leaves the others alone
    bad = native.moe_few(x, wr, w13, w2, 3)
    assert bad[2].isnan().all() and torch.equal(bad[[0, 1, 3]], got[[0, 1, 3]])


# ------------------------------------------------------------------------------------------------ streams, graphs, repeated calls
def _each():
    """(call, its inputs, inputs of another draw) of every operator."""
    a, b = (_experts(6, 8, 2, 512, 256, seed=s) for s in (1, 2))
    l1, l2 = (_logits(3, 32000, BF16, s) for s in (1, 2))
    t1 = [ints([5, 70], [3, 0], [1, -1], [1, 3]).cuda(), ints(4, 5, 6, 7).cuda()]
    t2 = [ints([70, 5], [0, 90], [-1, 0], [3, 1]).cuda(), ints(9, 8, 7, 6).cuda()]
    many = [_experts(3, 64, 8, 2048, 128, seed=s) for s in (3, 4)]      # (a router in a launch of its own)
    flat = lambda r: [x for f in r if f is not None for x in ([f] if isinstance(f, torch.Tensor) else [y for p in f for y in p])]
    return [(lambda *v: [native.moe_few(*v, 2)], list(a), list(b)),
            (lambda x, t: flat(native.token_scores(x, t, k=7)), list(l1), list(l2)),
            (lambda s, p: flat(native.step_tables(s, p, 75, 4, 32, tiles=((64, 3),), lora_tiles=3)), t1, t2),
            (lambda x, t: flat(native.token_scores(x, t)), list(l1), list(l2)),
            (lambda *v: [native.moe_few(*v, 8)], list(many[0]), list(many[1]))]


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4])
def test_captured_and_replayed(which):
    call, first, second = _each()[which]
    want1, want2 = ([x.clone() for x in call(*v)] for v in (first, second))
    held = [x.clone() for x in first]
    call(*held)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(*held)
    for want, inputs in ((want2, second), (want1, first), (want2, second)):
        for h, v in zip(held, inputs):
            h.copy_(v)
        g.replay()
        call(*(first if inputs is second else second))       # (an eager call in between shares nothing with the graph)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("which", [0, 1, 2, 3, 4])
def test_on_two_streams_at_once_and_again(which):
    call, first, second = _each()[which]
    want1, want2 = ([x.clone() for x in call(*v)] for v in (first, second))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for s, v, g in zip(streams, (first, second), got):
            with torch.cuda.stream(s):
                g.append(call(*v))
    torch.cuda.synchronize()
    for outs, want in zip(got, (want1, want2)):
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_inputs_of_the_kernel_in_front():
    """What the kernel directly in front wrote is there when an operator reads it."""
    for _ in range(5):
        for call, first, second in _each():
            want = [x.clone() for x in call(*second)]
            held = [x.clone() for x in first]
            for h, v in zip(held, second):
                h.copy_(v)
            got = call(*held)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------ a run of them together
def test_a_short_ragged_step():
    """Tables from lengths, keys and values to their slots, attention over the pages, a layer of experts, the head, the scores: every operator's result
    against 64 bits from what it was given."""
    nh, nkv, d, H, V, page, M = 8, 2, 128, 1024, 5003, 32, 4
    n, cached, slot, held = [4, 1, 5], [30, 70, 0], [2, -1, 0], [2, 3, 1]
    flat = [7, 3, 1, 9, 4, 6]
    T = sum(n)
    g = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(BF16)
    st = native.step_tables(ints(n, cached, slot, held).cuda(), ints(*flat).cuda(), T, M, page, tiles=((64, 3),), lora_tiles=2)
    want = reference.step_tables(ints(n, cached, slot, held), ints(*flat), T, M, page, tiles=((64, 3),), lora_tiles=2)
    assert torch.equal(st.slots.cpu(), want.slots) and torch.equal(st.lora_tiles.cpu(), want.lora_tiles)
    qkv, cache = r(T, (nh + 2 * nkv) * d), r(12, nkv, 2, page, d)
    before, raw = cache.clone(), qkv.clone()
    table = reference.rope_cache(d, 256, 1e4, device="cuda")
    native.rope_kvwrite(qkv, st.positions, table, cache, st.slots, nh, nkv, d, d)
    written = torch.zeros(12, page, dtype=torch.bool)
    for s in want.slots.tolist():
        written[s // page, s % page] = True
    assert torch.equal(cache.transpose(1, 3)[~written.cuda()], before.transpose(1, 3)[~written.cuda()])      # (pages of no request and rows behind the tokens stay)
    for t, s in enumerate(want.slots.tolist()):
        assert torch.equal(cache[s // page, :, 1, s % page], raw[t, (nh + nkv) * d:].view(nkv, d))
    att = native.attn_prefill(qkv, cache, st.block_tables, st.cu_q, ints(*cached).cuda(), *st.tiles[0], nh, nkv, d, d ** -0.5)
    at = 0
    for b in range(3):
        keys = cache[want.block_tables[b].long()].double()                       # [M, nkv, 2, page, d]
        for i in range(n[b]):
            for h in range(nh):
                k, v = (keys[:, h // (nh // nkv), o].reshape(-1, d)[: cached[b] + i + 1] for o in (0, 1))
                p = torch.softmax(k @ qkv[at, h * d:(h + 1) * d].double() * d ** -0.5, 0)
                ref = p @ v
                assert (att[at, h * d:(h + 1) * d].double() - ref).norm() <= 2.0 ** -7 * (p @ v.abs()).norm()      # weights and result rounded to bf16
            at += 1
    wr, w13, w2 = r(8, H, std=2 * H ** -0.5), r(8, 512, H, std=H ** -0.5), r(8, H, 256, std=256 ** -0.5)
    y = _check_experts((att, wr, w13, w2), 2)
    logits = native.gemm(y, r(V, H, std=0.2))
    targets = torch.randint(0, V, (T,), generator=g, device="cuda")
    _check_scores(logits, targets, 5, 30.0)
    native.workspace().check_status()


def test_scores_of_prompts_by_the_runner_with_experts():
    """`ModelRunner.score` on the kernels (a step of eight tokens: `moe_few`) against the fp32 CPU path of the same weights, and against its own logits."""
    from lorax_b200.runtime.runner import PrefillItem
    from tests.test_step_operators import _tiny
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (4, 1, 3)]
    outs = []
    for device, dtype in (("cuda", BF16), ("cpu", F32)):
        _, r = _tiny(device, dtype)
        item = lambda p, i: PrefillItem(p, 0, [1 + i])
        outs.append(r.score([item(p, i) for i, p in enumerate(prompts)], k=4))
        if device == "cuda":
            _, _, logits = r.prefill([PrefillItem(p, 0, [1 + i], all_logprobs=True) for i, p in enumerate(prompts)])
            lp, ent, ids, best = _scores_oracle(logits, torch.tensor([t for p in prompts for t in [*p[1:], -1]], device="cuda"), 4, 0.0)
            off = (512 / 512 + 80) * 2.0 ** -24
            assert torch.equal(outs[0].top_ids.long(), ids)
            _close(outs[0].logprobs, lp, off)
            _close(outs[0].entropy, ent, off * (2 + 2 * math.log(513)))
    a, b = outs[0].logprobs.cpu().double(), outs[1].logprobs.double()
    assert torch.equal(a.isnan(), b.isnan()) and ((a - b)[~a.isnan()].norm() / b[~b.isnan()].norm()).item() < 4e-2      # (the bound of the model's logits in bf16)


def test_decoding_with_experts_in_graphs_and_without():
    """Six rows through `moe_few`: a captured step and an eager one run the same kernels on the same data."""
    from lorax_b200.runtime.engine import Engine, EngineConfig
    from tests.test_step_operators import _tiny
    m, _ = _tiny("cuda", BF16)
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, 512, (3 + i,), generator=g).tolist() for i in range(6)]
    outs = [Engine(m, EngineConfig(max_total_tokens=128, max_batch_prefill_tokens=256), num_blocks=64, max_batch=8, use_graphs=graphs).generate(prompts, max_new_tokens=12)
            for graphs in (True, False)]
    assert outs[0] == outs[1] and all(len(o) == 12 for o in outs[0])
    native.workspace().check_status()


@pytest.mark.parametrize("k", [0, 5, 32, 40])      # (40: more than the kernel returns)
def test_scores_of_the_chooser(k):
    """Log-probabilities and alternatives of filtered, cooled and penalised rows against log_softmax of the same scores."""
    from lorax_b200.sampling.chooser import HeterogeneousNextTokenChooser, NextTokenParams
    V = 3001
    params = [NextTokenParams(return_k_alternatives=k), NextTokenParams(temperature=1e-4, do_sample=True, seed=1), NextTokenParams(top_k=3, do_sample=True, seed=2),
              NextTokenParams(repetition_penalty=1.3, top_p=0.4, do_sample=True, seed=3)]
    c = HeterogeneousNextTokenChooser(params, "cuda", V)
    logits, _ = _logits(4, V, BF16, 17)
    history = torch.randint(0, V, (4, 9), device="cuda")
    mask = torch.ones(4, 9, dtype=torch.bool, device="cuda")
    scores = c.warp(history, mask, logits.float(), history[:, -1])
    ids, lp, alts = HeterogeneousNextTokenChooser(params, "cuda", V)(history, mask, logits, history[:, -1])
    want, _, best, best_lp = _scores_oracle(scores, ids, max(k, 1), 0.0)
    # (a thread adds V / 256 terms at most; the form of log_softmax for more than 32 alternatives is PyTorch's own in fp32: as long a sum, in another order)
    off = (V / 256 + 80) * 2.0 ** -24
    _close(lp, want, off)
    assert (alts is None) == (k == 0)
    if k:
        _close(alts[1], best_lp, off)
        if k <= 32:
            assert torch.equal(alts[0].long(), best)
