"""Performance cases of the operators of short ragged steps: their tables, their experts and the scores of their tokens.

A speculative verification, the scoring of a prompt and the steps of a quiet server are ragged and short.  Each case is one call of one
operator: `step_tables` (block tables, slot maps and tile lists from the requests' lengths), `moe_few` (a mixture-of-experts layer for up to
sixteen tokens) or `token_scores` (log-probabilities of given tokens, the entropy of their distribution and its best alternatives).

With `own` false the operators are computed from elementary torch operations, with `own` true by the framework's kernels.
"""

import math
import random

import torch

own = False

PAGE = 32                        # tokens of a cache page
LORA_ROWS = 32                   # rows of an adapter tile
WEIGHT_LIMIT = 16 * 6144 * 10752      # experts x width x features of the largest expert case
LOGIT_LIMIT = 2048 * 128256


def _tables(prompts, tokens, cached, max_blocks, window=0, adapters=1, lead=0, **more):
    return dict(op="tables", prompts=prompts, tokens=tokens, cached=cached, max_blocks=max_blocks, window=window, adapters=adapters, lead=lead, **more)


def _experts(tokens, experts, top, width, features, act="silu", **more):
    return dict(op="experts", tokens=tokens, experts=experts, top=top, width=width, features=features, act=act, **more)


def _scores(rows, vocab, top, dtype="bf16", softcap=0.0, masked=0.0, padded=False, **more):
    return dict(op="scores", rows=rows, vocab=vocab, top=top, dtype=dtype, softcap=softcap, masked=masked, padded=padded, **more)


def listed():
    return [
        # time to first token of one short prompt: launch latency alone
        _tables(1, 137, 0, 65, name="tables_prompt"),
        # a speculative verification: 96 requests, four places each, contexts up to 8192, a third of the requests without adapter
        _tables(96, 384, 8192, 258, adapters=3, name="tables_verify"),
        # a prefill step of the serving benchmark beside 248 running rows
        _tables(7, 4001, 0, 129, adapters=100, lead=248, name="tables_prefill"),
        # many requests over pages that a sliding window recycles, prompts of 16384 tokens in all
        _tables(512, 16384, 30000, 1025, window=4096, adapters=100, name="tables_many"),
        # a lone user's next token
        _experts(1, 8, 2, 4096, 14336, name="experts_1"),
        # a verification of five places on the same layer
        _experts(5, 8, 2, 4096, 14336, name="experts_verify_5"),
        # many small experts, one token: latency of the routing and of two short products
        _experts(1, 64, 8, 2048, 1024, name="experts_small"),
        # wide experts and the most tokens
        _experts(16, 16, 4, 6144, 10752, name="experts_wide_16"),
        # one row with five alternatives: what a chat request with logprobs asks of every step
        _scores(1, 32000, 5, name="scores_1"),
        # prompt scoring: the log-probability of every token of a prompt
        _scores(4001, 32000, 0, name="scores_prompt"),
        # a batch of sampled rows: fp32 scores that filters have masked, twenty alternatives
        _scores(48, 128256, 20, dtype="f32", masked=0.9, name="scores_filtered"),
        # prompt scoring with alternatives over a large vocabulary
        _scores(2048, 128256, 20, name="scores_alternatives"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "experts", "scores"])
    if op == "tables":
        prompts = _log(rng, 1, 512)
        tokens = _log(rng, prompts, 16384)
        cached = rng.choice([0, _log(rng, 1, 30000), _log(rng, 1, 30000)])
        window = rng.choice([0, 0, _log(rng, 64, 8192)])
        max_blocks = (cached + tokens + PAGE - 1) // PAGE + 1 if prompts == 1 else (cached + tokens) // PAGE // rng.randint(1, 4) + 2
        return _tables(prompts, tokens, cached, min(max_blocks, 1025), window, rng.choice([0, 1, 3, 100]), rng.choice([0, _log(rng, 1, 256)]))
    if op == "experts":
        experts = rng.choice([4, 8, 16, 32, 64, 128])
        top = rng.randint(1, min(8, experts))
        width = 8 * _log(rng, 32, 768)
        most = max(16, min(14336, WEIGHT_LIMIT // (experts * width)))
        return _experts(_log(rng, 1, 16), experts, top, width, 8 * _log(rng, 2, most // 8), rng.choice(["silu", "silu", "gelu_tanh", "relu"]))
    vocab = _log(rng, 1000, 262144)
    rows = _log(rng, 1, min(4096, LOGIT_LIMIT // vocab))
    return _scores(rows, vocab, rng.choice([0, 0, 1, 5, 20, 32]), rng.choice(["bf16", "bf16", "f32"]) if rows * vocab * 2 <= LOGIT_LIMIT else "bf16",
                   rng.choice([0.0, 0.0, 30.0]), rng.choice([0.0, 0.0, 0.5]), rng.choice([False, True]))


# ------------------------------------------------------------------------------------------------ what a case's sizes mean

def _requests(case):
    """Tokens, cached tokens, adapter slot and pages of every request, from the case's numbers alone."""
    rng = random.Random("%(prompts)d %(tokens)d %(cached)d %(max_blocks)d %(window)d %(adapters)d" % case)
    n, total = case["prompts"], case["tokens"]
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    cached = [rng.randint(case["cached"] // 8, case["cached"]) for _ in range(n)]
    slots = [rng.randint(-1, case["adapters"] - 1) if case["adapters"] else -1 for _ in range(n)]
    pages = []
    for q, c in zip(lengths, cached):
        need = (c + q + PAGE - 1) // PAGE
        if case["window"]:                                   # (recycled pages: a window and the step's own tokens)
            need = min(need, (case["window"] + PAGE + PAGE - 1) // PAGE)
        pages.append(max(1, min(need, case["max_blocks"])))
    return lengths, cached, slots, pages


def _counts(case):
    """Entries of the lists that a step's tables hold: tiles of 64, of 128, adapter tiles."""
    lengths, _, slots, _ = _requests(case)
    up = lambda n, h: (n + h - 1) // h
    return (sum(up(n, 64) for n in lengths), sum(up(n, 128) for n in lengths), sum(up(n, LORA_ROWS) for n, a in zip(lengths, slots) if a >= 0))


def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + what) % (1 << 62))


def _rand(gen, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(std)


# ------------------------------------------------------------------------------------------------ preparing and running

def prepare(case, seed):
    return dict(tables=_prepare_tables, experts=_prepare_experts, scores=_prepare_scores)[case["op"]](case, seed)


def _prepare_tables(case, seed):
    lengths, cached, slots, pages = _requests(case)
    order = torch.randperm(sum(pages) + 1, generator=torch.Generator().manual_seed(seed * 31 + 7))[: sum(pages)] + 1
    n64, n128, lora = _counts(case)
    return dict(op="tables", seqs=torch.tensor([lengths, cached, slots, pages], dtype=torch.int32, device="cuda"),
                pages=order.to(torch.int32).cuda(), tokens=case["tokens"], max_blocks=case["max_blocks"], window=case["window"],
                n64=n64, n128=n128, lora=lora, lead=case["lead"])


def _prepare_experts(case, seed):
    T, E, H, I = case["tokens"], case["experts"], case["width"], case["features"]
    g = _gen(seed, 1)
    # normed rows; a router that is sharper than the other matrices, as a trained one is; down products that add to a residual stream
    return dict(op="experts", x=_rand(g, T, H), router=_rand(g, E, H, std=2.5 * H ** -0.5), up=_rand(g, E, 2 * I, H, std=1.25 * H ** -0.5),
                down=_rand(g, E, H, I, std=0.5 * I ** -0.5), top=case["top"], act=case["act"])


def _prepare_scores(case, seed):
    T, V = case["rows"], case["vocab"]
    g = _gen(seed, 2)
    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    wide = (V + 63) // 64 * 64 if case["padded"] else V      # a head padded to whole tiles: the rows lie further apart
    logits = torch.empty(T, wide, dtype=dtype, device="cuda")
    targets = torch.empty(T, dtype=torch.int32, device="cuda")
    for a in range(0, T, 256):
        n = min(256, T - a)
        x = _rand(g, n, wide, std=2.5, dtype=torch.float32)
        # a head is sure of a few tokens: how far they stand out differs by the row
        likely = torch.randint(0, V, (n, 8), generator=g, device="cuda")
        x.scatter_add_(1, likely, torch.rand(n, 1, generator=g, device="cuda") * torch.tensor([12.0, 9, 8, 7, 6, 5, 4, 3], device="cuda"))
        if case["masked"]:
            keep = torch.rand(n, wide, generator=g, device="cuda") >= case["masked"]
            keep[:, :64] = True                              # (what the filters leave: more than the alternatives that are asked for)
            keep.scatter_(1, likely, True)
            x.masked_fill_(~keep, float("-inf"))
        logits[a:a + n] = x
        targets[a:a + n] = likely[:, :1].squeeze(1).to(torch.int32)
    return dict(op="scores", logits=logits[:, :V], targets=targets, top=case["top"], softcap=case["softcap"])


def run(state):
    with torch.inference_mode():
        if own:
            return _run_own(state)
        return dict(tables=_plain_tables, experts=_plain_experts, scores=_plain_scores)[state["op"]](state)


_ops = None


def _run_own(state):
    global _ops
    if _ops is None:
        from lorax_b200.ops import get_ops
        _ops = get_ops("cuda")
    if state["op"] == "tables":
        s = state
        r = _ops.step_tables(s["seqs"], s["pages"], s["tokens"], s["max_blocks"], PAGE, window=s["window"], tiles=((64, s["n64"]), (128, s["n128"])),
                             lora_tiles=s["lora"], lora_rows=LORA_ROWS, row_offset=s["lead"])
        return dict(cu_q=r.cu_q, positions=r.positions, slots=r.slots, tok_slot=r.tok_slot, block_tables=r.block_tables, tiles=r.tiles,
                    lora_tiles=r.lora_tiles)
    if state["op"] == "experts":
        return _ops.moe_few(state["x"], state["router"], state["up"], state["down"], state["top"], act=state["act"])
    r = _ops.token_scores(state["logits"], state["targets"], k=state["top"], softcap=state["softcap"])
    return dict(logprobs=r.logprobs, entropy=r.entropy, top_ids=r.top_ids, top_logprobs=r.top_logprobs)


def _before(x):
    return torch.cumsum(x, 0) - x


def _plain_tables(s):
    n, cached, adapter, held = s["seqs"].long()
    pages, M, window, T, B = s["pages"].long(), s["max_blocks"], s["window"], s["tokens"], s["seqs"].shape[1]
    dev = n.device
    first, off = _before(n), _before(held)
    cu = torch.cat([first, first[-1:] + n[-1:]])
    j = torch.arange(M, device=dev)[None, :]
    own_pages = held[:, None]
    recycled = (own_pages < M) & (own_pages * PAGE >= window + PAGE) if window else torch.zeros(B, 1, dtype=torch.bool, device=dev)
    tables = torch.where((j < own_pages) | recycled, pages[off[:, None] + j % own_pages], torch.zeros_like(j))
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = cached[b] + t - first[b]
    slots = tables[b, (pos // PAGE).clamp(max=M - 1)] * PAGE + pos % PAGE

    def tiles(count, height, total):
        of = torch.repeat_interleave(torch.arange(B, device=dev), count, output_size=total)
        return of, (torch.arange(total, device=dev) - _before(count)[of]) * height
    up = lambda h: (n + h - 1) // h
    t64, t128 = tiles(up(64), 64, s["n64"]), tiles(up(128), 128, s["n128"])
    of, q0 = tiles(torch.where(adapter >= 0, up(LORA_ROWS), torch.zeros_like(n)), LORA_ROWS, s["lora"])
    lora = torch.stack([adapter[of], s["lead"] + first[of] + q0, (n[of] - q0).clamp(max=LORA_ROWS), torch.zeros_like(of)], 1)
    i32 = lambda x: x.to(torch.int32)
    return dict(cu_q=i32(cu), positions=i32(pos), slots=i32(slots), tok_slot=i32(adapter[b]), block_tables=i32(tables),
                tiles=tuple((i32(a), i32(q)) for a, q in (t64, t128)), lora_tiles=i32(lora))


def _act(x, act):
    if act == "relu":
        return x.clamp_min(0)
    if act == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x / (1 + torch.exp(-x))


def _route(x, router, top):
    """The routing weight of every expert for every token, zero for those that are not chosen; 64 bits: the choice lies at a border."""
    z = x.double() @ router.double().t()
    ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
    e = torch.exp(z.gather(1, ids) - z.max(1, keepdim=True).values)
    return torch.zeros_like(z).scatter_(1, ids, e / e.sum(1, keepdim=True))


def _plain_experts(s):
    w = _route(s["x"], s["router"], s["top"]).float()
    x, I = s["x"].float(), s["down"].shape[2]
    out = torch.zeros_like(x)
    for e in range(s["router"].shape[0]):
        z = x @ s["up"][e].float().t()
        out += w[:, e: e + 1] * ((_act(z[:, :I], s["act"]) * z[:, I:]) @ s["down"][e].float().t())
    return out.to(s["x"].dtype)


def _plain_scores(s):
    raw, k = s["logits"].float(), s["top"]
    x = s["softcap"] * torch.tanh(raw / s["softcap"]) if s["softcap"] else raw
    d = x - x.max(1, keepdim=True).values
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    logz = torch.log(total)
    entropy = logz - torch.where(e > 0, d * e, torch.zeros_like(d)).sum(1, keepdim=True) / total
    if k:
        ids = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :k]      # (equal logits: the lowest index first)
    else:
        ids = torch.empty(raw.shape[0], 0, dtype=torch.long, device=raw.device)
    return dict(logprobs=(d.gather(1, s["targets"].long()[:, None]) - logz)[:, 0], entropy=entropy[:, 0], top_ids=ids.to(torch.int32),
                top_logprobs=d.gather(1, ids) - logz)


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "tables":
        return None                                          # whole numbers
    with torch.inference_mode():
        state = prepare(case, seed)
        return _exact_experts(state) if case["op"] == "experts" else _exact_scores(state)


def _exact_experts(s):
    x, k, I = s["x"].double(), s["top"], s["down"].shape[2]
    scores = torch.einsum("th,eh->te", x, s["router"].double())
    chosen = [sorted(range(len(row)), key=lambda e: (-row[e], e))[:k] for row in scores.tolist()]
    out = torch.zeros_like(x)
    for e in sorted({i for row in chosen for i in row}):
        rows = [t for t, row in enumerate(chosen) if e in row]
        gate, up = s["up"][e, :I].double() @ x[rows].t(), s["up"][e, I:].double() @ x[rows].t()
        if s["act"] == "silu":
            gate = gate * torch.sigmoid(gate)
        elif s["act"] == "relu":
            gate = torch.relu(gate)
        else:
            gate = torch.nn.functional.gelu(gate, approximate="tanh")
        y = s["down"][e].double() @ (gate * up)
        for i, t in enumerate(rows):
            share = torch.softmax(scores[t, chosen[t]], 0)[chosen[t].index(e)]
            out[t] += share * y[:, i]
    return out


def _exact_scores(s):
    parts = []
    for a in range(0, s["logits"].shape[0], 128):
        raw = s["logits"][a:a + 128].double()
        x = torch.tanh(raw / s["softcap"]) * s["softcap"] if s["softcap"] else raw
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        ids = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, : s["top"]]
        parts.append((lp.gather(1, s["targets"][a:a + 128].long()[:, None])[:, 0], -torch.special.xlogy(p, p).sum(1), ids.to(torch.int32), lp.gather(1, ids)))
    logprobs, entropy, ids, best = (torch.cat(c) for c in zip(*parts))
    return dict(logprobs=logprobs, entropy=entropy, top_ids=ids, top_logprobs=best)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["op"] == "tables":
        n64, n128, lora = _counts(case)
        B, T, pages = case["prompts"], case["tokens"], sum(_requests(case)[3])
        return dict(bytes=4 * (4 * B + pages + B + 1 + 3 * T + B * case["max_blocks"] + 2 * (n64 + n128) + 4 * lora), flops=8 * T + 4 * B * case["max_blocks"])
    if case["op"] == "experts":
        T, E, k, H, I = (case[n] for n in ("tokens", "experts", "top", "width", "features"))
        reached = E * (1 - (1 - k / E) ** T)                 # experts that at least one token is routed to, on average
        return dict(bytes=2 * E * H + 6 * reached * H * I + 4 * T * H, flops=2.0 * T * E * H + 6.0 * T * k * H * I)
    T, V, k = case["rows"], case["vocab"], case["top"]
    return dict(bytes=T * V * (2 if case["dtype"] == "bf16" else 4) + T * (4 + 8 + 8 * k), flops=6.0 * T * V)
