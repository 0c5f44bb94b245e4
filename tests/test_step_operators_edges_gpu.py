"""Calls of the operators of short ragged steps that their documentation allows and that are easily answered wrongly: numbers that are not finite in some experts'
weights or in the router, activations, rings of few stages."""
import pytest
import torch

from lorax_b200.ops import reference
from tests.test_step_operators_gpu import BF16, INF, NAN, _check_experts, _experts, _experts_oracle

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from lorax_b200.ops import native


def _routes(x, wr, k):
    """Experts of every token, as the kernels choose them (inputs of these tests have no near ties)."""
    return torch.sort(x.double() @ wr.double().t(), dim=1, descending=True, stable=True).indices[:, :k].tolist()


def _one_expert(ids):
    """An expert that some token goes to and some other does not."""
    return next(e for row in ids for e in row if any(e not in r for r in ids))


SHAPES = [(6, 8, 2, 512, 256), (16, 8, 2, 1024, 768), (3, 8, 2, 520, 264), (13, 6, 3, 9480, 136), (2, 64, 8, 2048, 104)]


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("T,E,k,H,I", SHAPES)
def test_what_is_no_number_in_a_down_product_stays_with_its_experts_tokens(T, E, k, H, I, value):
    """One element of one expert: that feature of the tokens that the expert serves, nothing else, and an infinity stays one."""
    x, wr, w13, w2 = _experts(T, E, k, H, I, seed=3)
    ids = _routes(x, wr, k)
    e = _one_expert(ids)
    clean = native.moe_few(x, wr, w13, w2, k)
    want, off, _ = _experts_oracle(x, wr, w13, w2, k, 0, "silu", True, 1.0)
    for row, col in ((H - 1, 0), (7, I - 1)):
        bad = w2.clone()
        bad[e, row, col] = value
        got = native.moe_few(x, wr, w13, bad, k)
        for t in range(T):
            same = torch.ones(H, dtype=torch.bool, device="cuda")
            same[row] = False
            assert torch.equal(got[t][same], clean[t][same])
            if e not in ids[t]:
                assert abs(got[t, row].double() - want[t, row]) <= off[t, row]
                continue
            a = w13[e].double() @ x[t].double()
            h = torch.nn.functional.silu(a[col]) * a[I + col]
            assert abs(h) > 1e-6                             # (its sign is clear)
            expect = h * value
            assert got[t, row].isnan() if value != value else got[t, row].double() == expect
    native.workspace().check_status()


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("T,E,k,H,I", SHAPES)
def test_an_expert_without_numbers_spoils_its_own_tokens_only(T, E, k, H, I, value):
    x, wr, w13, w2 = _experts(T, E, k, H, I, seed=4)
    ids = _routes(x, wr, k)
    e = _one_expert(ids)
    want, off, _ = _experts_oracle(x, wr, w13, w2, k, 0, "silu", True, 1.0)
    whole, row = w2.clone(), w13.clone()
    whole[e] = value
    row[e, 3] = value
    for weights in ((w13, whole), (row, w2), (row, whole)):
        got = native.moe_few(x, wr, *weights, k)
        for t in range(T):
            if e in ids[t]:
                assert not got[t].isfinite().any()
            else:
                assert ((got[t].double() - want[t]).abs() <= off[t]).all()
    native.workspace().check_status()


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "relu2"])
@pytest.mark.parametrize("where", ["gate", "up"])
def test_a_token_of_an_expert_with_a_nan_in_front_of_its_activation_has_no_result(act, where):
    x, wr, w13, w2 = _experts(6, 8, 2, 512, 256, seed=9)
    ids = _routes(x, wr, 2)
    e = _one_expert(ids)
    bad = w13.clone()
    bad[e, 7 if where == "gate" else 263, 30] = NAN
    got, clean = native.moe_few(x, wr, bad, w2, 2, act=act), native.moe_few(x, wr, w13, w2, 2, act=act)
    plain = reference.moe_few(x.cpu(), wr.cpu(), bad.cpu(), w2.cpu(), 2, act=act)
    for t in range(6):
        assert got[t].isnan().all() and plain[t].isnan().all() if e in ids[t] else torch.equal(got[t], clean[t])


@pytest.mark.parametrize("T,E,k,H,I", SHAPES + [(4, 4, 4, 64, 40)])
@pytest.mark.parametrize("renorm", [True, False])
def test_a_router_row_without_numbers(T, E, k, H, I, renorm):
    """A token has no distribution over its experts if one of its logits is no number: no weights, and no result."""
    x, wr, w13, w2 = _experts(T, E, k, H, I, seed=5)
    bad = wr.clone()
    bad[E - 1, 5] = NAN
    got = native.moe_few(x, bad, w13, w2, k, renorm=renorm)
    plain = reference.moe_few(x.cpu(), bad.cpu(), w13.cpu(), w2.cpu(), k, renorm=renorm)
    assert got.isnan().all() and plain.isnan().all()
    some = x.clone()
    some[T - 1, 2] = INF                                     # (logits of both signs' infinities: only this token's)
    got, clean = native.moe_few(some, wr, w13, w2, k, renorm=renorm), native.moe_few(x, wr, w13, w2, k, renorm=renorm)
    assert torch.equal(got[:-1], clean[:-1]) and got[-1].isnan().all()


def test_a_router_row_without_numbers_on_ranks_of_experts():
    """What the ranks' shares sum up to is no number; a rank that has none of the chosen experts adds zeros."""
    x, wr, w13, w2 = _experts(5, 8, 2, 256, 64, seed=6)
    wr[2] = NAN
    total = torch.zeros(5, 256, dtype=torch.float64)
    for e0 in (0, 2, 4, 6):
        part = native.moe_few(x, wr, w13[e0:e0 + 2].contiguous(), w2[e0:e0 + 2].contiguous(), 2, e0).cpu()
        plain = reference.moe_few(x.cpu(), wr.cpu(), w13[e0:e0 + 2].cpu(), w2[e0:e0 + 2].cpu(), 2, e0)
        assert torch.equal(part.isnan(), plain.isnan()) and (part[~part.isnan()] == 0).all()
        total += part.double()
    assert total.isnan().all()


@pytest.mark.parametrize("T,E,k,H,I", [(5, 8, 2, 512, 256), (16, 8, 2, 1024, 264)])
def test_experts_of_squared_relu(T, E, k, H, I):
    """relu(x)^2: off by twice the activation times what the sum of the gate is off, and a step of the square."""
    x, wr, w13, w2 = _experts(T, E, k, H, I, seed=7)
    got = native.moe_few(x, wr, w13, w2, k, act="relu2").double()
    gamma = lambda K: (K / 128 + 32) * 2.0 ** -23
    z = x.double() @ wr.double().t()
    zerr = gamma(H) * (x.double().abs() @ wr.double().abs().t()).max()
    for t in range(T):
        order = torch.sort(z[t], descending=True).indices
        assert z[t, order[k - 1]] - z[t, order[k]] > 2 * zerr
        p = torch.softmax(z[t, order[:k]], 0)
        out, off = torch.zeros(H, dtype=torch.float64, device="cuda"), torch.zeros(H, dtype=torch.float64, device="cuda")
        for j, e in enumerate(order[:k].tolist()):
            a, mag = w13[e].double() @ x[t].double(), w13[e].double().abs() @ x[t].double().abs()
            r, u, d = a[:I].clamp_min(0), a[I:], gamma(H) * mag
            h = r * r * u
            herr = (2 * r * d[:I] + d[:I] ** 2) * (u.abs() + d[I:]) + r * r * d[I:] + h.abs() * (2.0 ** -16 + 4 * zerr) + 2.0 ** -120
            D = w2[e].double()
            out += p[j] * (D @ h)
            off += p[j] * (D.abs() @ (herr + gamma(I * min(E, T * k)) * h.abs()))
        off = off + 2.0 ** -8 * (out.abs() + off)
        assert ((got[t] - out).abs() <= off).all()


@pytest.mark.parametrize("T,E,k,H,I", [(16, 4, 2, 9480, 1024), (13, 8, 1, 9216, 1088), (16, 4, 2, 9480, 1160), (7, 8, 2, 4600, 2056), (16, 3, 3, 2304, 1096), (14, 8, 2, 2048, 4104)])
def test_all_tokens_at_the_same_experts_of_wide_layers(T, E, k, H, I):
    """What a stage of the second product's ring holds depends on the most tokens of an expert."""
    x, wr, w13, w2 = _experts(T, E, k, H, I, seed=8)
    x = (x[:1].float() + 0.02 * x.float()).to(BF16)
    ids = _routes(x, wr, k)
    assert max(sum(e in row for row in ids) for e in range(E)) == T
    _check_experts((x, wr, w13, w2), k)
    native.workspace().check_status()


@pytest.mark.parametrize("B,window", [(0, 0), (1, 0), (300, 64), (4096, 0)])
def test_tables_of_many_sequences_are_the_kernels(B, window):
    """Steps of more sequences than the kernel takes are tabled by whole arrays on the device."""
    g = torch.Generator().manual_seed(B)
    draw = lambda lo, hi: torch.randint(lo, hi, (B,), generator=g, dtype=torch.int32)
    seqs = torch.stack([draw(0, 40), draw(0, 200), draw(-1, 4), draw(0, 9)]).cuda()
    pages = torch.randint(1, 10000, (int(seqs[3].sum()),), generator=g, dtype=torch.int32).cuda()
    args = dict(tokens=int(seqs[0].sum()) + 3, max_blocks=8, page=16, window=window, tiles=((64, B + 2), (8, 4 * B)), lora_tiles=B + 1, lora_rows=32, row_offset=7,
                lead=torch.tensor([[2, 0, 7, 0]], dtype=torch.int32, device="cuda"))
    a, b = native.step_tables(seqs, pages, **args), reference.step_tables_of_many(seqs, pages, **args)
    for x, y in zip(a, b):
        assert all(torch.equal(p, q) for s, t in zip(x, y) for p, q in zip(s, t)) if isinstance(x, tuple) else torch.equal(x, y)


@pytest.mark.parametrize("T,E,H,kernels", [(1, 8, 512, 2), (8, 8, 4096, 2), (9, 8, 4096, 3), (1, 64, 2048, 3)])
def test_launches_of_small_and_of_large_routers(T, E, H, kernels):
    a = _experts(T, E, 2, H, 64)
    native.moe_few(*a, 2)
    before = native.launch_count
    native.moe_few(*a, 2)
    assert native.launch_count - before == kernels
