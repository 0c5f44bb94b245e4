"""Operators of layers in 8-bit integers on the GPU: rows at the ends of the numbers' range, and what other rows, forms and plans may change."""
import pytest
import torch

from lorax_b200.ops import native, native_int8  # noqa: F401  (the bindings of every operator first)
from lorax_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from lorax_b200.ops import native
    native.load()
    yield native
    native.workspace().check_status()


# A scale of few units of 2^-149 is off from max / 127 by up to half a unit, so that quotients pass 127: of 190 units, whose scale is one, 190.
TOPS = [1, 63, 64, 100, 127, 128, 129, 150, 190, 191, 255, 256, 300, 400, 513, 1000, 2039, 4000, 5000, 8000, 12345, 16002, 20000, 40000]


@pytest.mark.parametrize("I", [8, 100, 1001, 4096, 17000])
@pytest.mark.parametrize("copies", [1, 30])
@pytest.mark.parametrize("ring", [0, 1])
def test_rows_of_few_units_of_the_least_number(ops, I, copies, ring):
    """Products of two small halves, whole units of 2^-149, by a block per row and by blocks that stay: the bits of the plain form, whose quotients end at 127."""
    g = torch.Generator().manual_seed(I)
    tops = torch.tensor(TOPS * copies, dtype=torch.float64)
    # a unit is 2^-70 of the gate times 2^-79 of the other half; both hold 8 bits, so a row's largest is the nearest such product
    a = (tops.sqrt().floor()).clamp(1, 255)
    b = (tops / a).round().clamp(1, 255)
    up = torch.randint(-255, 256, (len(tops), I), generator=g).double()
    up = torch.minimum(torch.maximum(up, -b[:, None]), b[:, None])
    at = torch.arange(len(tops)) % I
    sign = torch.where(torch.arange(len(tops)) % 2 == 0, 1.0, -1.0).double()
    up[torch.arange(len(tops)), at] = b * sign
    x = torch.cat([(a[:, None] * 2.0 ** -70).expand(-1, I), up * 2.0 ** -79], 1).to(BF)
    want = ref.act_mul_int8(x, I, "relu")
    x = x.cuda()
    got = native_int8._on(x, native_int8._rows, x, x.stride(0), len(tops), I, 3, True, None, ring)
    assert torch.equal(got.scale.cpu(), want.scale) and torch.equal(got.q.cpu(), want.q)
    pub = ops.act_mul_int8(x, I, "relu")
    assert torch.equal(pub.q, got.q) and torch.equal(pub.scale, got.scale)


def _beside_borders():
    """(a row's largest value, its scale, a value half a unit from the border between two steps), in units of 2^-149, the values as (a, b, e): a * b * 2^e with a and b of 8
    bits.  The scales are odd and below 2^24 units, so that half of one lies between two numbers of 32 bits."""
    halves = {a * b: (a, b) for a in range(1, 256) for b in range(a, 256)}
    found = []
    for top in sorted(m for m in halves if m >= 1 << 14):
        for e in (13, 14, 15, 16):
            k = ((top << (e + 1)) + 127) // 254
            if 2500000 < k < 1 << 24 and k % 2:
                for v in (((2 * q + 1) * k + s) // 2 for q in range(126) for s in (-1, 1)):
                    z = (v & -v).bit_length() - 1
                    if v >> z in halves:
                        found.append(((*halves[top], e), k, (*halves[v >> z], z)))
    return found


@pytest.mark.parametrize("I", [2, 16])
def test_values_beside_the_border_of_steps_that_are_odd(ops, I):
    rows = _beside_borders()
    assert len(rows) > 200
    x = torch.zeros(len(rows), 2 * I, dtype=torch.float64)
    for t, (top, _, v) in enumerate(rows):
        for c, (a, b, e) in enumerate((top, v)):
            x[t, c], x[t, I + c] = a * 2.0 ** -70, b * 2.0 ** (e - 79)
    x = x.to(BF)
    want = ref.act_mul_int8(x, I, "relu")
    assert (want.scale.double() * 2.0 ** 149).tolist() == [k for _, k, _ in rows]
    got = ops.act_mul_int8(x.cuda(), I, "relu")
    assert torch.equal(got.scale.cpu(), want.scale) and torch.equal(got.q.cpu(), want.q)


@pytest.mark.parametrize("T,H", [(5, 64), (40, 65), (700, 2048), (700, 2049), (6, 16384)])
@pytest.mark.parametrize("layernorm", [False, True])
def test_norms_of_few_units_of_the_least_number(ops, T, H, layernorm):
    """Weights of 2^-133 behind a root of 2^20: a value of the stream of n / 64 is n units of 2^-149, give or take a millionth."""
    g = torch.Generator().manual_seed(H)
    n = torch.randint(-90, 91, (T, H), generator=g).double()
    tops = torch.tensor([100, 128, 150, 190, 255, 64, 129]).double()[torch.arange(T) % 7]
    n[:, 0] = tops * torch.where(torch.arange(T) % 2 == 0, 1.0, -1.0)
    n[:, 1] = -n[:, 0]
    if layernorm:                                  # (a mean of zero, which leaves whole units)
        n[:, 2::2] = -n[:, 3::2] if H % 2 == 0 else -torch.cat([n[:, 3::2], torch.zeros(T, 1, dtype=torch.float64)], 1)
    res = (n / 64).to(BF)
    w = torch.full((H,), 2.0 ** -133, dtype=BF)
    want = ref.norm_block(None, res, w, 2.0 ** 20, layernorm=layernorm, int8=True)
    got = ops.norm_block(None, res.cuda(), w.cuda(), 2.0 ** 20, layernorm=layernorm, int8=True)
    assert torch.equal(got.scale.cpu(), want.scale) and torch.equal(got.q.cpu(), want.q)


# ------------------------------------------------------------------------------------------------ other rows, forms and plans
def _plan(T, N, K, clusters, sms):
    import ctypes
    out = (ctypes.c_int * 4)()
    assert native.load().lx_gemm_int8_plan(T, N, K, sms, (ctypes.c_int * 4)(*clusters), out) == 0
    return tuple(out)


def _clusters():
    """Clusters of 1 to 4 pairs that run at the same time here, and SMs."""
    lib = native.load()
    return tuple(lib.lx_gemm_int8_clusters(p) for p in (1, 2, 3, 4)), native.workspace().num_sms


SIZES = [(1, 6144, 4096), (64, 4096, 14336), (256, 4096, 14336), (300, 1024, 8192), (512, 4096, 14336), (700, 4096, 4096), (1500, 2050, 1030), (33, 256, 512)]


def test_plans_go_by_the_clusters_that_the_device_runs(ops):
    clusters, sms = _clusters()
    assert all(0 <= 2 * p * n <= sms for p, n in enumerate(clusters, 1)) and clusters[0] > 0 and sorted(clusters, reverse=True) == list(clusters)
    shared = 0
    for T, N, K in SIZES + [(t, n, k) for t in (40, 130, 260, 520, 1030) for n in (256, 1000, 4096, 6144) for k in (512, 4096, 14336)]:
        pairs, bn, parts, _ = _plan(T, N, K, clusters, sms)
        assert pairs <= clusters[0]
        if pairs and parts > 1:
            shared += 1
            assert -(-N // 256) * -(-T // bn) <= clusters[parts - 1]
    assert shared
    for bad in (0, 5, -1):
        assert native.load().lx_gemm_int8_clusters(bad) < 0


@pytest.mark.parametrize("n", [4096, 1001])
def test_a_row_s_bytes_do_not_depend_on_other_rows_or_the_form(ops, n):
    """Rows and activations of 700 rows (at a width of a multiple of eight by blocks that stay), and of one row and a few of them by a block per row."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = (torch.randn(700, 2 * n, generator=g, device="cuda") * 3).to(BF)
    plain, gated = ops.quant_rows_int8(x[:, :n]), ops.act_mul_int8(x, n)
    for a, b in ((0, 1), (3, 20), (500, 700)):
        for whole, part in ((plain, ops.quant_rows_int8(x[a:b, :n])), (gated, ops.act_mul_int8(x[a:b], n))):
            assert torch.equal(part.q, whole.q[a:b]) and torch.equal(part.scale, whole.scale[a:b])


@pytest.mark.parametrize("N,K", [(4096, 4096), (1000, 1030)])
def test_a_row_s_product_does_not_depend_on_other_rows_or_the_plan(ops, N, K):
    g = torch.Generator(device="cuda").manual_seed(N)
    x = ops.quant_rows_int8(torch.randn(1500, K, generator=g, device="cuda").to(BF))
    w, ws = ref.quantize_weight_int8(torch.randn(N, K, generator=g, device="cuda"))
    b = torch.randn(N, generator=g, device="cuda").to(BF)
    whole = ops.gemm_int8(x, w, ws, bias=b)
    clusters, sms = _clusters()
    plans = {_plan(1500, N, K, clusters, sms)[:3]}
    for a, e in ((0, 1), (3, 20), (7, 100), (500, 800)):
        plans.add(_plan(e - a, N, K, clusters, sms)[:3])
        part = ops.gemm_int8(ref.Int8Rows(x.q[a:e], x.scale[a:e]), w, ws, bias=b)
        assert torch.equal(part, whole[a:e])
    assert len(plans) >= 4


@pytest.mark.parametrize("H,switch", [(512, False), (4096, True), (2049, True)])
@pytest.mark.parametrize("layernorm", [False, True])
def test_a_row_s_norm_differs_by_its_sums_order_alone(ops, H, switch, layernorm):
    """Of 2500 rows of 4096 and of 2049 the norms come from blocks that stay, of a few rows from a block each (of 512: from a block each, always): the same stream to the bit, as
    there is no norm in front of it, and the same result but for the order in which 32-bit sums are formed."""
    g = torch.Generator(device="cuda").manual_seed(H)
    T = 2500 if switch else 500
    y, res, w, b = ((torch.randn(*s, generator=g, device="cuda")).to(BF) for s in ((T, H), (T, H), (H,), (H,)))
    h = torch.empty_like(res)
    whole = ops.norm_block(y, res, w, 1e-5, bias=b, layernorm=layernorm, residual_out=h)
    for lo, hi in ((0, 1), (8, 21), (T - 30, T)):
        part_h = torch.empty_like(res[lo:hi])
        part = ops.norm_block(y[lo:hi], res[lo:hi], w, 1e-5, bias=b, layernorm=layernorm, residual_out=part_h)
        assert torch.equal(part_h, h[lo:hi])
        if not switch:
            assert torch.equal(part, whole[lo:hi])
            continue
        v = h[lo:hi].double()
        mean = v.mean(1, keepdim=True) if layernorm else 0
        scaled = (v - mean) / ((v - mean).square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
        # a sum passes 16 values in a thread, 5 and 5 levels of a block: 26 roundings, of the mean and of half the squares' sum; the root, and three factors and the
        # bias: 45 of 2^-24 for each of the two, the mean's of the row's largest; then a rounding to bf16 each
        loose = 45 * 2.0 ** -24 * (scaled.abs() + (v.abs().amax(1, keepdim=True) / (v - mean).square().mean(1, keepdim=True).sqrt() * w.double().abs() if layernorm else 0))
        want = scaled + b.double()
        assert ((part.double() - whole[lo:hi].double()).abs() <= 2 * (2.0 ** -8 * (want.abs() + loose) + loose)).all()
