"""Layers in 8-bit integers: products beside cuBLAS, both forms of the operators on rows, plans of products, and a model's steps.

    python benchmarks/bench_int8.py [products] [forms] [plans] [steps]

Operators: microseconds a call in a CUDA graph, over inputs larger than the 126 MB of L2, best of 5 replays, CUDA events on the launching stream.  Steps: microseconds a
step of eight layers of a 7B decoder with random weights, decode steps in graphs over contexts of 700 tokens, prompts as the engine runs them."""
import os
import random
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch

from lorax_b200.ops import native, native_int8
from lorax_b200.ops import reference as ref

BF = torch.bfloat16
L2 = 300e6


def timeit(fn, copies, reps=5):
    """Of fn(i), i below `copies`; results of the last captured calls are kept, so that no call's output takes the place of another's."""
    n = max(copies, 8)
    for i in range(3):
        fn(i % copies)
    torch.cuda.synchronize()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        for i in range(n):
            fn(i % copies)
    g.replay()
    torch.cuda.synchronize()
    best = 1e9
    for _ in range(reps):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / n)
    return best


def _copies(nbytes):
    return max(1, min(100, -(-int(L2) // int(nbytes))))


def _up(a, b):
    return -(-a // b)


class Product:
    def __init__(self, T, N, K):
        c = self.copies = _copies(N * K + T * K)
        pitch = _up(K, 16) * 16
        self.sizes = (T, N, K, pitch, pitch)
        self.w = [torch.randint(-127, 128, (N, pitch), device="cuda", dtype=torch.int8)[:, :K] for _ in range(c)]
        self.q = [torch.randint(-127, 128, (T, pitch), device="cuda", dtype=torch.int8)[:, :K] for _ in range(c)]
        self.ws, self.xs = torch.rand(N, device="cuda"), torch.rand(T, device="cuda")
        self.out = torch.empty(T, _up(N, 8) * 8, device="cuda", dtype=BF)[:, :N]

    def time(self, plan=None, reps=5):
        return timeit(lambda i: native_int8._on(self.w[0], native_int8._gemm_int8, ref.Int8Rows(self.q[i], self.xs), self.w[i], self.ws, None, self.out, self.sizes, True, plan),
                      self.copies, reps)


def products():
    print("products: T x N x K, here, torch._int_mm (sums of 32 bits, no scales), torch.matmul in bf16")
    for T, N, K in ((1, 28672, 4096), (1, 4096, 14336), (1, 6144, 4096), (48, 28672, 4096), (256, 28672, 4096), (256, 4096, 14336), (512, 4096, 4096), (2048, 28672, 4096),
                    (2048, 4096, 14336), (4001, 28672, 4096)):
        p = Product(T, N, K)
        ours = p.time()
        theirs = timeit(lambda i: torch._int_mm(p.q[i], p.w[i].t()), p.copies) if T > 16 else float("nan")
        c = _copies(2 * N * K + 2 * T * K)
        w, x = [torch.randn(N, K, device="cuda").to(BF) for _ in range(c)], torch.randn(T, K, device="cuda").to(BF)
        out = torch.empty(T, N, device="cuda", dtype=BF)
        dense = timeit(lambda i: torch.matmul(x, w[i].t(), out=out), c)
        print(f"  {T} x {N} x {K}: {ours:.1f}  {theirs:.1f}  {dense:.1f}", flush=True)
        del p, w
        torch.cuda.empty_cache()


def _rows(T, n, act, ring):
    c = _copies(T * n * (5 if act else 3))
    x = [torch.randn(T, n * (2 if act else 1), device="cuda").to(BF) for _ in range(c)]
    a = native._ACTS[act] if act else -1
    return timeit(lambda i: native_int8._on(x[0], native_int8._rows, x[i], x[0].stride(0), T, n, a, bool(act), None, ring), c)


def _norms(T, H, ring, int8=False, layernorm=False, post=True, gate=False):
    c = _copies(T * H * 7)
    new = lambda *s: torch.randn(*s, device="cuda").to(BF)
    y, res, out, h = ([new(T, H) for _ in range(c)] for _ in range(4))
    w, pw, b, pb, g = (new(H) for _ in range(5))

    def call(i):
        o = None if int8 else out[i]
        vectors = (pw if post else None, g if gate else None, 1.0, b if layernorm else None, pb if layernorm and post else None)
        checked = ref.check_norm_block(y[i], res[i], w, *vectors, h[i], o, int8)
        native_int8._on(w, native_int8._norm_block, checked, 1e-5, 1.0, 0.0, layernorm, o, int8, ring)
    return timeit(call, c)


def forms():
    pair = lambda f, *a, **k: "%.1f / %.1f" % tuple(f(*a, **k, ring=r) for r in (0, 1))
    print("quantisers: a block per row / blocks that stay")
    for n, act in ((1024, None), (4096, None), (8192, None), (14336, None), (4096, "silu"), (8192, "silu"), (14336, "silu")):
        print(f"  {n} {act or 'rows'}: " + ", ".join(f"{T} rows {pair(_rows, T, n, act)}" for T in (148, 200, 256, 300, 400, 500, 592, 700, 1000, 4001)), flush=True)
    print("norms on both sides: a block per row / blocks that stay (from 9600 values an SM)")
    for more in (dict(), dict(int8=True), dict(layernorm=True), dict(layernorm=True, int8=True)):
        for H in (1024, 4096, 8192):
            print(f"  {H} {more}: " + ", ".join(f"{T} rows ({T * H / 148 / 9600:.2f}) {pair(_norms, T, H, **more)}" for T in (200, 300, 400, 600, 1200, 1500, 4001)), flush=True)
    print("norms of odd widths: a block per row / blocks that stay")
    for more in (dict(post=False), dict(), dict(layernorm=True, gate=True)):
        for H in (1021, 1279, 1535, 1791, 2049, 4097):
            print(f"  {H} {more}: " + ", ".join(f"{T} rows {pair(_norms, T, H, **more)}" for T in (1500, 3000, 6000)), flush=True)


def _allowed(T, N, K):
    """Plans to try: tiles that even the rows out, shares of K up to eight CTAs or three pairs, as far as they run at the same time."""
    lib = native.load()
    fit, found, most, blocks = [0] + [lib.lx_gemm_int8_clusters(p) for p in (1, 2, 3, 4)], [], 256, _up(K, 128)
    while most >= 16:
        bn = _up(_up(T, _up(T, most)), 16) * 16
        if _up(T, most) <= 64:
            tiles, pairs = _up(N, 128) * _up(T, bn), _up(N, 256) * _up(T, _up(bn, 32) * 32)
            found += [(False, bn, p) for p in (1, 2, 3, 4, 8) if p <= blocks and tiles * p <= (1500 if p == 1 else 420)]
            found += [(True, _up(bn, 32) * 32, p) for p in (1, 2, 3) if T > 32 and p <= blocks and (pairs <= fit[p] if p > 1 else pairs < 2000)]
        most -= 32 if most > 64 else 16
    return sorted(set(found))


def plans():
    rng, worse, tried = random.Random(11), [], 0
    shapes = [(T, N, K) for T in (1, 48, 137, 256, 512, 1500) for N, K in ((4096, 4096), (6144, 4096), (28672, 4096), (4096, 14336), (2050, 1024), (512, 512))]
    while len(shapes) < 100:
        T, K, N = int(2 ** rng.uniform(0, 11.9)), int(2 ** rng.uniform(7, 13.8)), int(2 ** rng.uniform(7, 14.8))
        if N * K < 120e6 and T * N * K < 3e11:
            shapes.append((T, N // 2 * 2, K))
    for T, N, K in shapes:
        p = Product(T, N, K)
        times = {plan: p.time(plan, reps=2) for plan in _allowed(T, N, K)}
        tried += len(times)
        worse.append((p.time(reps=2) / min(times.values()), (T, N, K)))
        del p
        torch.cuda.empty_cache()
    worse.sort(reverse=True)
    print(f"plans: {tried} of {len(shapes)} shapes; the chosen one is {sum(w for w, _ in worse) / len(worse) - 1:.1%} slower than the quickest on average, over 10 % in "
          f"{sum(w > 1.1 for w, _ in worse)}; the worst: " + ", ".join(f"{s} {w:.2f}" for w, s in worse[:5]), flush=True)


def _adapters(cfg, model, count, rank=16):
    from lorax_b200.adapters.lora import random_adapter
    from lorax_b200.adapters.manager import AdapterManager
    mgr = AdapterManager(model, arena_bytes=1 << 30, host_bytes=1 << 30)
    for i in range(count):
        c, m = random_adapter(cfg, r=rank, alpha=16, seed=i, target_modules=["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"])
        mgr.register(f"a{i}", c, m)
        assert mgr.load(i + 1, f"a{i}")


def steps():
    from lorax_b200 import config as cfgs
    from lorax_b200.models.decoder import DecoderModel
    from lorax_b200.runtime.kv_cache import KVCache
    from lorax_b200.runtime.runner import ModelRunner, PrefillItem
    dev, page, ctx = torch.device("cuda", 0), 32, 700
    blocks = _up(ctx + 64, page)
    for adapters in (0, 8):
        print(f"steps, {adapters} adapters" + (" of rank 16 on every projection, a row's own in turn" if adapters else ""))
        for method in (None, "fp8", "eetq", "w8a8"):
            cfg = cfgs.mistral_7b()
            cfg.num_hidden_layers = 8
            model = DecoderModel.random_init_on_device(cfg, dev, BF, max_positions=4096)
            if method:
                model.quantize(method)
            if adapters:
                _adapters(cfg, model, adapters)
            torch.cuda.empty_cache()
            took = []
            for B in (1, 48, 256):
                kv = KVCache(cfg.num_hidden_layers, B * blocks + 300, model.nkv, model.d, BF, dev)
                r = ModelRunner(model, kv, max_batch=B, max_seq_tokens=4200, max_prefill_tokens=4096, use_graphs=True)
                rows = [r.state.take_row(i) for i in range(B)]
                r.install(rows, [1] * B, [ctx] * B, [[1 + i * blocks + j for j in range(blocks)] for i in range(B)], [1 + i % adapters if adapters else 0 for i in range(B)])
                r.resort()
                took.append((f"decode of {B}", _best(lambda: [r.decode() for _ in range(20)], 3) / 20))
            for T in (512, 4096):
                items = [PrefillItem(torch.randint(0, 32000, (T,)).tolist(), 0, [1 + j for j in range(_up(T, page))], adapter_index=1 if adapters else 0)]
                took.append((f"prompt of {T}", _best(lambda: r.prefill(items), 5)))
            native.workspace().check_status()
            print(f"  {method or 'bf16'}: " + ", ".join(f"{name} {us:.0f}" for name, us in took), flush=True)
            del model, kv, r
            torch.cuda.empty_cache()


def _best(fn, reps):
    for _ in range(2):
        fn()
    torch.cuda.synchronize()
    best = 1e9
    for _ in range(reps):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        fn()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3)
    return best


if __name__ == "__main__":
    for what in sys.argv[1:] or ("products", "forms", "plans", "steps"):
        dict(products=products, forms=forms, plans=plans, steps=steps)[what]()
    native.workspace().check_status()
