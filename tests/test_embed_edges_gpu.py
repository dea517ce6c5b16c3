"""Embedding tables and linear adapters (quiver_b200.embed): calls side by side, wide ranges,
infinities, float32 results of 16-bit inputs, waits that run out. Against 64-bit computations;
bounds are derived as in test_embed_gpu.py (u = 2^-24, half a step of the result's type)."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(scope="module")
def embed(gpu):
    from quiver_b200 import embed as e
    return e


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, t=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)


def assert_within(got, want, bound, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float((off / bound.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} "
                           f"of the bound")


def test_threads_with_tables_of_different_sizes(embed):
    """Gradients of narrow and wide tables side by side: their sorts need different amounts of
    shared memory. (Calls of the C ABI with their arguments ready, so that they follow each other
    closely.)"""
    import ctypes as C
    from quiver_b200 import _native
    lib = _native.lib()
    n, dim = 9000, 4
    ids = torch.randint(0, 3, (n,), generator=gen(1), device="cuda")
    up = normal(gen(2), n, dim)
    tables = (3, 2047) * 4  # digits of 2 and of 11 bits
    want = [embed.embedding_grad(up, ids, r) for r in tables]
    torch.cuda.synchronize()
    bad = []

    def work(rows, want):
        s = torch.cuda.Stream()
        size = C.c_size_t()
        _native.check(lib.qv_embedding_grad_workspace(n, rows, dim, C.byref(size)))
        with torch.cuda.stream(s):
            out = torch.empty(rows, dim, device="cuda")
            ws = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        args = (0, 0, up.data_ptr(), dim, 1, ids.data_ptr(), n, rows, dim, C.c_float(1.0),
                out.data_ptr(), dim, ws.data_ptr(), size.value, s.cuda_stream)
        for _ in range(3000):
            if lib.qv_embedding_grad_device(*args) != 0:
                bad.append((rows, lib.qv_last_error()))
                break
        s.synchronize()
        if not torch.equal(out, want):
            bad.append(rows)

    threads = [threading.Thread(target=work, args=a) for a in zip(tables, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


@pytest.mark.parametrize("m,k,n,t", [(32768, 128, 2048, "bf16"), (32768, 192, 2048, "f16"),
                                     (32768, 1024, 2048, "bf16"), (16384, 16384, 1024, "bf16"),
                                     (20000, 200, 640, "f32"), (32768, 512, 1024, "f32")])
def test_wait_that_runs_out_over_many_units(embed, monkeypatch, m, k, n, t):
    """Blocks (of 64 and 128 columns, and pairs) with six units and more each: whatever a pipeline
    that gave up still returns is right, and the rest is NaN."""
    x = normal(gen(1), m, k, t=TYPES[t])
    w = normal(gen(2), n, k, t=TYPES[t])
    b = normal(gen(3), n, t=TYPES[t])
    r = normal(gen(4), m, n, t=TYPES[t])
    calls = (lambda: (embed.linear(x, w),), lambda: (embed.linear(x, w, b, residual=r),),
             lambda: embed.linear_preact(x, w, b, activation="relu"),
             lambda: embed.linear_preact(x, w, b, residual=r, activation="relu"),
             lambda: embed.linear_grad(r, x, w, need=(True, True, False))[:2])
    want = [c() for c in calls]
    torch.cuda.synchronize()
    lost = 0
    for limit in ("1", "2", "4", "8"):
        monkeypatch.setenv("QV_TC_WAIT_LIMIT_US", limit)
        got = [c() for c in calls]
        torch.cuda.synchronize()
        monkeypatch.delenv("QV_TC_WAIT_LIMIT_US")
        for i, (g, v) in enumerate(zip(got, want)):
            for p, q in zip(g, v):
                gone = p.isnan()
                lost += int(gone.sum())
                assert torch.equal(p[~gone], q[~gone]), (limit, i)
    assert lost > 0
    for c, v in zip(calls, want):
        assert all(torch.equal(p, q) for p, q in zip(c(), v))


def product_bound(x, w):
    """What a float32 product of k terms in any order and its parts may be off by, from sum |x||w|
    alone: 2u a term where the accumulator cuts, and 2^-21 for parts that leave out up to 2^-22 and
    2^-23 of a term."""
    return (x.double().abs() @ w.double().abs().t()) * ((x.shape[1] + 8) * 2 * U + 2.0 ** -21) \
        + TINY[torch.float32]


def wide_inputs(kind, m, n, k):
    g = gen(m + n + k)
    x, w = normal(g, m, k), normal(g, n, k)
    if kind == "column":  # one feature far above the others, its weights as far below
        for i, p in enumerate((20, 25, 30, 60)):
            x[:, i] *= 2.0 ** p
            w[:, i] *= 2.0 ** -p
    elif kind == "columns":  # every feature its own unit
        e = torch.linspace(-40, 40, k, device="cuda").round()
        x, w = x * 2.0 ** e, w * 2.0 ** -e
    elif kind == "row":  # a single row of the batch, its large element without a weight
        x[m // 2] = 1
        x[m // 2, 0] = 2.0 ** 40
        w[:, 0] = 0
    elif kind == "weight":
        w[n // 2] = 1
        w[n // 2, k - 1] = 2.0 ** 45
        x[:, k - 1] = 0
    elif kind == "one-hot":
        x.zero_()
        x[:, 1] = 1
        w[:, 0] = 2.0 ** 50
    elif kind == "tiny":  # rows of subnormal elements and weights that bring them back
        x = x * 2.0 ** -135
        x[:, 0] = 2.0 ** -112
        w = w * 2.0 ** 100
        w[:, 0] = 2.0 ** 60
    elif kind == "sparse":
        x = x.clamp(min=0) * (torch.rand(m, k, generator=g, device="cuda") < 0.3)
        w = w * 2.0 ** torch.randint(-30, 1, (1, k), generator=g, device="cuda")
    return x, w


@pytest.mark.parametrize("kind", ["plain", "column", "columns", "row", "weight", "one-hot", "tiny",
                                  "sparse"])
@pytest.mark.parametrize("m,k,n", [(300, 80, 72), (140, 129, 130), (6000, 512, 768),
                                   (1001, 1027, 515), (64, 8192, 128)])
def test_linear_float32_wide_rows(embed, kind, m, k, n):
    """Elements of very different magnitudes within a row keep float32's accuracy of the sum."""
    x, w = wide_inputs(kind, m, n, k)
    want = x.double() @ w.double().t()
    got = embed.linear(x, w)
    assert_within(got, want, product_bound(x, w), kind)
    assert torch.equal(got, embed.linear(x, w))
    y, z = embed.linear_preact(x, w, None, residual=got, activation="relu")
    assert torch.equal(z, got)


@pytest.mark.parametrize("m,n,k", [(300, 72, 80), (1500, 520, 1024)])
def test_linear_float32_wide_rows_alternate(embed, m, n, k):
    """Batches that need the planes and batches that do not, in turn and from replayed graphs with
    one workspace each: nothing of one call is left for the next."""
    plain, wide = wide_inputs("plain", m, n, k), wide_inputs("row", m, n, k)
    want = [embed.linear(*v) for v in (plain, wide)]
    held = [v.clone() for v in plain]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = embed.linear(*held)
    for i in (0, 1, 0, 1, 1, 0):
        for h, v in zip(held, (plain, wide)[i]):
            h.copy_(v)
        graph.replay()
        assert torch.equal(out, want[i])
        assert torch.equal(embed.linear(*(plain, wide)[i]), want[i])


def same_special(got, want, what=""):
    """Infinities and NaN exactly where the definition has them, and nowhere else."""
    assert torch.equal(got.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(got.isinf(), inf), what
    assert torch.equal(got[inf].double(), want[inf]), what


def plain_product(x, w):
    """x w^T in 64 bits with every term's own infinities (a library product may skip zeros)."""
    return torch.cat([(p[:, None, :] * w.double()[None]).sum(-1) for p in x.double().split(64)])


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(3, 40, 50), (140, 72, 130), (40, 4096, 72), (700, 129, 257)])
def test_linear_infinities(embed, t, m, k, n):
    """Infinite elements of x and of the weights: alone, beside large finite ones, of both signs,
    against zeros."""
    t = TYPES[t]
    g = gen(m + k)
    x, w = normal(g, m, k, t=t), normal(g, n, k, t=t)
    w[:, ::7] = 1  # values one part holds
    clean = embed.linear(x, w)
    inf = math.inf
    x[0, 0] = inf
    x[1, [3, 5]] = torch.tensor([-inf, -inf], device="cuda", dtype=t)
    x[2, [2, 7]] = torch.tensor([inf, -inf], device="cuda", dtype=t)
    if m > 8:
        x[m - 1, 1], x[m - 1, 2] = inf, (1e6 if t != torch.float16 else 6e4)
        x[5, 4], x[6, k - 1] = math.nan, inf
        w[n - 1, 9] = -inf
        w[n - 2, 11], w[n - 2, 12] = inf, 0
        w[3, 0] = 0  # against x[0, 0]
        x[7, 9] = 0
    want = plain_product(x, w)
    got = embed.linear(x, w)
    same_special(got, want)
    keep = torch.isfinite(x).all(1)[:, None] & torch.isfinite(w).all(1)[None] & (w[:, 0] != 0)
    if m > 8:
        keep[7] = False
    assert torch.equal(got[keep], clean[keep])
    # through bias, residual and preactivations, whole and unaligned rows
    b, r = normal(g, n, t=t), normal(g, m, n, t=t)
    z = want + b.double()
    y, pre = embed.linear_preact(x, w, b, residual=r, activation="relu")
    same_special(pre, z)
    same_special(y, torch.where(z.isnan(), z, z.clamp(min=0)) + r.double())
    # gradients: dz holds the infinities
    dy = normal(g, m, n, t=t)
    dy[0, 0] = inf
    dy[1, 1], dy[1, 2] = -inf, -inf
    fx, fw = normal(g, m, k, t=t), normal(g, n, k, t=t)
    fx[0, 0] = 0
    fw[:, ::5] = -1
    dx, dw, db = embed.linear_grad(dy, fx, fw)
    same_special(dx, plain_product(dy, fw.t()), "dx")
    same_special(dw, plain_product(dy.t(), fx.t()), "dw")
    same_special(db, dy.double().sum(0), "db")


def test_linear_all_special(embed):
    """Nothing but NaN, and nothing but infinities, at a size of many tiles."""
    x, w = torch.full((3000, 256), math.nan, device="cuda"), normal(gen(1), 500, 256)
    assert embed.linear(x, w).isnan().all()
    x.fill_(math.inf)
    assert embed.linear(x, w.abs() + 1).eq(math.inf).all()
    same_special(embed.linear(x[:100], w), plain_product(x[:100], w))


def act_ref(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":  # by erfc, which keeps the tail
        return z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
    if act == "gelu_tanh":  # z / (1 + exp(-2u)): the tanh form without its cancellation
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def activations_on_a_grid(embed, t, act, out_dtype, m, relative):
    """act(z) by a layer of zero weights whose bias is z."""
    z = torch.cat([torch.linspace(-90, 90, 24001), torch.linspace(-14, 14, 40001),
                   torch.linspace(-0.01, 0.01, 2001)]).cuda().to(t)
    for z in z.split(65536):
        got = embed.linear(torch.zeros(m, 16, device="cuda", dtype=t),
                           torch.zeros(len(z), 16, device="cuda", dtype=t), z, activation=act,
                           out_dtype=out_dtype)
        want = act_ref(z.double(), act).expand(m, len(z))
        # factors below 2^-126 are flushed to zero: up to |z| 2^-126 <= 90 * 2^-126 < 2^-119
        assert_within(got, want, want.abs() * relative + 2.0 ** -119 + TINY[got.dtype], act)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m", [1, 200])
def test_activation_tails(embed, t, act, m):
    """16-bit activations to their own half step in the tails too. The exponents reach 126 in units
    of log2, with up to three roundings of 2^-24: 1.6e-5; with the fitted tail's 4.3e-6 less than
    2^-15 of the value."""
    t = TYPES[t]
    activations_on_a_grid(embed, t, act, None, m, half_step(t) + 2.0 ** -15)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m", [1, 200])
def test_activations_to_float32(embed, t, act, m):
    """Float32 results, of 16-bit inputs too: the math library's few ulp (2^-21) and the exponents'
    roundings, which grow with them: |x| <= 4 gelu_tanh's argument has at most 2^3.4 and three
    roundings of 2^-24."""
    t = TYPES[t]
    z = torch.linspace(-4, 4, 40001).cuda().to(t)
    got = embed.linear(torch.zeros(m, 16, device="cuda", dtype=t),
                       torch.zeros(len(z), 16, device="cuda", dtype=t), z, activation=act,
                       out_dtype=torch.float32)
    want = act_ref(z.double(), act).expand(m, len(z))
    assert_within(got, want, want.abs() * 2.0 ** -18.5 + 2.0 ** -140, act)
    activations_on_a_grid(embed, t, act, torch.float32, m, 2.0 ** -15)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(3, 500, 70), (300, 1000, 96), (300, 4096, 1000),
                                   (5000, 8192, 520), (260, 8190, 257)])
def test_float32_results_of_16_bit_inputs(embed, t, m, k, n):
    """Sums of one sign, with bias, activation and residual. The accumulator cuts its sum so far by
    at most 2u, and at most once for every four terms (at 4096 terms it loses 436u, which are 1.7u
    of the mean sum for every eight: cuts lose half of what they may at the mean). 512 terms stay
    there: 128 cuts, at half of the last sum on average, 128u; then the sums are added, rounding."""
    t = TYPES[t]
    g = gen(m + n)
    x, w = normal(g, m, k, t=t).abs(), normal(g, n, k, t=t, scale=1 / k).abs()
    b, r = normal(g, n, t=t), normal(g, m, n, t=t)
    mass = x.double() @ w.double().t()
    sums = mass * (128 + k / 512 + 8) * U
    got = embed.linear(x, w, out_dtype=torch.float32)
    assert_within(got, mass, sums)
    z = mass + b.double()
    zerr = sums + z.abs() * U
    for act in ("none", "silu"):
        want = act_ref(z, act) + r.double()
        err = 1.13 * zerr + (z.abs() + want.abs()) * (2.0 ** -21 + U)
        got = embed.linear(x, w, b, residual=r, activation=act, out_dtype=torch.float32)
        assert_within(got, want, err, act)


def act_slope(z, act):
    """act'(z) and act in 64 bits, by autograd of the definition."""
    z = z.clone().requires_grad_()
    (d,) = torch.autograd.grad(act_ref(z, act).sum(), z)
    return d


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(1, 16, 24), (40, 64, 72), (300, 40, 57), (2000, 96, 260)])
def test_gradients_of_float32_results(embed, t, act, m, k, n):
    """A float32 gradient is rounded once, with the derivative on it: values that the 16-bit type
    cannot hold do not become infinite or zero ahead of it."""
    t = TYPES[t]
    h = half_step(t)
    g = gen(m + n)
    x, w = normal(g, m, k, t=t), normal(g, n, k, t=t, scale=k ** -0.5)
    z = normal(g, m, n, t=t)
    dy = normal(g, m, n)
    if t == torch.float16:  # past the type's range where the derivative is small
        z[:, ::3] = -4.0
        dy[:, ::3] *= 1e5 / (1.0 if act in ("gelu", "silu") else 1e5)
    dx, dw, db = embed.linear_grad(dy, x, w, z, act)
    dz = dy.double() * act_slope(z.double(), act)
    # the derivative to 2^-15 (+ as much of 1 where it crosses 0), one rounding of dz, the sums
    off = dy.double().abs() * 2.0 ** -14 * (0 if act in ("none", "relu") else 1)
    rounded = off + (dz.abs() + off) * (h + 2 * U) + TINY[t]

    def check(got, a, b, err, what):
        want = a @ b
        bound = err @ b.abs() + (a.abs() + err) @ b.abs() * ((a.shape[1] + 8) * 2 * U)
        held = (want.abs() + bound) < torch.finfo(t).max
        bound = bound + (want.abs() + bound) * h + TINY[t]
        assert_within(got[held], want[held], bound[held], what)

    check(dx, dz, w.double(), rounded, "dx")
    check(dw, dz.t(), x.double(), rounded.t(), "dw")
    ones = torch.ones(m, 1, dtype=torch.float64, device="cuda")
    check(db[:, None], dz.t(), ones, (off + dz.abs() * 2 * U).t(), "db")
    # autograd takes the same way, also strided and broadcast
    leaves = [v.clone().requires_grad_() for v in (x, w, normal(g, n, t=t), normal(g, m, n, t=t))]
    y = embed.linear(*leaves[:3], residual=leaves[3], activation=act, out_dtype=torch.float32)
    _, pre = embed.linear_preact(*[v.detach() for v in leaves[:3]], activation=act,
                                 out_dtype=torch.float32)
    dy = normal(g, m, n)  # in range for these preactivations: NaN would equal nothing
    for up in (dy, dy[:1].expand(m, n), torch.cat([dy, dy], 1)[:, 1:n + 1]):
        got = torch.autograd.grad(y, leaves, up, retain_graph=True)
        want = embed.linear_grad(up.contiguous(), x, w, pre, act)
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        assert torch.equal(got[3], up.to(t))


def test_gradients_of_float32_results_hold_the_range(embed):
    """Upstream values outside float16's range whose gradients are inside it."""
    x = torch.full((40, 16), 2.0 ** -8, device="cuda", dtype=torch.float16)
    w = torch.full((24, 16), 2.0 ** -8, device="cuda", dtype=torch.float16)
    z = torch.full((40, 24), -4.0, device="cuda", dtype=torch.float16)
    dy = torch.full((40, 24), 2.0 ** 18, device="cuda")
    dx, dw, db = embed.linear_grad(dy, x, w, z, "gelu")
    d = float(act_slope(torch.tensor([-4.0], dtype=torch.float64), "gelu")) * 2.0 ** 18
    for got, want in ((dx, d * 24 / 256), (dw, d * 40 / 256), (db, d * 40)):
        assert ((got.double() / want - 1).abs() <= 2 * 2.0 ** -11 + 2.0 ** -13).all()
    dx, dw, db = embed.linear_grad(dy * 2.0 ** -50, x, w, z, "gelu")
    assert (db != 0).logical_or(torch.tensor(abs(d) * 40 * 2.0 ** -50 < 2.0 ** -25)).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 40), (6, 64, 33), (300, 96, 96), (1000, 64, 257)])
def test_float32_residual(embed, t, m, k, n):
    """A 16-bit layer with a float32 result adds a float32 residual with all its bits: whole and
    unaligned rows, one row for all, windows, with preactivations."""
    t = TYPES[t]
    g = gen(m + n)
    x, w, b = normal(g, m, k, t=t), normal(g, n, k, t=t, scale=k ** -0.5), normal(g, n, t=t)
    plain, z = embed.linear_preact(x, w, b, activation="silu", out_dtype=torch.float32)
    wide = normal(g, m, n + 7)
    for r in (normal(g, m, n), wide[:, 3:n + 3], wide[:1, :n].expand(m, n)):
        got = embed.linear(x, w, b, residual=r, activation="silu", out_dtype=torch.float32)
        assert torch.equal(got, plain + r)  # the same sum, one float32 addition
        y, pre = embed.linear_preact(x, w, b, residual=r, activation="silu", out_dtype=torch.float32)
        assert torch.equal(y, got) and torch.equal(pre, z)
    leaf = normal(g, m, n).requires_grad_()
    dy = normal(g, m, n)
    (dr,) = torch.autograd.grad(embed.linear(x, w, b, residual=leaf, out_dtype=torch.float32), leaf,
                                dy)
    assert dr.dtype == torch.float32 and torch.equal(dr, dy)
    for bad in (lambda: embed.linear(x, w, residual=leaf.detach()),  # a 16-bit result
                lambda: embed.linear(x, w, residual=leaf.detach()[:, 1:], out_dtype=torch.float32),
                lambda: embed.linear(x, w, residual=leaf.detach().double(),
                                     out_dtype=torch.float32)):
        with pytest.raises(ValueError):
            bad()


def test_adapter_adds_the_vector_itself(embed):
    """A 16-bit adapter with a skip keeps the float32 vector's bits; zero weights give it back."""
    for t in TYPES.values():
        for m in (1, 500):
            v = normal(gen(m), m, 96)
            a = embed.Adapter(torch.zeros(96, 96, device="cuda", dtype=t), residual=True)
            assert torch.equal(a(v), v)
            w, b = normal(gen(1), 96, 96, t=t, scale=0.1), normal(gen(2), 96, t=t)
            got = embed.Adapter(w, b, activation="gelu", residual=True)(v)
            x = v.to(t)
            assert torch.equal(got, embed.linear(x, w, b, activation="gelu",
                                                 out_dtype=torch.float32) + v)
            assert embed.Adapter(w, residual=True)(x).dtype == torch.float32


def test_rows_of_answers(gpu, embed):
    """From answers to their stored rows, with labels of one's own, unfilled slots and an adapter."""
    base = normal(gen(1), 400, 48)
    labels = torch.randperm(400, generator=torch.Generator().manual_seed(1)).cuda() + 10_000
    ix = gpu.FlatIndex(48, "l2")
    ix.add_device(base[:250], labels[:250])
    ix.add_device(base[250:], labels[250:])
    at = torch.tensor([7, 399, 250], device="cuda")
    dist, label, rows = ix.search_device(base[at], 5, return_rows=True)
    assert rows.dtype == torch.int64 and rows.shape == (3, 5)
    assert torch.equal(rows[:, 0], at) and torch.equal(labels[rows], label)
    assert torch.equal(ix.lookup_device(rows), base[rows])
    d2, l2 = ix.search_device(base[at], 5)
    assert torch.equal(dist, d2) and torch.equal(label, l2)
    few = gpu.FlatIndex(48, "l2")
    few.add_device(base[:3], labels[:3])
    eye = embed.Adapter(torch.eye(48, device="cuda"))
    dist, label, rows = few.search_device(base[:2], 7, adapter=eye, return_rows=True)
    assert (rows[:, 3:] == -1).all() and (rows[:, :3].sort(1)[0] == torch.arange(3).cuda()).all()
    near = few.lookup_device(rows)
    assert (near[:, 3:] == 0).all() and torch.equal(near[:, :3], base[rows[:, :3]])
    none = few.search_device(base[:0], 7, return_rows=True)
    assert [tuple(v.shape) for v in none] == [(0, 7)] * 3


@pytest.mark.parametrize("m,k,n", [(20, 40, 50), (140, 72, 130), (3000, 512, 520), (64, 8192, 128)])
def test_linear_float32_next_to_the_largest(embed, m, k, n):
    """Products just below float32's end, whose operands' first parts multiply to infinity."""
    v = 1.9995 * 2.0 ** 63  # v^2 = 1.999 * 2^127; bfloat16 rounds v up to 2^64
    x, w = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    x[:, 3], w[:, 3] = v, v
    x[1::3, 3] = -v
    w[:, 5] = 2.0 ** -126
    b = torch.full((n,), -2.0 ** 126, device="cuda")
    want = x.double() @ w.double().t()
    same = lambda got, want: assert_within(got, want, want.abs() * 2.0 ** -21)  # noqa: E731
    same(embed.linear(x, w), want)
    y, z = embed.linear_preact(x, w, b.abs() * torch.where(x[0, 3] > 0, -1, 1), activation="relu")
    keep = x[:, 3] > 0
    same(z[keep], want[keep] - 2.0 ** 126)
    same(y[keep], want[keep] - 2.0 ** 126)
    assert (y[~keep] == 0).all()
    dy = torch.zeros(m, n, device="cuda")
    dy[:, 3], w[3] = v, v
    dx, _, _ = embed.linear_grad(dy, x, w, need=(True, False, False))
    same(dx, dy.double() @ w.double())
    dy.zero_()
    dy[3] = v
    x[3] = -v
    _, dw, _ = embed.linear_grad(dy, x, w, need=(False, True, False))
    same(dw, dy.double().t() @ x.double())


def test_float32_far_offsets(embed):
    """Float32 operands, parts and results past 2^31 elements, infinities at their end, and their
    gradients."""
    m, k, n = 17_000_000, 136, 130
    x = torch.zeros(m, k, device="cuda")
    x[-300:] = normal(gen(1), 300, k)
    w = normal(gen(2), n, k)
    for wide in (False, True):
        if wide:
            x[-300:, 0], w[:, 0] = 2.0 ** 40, 0
            x[-300:, 1:] = 1
        y = embed.linear(x, w, activation="relu")
        want = (x[-300:].double() @ w.double().t()).clamp(min=0)
        assert_within(y[-300:], want, product_bound(x[-300:], w))
        assert (y[:1000] == 0).all() and (y[m // 2:m // 2 + 1000] == 0).all()
        del y
    x[-7, 5] = math.inf
    y = embed.linear(x, w)
    same_special(y[-300:], plain_product(x[-300:], w))
    dx, dw, db = embed.linear_grad(y, x, w)
    assert dx[-7].isnan().any() and torch.isfinite(dx[-6:]).all() and (dx[:1000] == 0).all()
    assert_within(dx[-6:], y[-6:].double() @ w.double(), product_bound(y[-6:], w.t()))
    same_special(db, y[-300:].double().sum(0))


def test_flags_of_the_c_interface(embed):
    """QV_RESIDUAL_F32 goes with float32 results, QV_GRAD_F32 with every type; other bits are refused."""
    import ctypes as C
    from quiver_b200 import _native
    lib, size = _native.lib(), C.c_size_t()
    x, w, y = normal(gen(1), 20, 16), normal(gen(2), 24, 16), torch.empty(20, 24, device="cuda")
    p = [v.data_ptr() for v in (x, w, y)]

    def forward(dtype, out_dtype):
        a = _native.qv_linear(dtype, out_dtype, 0, 20, 24, 16, p[0], 16, p[1], 16, None, p[2], 24, p[2],
                              24, None, 24)
        return lib.qv_linear_workspace(0, C.byref(a), C.byref(size))

    def backward(dtype):
        a = _native.qv_linear_grad(dtype, 0, 20, 24, 16, p[2], 24, p[0], 16, p[1], 16, None, 0, p[0],
                                   16, p[1], 16, None)
        return lib.qv_linear_grad_workspace(0, C.byref(a), C.byref(size))

    for good in (lambda: forward(2, 0x100), lambda: forward(0, 0x100), lambda: forward(1, 0),
                 lambda: backward(0x100), lambda: backward(0x102), lambda: backward(1)):
        _native.check(good())
    for bad in (lambda: forward(2, 0x102), lambda: forward(0x102, 2), lambda: forward(2, 0x200),
                lambda: forward(2, 1), lambda: backward(0x202), lambda: backward(3),
                lambda: backward(0x103)):
        with pytest.raises(ValueError):
            _native.check(bad())
