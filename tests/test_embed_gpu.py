"""Embedding tables and linear adapters (quiver_b200.embed) against plain 64-bit computations.

Tolerances are bounds, not fits: u = 2^-24 for a float32 operation (2u where an accumulator cuts
instead of rounding), half a step of the result's type, and the propagation of both through the
formulas."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Half the spacing of a type's smallest values: what a result near zero may be off by.
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


# ---- lookup -------------------------------------------------------------------------------------


def lookup_ref(table, ids, scale):
    s = float(np.float32(scale))
    out = torch.zeros(tuple(ids.shape) + (table.shape[1],), dtype=torch.float64, device="cuda")
    ok = (ids >= 0) & (ids < table.shape[0])
    out[ok] = table.double()[ids[ok].long()] * s
    out[ids >= table.shape[0]] = math.nan
    return out


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 33, 100, 128, 768])
@pytest.mark.parametrize("n", [1, 5, 1000])
def test_lookup(embed, t, dim, n):
    t = TYPES[t]
    g = gen(dim * 1000 + n)
    table = normal(g, 777, dim, t=t)
    ids = torch.randint(0, 777, (n,), generator=g, device="cuda")
    for i in (ids, ids.int()):
        got = embed.embedding_lookup(table, i, 27.7)
        want = lookup_ref(table, ids, 27.7)
        assert got.dtype == t and got.shape == (n, dim)
        # one float32 product and one rounding
        assert_within(got, want, want.abs() * (half_step(t) + 2 * U) + TINY[t])
    assert torch.equal(embed.embedding_lookup(table, ids), table[ids])


def test_lookup_slots_shapes_and_strides(embed):
    g = gen(3)
    table = normal(g, 50, 24, t=torch.float32)
    ids = torch.tensor([[0, -1, 49], [50, 7, -2 ** 62]], device="cuda")
    got = embed.embedding_lookup(table, ids)
    assert got.shape == (2, 3, 24)
    assert torch.equal(got[0, 1], torch.zeros(24, device="cuda"))
    assert torch.equal(got[1, 2], torch.zeros(24, device="cuda"))
    assert got[1, 0].isnan().all()
    assert torch.equal(got[0, 0], table[0]) and torch.equal(got[1, 1], table[7])
    # a window of wider rows, at an odd offset, and a transposed table
    wide = normal(g, 50, 40, t=torch.bfloat16)
    i = torch.tensor([3, 3, 49, 0], device="cuda")
    assert torch.equal(embed.embedding_lookup(wide[:, 3:30], i), wide[:, 3:30][i])
    assert torch.equal(embed.embedding_lookup(wide.t(), i.clamp(max=39)),
                       wide.t()[i.clamp(max=39)])
    assert torch.equal(embed.embedding_lookup(wide[:1].expand(50, 40), i), wide[:1].expand(4, 40))
    # none, an empty table, and a caller's result
    assert embed.embedding_lookup(table, ids[:0]).shape == (0, 3, 24)
    none = torch.empty(0, 24, device="cuda")
    assert embed.embedding_lookup(none, i).isnan().all()
    out = torch.empty(4, 24, device="cuda")
    assert embed.embedding_lookup(table, i, 2.0, out=out) is out
    assert torch.equal(out, table[i] * 2)


def test_lookup_special_values(embed):
    table = torch.tensor([[math.inf, -math.inf, math.nan, 6e4]], device="cuda").half()
    got = embed.embedding_lookup(table, torch.zeros(1, dtype=torch.long, device="cuda"), 2.0)
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and got[0, 2].isnan()
    assert got[0, 3] == math.inf  # past float16's range


# ---- gradient ------------------------------------------------------------------------------------


def grad_ref(up, ids, rows, scale):
    """(gradient, bound of the float32 sum's error) in 64 bits."""
    s = float(np.float32(scale))
    up = up.reshape(-1, up.shape[-1]).double()
    ids = ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < rows)
    want = torch.zeros(rows, up.shape[1], dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(want)
    want.index_add_(0, ids[ok], up[ok] * s)
    mass.index_add_(0, ids[ok], up[ok].abs() * s)
    count = torch.bincount(ids[ok], minlength=rows)[:, None].double()
    # a sum of `count` terms in any order is off by at most (count - 1) u of their magnitudes,
    # the joins of partial sums included; one more for the scale
    return want, mass * (count + 2) * U


def check_grad(embed, up, ids, rows, scale=1.0):
    got = embed.embedding_grad(up, ids, rows, scale)
    want, err = grad_ref(up, ids, rows, scale)
    t = up.dtype
    assert got.dtype == t and got.shape == (rows, up.shape[-1])
    assert_within(got, want, err + want.abs() * (half_step(t) + 2 * U) + TINY[t])
    assert torch.equal(got, embed.embedding_grad(up, ids, rows, scale))  # the same bits again
    return got


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("dim", [1, 3, 8, 100, 129, 768])
@pytest.mark.parametrize("n,rows", [(1, 1), (1, 5000), (33, 7), (700, 5000), (3000, 40),
                                    (5000, 70000)])
def test_grad(embed, t, dim, n, rows):
    g = gen(dim + n * 7 + rows)
    up = normal(g, n, dim, t=TYPES[t])
    ids = torch.randint(-1, rows, (n,), generator=g, device="cuda")
    check_grad(embed, up, ids, rows, 1.7)
    check_grad(embed, up, ids.int(), rows)


@pytest.mark.parametrize("n", [511, 512, 2047, 2048, 2049, 20011, 70001])
@pytest.mark.parametrize("kind", ["one", "two", "power", "last", "none"])
def test_grad_distributions(embed, n, kind):
    """Every id the same row, two rows, a power law, the table's last row, no valid id."""
    rows, dim = 3001, 40
    g = gen(n)
    up = normal(g, n, dim, t=torch.bfloat16)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = {"one": torch.full((n,), 17, device="cuda"), "two": (u < 0.3).long() * 2999,
           "power": (torch.exp(u * math.log(rows + 1.0)) - 1).long().clamp(max=rows - 1),
           "last": torch.full((n,), rows - 1, device="cuda"),
           "none": torch.where(u < 0.5, -1, rows + 5)}[kind]
    got = check_grad(embed, up, ids, rows, 0.5)
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[ids[(ids >= 0) & (ids < rows)]] = True
    assert (got[~hit] == 0).all()


def test_grad_wide_table(embed):
    """More rows than one radix pass tells apart, and than 2^22."""
    for rows in (2047, 2048, 2049, 3_000_000, 4_200_000):
        for n in (9000, 300):
            g = gen(rows)
            ids = torch.randint(0, rows, (n,), generator=g, device="cuda")
            ids[::3] = ids[0]
            check_grad(embed, normal(g, n, 4), ids, rows)


def test_grad_strides_and_empty(embed):
    g = gen(8)
    ids = torch.randint(0, 30, (4, 25), generator=g, device="cuda")
    wide = normal(g, 4, 25, 64, t=torch.bfloat16)
    check_grad(embed, wide[..., 5:50], ids, 30)
    check_grad(embed, normal(g, 1, 1, 16).expand(4, 25, 16), ids, 30)
    assert (embed.embedding_grad(wide[:0], ids[:0], 9) == 0).all()
    assert embed.embedding_grad(wide, ids, 0).shape == (0, 64)
    out = torch.full((30, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    assert embed.embedding_grad(wide, ids, 30, out=out) is out
    assert torch.equal(out, embed.embedding_grad(wide, ids, 30))


def test_lookup_autograd_matches_differences(embed):
    g = gen(5)
    table = normal(g, 40, 12).requires_grad_()
    ids = torch.tensor([3, 3, 39, -1, 0], device="cuda")
    weight = normal(g, 5, 12)
    y = embed.embedding_lookup(table, ids, 3.0)
    (y * weight).sum().backward()
    want, err = grad_ref(weight, ids, 40, 3.0)
    assert_within(table.grad, want, err + want.abs() * 2 * U)
    # the loss is linear in the table: a difference is the gradient up to the sums' rounding
    step = normal(g, 40, 12)
    with torch.no_grad():
        l0 = (embed.embedding_lookup(table, ids, 3.0).double() * weight.double()).sum()
        l1 = (embed.embedding_lookup(table + step, ids, 3.0).double() * weight.double()).sum()
    slope = (table.grad.double() * step.double()).sum()
    mass = float((want.abs() * (table.detach().abs() + step.abs()).double()).sum())
    assert abs(float(l1 - l0 - slope)) <= 8 * U * mass


# ---- linear ----------------------------------------------------------------------------------------

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def act_ref(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def act_error(z, t):
    """What evaluating an activation or its derivative may add, per unit of |z| or 1: the 16-bit
    forms use a 1.5e-7 formula and fast exponentials (relative error up to 2^-21 + 2^-22 |x|, with
    |x| at most about 90 where the result is not negligible); float32 a few ulp."""
    return 2.0 ** -15 if t != torch.float32 else 2.0 ** -20


def linear_ref(x, w, b, r, act, t):
    """y, its bound before the last rounding, z and z's bound, in 64 bits."""
    k = x.shape[1]
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    mass = xd.abs() @ wd.abs().t()
    zerr = mass * (k + 8) * 2 * U
    if b is not None:
        z = z + b.double()
        zerr = zerr + (mass + b.double().abs()) * 2 * U
    y = act_ref(z, act)
    yerr = 1.13 * zerr  # the steepest slope of the activations
    if act not in ("none", "relu"):
        yerr = yerr + z.abs() * act_error(z, t)
    if r is not None:
        y = y + r.double()
        yerr = yerr + (y.abs() + r.double().abs()) * 2 * U
    return y, yerr, z, zerr


def make(seed, m, k, n, t, bias=True, residual=True, scale=1.0):
    g = gen(seed)
    x = normal(g, m, k, t=t, scale=scale)
    w = normal(g, n, k, t=t, scale=k ** -0.5)
    b = normal(g, n, t=t, scale=0.2) if bias else None
    r = normal(g, m, n, t=t) if residual else None
    return x, w, b, r


def check_linear(embed, x, w, b, r, act, out_dtype=None):
    t = x.dtype
    got = embed.linear(x, w, b, residual=r, activation=act, out_dtype=out_dtype)
    y, yerr, _, _ = linear_ref(x, w, b, r, act, t)
    ot = out_dtype or t
    assert got.dtype == ot
    assert_within(got, y, yerr + (y.abs() + yerr) * half_step(ot) + TINY[ot])
    return got


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 768, 768), (2, 100, 33), (7, 257, 130),
                                   (8, 64, 64), (9, 64, 64), (127, 100, 100), (128, 128, 128),
                                   (129, 65, 257), (300, 768, 96), (1000, 33, 7)])
def test_linear(embed, t, m, k, n):
    x, w, b, r = make(m + k + n, m, k, n, TYPES[t])
    check_linear(embed, x, w, b, r, "gelu")
    check_linear(embed, x, w, None, None, "none")


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [3, 200])
def test_linear_activations(embed, t, act, m):
    x, w, b, r = make(7, m, 72, 80, TYPES[t], scale=3.0)
    check_linear(embed, x, w, b, r, act)
    check_linear(embed, x, w, b, None, act, torch.float32)
    check_linear(embed, x, w, None, r, act)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(64, 8192, 128), (40, 4096, 520), (2500, 256, 1100),
                                   (5000, 1024, 264), (6000, 16500, 520), (9000, 20000, 256)])
def test_linear_splits_and_waves(embed, t, m, k, n):
    """Long sums split over several blocks, and more tiles than the GPU holds at once."""
    x, w, b, r = make(9, m, k, n, TYPES[t])
    got = check_linear(embed, x, w, b, r, "silu")
    assert torch.equal(got, embed.linear(x, w, b, residual=r, activation="silu"))


def test_linear_shapes_and_strides(embed):
    for t in TYPES.values():
        g = gen(11)
        x = normal(g, 3, 50, 96, t=t)
        w = normal(g, 70, 96, t=t, scale=0.1)
        flat = embed.linear(x.reshape(150, 96), w)
        assert torch.equal(embed.linear(x, w), flat.view(3, 50, 70))
        # windows at odd offsets, padded rows, a transposed weight
        xw, ww = normal(g, 150, 131, t=t), normal(g, 70, 203, t=t, scale=0.1)
        for a, b in ((1, 2), (8, 16), (4, 4)):
            check_linear(embed, xw[:, a:a + 96], ww[:, b:b + 96], None, None, "none")
        check_linear(embed, x[0], normal(g, 96, 70, t=t, scale=0.1).t(), None, None, "none")
        # one residual row for all, and a strided residual
        row = normal(g, 1, 70, t=t)
        check_linear(embed, x[0], w, None, row.expand(50, 70), "relu")
        check_linear(embed, x[0], w, None, normal(g, 50, 99, t=t)[:, 7:77], "relu")
        check_linear(embed, x[0, :1], w, None, row, "relu")
        assert embed.linear(x[:, :0], w).shape == (3, 0, 70)
        out = torch.empty(50, 70, dtype=t, device="cuda")
        assert embed.linear(x[0], w, out=out) is out
        assert torch.equal(out, embed.linear(x[0], w))


def test_linear_float32_ranges(embed):
    """Rows of very different magnitudes, up to float32's ends: each row keeps float32's accuracy
    relative to its own largest element."""
    g = gen(23)
    m, k, n = 200, 80, 72
    for xs, ws in ((120, -110), (-120, 100), (0, -126), (-126, 126), (60, 60)):
        x = normal(g, m, k) * 2.0 ** torch.linspace(xs - 6, xs, m, device="cuda")[:, None]
        w = normal(g, n, k) * 2.0 ** torch.linspace(ws - 4, ws - 2, n, device="cuda")[:, None]
        x[5], w[7] = 0, 0
        want = x.double() @ w.double().t()
        bound = (x.double().abs() @ w.double().abs().t()) * (k + 8) * 2 * U \
            + x.double().abs().amax(1, keepdim=True) * w.double().abs().sum(1) * 2.0 ** -38 \
            + x.double().abs().sum(1, keepdim=True) * w.double().abs().amax(1) * 2.0 ** -38 \
            + TINY[torch.float32]
        got = embed.linear(x, w)
        top = torch.finfo(torch.float32).max
        inside = (want.abs() + bound) < top
        assert_within(got[inside], want[inside], bound[inside])
        assert (got[want.abs() > top * 1.01].isinf()).all()


def test_linear_special_values(embed):
    """A row holding NaN or infinity leaves the other rows alone; magnitudes at the types' ends."""
    for t in TYPES.values():
        for m in (4, 140):
            x, w, b, _ = make(21, m, 64, 72, t, residual=False)
            clean = embed.linear(x, w, b, activation="relu")
            x = x.clone()
            x[1, 5] = math.nan
            x[3, 6] = math.inf
            got = embed.linear(x, w, b, activation="relu")
            assert got[1].isnan().all()
            # an infinite sum is +inf, ReLU's 0 or, for float32 parts, NaN
            assert (got[3].isnan() | got[3].isinf() | (got[3] == 0)).all()
            keep = torch.ones(m, dtype=torch.bool, device="cuda")
            keep[[1, 3]] = False
            assert torch.equal(got[keep], clean[keep])
            # gradients: the NaN row's dx is NaN, an infinite z has a finite derivative
            dy = normal(gen(22), m, 72, t=t)
            for act in ACTS[1:]:
                z = normal(gen(23), m, 72, t=t)
                clean = embed.linear_grad(dy, x, w, z, act, need=(True, False, False))[0]
                z[1, 3], z[2, 4], z[3, 5] = math.nan, math.inf, -math.inf
                z[0, 6], z[0, 7] = 6e4, -6e4
                dx = embed.linear_grad(dy, x, w, z, act, need=(True, False, False))[0]
                assert dx[1].isnan().all() and dx[[0, 2, 3]].isfinite().all()
                assert torch.equal(dx[4:], clean[4:])
                one = torch.zeros(m, 72, device="cuda", dtype=t)
                one[2, 4] = one[3, 5] = one[0, 6] = one[0, 7] = 1
                db = embed.linear_grad(one, x, w, z, act, need=(False, False, True))[2]
                assert db[[4, 6]].tolist() == [1, 1] and db[[5, 7]].abs().max() <= 2.0 ** -100
    big = torch.full((130, 64), torch.finfo(torch.float32).max, device="cuda")
    eye = torch.eye(64, device="cuda")
    assert torch.equal(embed.linear(big, eye), big)
    for act in ACTS:  # far tails
        z = torch.tensor([-300.0, -90.0, -20.0, 0.0, 20.0, 90.0, 300.0], device="cuda")
        for t in TYPES.values():
            for m in (1, 20):
                x = torch.zeros(m, 16, device="cuda", dtype=t)
                got = embed.linear(x, torch.zeros(7, 16, device="cuda", dtype=t), z.to(t),
                                   activation=act)
                want = act_ref(z.to(t).double(), act).expand(m, 7)
                assert_within(got, want, want.abs() * (half_step(t) + 4 * U) + 2.0 ** -20)


# ---- gradients of linear --------------------------------------------------------------------------

SLOPE2 = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.85, "silu": 0.5}  # max |act''|


def grads_ref(x, w, b, dy, act):
    """Gradients with elementwise bounds, in 64 bits, by autograd of the definition."""
    t = x.dtype
    h = half_step(t)
    m, k = x.shape
    n = w.shape[0]
    _, _, z, zerr = linear_ref(x, w, b, None, act, t)
    zz = z.clone().requires_grad_()
    (d1,) = torch.autograd.grad(act_ref(zz, act).sum(), zz)
    dyd = dy.double()
    dz = dyd * d1
    # the stored z is rounded once; act' follows with its largest slope
    zoff = zerr + (z.abs() + zerr) * h + TINY[t]
    derr = dyd.abs() * (SLOPE2[act] * zoff + (0 if act in ("none", "relu") else
                                              act_error(z, t) * (1 + z.abs())))
    if act == "relu":
        derr = derr + dyd.abs() * (z.abs() <= zoff)
    derr = derr + dz.abs() * 2 * U
    # the products see dz rounded to 16 bits (float32: parts that lose 2^-24)
    perr = derr + (dz.abs() + derr) * (h if t != torch.float32 else 2 * U) + TINY[t]
    xd, wd = x.double(), w.double()
    dx = dz @ wd
    dxe = perr @ wd.abs() + (dz.abs() + perr) @ wd.abs() * (n + 8) * 2 * U
    dw = dz.t() @ xd
    dwe = perr.t() @ xd.abs() + (dz.abs() + perr).t() @ xd.abs() * (m + 8) * 2 * U
    db = dz.sum(0)
    dbe = derr.sum(0) + (dz.abs() + derr).sum(0) * (m + 8) * U
    fin = lambda v, e: e + (v.abs() + e) * h + TINY[t]  # noqa: E731
    return (dx, fin(dx, dxe)), (dw, fin(dw, dwe)), (db, fin(db, dbe))


def check_grads(embed, x, w, b, r, dy, act):
    leaves = [v.clone().requires_grad_() if v is not None else None for v in (x, w, b, r)]
    y = embed.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
    held = [v for v in leaves if v is not None]
    got = dict(zip([i for i, v in enumerate(leaves) if v is not None],
                   torch.autograd.grad(y, held, dy)))
    want = grads_ref(x, w, b, dy, act)
    for i, name in enumerate(("dx", "dw", "db")):
        if i in got:
            assert got[i].dtype == x.dtype
            assert_within(got[i], want[i][0], want[i][1], name)
    if 3 in got:
        assert torch.equal(got[3], dy)
    return got


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 40), (5, 100, 100), (130, 100, 100),
                                   (257, 65, 130), (1000, 128, 264), (3000, 40, 56),
                                   (64, 1024, 72)])
def test_linear_gradients(embed, t, m, k, n):
    x, w, b, r = make(m * 3 + k + n, m, k, n, TYPES[t])
    dy = normal(gen(m), m, n, t=TYPES[t], scale=0.1)
    check_grads(embed, x, w, b, r, dy, "gelu")
    check_grads(embed, x, w, None, None, dy, "none")


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("act", ACTS)
def test_linear_gradient_activations(embed, t, act):
    x, w, b, r = make(31, 150, 48, 72, TYPES[t], scale=2.0)
    dy = normal(gen(1), 150, 72, t=TYPES[t])
    got = check_grads(embed, x, w, b, r, dy, act)
    again = check_grads(embed, x, w, b, r, dy, act)
    for i in got:
        assert torch.equal(got[i], again[i])


def test_linear_gradient_differences(embed):
    """Central differences of the 64-bit definition agree with the float32 gradients."""
    x, w, b, _ = make(41, 20, 24, 16, torch.float32, residual=False)
    for act in ("gelu", "gelu_tanh", "silu"):
        dy = normal(gen(2), 20, 16)
        leaves = [v.clone().requires_grad_() for v in (x, w, b)]
        grads = torch.autograd.grad(embed.linear(*leaves, activation=act), leaves, dy)
        for i, (leaf, grad) in enumerate(zip((x, w, b), grads)):
            step = normal(gen(50 + i), *leaf.shape).double()
            h = 1e-4

            def loss(s):
                v = [u.double() for u in (x, w, b)]
                v[i] = v[i] + s * step
                return (act_ref(v[0] @ v[1].t() + v[2], act) * dy.double()).sum()

            slope = float((loss(h) - loss(-h)) / (2 * h))
            got = float((grad.double() * step).sum())
            # h^2 / 6 times a third derivative of order 10 per unit step, and float32 gradients
            mass = float((grad.double().abs() * step.abs()).sum())
            assert abs(got - slope) <= mass * 2.0 ** -16 + h * h * 1e3


def test_linear_grad_parts_and_strides(embed):
    for t in TYPES.values():
        x, w, b, _ = make(51, 60, 40, 48, t, residual=False)
        dy = normal(gen(3), 60, 48, t=t)
        y, z = embed.linear_preact(x, w, b, activation="silu")
        assert torch.equal(y, embed.linear(x, w, b, activation="silu"))
        full = embed.linear_grad(dy, x, w, z, "silu")
        for need in ((True, False, False), (False, True, False), (False, False, True),
                     (True, False, True)):
            part = embed.linear_grad(dy, x, w, z, "silu", need=need)
            for p, f, want in zip(part, full, need):
                assert (p is None) == (not want)
                assert p is None or torch.equal(p, f)
        # strided and broadcast gradients, three-dimensional inputs
        wide = normal(gen(4), 60, 70, t=t)
        for gy in (wide[:, 5:53], wide[:1, :48].expand(60, 48), wide[:, :1].expand(60, 48)):
            a = embed.linear_grad(gy, x, w, z, "silu")
            c = embed.linear_grad(gy.contiguous(), x, w, z, "silu")
            for p, q in zip(a, c):
                assert torch.equal(p, q)
        a = embed.linear_grad(dy.view(3, 20, 48), x.view(3, 20, 40), w, z.view(3, 20, 48), "silu")
        assert a[0].shape == (3, 20, 40) and torch.equal(a[1], full[1])
        # no rows
        e = embed.linear_grad(dy[:0], x[:0], w)
        assert e[0].shape == (0, 40) and (e[1] == 0).all() and (e[2] == 0).all()
    # a float32 result's gradient is taken in the inputs' type
    x, w, b, _ = make(52, 20, 32, 32, torch.bfloat16, residual=False)
    x.requires_grad_()
    embed.linear(x, w, b, out_dtype=torch.float32).sum().backward()
    assert x.grad.dtype == torch.bfloat16


def test_broadcast_residual_gradient(embed):
    x, w, _, _ = make(61, 30, 16, 24, torch.float32)
    row = normal(gen(6), 24).requires_grad_()
    dy = normal(gen(7), 30, 24)
    y = embed.linear(x, w, residual=row.expand(30, 24))
    (g,) = torch.autograd.grad(y, row, dy)
    want = dy.double().sum(0)
    assert_within(g, want, dy.double().abs().sum(0) * 30 * U)


# ---- with the index --------------------------------------------------------------------------------


def test_flat_lookup_and_adapter(gpu, embed):
    g = gen(71)
    base = normal(g, 500, 48)
    ix = gpu.FlatIndex(48, "cosine")
    ix.add_device(base)
    ids = torch.tensor([0, 499, -1, 500, 7], device="cuda")
    got = ix.lookup_device(ids)
    stored = torch.from_numpy(ix.rows()[0]).cuda()
    assert torch.equal(got[0], stored[0]) and torch.equal(got[1], stored[499])
    assert (got[2] == 0).all() and got[3].isnan().all() and torch.equal(got[4], stored[7])
    # tokens -> table -> adapter -> index -> neighbours' vectors: the run of an encoder
    table = normal(g, 300, 32, t=torch.bfloat16)
    w = normal(g, 48, 32, t=torch.bfloat16, scale=32 ** -0.5)
    adapter = embed.Adapter(w, normal(g, 48, t=torch.bfloat16), activation="gelu")
    items = embed.embedding_lookup(table, torch.arange(300, device="cuda"), 32 ** 0.5)
    ax = gpu.FlatIndex(48, "l2")
    ax.add_device(items, adapter=adapter)
    assert torch.equal(torch.from_numpy(ax.rows()[0]).cuda(), adapter(items))
    query = embed.embedding_lookup(table, torch.tensor([5, 250], device="cuda"), 32 ** 0.5)
    dist, label = ax.search_device(query, 3, adapter=adapter)
    assert label[:, 0].tolist() == [5, 250] and dist.shape == (2, 3)
    d2, l2 = ax.search_device(adapter(query), 3)
    assert torch.equal(dist, d2) and torch.equal(label, l2)
    near = ax.lookup_device(label, 0.5)
    assert near.shape == (2, 3, 48) and torch.equal(near[0, 0], ax.lookup_device(label[0, :1])[0] / 2)


def test_flat_adapter_on_a_side_stream(gpu, embed, tmp_path):
    """The map and the add or search that takes it run on one stream, PyTorch's current one."""
    g = gen(72)
    w = normal(g, 64, 512, t=torch.bfloat16, scale=512 ** -0.5)
    adapter = embed.Adapter(w)
    x = normal(g, 40_000, 512, t=torch.bfloat16)
    want = adapter(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = x * 1  # work ahead of the map on the same stream
        for _ in range(20):
            y = y * 1
        ix = gpu.FlatIndex(64, "l2")
        ix.add_device(y, adapter=adapter)
        dist, label = ix.search_device(y[:50] * 1, 1, adapter=adapter)
    side.synchronize()
    assert torch.equal(torch.from_numpy(ix.rows()[0]).cuda(), want)
    # The query batch and the row batch may sum in different orders: each element is off by at most
    # yerr + half a float32 step in both, the squared distance by the squares of twice that (and its
    # own 64 roundings).
    ref, yerr, _, _ = linear_ref(x[:50], w, None, None, "none", torch.float32)
    off = 2 * (yerr + ref.abs() * U)
    assert (dist[:, 0].double() <= (off * off).sum(1) * (1 + 2.0 ** -16)).all()
    assert label[:, 0].tolist() == list(range(50))
    assert torch.equal(ix.lookup_device(label[:, 0]), want[label[:, 0]])
    path = str(tmp_path / "a.qvr")
    ix.save(path)
    again = gpu.FlatIndex.load(path)
    assert torch.equal(again.lookup_device(label[:, 0].int()), want[label[:, 0]])
    for bad in (label.cpu(), label.float()):
        with pytest.raises(ValueError):
            ix.lookup_device(bad)
    with pytest.raises(ValueError):
        ix.search_device(x, 1)
    with pytest.raises(ValueError):
        ix.search_device(want[:3], 0)


# ---- streams, graphs, threads, refusals -------------------------------------------------------------


def test_streams_and_graph(embed):
    """The same bits on a side stream and from a replayed graph with new inputs, two graphs alive."""
    g = gen(81)
    table = normal(g, 900, 64, t=torch.bfloat16)
    x, w, b, r = make(82, 150, 64, 64, torch.float32)

    def step(ids, x, dy):
        e = embed.embedding_lookup(table, ids, 8.0)
        eg = embed.embedding_grad(e, ids, 900, 8.0)
        y, z = embed.linear_preact(x, w, b, residual=r, activation="gelu")
        return (e, eg, y) + embed.linear_grad(dy, x, w, z, "gelu")

    def inputs(seed):
        g = gen(seed)
        return (torch.randint(-1, 900, (3000,), generator=g, device="cuda"),
                normal(g, 150, 64), normal(g, 150, 64))

    want = [step(*inputs(s)) for s in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*inputs(1))
    side.synchronize()
    for p, q in zip(got, want[0]):
        assert torch.equal(p, q)
    graphs = []
    for _ in range(2):
        held = [v.clone() for v in inputs(1)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(*held)
        graphs.append((graph, held, res))
    for s in (0, 1):
        for graph, held, _ in graphs:
            for h, v in zip(held, inputs(s + 1)):
                h.copy_(v)
            graph.replay()
        torch.cuda.synchronize()
        for _, _, res in graphs:
            for p, q in zip(res, want[s]):
                assert torch.equal(p, q)


def test_captured_training_step(embed):
    """A step with autograd, captured after a warm-up on a side stream and replayed on new inputs."""
    table = normal(gen(1), 500, 64, t=torch.bfloat16).requires_grad_()
    x0, w, b, _ = make(2, 300, 64, 64, torch.bfloat16, residual=False)
    w.requires_grad_(), b.requires_grad_()
    ids = torch.zeros(300, dtype=torch.long, device="cuda")
    dy = torch.zeros(300, 64, dtype=torch.bfloat16, device="cuda")

    def step():
        e = embed.embedding_lookup(table, ids, 8.0)
        y = embed.linear(e, w, b, residual=e, activation="silu")
        return [y.detach()] + list(torch.autograd.grad(y, (table, w, b), dy))

    def fill(seed):
        g = gen(seed)
        ids.copy_(torch.randint(-1, 500, (300,), generator=g, device="cuda"))
        dy.copy_(normal(g, 300, 64, t=torch.bfloat16))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (5, 6):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [v.clone() for v in got]
        for p, q in zip(replayed, step()):
            assert torch.equal(p, q)


def test_threads(embed):
    import threading
    x, w, b, r = make(91, 500, 96, 100, torch.float32)
    ids = torch.randint(0, 700, (6000,), generator=gen(92), device="cuda")
    up = normal(gen(93), 6000, 32)
    want = (embed.linear(x, w, b, residual=r), embed.embedding_grad(up, ids, 700))
    torch.cuda.synchronize()
    bad = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = (embed.linear(x, w, b, residual=r), embed.embedding_grad(up, ids, 700))
                s.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(got, want)):
                    bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_rows_behind_the_result_stay(embed):
    """Strided results through the C ABI: what lies between and behind the rows is not written."""
    import ctypes as C
    from quiver_b200 import _native
    lib = _native.lib()
    g = gen(95)
    st = torch.cuda.current_stream().cuda_stream
    for m in (3, 140):
        x, w, _, _ = make(96, m, 64, 40, torch.bfloat16)
        buf = torch.full((m + 2, 64), 5.0, device="cuda", dtype=torch.bfloat16)
        a = _native.qv_linear(2, 2, 0, m, 40, 64, x.data_ptr(), 64, w.data_ptr(), 64)
        a.out, a.out_stride = buf.data_ptr(), 64
        size = C.c_size_t()
        _native.check(lib.qv_linear_workspace(0, C.byref(a), C.byref(size)))
        ws = torch.empty(size.value + 256, dtype=torch.uint8, device="cuda")
        _native.check(lib.qv_linear_device(0, C.byref(a), ws.data_ptr(), size.value, st))
        assert torch.equal(buf[:m, :40], embed.linear(x, w))
        assert (buf[:m, 40:] == 5).all() and (buf[m:] == 5).all()
    ids = torch.randint(0, 30, (5000,), generator=g, device="cuda")
    up = normal(g, 5000, 24)
    buf = torch.full((33, 32), 5.0, device="cuda")
    _native.check(lib.qv_embedding_grad_workspace(5000, 30, 24, C.byref(size)))
    ws = torch.full((size.value + 256,), 77, dtype=torch.uint8, device="cuda")
    _native.check(lib.qv_embedding_grad_device(0, 0, up.data_ptr(), 24, 1, ids.data_ptr(), 5000,
                                               30, 24, 1.0, buf.data_ptr(), 32, ws.data_ptr(),
                                               size.value, st))
    assert torch.equal(buf[:30, :24], embed.embedding_grad(up, ids, 30))
    assert (buf[:30, 24:] == 5).all() and (buf[30:] == 5).all()
    assert (ws[size.value:] == 77).all()
    out = torch.full((7, 40), 5.0, device="cuda")
    _native.check(lib.qv_embedding_lookup_device(0, 0, up.data_ptr(), 5000, 24, 24, 1,
                                                 ids.data_ptr(), 5, 1.0, out.data_ptr(), 40, st))
    assert torch.equal(out[:5, :24], up[ids[:5]])
    assert (out[:5, 24:] == 5).all() and (out[5:] == 5).all()


def test_far_offsets(embed):
    """Tables, results and gradients past 2^31 elements."""
    rows, dim = 4_300_000, 512
    table = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, rows - 1, 4_194_304, rows - 1], device="cuda")
    g = gen(98)
    mark = normal(g, 3, dim, t=torch.bfloat16)
    table[ids[:3]] = mark
    assert torch.equal(embed.embedding_lookup(table, ids), mark[[0, 1, 2, 1]])
    many = torch.arange(rows, device="cuda").flip(0)
    got = embed.embedding_lookup(table, many)
    assert torch.equal(got[[rows - 1, 0, rows - 1 - 4_194_304]], mark)
    del got
    up = normal(g, 4, dim, t=torch.bfloat16)
    grad = embed.embedding_grad(up, ids, rows)
    assert torch.equal(grad[ids[[0, 2]]], up[[0, 2]])
    assert torch.equal(grad[rows - 1], (up[1].float() + up[3].float()).bfloat16())
    assert int((grad != 0).any(1).sum()) == 3
    del grad
    # the table as upstream rows: few targets, the same sums
    target = (many % 3).int()
    grad = embed.embedding_grad(table, target, 3)
    want = torch.zeros(3, dim, dtype=torch.float64, device="cuda")
    want.index_add_(0, target[ids[:3]].long(), mark.double())
    assert_within(grad, want, want.abs() * half_step(torch.bfloat16) + 2.0 ** -12)
    del table, grad, many, target
    # a result past 2^31 elements, and its gradients
    m, n = 2_200_000, 1024
    x = normal(g, m, 16, t=torch.bfloat16)
    w = normal(g, n, 16, t=torch.bfloat16)
    y = embed.linear(x, w, activation="relu")
    tail = slice(m - 300, m)
    assert torch.equal(y[tail], embed.linear(x[tail], w, activation="relu"))
    dx, dw, _ = embed.linear_grad(y, x, w, need=(True, True, False))
    want = y[tail].double() @ w.double()
    mass = y[tail].double().abs() @ w.double().abs()
    assert_within(dx[tail], want, want.abs() * half_step(torch.bfloat16) + mass * 1032 * 2 * U)
    part = torch.zeros(n, 16, dtype=torch.float64, device="cuda")
    for i in range(0, m, 100_000):
        part += y[i:i + 100_000].double().t() @ x[i:i + 100_000].double()
    # every partial sum is cut at most once per 16 terms, at 2^-23 of its magnitude
    mass = torch.zeros_like(part)
    for i in range(0, m, 100_000):
        mass += y[i:i + 100_000].double().t() @ x[i:i + 100_000].double().abs()
    assert_within(dw, part, part.abs() * half_step(torch.bfloat16) + mass * 1024 * 2 * U)


@pytest.mark.parametrize("m,k,n,t", [(2000, 512, 512, "bf16"), (8192, 1024, 1024, "bf16"),
                                     (600, 512, 300, "f32"), (6000, 512, 768, "f32")])
def test_wait_limit_runs_out(embed, monkeypatch, m, k, n, t):
    """A pipeline wait that runs out marks its results NaN; the next call is right again. (Single
    blocks and pairs of them, sums of one chunk and of several.)"""
    x, w, _, _ = make(99, m, k, n, TYPES[t])
    want = embed.linear(x, w)
    r = normal(gen(1), m, n, t=TYPES[t])
    monkeypatch.setenv("QV_TC_WAIT_LIMIT_US", "1")
    for res in (None, r):
        got = embed.linear(x, w, residual=res)
        ref = want if res is None else embed.linear(x, w, residual=res)
        torch.cuda.synchronize()
        ok = got.isnan() | ref.isnan() | (got == ref)
        assert ok.all()
    monkeypatch.delenv("QV_TC_WAIT_LIMIT_US")
    assert torch.equal(embed.linear(x, w), want)


def test_bad_device_leaves_no_error(embed):
    import ctypes as C
    from quiver_b200 import _native
    lib = _native.lib()
    t = torch.ones(4, 8, device="cuda")
    ids = torch.zeros(2, dtype=torch.long, device="cuda")
    out = torch.empty(2, 8, device="cuda")
    with pytest.raises(RuntimeError):
        _native.check(lib.qv_embedding_lookup_device(97, 0, t.data_ptr(), 4, 8, 8, 1,
                                                     ids.data_ptr(), 2, 1.0, out.data_ptr(), 8,
                                                     C.c_void_p(0)))
    assert torch.equal(embed.embedding_lookup(t, ids), t[:2])


def test_refusals(embed):
    x, w, b, r = make(97, 20, 16, 24, torch.float32)
    ids = torch.zeros(3, dtype=torch.long, device="cuda")
    E = ValueError
    for f in (lambda: embed.linear(x.cpu(), w), lambda: embed.linear(x, w.half()),
              lambda: embed.linear(x, w[:, :8]), lambda: embed.linear(x, w, b[:5]),
              lambda: embed.linear(x, w, residual=r[:, :5]),
              lambda: embed.linear(x, w, activation="tanh"),
              lambda: embed.linear(x, w, out_dtype=torch.float16),
              lambda: embed.linear(x.double(), w.double()),
              lambda: embed.linear(x, w, out=r.t()),
              lambda: embed.linear_grad(r, x, w, None, "gelu"),
              lambda: embed.linear_grad(r[:, :3], x, w),
              lambda: embed.embedding_lookup(w, ids.float()),
              lambda: embed.embedding_lookup(w, ids.cpu()),
              lambda: embed.embedding_lookup(w[0], ids),
              lambda: embed.embedding_lookup(w.int(), ids),
              lambda: embed.embedding_grad(x, ids, 5),
              lambda: embed.embedding_grad(x[:3], ids, -1),
              lambda: embed.embedding_grad(x[:3], ids, 2 ** 31),
              lambda: embed.Adapter(w, b, residual=True),
              lambda: embed.linear(x, x[:16], out=x[:, :].view(20, 16)),
              lambda: embed.linear(x, w, residual=r, out=r),
              lambda: embed.embedding_grad(x[:3], ids, 3, out=x[:3]),
              lambda: embed.embedding_lookup(x, ids, out=x[2:5]),
              lambda: embed.Adapter(w, b[:4])):
        with pytest.raises(E):
            f()
