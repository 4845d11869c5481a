"""The token operators (sparse_amd.tokens) against their definitions in 64 bits, at the sizes, masks and layouts where they
can go wrong.

Tolerances.  A result is a 32-bit sum rounded once to its type: with u = 2^-24, a sum of k products is off by at most
(k + 2) u times the sum of their magnitudes (each product and each addition rounds once; the factor scale * val adds two
roundings), and the last step by half a step of the type, eps / 2 relative, or half its smallest subnormal."""
import itertools

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
NAN = float("nan")


@pytest.fixture(scope="module")
def ctx():
    from sparse_amd import Context
    c = Context(0)
    yield c
    c.sync()


@pytest.fixture(scope="module")
def tk(ctx):
    from sparse_amd import mk_tokens
    made = {}

    def get(t):
        if t not in made:
            made[t] = mk_tokens(t, ctx)
        return made[t]
    return get


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def close(got, want, magnitude, k):
    """got: of its type; want: 64 bits; magnitude: the sum of the magnitudes of the k products behind every value."""
    assert got.shape == want.shape
    half = torch.finfo(got.dtype).eps / 2
    bound = (k + 4) * U * magnitude + half * want.abs() * (1 + 2.0 ** -9) + SMALLEST[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%d of %d values off, worst %.3g of its bound" % (int(bad.sum()), bad.numel(), float((off / bound).max()))


def strided(a, pad, shift):
    """The same values in rows `pad` elements further apart, the first `shift` elements into the memory; NaN around them."""
    n, d = a.shape
    base = torch.full((n * (d + pad) + shift,), NAN, dtype=a.dtype, device="cuda")
    v = base[shift:].as_strided((n, d), (d + pad, 1))
    v.copy_(a)
    return v


# ------------------------------------------------------------------------------------------------ lookup
def lookup_ref(E, ids, f):
    ids = ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < E.shape[0])
    return torch.where(ok[:, None], E.double()[torch.where(ok, ids, 0)] * f.reshape(-1, 1), 0.0)


def make_ids(g, n, V, kind, bits):
    if kind == "uniform":
        ids = torch.randint(0, V, (n,), generator=g, device="cuda")
    elif kind == "one":
        ids = torch.full((n,), V // 2, device="cuda")
    elif kind == "skew":
        ids = ((V + 1) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64) - 1).long().clamp(0, V - 1)
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.3, torch.full_like(ids, -1), ids)
    elif kind == "none":
        ids = torch.full((n,), -1, device="cuda")
    else:                                                          # "wild": far out of range on both sides
        ids = torch.randint(-3 * V, 3 * V, (n,), generator=g, device="cuda")
        if bits == 64 and n > 3:
            ids[0], ids[1], ids[2] = 2 ** 40, -2 ** 40, 2 ** 32    # low 32 bits of the last: a valid id
    return ids.to(torch.int64 if bits == 64 else torch.int32)


LOOKUPS = [(1, 1, 1), (1, 1000, 4096), (3, 7, 5), (64, 100, 8), (63, 33, 64), (129, 5, 65), (17, 300, 511), (5, 40, 513), (300, 1000, 1001),
           (1000, 50, 2048), (2500, 200, 4100), (7, 9, 20000)]


@pytest.mark.parametrize("n,V,D", LOOKUPS)
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_lookup(tk, t, n, V, D):
    g = gen(n * 7 + D)
    E = normal(g, (V, D), DT[t])
    for kind, bits, with_vals, lay in [("uniform", 64, False, 0), ("wild", 32, True, 1), ("skew", 64, True, 2)]:
        ids = make_ids(g, n, V, kind, bits)
        vals = torch.randn(n, generator=g, device="cuda") if with_vals else None
        scale = 1.0 if kind == "uniform" else 3.7
        table = E if lay == 0 else strided(E, 3, 1) if lay == 1 else strided(E, 8, 8)
        y = tk(t).lookup(table, ids, vals=vals, scale=scale)
        f = scale * (vals.double() if with_vals else torch.ones(n, device="cuda", dtype=torch.float64))
        want = lookup_ref(E, ids, f)
        if kind == "uniform":
            assert torch.equal(y, want.to(DT[t]))                  # no factor: the row itself
        else:
            close(y, want, want.abs(), 1)
        out = strided(torch.zeros(n, D, dtype=DT[t], device="cuda"), 5, 3)
        around = out.as_strided((n, D + 5), (D + 5, 1)) if n > 1 else None
        assert tk(t).lookup(table, ids, vals=vals, scale=scale, out=out) is out and torch.equal(out, y)
        if around is not None:
            assert torch.isnan(around[:-1, D:]).all()              # nothing is written between the rows


def test_lookup_keeps_shape_and_special_values(tk):
    E = torch.tensor([[float("inf"), -0.0, 1.0], [NAN, 2.0, -float("inf")], [NAN, NAN, NAN]], device="cuda")
    ids = torch.tensor([[0, 1, -1], [1, 0, 0]], device="cuda")
    y = tk("f32").lookup(E, ids)
    assert y.shape == (2, 3, 3) and torch.equal(y[0, 0], E[0]) and torch.equal(y[0, 2], torch.zeros(3, device="cuda"))
    assert torch.equal(y[0, 1].isnan(), E[1].isnan()) and not y[1, 1].isnan().any()
    assert tk("f32").lookup(E, ids[:0]).shape == (0, 3, 3)


# ------------------------------------------------------------------------------------------------ lookup's gradients
def lookup_grad_ref(dy, ids, V, f):
    ids = ids.reshape(-1).long()
    ok = (ids >= 0) & (ids < V)
    rows = torch.where(ok[:, None], dy.double() * f.reshape(-1, 1), 0.0)
    at = torch.where(ok, ids, 0)
    z = torch.zeros((V, dy.shape[1]), dtype=torch.float64, device="cuda")
    count = torch.bincount(at, weights=ok.double(), minlength=V)
    return z.clone().index_add_(0, at, rows), z.index_add_(0, at, rows.abs()), count[:, None]


GRADS = [(1, 1, 1, "uniform"), (1, 5000, 64, "uniform"), (5, 3, 7, "wild"), (100, 40, 65, "skew"), (300, 17, 1001, "uniform"), (1000, 1, 130, "one"), (256, 1, 40, "one"), (256, 9, 72, "skew"), (257, 9, 72, "skew"), (200, 70000, 8, "skew"), (33, 50, 3001, "uniform"), (100, 20000000, 1, "wild"), (2048, 300, 56, "skew"), (2049, 300, 56, "skew"), (5000, 70, 33, "wild"), (3000, 5000000, 2, "skew"),
         (1025, 700, 520, "wild"), (4096, 300000, 24, "skew"), (4097, 300000, 24, "skew"), (8192, 50, 96, "skew"), (8193, 1000, 40, "skew"), (16384, 1000, 40, "skew"), (16385, 9000, 24, "skew"), (20000, 131072, 64, "skew"),
         (30000, 3, 33, "one"), (600000, 2000, 8, "uniform"), (9000, 100, 16, "none"), (70, 9, 12, "none"), (9000, 3000000, 1, "wild"),
         (2048, 64, 4096, "uniform")]


@pytest.mark.parametrize("n,V,D,kind", GRADS)
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_lookup_grad(tk, t, n, V, D, kind):
    g = gen(n + V + D)
    ids = make_ids(g, n, V, kind, 32 if D % 2 else 64)
    dy = normal(g, (n, D), DT[t])
    vals = torch.randn(n, generator=g, device="cuda") if n % 2 else None
    f = 0.5 * (vals.double() if vals is not None else torch.ones(n, device="cuda", dtype=torch.float64))
    want, magnitude, count = lookup_grad_ref(dy, ids, V, f)
    dead = ((ids < 0) | (ids >= V)).nonzero().reshape(-1)
    rows = strided(dy, 8, 0) if n % 3 else dy
    rows[dead] = NAN                                               # what no id names is not part of any sum
    got = tk(t).lookup_grad(rows, ids, V, vals=vals, scale=0.5)
    close(got, want, magnitude, count)
    assert torch.equal(got, tk(t).lookup_grad(rows, ids, V, vals=vals, scale=0.5))   # the same bits every time
    wide = tk(t).lookup_grad(rows, ids, V, vals=vals, scale=0.5, dtype=torch.float32)
    assert wide.dtype == torch.float32
    close(wide, want, magnitude, count)
    # added to what is there: rows without an id keep their bits (NaN among them)
    for dtype in {DT[t], torch.float32}:
        start = normal(g, (V, D), dtype)
        out = strided(start, 3, 1)
        named = torch.zeros(V, dtype=torch.bool, device="cuda")
        named[ids[(ids >= 0) & (ids < V)].long()] = True
        out[~named] = NAN
        tk(t).lookup_grad(rows, ids, V, vals=vals, scale=0.5, out=out, accumulate=True)
        assert torch.isnan(out[~named]).all()
        s = start.double()
        close(out[named], (want + s)[named], (magnitude + s.abs())[named], (count + 1)[named])


def test_lookup_grad_without_ids_is_zero(tk):
    out = torch.full((50, 9), NAN, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert not tk("f32").lookup_grad(torch.zeros(0, 9, device="cuda"), none, 50, out=out).any()
    out.fill_(2.0)
    tk("f32").lookup_grad(torch.zeros(0, 9, device="cuda"), none, 50, out=out, accumulate=True)
    assert (out == 2.0).all()


@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (37, 10, 64), (130, 9, 1001), (2000, 64, 777)])
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_lookup_vals_grad(tk, t, n, V, D):
    g = gen(n + D)
    E, dy, ids = normal(g, (V, D), DT[t]), normal(g, (n, D), DT[t]), make_ids(g, n, V, "skew", 64)
    got = tk(t).lookup_vals_grad(strided(dy, 2, 1), strided(E, 1, 0), ids, scale=2.5)
    rows = lookup_ref(E, ids, torch.full((n,), 2.5, device="cuda", dtype=torch.float64)) * dy.double()
    close(got, rows.sum(1), rows.abs().sum(1), D)


# ------------------------------------------------------------------------------------------------ routing
def choices(g, n, K, X, drop, kind="uniform", bits=64):
    if kind == "one":
        c = torch.full((n, K), X - 1, device="cuda")
    else:
        c = torch.randint(0, X, (n, K), generator=g, device="cuda")
        if kind == "skew":
            c = (c * torch.rand((n, K), generator=g, device="cuda")).long()
    c = torch.where(torch.rand((n, K), generator=g, device="cuda") < drop, torch.randint(-5, 0, (n, K), generator=g, device="cuda"), c)
    if drop and n > 1 and bits == 64:
        c[0, 0], c[1, 0] = X, 2 ** 32                              # beyond the last expert; low 32 bits: expert 0
    return c.to(torch.int64 if bits == 64 else torch.int32)


def route_ref(c, X):
    flat = c.reshape(-1).cpu().numpy().astype(np.int64)
    key = np.where((flat >= 0) & (flat < X), flat, X)
    order = np.argsort(key, kind="stable")
    live = int((key < X).sum())
    pos = np.full(len(flat), -1)
    pos[order[:live]] = np.arange(live)
    src = np.full(len(flat), -1)
    src[:live] = order[:live]
    return pos.reshape(c.shape), src, np.searchsorted(key[order], np.arange(X + 1))

# nearly all of the result is zeros, whole and with rows apart
@pytest.mark.parametrize("V,D,pad", [(70001, 2048, 0), (40003, 1801, 7)])
def test_few_ids_of_a_large_table(tk, V, D, pad):
    g = gen(V)
    ids = torch.tensor([V - 1, 0, -1, 5, V, 5, V // 2], device="cuda")
    dy = torch.randn((len(ids), D), generator=g, device="cuda")
    base = torch.full((V, D + pad), 7.0, device="cuda")
    out = base[:, :D]
    assert tk("f32").lookup_grad(dy, ids, V, out=out) is out
    want = {V - 1: dy[0], 0: dy[1], 5: dy[3] + dy[5], V // 2: dy[6]}
    for v, row in want.items():
        assert torch.equal(out[v], row)
    out[list(want)] = 0.0
    assert not out.any() and (base[:, D:] == 7.0).all()



ROUTES = [(0, 2, 4), (1, 1, 1), (1, 8, 64), (64, 4, 1024), (65, 4, 3), (256, 4, 256), (1000, 8, 17), (1025, 8, 1000), (4096, 2, 8), (4097, 2, 8), (8192, 2, 64), (8193, 2, 1000), (5461, 3, 1024),
          (30001, 3, 128), (150000, 4, 1024), (600000, 2, 5)]


@pytest.mark.parametrize("n,K,X", ROUTES)
@pytest.mark.parametrize("kind,drop,bits", [("uniform", 0.0, 64), ("skew", 0.3, 32), ("one", 0.0, 64), ("uniform", 1.0, 64), ("uniform", 0.1, 64)])
def test_route(tk, n, K, X, kind, drop, bits):
    c = choices(gen(n + X), n, K, X, drop, kind, bits)
    r = tk("bf16").route(c, X)
    pos, src, offsets = route_ref(c, X)
    assert r.pos.dtype == r.src.dtype == r.offsets.dtype == torch.int32
    assert np.array_equal(r.pos.cpu().numpy(), pos) and np.array_equal(r.src.cpu().numpy(), src) and np.array_equal(r.offsets.cpu().numpy(), offsets)


MOVES = [(1, 1, 1, 1), (1, 3, 2, 4096), (5, 2, 3, 7), (64, 4, 16, 64), (33, 9, 4, 65), (100, 2, 8, 1001), (700, 8, 32, 2048), (3000, 3, 5, 520), (40, 17, 64, 9000)]


@pytest.mark.parametrize("n,K,X,D", MOVES)
@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_dispatch_and_combine_and_their_gradients(tk, t, n, K, X, D):
    g = gen(n + D)
    d = torch.float64
    for drop, lay in [(0.0, 0), (0.35, 1)]:
        r = tk(t).route(choices(g, n, K, X, drop), X)
        live = int(r.offsets[-1])
        x, ys, w = normal(g, (n, D), DT[t]), normal(g, (n * K, D), DT[t]), torch.randn((n, K), generator=g, device="cuda")
        ok = r.pos >= 0
        at = r.pos.clamp(min=0).long()
        w[~ok] = NAN                                               # the weight of a dropped choice is not used
        wz = torch.where(ok, w, 0.0).to(d)
        if lay:
            x, ys = strided(x, 5, 3), strided(ys, 1, 1)
        ys[live:] = NAN                                            # nor is a row behind the last place
        out = torch.full((n * K, D), 7.0, dtype=DT[t], device="cuda")
        out = strided(out, 3, 2) if lay else out
        assert tk(t).dispatch(x, r, out=out) is out
        token = (r.src[:live] // K).long()
        assert torch.equal(out[:live], x[token]) and (out[live:] == 7.0).all()
        factor = w.reshape(-1)[r.src[:live].long()].to(d)
        weighted = tk(t).dispatch(x, r, weights=w)[:live]
        want = x[token].to(d) * factor[:, None]
        close(weighted, want, want.abs(), 1)

        terms = torch.where(ok[..., None], ys[at].to(d) * wz[..., None], 0.0)
        close(tk(t).combine(ys, r, w), terms.sum(1), terms.abs().sum(1), K)
        terms = torch.where(ok[..., None], ys[at].to(d), 0.0)
        close(tk(t).dispatch_grad(ys, r), terms.sum(1), terms.abs().sum(1), K)

        dys, dw = tk(t).combine_grad(x, ys, r, w, out=out)
        assert dys is out and (out[live:] == 7.0).all()
        close(dys[:live], want, want.abs(), 1)
        terms = torch.where(ok[..., None], ys[at].to(d) * x.to(d)[:, None, :], 0.0)
        close(dw, terms.sum(2), terms.abs().sum(2), D)
        assert not dw[~ok].any()


def test_a_token_without_a_place_has_zeros(tk):
    r = tk("f32").route(torch.full((3, 2), -1, device="cuda"), 4)
    ys = torch.full((6, 33), NAN, device="cuda")
    assert not tk("f32").combine(ys, r, torch.full((3, 2), NAN, device="cuda")).any()
    dys, dw = tk("f32").combine_grad(torch.ones(3, 33, device="cuda"), ys, r, torch.ones(3, 2, device="cuda"), out=torch.ones(6, 33, device="cuda"))
    assert (dys == 1).all() and not dw.any()


# ------------------------------------------------------------------------------------------------ experts
#          rows of each expert, dropped choices, D, F
EXPERTS = [([1], 0, 8, 8), ([3], 0, 1, 1), ([0, 0, 5, 0], 2, 64, 64), ([1, 2, 3, 0, 40], 3, 72, 136), ([31, 0, 33, 64, 1], 0, 200, 328),
           ([16, 17, 15] * 5, 1, 128, 256), ([100, 0, 129, 128], 7, 264, 136), ([40, 300, 1, 60], 0, 65, 77), ([5, 2, 9], 1, 1001, 13),
           ([300, 700, 1, 511], 30, 136, 520), ([2000], 0, 512, 264), ([257, 0, 1024], 5, 192, 257), ([900, 300], 9, 515, 384),
           ([700, 500], 0, 64, 15350), ([513, 0, 511], 3, 15360, 72), ([300, 260, 10, 90], 0, 8200, 8192), ([64] * 40, 0, 96, 264),
           ([1] * 200, 0, 64, 128), ([0, 0], 10, 64, 64), ([600], 600, 96, 80)]


def routed(tk, g, counts, dropped):
    """A routing of one choice a row with so many rows for each expert, the choices in a random order."""
    c = torch.cat([torch.full((k,), e, device="cuda", dtype=torch.int64) for e, k in enumerate(counts)] + [torch.full((dropped,), -1, device="cuda", dtype=torch.int64)])
    c = c[torch.randperm(len(c), generator=g, device="cuda")].reshape(-1, 1)
    return tk.route(c, len(counts))


@pytest.mark.parametrize("counts,dropped,D,F", EXPERTS)
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("lay", ["plain", "strided", "unaligned"])
def test_experts_and_their_gradients(tk, t, counts, dropped, D, F, lay):
    g = gen(D + F)
    X, n, live = len(counts), sum(counts) + dropped, sum(counts)
    r = routed(tk(t), g, counts, dropped)
    xs, dys, W = normal(g, (n, D), DT[t]), normal(g, (n, F), DT[t]), normal(g, (X, F, D), DT[t])
    xs[live:], dys[live:] = NAN, NAN                               # rows behind the last place
    x64, g64, w64 = xs.double(), dys.double(), W.double()
    out, out_x = torch.full((n, F), 7.0, dtype=DT[t], device="cuda"), torch.full((n, D), 7.0, dtype=DT[t], device="cuda")
    if lay != "plain":
        pad = 8 if lay == "strided" else 3
        xs, dys = strided(xs, pad, pad), strided(dys, pad, 0)
        out, out_x = strided(out, pad, 0), strided(out_x, pad, pad)
        base = torch.full((X, F + 2, D + pad), NAN, dtype=DT[t], device="cuda")
        base[:, :F, :D] = W
        W = base[:, :F, :D]
    ys, dxs = tk(t).experts(xs, W, r, out=out), tk(t).experts_grad_x(dys, W, r, out=out_x)
    dW = tk(t).experts_grad_w(dys, xs, r)
    wide = tk(t).experts_grad_w(dys, xs, r, dtype=torch.float32)
    start = normal(g, (X, F, D), torch.float32)
    added = tk(t).experts_grad_w(dys, xs, r, out=start.clone(), accumulate=True)
    assert ys is out and (out[live:] == 7.0).all() and (out_x[live:] == 7.0).all()
    at = 0
    for e, k in enumerate(counts):
        a, b, w = x64[at:at + k], g64[at:at + k], w64[e]
        close(ys[at:at + k], a @ w.t(), a.abs() @ w.abs().t(), D)
        close(dxs[at:at + k], b @ w, b.abs() @ w.abs(), F)
        want, magnitude = b.t() @ a, b.abs().t() @ a.abs()
        close(dW[e], want, magnitude, k)
        close(wide[e], want, magnitude, k)
        s = start[e].double()
        close(added[e], want + s, magnitude + s.abs(), k + 1)
        if k == 0:
            assert not dW[e].any() and torch.equal(added[e], start[e])
        at += k

# ------------------------------------------------------------------------------------------------ experts in padded rows
def padded(a, fill=NAN):
    """The same values in rows (of blocks, one more row apart) that begin on 16 bytes, the next multiple of 8 elements long."""
    base = torch.full((*a.shape[:-2], a.shape[-2] + (a.dim() == 3), (a.shape[-1] + 7) // 8 * 8), fill, dtype=a.dtype, device="cuda")
    v = base[..., :a.shape[-2], :a.shape[-1]]
    v.copy_(a)
    return base, v


def untouched(base, v, fill):
    """What lies between the rows and blocks of v, a view of base, is `fill` still."""
    around = torch.ones(base.shape, dtype=torch.bool, device="cuda")
    around[..., :v.shape[-2], :v.shape[-1]] = False
    return bool((base[around] == fill).all())


# The last rows of an operand end inside a piece of 16 bytes, and inside one of 4: nothing of them may be lost.  The experts'
# rows fill the last step of the sums exactly, by one row more and by one less; few and many of them (all tiles of the gradients).
@pytest.mark.parametrize("counts,D,F", [([128, 64, 1, 0, 32], 65, 77), ([127, 129], 68, 257), ([64, 33], 257, 68), ([512, 1024], 130, 77), ([700, 511, 0, 641], 516, 259),
                                        ([300, 1000], 1030, 2049), ([192], 4093, 4090), ([40, 24] * 8, 1027, 515), ([1, 2, 0, 3], 2051, 1025), ([1024, 2048, 1500], 1036, 2044)])
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_experts_of_any_width_in_padded_rows(tk, t, counts, D, F):
    g = gen(D + F)
    X, n = len(counts), sum(counts)
    r = routed(tk(t), g, counts, 0)
    xs, dys, W = (padded(normal(g, shape, DT[t]))[1] for shape in ((n, D), (n, F), (X, F, D)))
    ys, dxs, dW = tk(t).experts(xs, W, r), tk(t).experts_grad_x(dys, W, r), tk(t).experts_grad_w(dys, xs, r)
    at = 0
    for e, k in enumerate(counts):
        a, b, w = xs[at:at + k].double(), dys[at:at + k].double(), W[e].double()
        close(ys[at:at + k], a @ w.t(), a.abs() @ w.abs().t(), D)
        close(dxs[at:at + k], b @ w, b.abs() @ w.abs(), F)
        close(dW[e], b.t() @ a, b.abs().t() @ a.abs(), k)
        at += k


# Every kernel of the gradient by W, into every kind of result.
@pytest.mark.parametrize("counts,D,F", [([20, 0, 7], 72, 136), ([200, 0, 300], 72, 136), ([200, 0, 300, 180], 1040, 1288), ([400, 0, 170], 4096, 2048), ([40, 0, 30], 65, 77),
                                        ([700, 0, 600], 65, 77), ([300, 0, 170], 2051, 1025), ([25, 3, 0, 9], 517, 1026)])
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("lay", ["rows", "padded"])
def test_weight_gradients_into_and_onto_every_result(tk, t, counts, D, F, lay):
    g = gen(D + F)
    X, n = len(counts), sum(counts)
    r = routed(tk(t), g, counts, 0)
    xs, dys = normal(g, (n, D), DT[t]), normal(g, (n, F), DT[t])
    if lay == "padded":
        xs, dys = padded(xs)[1], padded(dys)[1]
    for dtype, add in itertools.product((DT[t], torch.float32), (False, True)):
        start = normal(g, (X, F, D), dtype)
        base, out = padded(start, 3.0) if lay == "padded" else (None, start.clone())
        assert tk(t).experts_grad_w(dys, xs, r, out=out, accumulate=add) is out
        assert base is None or untouched(base, out, 3.0)
        at = 0
        for e, k in enumerate(counts):
            a, b, s = xs[at:at + k].double(), dys[at:at + k].double(), start[e].double() * add
            close(out[e], b.t() @ a + s, b.abs().t() @ a.abs() + s.abs(), k + add)
            if k == 0:
                assert torch.equal(out[e], start[e] if add else torch.zeros_like(start[e]))
            at += k


# many experts, so that the card has more than one round of tiles: a last round of half tiles, sums that begin at another column
# for every expert, results written past the caches
@pytest.mark.parametrize("counts,D,F", [([400, 389, 511, 257] * 5, 2056, 2048), ([20, 100, 130, 64] * 15, 1528, 328), ([3, 0, 1] * 17, 2048, 1032), ([170, 1, 350] * 12, 1032, 2064)])
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_rounds_of_tiles(tk, t, counts, D, F):
    g = gen(D + F + len(counts))
    X, n = len(counts), sum(counts)
    r = routed(tk(t), g, counts, 0)
    xs, dys, W = normal(g, (n, D), DT[t]), normal(g, (n, F), DT[t]), normal(g, (X, F, D), DT[t])
    ys, dxs, dW = tk(t).experts(xs, W, r), tk(t).experts_grad_x(dys, W, r), tk(t).experts_grad_w(dys, xs, r)
    at = 0
    for e, k in enumerate(counts):
        a, b, w = xs[at:at + k].double(), dys[at:at + k].double(), W[e].double()
        close(ys[at:at + k], a @ w.t(), a.abs() @ w.abs().t(), D)
        close(dxs[at:at + k], b @ w, b.abs() @ w.abs(), F)
        close(dW[e], b.t() @ a, b.abs().t() @ a.abs(), k)
        at += k


def test_an_experts_nan_stays_with_it(tk):
    g = gen(3)
    counts = [40, 50, 70]
    r = routed(tk("bf16"), g, counts, 0)
    xs, dys, W = normal(g, (160, 96), DT["bf16"]), normal(g, (160, 80), DT["bf16"]), normal(g, (3, 80, 96), DT["bf16"])
    W[1], xs[40:90], dys[40:90] = NAN, float("inf"), NAN
    for got in (tk("bf16").experts(xs, W, r), tk("bf16").experts_grad_x(dys, W, r)):
        assert torch.isfinite(got[:40]).all() and torch.isfinite(got[90:]).all() and not torch.isfinite(got[40:90]).any()
    dW = tk("bf16").experts_grad_w(dys, xs, r)
    assert torch.isfinite(dW[0]).all() and torch.isfinite(dW[2]).all() and not torch.isfinite(dW[1]).any()


@pytest.mark.parametrize("D,F", [(0, 16), (16, 0), (0, 0)])
def test_products_of_nothing(tk, D, F):
    r = routed(tk("bf16"), gen(1), [3, 0, 2], 1)
    z = lambda *s: torch.zeros(s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    assert not tk("bf16").experts(z(6, D), z(3, F, D), r, out=torch.zeros_like(z(6, F)) + 1)[:5].any()
    assert not tk("bf16").experts_grad_x(z(6, F), z(3, F, D), r, out=z(6, D) + 1)[:5].any()
    assert tk("bf16").experts_grad_w(z(6, F), z(6, D), r).shape == (3, F, D)
    none = tk("bf16").route(torch.zeros(4, 0, device="cuda", dtype=torch.int64), 3)
    assert not none.offsets.any() and not tk("bf16").combine(z(0, 16), none, torch.zeros(4, 0, device="cuda")).any()
    assert tk("bf16").dispatch(z(4, 16), none).shape == (0, 16) and not tk("bf16").experts_grad_w(z(0, 4), z(0, 8), none).any()


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_products_keep_small_values(tk, t):
    """Values below the type's smallest normal one are values too, in and out of the matrix cores."""
    r = routed(tk(t), gen(2), [20, 30], 0)
    small = 2.0 ** -20 if t == "f16" else 2.0 ** -130
    x = torch.full((50, 64), small, device="cuda").to(DT[t])
    assert (x == small).all()
    W = torch.ones(2, 40, 64, device="cuda", dtype=DT[t])
    assert (tk(t).experts(x, W, r) == 64 * small).all()
    assert (tk(t).experts_grad_x(torch.ones(50, 40, device="cuda", dtype=DT[t]), W * x[0, 0], r) == 40 * small).all()


def test_inputs_that_are_one_row_for_all(tk):
    """Expanded rows and blocks: what the gradient of a sum over rows, or experts with the same weights, look like."""
    g, k = gen(4), tk("bf16")
    r = routed(k, g, [40, 3, 90], 2)
    row, W = normal(g, (1, 64), DT["bf16"]), normal(g, (1, 72, 64), DT["bf16"])
    xs, Ws = row.expand(135, 64), W.expand(3, 72, 64)
    assert torch.equal(k.experts(xs, Ws, r)[:133], k.experts(xs.contiguous(), Ws.contiguous(), r)[:133])
    dys = normal(g, (1, 72), DT["bf16"]).expand(135, 72)
    assert torch.equal(k.experts_grad_x(dys, Ws, r)[:133], k.experts_grad_x(dys.contiguous(), Ws.contiguous(), r)[:133])
    assert torch.equal(k.experts_grad_w(dys, xs, r), k.experts_grad_w(dys.contiguous(), xs.contiguous(), r))
    ids = make_ids(g, 500, 40, "skew", 64)
    assert torch.equal(k.lookup_grad(row.expand(500, 64), ids, 40), k.lookup_grad(row.expand(500, 64).contiguous(), ids, 40))
    assert torch.equal(k.combine(xs, r), k.combine(xs.contiguous(), r))


def test_far_rows(tk):
    """Tables and blocks whose elements are counted beyond 32 bits."""
    k, g = tk("bf16"), gen(8)
    V, D = 4300000, 1024                                           # 4.4e9 elements
    E = torch.empty(V, D, device="cuda", dtype=torch.bfloat16)
    ids = torch.tensor([V - 1, 0, V - 7, 4194304, 4194303], device="cuda")
    E[ids] = normal(g, (5, D), torch.bfloat16)
    want = E[ids]
    assert torch.equal(k.lookup(E, ids), want)
    dy = normal(g, (5, D), torch.bfloat16)
    k.lookup_grad(dy, ids, V, out=E, accumulate=True)
    assert torch.equal(E[ids], (want.float() + dy.float()).bfloat16())
    many = ids.repeat(100)                                         # through the ordered path
    E[ids] = 0
    k.lookup_grad(dy.repeat(100, 1), many, V, out=E, accumulate=True)
    assert torch.equal(E[ids], (100.0 * dy.double()).bfloat16())
    xs, w = E[:4200000], torch.full((4200000, 1), 2.0, device="cuda")
    r = k.route(torch.zeros(4200000, 1, device="cuda", dtype=torch.int32), 1)
    xs[-3:] = want[:3]
    y = k.combine(xs, r, w)
    assert torch.equal(y[-3:], want[:3] * 2)
    out = k.dispatch(y, r, out=xs)
    assert torch.equal(out[-3:], want[:3] * 2)
    W = torch.empty(5, 16384, 65536, device="cuda", dtype=torch.bfloat16)   # 5.4e9 elements
    W[4, -40:] = 0
    W[4, -40:, 5] = 3.0
    r = routed(k, g, [0, 0, 0, 0, 2], 0)
    x = torch.zeros(2, 65536, device="cuda", dtype=torch.bfloat16)
    x[:, 5] = 2.0
    y = k.experts(x, W, r)
    assert (y[:, -40:] == 6.0).all()
    dys = torch.zeros(2, 16384, device="cuda", dtype=torch.bfloat16)
    dys[:, -1] = 1.0
    assert (k.experts_grad_x(dys, W.nan_to_num_(0.0, 0.0, 0.0), r)[:, 5] == 3.0).all()
    k.experts_grad_w(dys, x, r, out=W)
    assert (W[4, -1, 5] == 4.0) and not W[4, -2].any() and not W[0].any()


# 2^26 and a few rows, a wave each: more threads than the first dimension of a grid can have.  What is read is one row for all
# of them, what is written (35 GB) has a different value in every few rows.
MANY = (1 << 26) + 6


def every_row_is(out, value):
    """All columns of row i are value[i], looked at in parts."""
    step = 1 << 22
    return all(bool((out[i:i + step] == value[i:i + step, None]).all()) for i in range(0, len(out), step))


@pytest.mark.parametrize("op", ["lookup", "dispatch", "combine", "combine_grad", "combine_grad wide", "lookup_vals_grad", "lookup_grad"])
def test_more_rows_than_a_grid_has_in_a_row(tk, op):
    k, n = tk("bf16"), MANY if op != "combine_grad wide" else (1 << 24) + 6
    torch.cuda.empty_cache()
    one = lambda D, n=n: torch.ones(1, D, device="cuda", dtype=torch.bfloat16).expand(n, D)  # noqa: E731
    v = torch.arange(n, device="cuda", dtype=torch.int32) % 251     # exact in 8 bits
    zero = torch.zeros(n, device="cuda", dtype=torch.int32)
    if op == "lookup":
        assert every_row_is(k.lookup(one(264, 1), zero, vals=v.float()), v)
    elif op == "lookup_vals_grad":
        assert torch.equal(k.lookup_vals_grad(v.bfloat16()[:, None], one(1, 1), zero, scale=2.0), 2.0 * v)
    elif op == "lookup_grad":                                       # nearly all of it is zeros
        ids = torch.arange(300, device="cuda") * (n // 300)
        ids[-1] = n - 1
        got = k.lookup_grad(one(264, 300), ids, n)
        want = torch.zeros(n, device="cuda").index_fill_(0, ids, 1.0)
        assert every_row_is(got, want)
    else:
        r = k.route(zero[:, None], 1)
        if op == "dispatch":
            assert every_row_is(k.dispatch(one(264), r, v.float()[:, None]), v)
        elif op == "combine":
            assert every_row_is(k.combine(one(264), r, v.float()[:, None]), v)
        else:
            D = 1 if op == "combine_grad" else 1040
            dys, dw = k.combine_grad(one(D), one(D), r, v.float()[:, None])
            assert every_row_is(dys, v) and bool((dw == D).all())
    torch.cuda.empty_cache()


def test_more_parts_of_runs_than_a_grid_has_in_a_row(tk):
    """2^29 ids and a few: a workgroup for every 32 of them joins the sums that cross parts.  Sums of ones stay exact."""
    k, n, V = tk("bf16"), (1 << 29) + 70, 1000
    torch.cuda.empty_cache()
    ids = torch.arange(n, device="cuda", dtype=torch.int32) % V
    got = k.lookup_grad(torch.ones(1, 1, device="cuda", dtype=torch.bfloat16).expand(n, 1), ids, V, dtype=torch.float32)
    assert torch.equal(got[:, 0], (n // V + (torch.arange(V, device="cuda") < n % V)).float())
    del ids, got
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ gradients against differences
def test_gradients_are_the_differences(tk):
    """Every operator is linear in each argument: with small whole numbers nothing is rounded, and a difference over a step
    of one is the derivative, exactly."""
    g = gen(11)
    k = tk("f16")
    whole = lambda *s: torch.randint(-2, 3, s, generator=g, device="cuda").half()  # noqa: E731
    n, V, D, K, X, F = 6, 5, 8, 2, 3, 8
    ids, c = torch.randint(0, V, (n,), generator=g, device="cuda"), torch.randint(0, X, (n, K), generator=g, device="cuda")
    r = k.route(c, X)
    E, gy, f = whole(V, D), whole(n, D), whole(n).float()
    x, ys, w, W = whole(n, D), whole(n * K, F), whole(n, K).float(), whole(X, F, D)
    gx, gs, gf = whole(n * K, D), whole(n, F), whole(n * K, F)
    xs = whole(n * K, D)
    dot = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731

    def differences(f, a):
        d = torch.zeros_like(a)
        for i in itertools.product(*map(range, a.shape)):
            b = a.clone()
            b[i] += 1
            d[i] = f(b) - f(a)
        return d

    assert torch.equal(differences(lambda E: dot(gy, k.lookup(E, ids, vals=f, scale=2.0)), E), k.lookup_grad(gy, ids, V, vals=f, scale=2.0))
    assert torch.equal(differences(lambda f: dot(gy, k.lookup(E, ids, vals=f, scale=2.0)), f), k.lookup_vals_grad(gy, E, ids, scale=2.0))
    assert torch.equal(differences(lambda x: dot(gx, k.dispatch(x, r)), x), k.dispatch_grad(gx, r))
    dys, dw = k.combine_grad(gs, ys, r, w)
    assert torch.equal(differences(lambda ys: dot(gs, k.combine(ys, r, w)), ys), dys)
    assert torch.equal(differences(lambda w: dot(gs, k.combine(ys, r, w)), w), dw)
    assert torch.equal(differences(lambda xs: dot(gf, k.experts(xs, W, r)), xs), k.experts_grad_x(gf, W, r))
    assert torch.equal(differences(lambda W: dot(gf, k.experts(xs, W, r)), W), k.experts_grad_w(gf, xs, r))


# ------------------------------------------------------------------------------------------------ together
def layer(k, s):
    """Token ids to the output of a layer of routed experts, and every gradient back."""
    x = k.lookup(s["E"], s["ids"], scale=2.0)
    r = k.route(s["chosen"], s["W"].shape[0])
    xs = k.dispatch(x, r)
    ys = k.experts(xs, s["W"], r)
    y = k.combine(ys, r, s["w"])
    dys, dw = k.combine_grad(s["dy"], ys, r, s["w"])
    dW = k.experts_grad_w(dys, xs, r, dtype=torch.float32)
    dx = k.dispatch_grad(k.experts_grad_x(dys, s["W"], r), r)
    return y, dw, dW, dx, k.lookup_grad(dx, s["ids"], s["E"].shape[0], scale=2.0, dtype=torch.float32)


def layer_state(seed, n=50, V=40, D=64, F=64, X=6, K=2):
    g = gen(seed)
    c = choices(g, n, K, X, 0.1)
    ids = make_ids(g, n, V, "skew", 64)
    bf = torch.bfloat16
    return {"E": normal(g, (V, D), bf), "ids": ids, "chosen": c, "W": normal(g, (X, F, D), bf) / 8, "w": torch.rand((n, K), generator=g, device="cuda"), "dy": normal(g, (n, F), bf)}


def test_a_layer_of_experts_and_its_gradients(tk):
    """A layer in bf16 against torch's autograd of its definition in 64 bits: two roundings to bf16 in a row on the way
    forward and three on the way back, each 2^-9 of its value, taken over the norms."""
    s = layer_state(5)
    y, dw, dW, dx, dE = layer(tk("bf16"), s)
    E, W, w = (s[k].double().requires_grad_() for k in ("E", "W", "w"))
    ok = s["ids"] >= 0
    x = torch.where(ok[:, None], 2.0 * E[s["ids"].clamp(min=0)], 0.0)
    x.retain_grad()
    X = W.shape[0]
    use = (s["chosen"] >= 0) & (s["chosen"] < X)
    blocks = W[torch.where(use, s["chosen"], 0)]                   # [n, K, F, D]
    out = (torch.matmul(blocks, x[:, None, :, None]).squeeze(-1) * torch.where(use, w, 0.0)[..., None]).sum(1)
    out.backward(s["dy"].double())
    for got, want, roundings in ((y, out, 2), (dw, w.grad, 1), (dW, W.grad, 1), (dx, x.grad, 3), (dE, E.grad, 3)):
        off = float((got.double() - want.detach()).norm() / want.detach().norm())
        assert off <= roundings * 2.0 ** -8, off


def test_a_captured_layer_replays(tk):
    """One graph of the whole layer, replayed on new inputs in the same buffers with eager calls between the replays."""
    s = layer_state(1)
    k = tk("bf16")
    layer(k, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(k, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer(k, s)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        outs2 = layer(k, s)
    for seed in (2, 3, 4):
        for name, v in layer_state(seed).items():
            s[name].copy_(v)
        graph.replay()
        second.replay()
        want = layer(k, s)
        torch.cuda.synchronize()
        live = int(k.route(s["chosen"], 6).offsets[-1])
        assert live > 0
        for a, b, c in zip(outs, outs2, want):
            assert torch.equal(a, c) and torch.equal(b, c)


def test_calls_follow_torchs_stream(tk):
    """Two streams at once, each with inputs made on it: every call has to run behind what made its arguments."""
    k = tk("bf16")
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            big = torch.zeros(1 << 24, device="cuda")
            for _ in range(10):
                big = big + 1.0
            s = layer_state(i, n=3000, V=500)
            got.append((s, layer(k, s)))
    torch.cuda.synchronize()
    for s, outs in got:
        for a, b in zip(outs, layer(k, s)):
            assert torch.equal(a, b)


def test_the_context_and_its_device_are_left_alone(tk, ctx):
    before, held = ctx.get_stream(), ctx.report().split("device memory held")[1]
    layer(tk("bf16"), layer_state(9))
    assert ctx.get_stream() == before and ctx.report().split("device memory held")[1] == held and torch.cuda.current_device() == 0


def test_refusals_on_tensors(tk):
    from sparse_amd.compressed import SparseError
    k = tk("bf16")
    E, ids = torch.zeros(9, 16, device="cuda", dtype=torch.bfloat16), torch.zeros(4, device="cuda", dtype=torch.int64)
    r = k.route(ids.view(2, 2), 3)
    x, ys, w, W = E[:2], E[:4], torch.zeros(2, 2, device="cuda"), torch.zeros(3, 8, 16, device="cuda", dtype=torch.bfloat16)
    for words, call in [("bfloat16", lambda: k.lookup(E.float(), ids)), ("int64", lambda: k.lookup(E, ids.float())), ("side by side", lambda: k.lookup(E.t(), ids)),
                        ("not contiguous", lambda: k.lookup(E, ids[::2])), ("shape", lambda: k.lookup(E, ids, vals=torch.ones(3, device="cuda"))),
                        ("overlaps", lambda: k.lookup(E, ids, out=E[:4])), ("expected 4 x 16", lambda: k.lookup(E, ids, out=E[:3])),
                        ("accumulate", lambda: k.lookup_grad(ys, ids, 9, accumulate=True)), ("float32", lambda: k.lookup_grad(ys, ids, 9, dtype=torch.float16)),
                        ("rows|expected", lambda: k.dispatch(E, r)), ("overlaps", lambda: k.dispatch(x, r, out=E[:4])), ("shape", lambda: k.combine(ys, r, w[:1])),
                        ("no weights", lambda: k.combine_grad(x, ys, r, None)), ("blocks for", lambda: k.experts(ys, W[:2], r)), ("expected", lambda: k.experts(ys, W[:, :, :8], r)),
                        ("16-bit", lambda: tk("f32").experts(ys.float(), W.float(), r)), ("experts", lambda: k.route(ids.view(2, 2), 1025)),
                        ("Routing", lambda: k.experts(ys, W, None)), ("overlap", lambda: k.experts_grad_w(E[:4, :8], ys, r, out=W[:1].expand(3, 8, 16))),
                        ("apart", lambda: k.lookup(E, ids, out=torch.zeros(1, 16, device="cuda", dtype=torch.bfloat16).expand(4, 16))), ("-1 rows", lambda: k.lookup_grad(ys, ids, -1)),
                        ("expected", lambda: k.lookup_grad(ys.view(2, 2, 16), ids, 9))]:
        with pytest.raises(SparseError, match=words):
            call()
    assert not k.lookup(E, ids).any()                              # and the module still works
