"""Arguments the token entries refuse (include/sparse_amd.h, group 7), without a GPU: the checks come before anything that
touches a device, the addresses below are never followed.  A call that passes them fails only for want of a device."""
import ctypes

import pytest

from sparse_amd.compressed import load_library

VP, I64 = ctypes.c_void_p, ctypes.c_int64
F32, F16, BF16 = 0, 1, 2
A, B, C, D, E, W = (0x10000000 * k for k in range(1, 7))


@pytest.fixture(scope="module")
def call():
    import torch
    if torch.cuda.is_available():
        pytest.skip("with a GPU at hand a call that passes the checks would launch on these made-up addresses")
    from sparse_amd.tokens import _SIGNATURES
    L = load_library()
    cfg = VP(L.futhark_context_config_new())
    ctx = VP(L.futhark_context_new(cfg))
    free = ctypes.CDLL(None).free
    free.argtypes = [VP]

    def go(name, *args):
        f = getattr(L, "sparse_amd_tokens_" + name)
        f.argtypes = _SIGNATURES[name]
        rc = f(ctx, None, *args)
        p = L.futhark_context_get_error(ctx)
        text = ctypes.string_at(p).decode() if p else ""
        free(VP(p))
        return rc, text

    go.lib = L
    return go


def lookup(call, type=BF16, y=A, ldy=64, table=B, V=100, D=64, ldt=64, ids=C, bits=64, n=10, vals=None, scale=1.0):
    return call("lookup", type, y, ldy, table, V, D, ldt, ids, bits, n, vals, scale)


def grad(call, type=BF16, out=F32, acc=0, dt=A, V=100, D=64, ldt=64, dy=B, ldy=64, ids=C, bits=64, n=10, vals=None, work=W, size=1 << 20):
    return call("lookup_grad", type, out, acc, dt, V, D, ldt, dy, ldy, ids, bits, n, vals, 1.0, work, size)


def route(call, chosen=A, bits=64, n=100, X=8, pos=B, src=C, offsets=D, work=W, size=1 << 20):
    return call("route", chosen, bits, n, X, pos, src, offsets, work, size)


def combine(call, type=BF16, y=A, ldy=64, ys=B, ldys=64, slots=20, n=10, D=64, K=2, pos=C, w=D):
    return call("combine", type, y, ldy, ys, ldys, slots, n, D, K, pos, w)


def experts(call, type=BF16, ys=A, ldy=32, xs=B, ldx=64, rows=20, w=C, X=4, F=32, Dd=64, ldw=64, block=2048, offsets=D):
    return call("experts", type, ys, ldy, xs, ldx, rows, w, X, F, Dd, ldw, block, offsets)


def grad_w(call, type=BF16, out=F32, acc=0, dw=A, X=4, F=32, Dd=64, ldw=64, block=2048, dys=B, ldy=32, xs=C, ldx=64, rows=20, offsets=D):
    return call("experts_grad_w", type, out, acc, dw, X, F, Dd, ldw, block, dys, ldy, xs, ldx, rows, offsets)


@pytest.mark.parametrize("f", [lookup, grad, route, combine, experts, grad_w])
def test_what_passes_the_checks_asks_for_a_device(call, f):
    rc, text = f(call)
    assert rc != 0 and "no usable HIP device" in text


REFUSED = [
    (lookup, dict(type=7), "element type"), (lookup, dict(bits=16), "32 or 64 bits"), (lookup, dict(ldt=-1), "negative stride"),
    (lookup, dict(ldy=63), "apart"), (lookup, dict(n=-1), "negative"), (lookup, dict(y=None), "null"), (lookup, dict(ids=None), "null"),
    (lookup, dict(table=None), "null"), (lookup, dict(y=B + 64), "overlaps"), (lookup, dict(y=C), "overlaps"), (lookup, dict(y=A + 1), "aligned"),
    (lookup, dict(vals=A + 8), "overlaps"), (lookup, dict(ids=C + 4), "aligned"), (lookup, dict(ldt=1 << 50), "too large"),
    (grad, dict(out=F16), "32 bits"), (grad, dict(n=300, size=100), "workspace of"), (grad, dict(n=300, work=None), "workspace of"),
    (grad, dict(n=300, work=W + 8), "aligned to 256"), (grad, dict(work=A), "overlaps"), (grad, dict(dt=B), "overlaps"), (grad, dict(V=1 << 31), "31 bits"),
    (grad, dict(n=1 << 31), "31 bits"), (grad, dict(bits=8), "32 or 64 bits"),
    (route, dict(X=0), "experts"), (route, dict(X=1025), "experts"), (route, dict(n=-1), "negative"), (route, dict(n=1 << 31), "31 bits"),
    (route, dict(pos=A), "overlaps"), (route, dict(src=B), "overlaps"), (route, dict(n=100000, size=64), "workspace of"), (route, dict(offsets=None), "null"),
    (combine, dict(K=-1), "places a row"), (combine, dict(ldy=10), "apart"), (combine, dict(y=B), "overlaps"), (combine, dict(pos=None), "null"),
    (experts, dict(type=F32), "16-bit"), (experts, dict(X=2000), "experts"), (experts, dict(offsets=None), "null"), (experts, dict(block=-8), "negative stride"),
    (experts, dict(ldy=31), "apart"), (experts, dict(ldx=-64), "negative stride"), (experts, dict(ys=B), "overlaps"), (experts, dict(rows=-1), "negative"), (experts, dict(F=1 << 31), "too large"),
    (experts, dict(w=None), "null"),
    (grad_w, dict(out=F16), "32 bits"), (grad_w, dict(block=100), "overlap"), (grad_w, dict(dw=C), "overlaps"), (grad_w, dict(ldw=10, block=4096), "apart"),
]


@pytest.mark.parametrize("f,change,words", REFUSED)
def test_refused(call, f, change, words):
    rc, text = f(call, **change)
    assert rc != 0 and words in text, text


def test_combine_grad_and_grad_x_refuse_overlaps(call):
    rc, text = call("combine_grad", BF16, A, 64, E, B, 64, A, 64, 20, 10, 64, 2, C, D)
    assert rc != 0 and "overlaps" in text
    rc, text = call("combine_grad", BF16, A, 64, A + 64, B, 64, W, 64, 20, 10, 64, 2, C, D)
    assert rc != 0 and "overlaps" in text
    rc, text = call("experts_grad_x", BF16, A, 64, A, 32, 20, C, 4, 32, 64, 64, 2048, D)
    assert rc != 0 and "overlaps" in text


# a grid has fewer than 2^32 threads in its first dimension: tiles of 512 threads reach that before their number does
@pytest.mark.parametrize("rows,words", [(1 << 22, "no usable HIP device"), (1 << 24, "more work than one launch"), (1 << 30, "more work than one launch")])
def test_a_launch_of_tiles_too_many_is_refused(call, rows, words):
    rc, text = experts(call, ys=1 << 58, ldy=1 << 16, xs=1 << 44, rows=rows, X=1, F=1 << 16)
    assert rc != 0 and words in text, text


# the workspace is written while the inputs are still read; where none is needed, what is given for one is not touched
@pytest.mark.parametrize("f,change,words", [(grad, dict(n=300, work=B), "workspace overlaps dy"), (grad, dict(n=300, dy=W - 300 * 128 + 128, work=W), "workspace overlaps dy"),
                                            (grad, dict(n=300, work=C), "workspace overlaps ids"), (grad, dict(n=300, vals=D + 512, work=D), "workspace overlaps vals"),
                                            (route, dict(n=10000, work=A), "workspace overlaps chosen"), (route, dict(n=10000, work=A + 65536), "workspace overlaps chosen"),
                                            (grad, dict(n=256, work=B), "no usable HIP device"), (route, dict(n=8192, work=A), "no usable HIP device"),
                                            (grad, dict(n=300, dy=W - 300 * 128, work=W), "no usable HIP device")])
def test_a_workspace_shares_nothing_with_what_is_read(call, f, change, words):
    rc, text = f(call, **change)
    assert rc != 0 and words in text, text


@pytest.mark.parametrize("f,change", [(lookup, dict(n=0)), (lookup, dict(D=0)), (combine, dict(n=0)), (experts, dict(rows=0)), (experts, dict(F=0)),
                                      (grad, dict(n=0, acc=1)), (grad, dict(V=0)), (grad_w, dict(F=0))])
def test_nothing_to_do_is_no_success_without_a_device(call, f, change):
    rc, text = f(call, **change)
    assert rc != 0 and "no usable HIP device" in text


def test_workspaces():
    L = load_library()
    f = L.sparse_amd_tokens_lookup_grad_workspace
    f.argtypes, f.restype = (ctypes.c_int, I64, I64, I64), I64
    assert f(BF16, 256, 100, 64) == 0 and f(BF16, 257, 100, 64) > 0 and f(BF16, 10, 100, 0) == 0 and f(BF16, -1, 100, 64) == 0
    # keys and items at least, and two rows of 32-bit sums for every chunk
    assert f(BF16, 10000, 1000, 64) > 8 * 10000 + 2 * (10000 // 32) * 64 * 4
    g = L.sparse_amd_tokens_route_workspace
    g.argtypes, g.restype = (I64, I64), I64
    assert g(8192, 1024) == 0 and g(8193, 1024) >= 4 * 1025 and g(1 << 30, 1024) <= 2 << 20


def test_the_python_side_refuses_what_is_not_on_the_device():
    import torch
    from sparse_amd.compressed import SparseError
    from sparse_amd.tokens import mk_tokens

    class Ctx:
        L, h, device = load_library(), None, 0
    tk = mk_tokens("bf16", Ctx())
    E_, ids = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(SparseError, match="cuda:0"):
        tk.lookup(E_, ids)
    with pytest.raises(SparseError, match="2 dimensions"):
        tk.route(ids, 4)
    with pytest.raises(SparseError, match="Routing"):
        tk.combine(E_, ids)
    with pytest.raises(AssertionError):
        mk_tokens("f64", Ctx())


@pytest.mark.parametrize("name", ["dispatch", "combine", "dispatch_grad", "combine_grad", "experts", "experts_grad_x", "experts_grad_w"])
def test_a_routing_of_another_device_is_refused(name):
    """Its addresses are another device's: every operator that takes one looks where it is before anything else."""
    import torch
    from sparse_amd.compressed import SparseError
    from sparse_amd.tokens import Routing, mk_tokens

    class Ctx:
        L, h, device = load_library(), None, 0
    buf = torch.zeros(2 * 4 + 4, dtype=torch.int32)
    r = Routing(buf, buf.data_ptr(), 2, 2, 3)
    a = torch.zeros(4, 8, dtype=torch.bfloat16)
    args = {"combine_grad": (a, a, r, None), "experts": (a, a, r), "experts_grad_x": (a, a, r), "experts_grad_w": (a, a, r)}.get(name, (a, r))
    with pytest.raises(SparseError, match="routing: expected one on cuda:0"):
        getattr(mk_tokens("bf16", Ctx()), name)(*args)


@pytest.mark.parametrize("X", [-1, 0, 1025, 2 ** 40, 2 ** 64 + 4])
def test_too_many_experts_or_rows_are_refused_before_they_are_allocated(X):
    import torch
    from sparse_amd.compressed import SparseError
    from sparse_amd.tokens import mk_tokens

    class Ctx:
        L, h, device = load_library(), None, 0
    tk, ids = mk_tokens("bf16", Ctx()), torch.zeros(2, 2, dtype=torch.int64)
    with pytest.raises(SparseError, match="experts"):
        tk.route(ids, X)
    if X < 0 or X > 2 ** 31:
        with pytest.raises(SparseError, match="rows"):
            tk.lookup_grad(torch.zeros(4, 8, dtype=torch.bfloat16), ids, X)
