"""Products with the sparse records a language model makes anew at every step, on torch CUDA tensors.

    tk = mk_tokens("bf16")                      # element type of the panels: bf16, f16, f32
    y  = tk.lookup(E, ids, vals, scale)         # a mono record (one entry per row: ids, vals) times the panel E
    dE = tk.lookup_grad(dy, ids, len(E), vals, scale)
    r  = tk.route(chosen, X)                    # K entries per row: every choice's place, an expert's places side by side
    xs = tk.dispatch(x, r)                      # rows into the order of their experts
    ys = tk.experts(xs, W, r)                   # times the block-diagonal matrix of the experts' blocks W[X, F, D]
    y  = tk.combine(ys, r, weights)             # and back, weighted

and the gradients: lookup_vals_grad, combine_grad, experts_grad_x, experts_grad_w, dispatch_grad.

Neighbours of sparse_amd.mono (a record of col_idx[n] and vals[n], mono.fut:95) and of `smm`, behind the same library; every
call is one entry of include/sparse_amd.h, group (7), where the formulas stand.  What differs from the other modules:

* arguments and results are torch CUDA tensors (numpy knows no bf16), on the context's device; a row of a panel is
  contiguous, its rows may be any stride apart (expanded rows too, where they are only read).  Ids, choices, values and
  weights are contiguous;
* a call runs on torch's current stream of that device, like torch's own operations, whatever stream the context is on; it
  allocates from torch's allocator only, never waits, and may be captured into a graph.  Rows of a result it does not
  define (behind the last routed slot) are whatever the memory held, or what `out` held;
* an id or an expert out of range selects nothing (row of zeros, place -1); there is no error for it, since that would
  have to wait for the device;
* `out` shares no memory with an argument, and does not lie between an argument's rows;
* nothing is recorded for torch's autograd: the gradients are calls of their own.

Arguments that do not fit (type, shape, device, overlap) raise SparseError before anything is launched.
"""
import ctypes
import functools

import torch

from .compressed import SparseError, default_context

_VP, _I64, _INT, _F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
_MAX_EXPERTS, _MAX_ROWS = 1024, 2 ** 31 - 2      # as the library has them: refused before a result of such a size is allocated
_TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}

_SIGNATURES = {
    "lookup": (_VP, _VP, _INT, _VP, _I64, _VP, _I64, _I64, _I64, _VP, _INT, _I64, _VP, _F32),
    "lookup_dots": (_VP, _VP, _INT, _VP, _VP, _I64, _VP, _I64, _I64, _I64, _VP, _INT, _I64, _F32),
    "lookup_grad": (_VP, _VP, _INT, _INT, _INT, _VP, _I64, _I64, _I64, _VP, _I64, _VP, _INT, _I64, _VP, _F32, _VP, _I64),
    "route": (_VP, _VP, _VP, _INT, _I64, _I64, _VP, _VP, _VP, _VP, _I64),
    "dispatch": (_VP, _VP, _INT, _VP, _I64, _I64, _VP, _I64, _I64, _I64, _I64, _VP, _VP),
    "combine": (_VP, _VP, _INT, _VP, _I64, _VP, _I64, _I64, _I64, _I64, _I64, _VP, _VP),
    "combine_grad": (_VP, _VP, _INT, _VP, _I64, _VP, _VP, _I64, _VP, _I64, _I64, _I64, _I64, _I64, _VP, _VP),
    "experts": (_VP, _VP, _INT, _VP, _I64, _VP, _I64, _I64, _VP, _I64, _I64, _I64, _I64, _I64, _VP),
    "experts_grad_x": (_VP, _VP, _INT, _VP, _I64, _VP, _I64, _I64, _VP, _I64, _I64, _I64, _I64, _I64, _VP),
    "experts_grad_w": (_VP, _VP, _INT, _INT, _INT, _VP, _I64, _I64, _I64, _I64, _I64, _VP, _I64, _VP, _I64, _I64, _VP),
}


def _current_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


# the same number without the object around it, where this torch has it
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)


class Routing:
    """Where a batch's choices go (tk.route).  pos[tokens, K]: the place of every choice, -1 where it names no expert;
    src[tokens * K]: the choice (token * K + j) at every place, -1 behind the last; offsets[X + 1]: expert e has the places
    offsets[e] .. offsets[e + 1] - 1.  All int32, on the device, in one buffer."""
    __slots__ = ("tokens", "K", "X", "slots", "_buf", "_pos", "_offsets", "_on")

    def __init__(self, buf, address, tokens, K, X):
        self.tokens, self.K, self.X, self.slots = tokens, K, X, tokens * K
        self._buf, self._pos, self._offsets, self._on = buf, address, address + 8 * tokens * K, buf.get_device()

    @property
    def pos(self):
        return self._buf[:self.slots].view(self.tokens, self.K)

    @property
    def src(self):
        return self._buf[self.slots:2 * self.slots]

    @property
    def offsets(self):
        return self._buf[2 * self.slots:]


class mk_tokens:
    """The products of this module for panels of element type T: bf16, f16 or f32 (the experts' products: bf16, f16)."""

    def __init__(self, T, ctx=None):
        assert T in _TYPES, T
        self.t = T
        self._code, self._dtype = _TYPES[T]
        self.ctx = ctx if ctx is not None else default_context()
        self._dev = self.ctx.device
        self._device = torch.device("cuda", self._dev)
        L = self.ctx.L
        for name, types in _SIGNATURES.items():
            f = getattr(L, "sparse_amd_tokens_" + name)
            f.argtypes = types
            setattr(self, "_c_" + name, f)
        # how much a workspace takes depends on the sizes alone: asked once for each of the last ones
        f = L.sparse_amd_tokens_lookup_grad_workspace
        f.argtypes, f.restype = (_INT, _I64, _I64, _I64), _I64
        self._c_grad_work = functools.lru_cache(256)(f)
        f = L.sparse_amd_tokens_route_workspace
        f.argtypes, f.restype = (_I64, _I64), _I64
        self._c_route_work = functools.lru_cache(256)(f)

    # ---- arguments: what fits is taken with a handful of attribute reads, since a small call costs as much as they do; what
    # does not is looked at again for the message
    def _refuse(self, a, name, dtypes, why):
        if not isinstance(a, torch.Tensor) or a.get_device() != self._dev:
            raise SparseError("%s: expected a tensor on cuda:%d" % (name, self._dev))
        if a.dtype not in dtypes:
            raise SparseError("%s: expected %s, got %s" % (name, " or ".join(str(d) for d in dtypes), a.dtype))
        raise SparseError("%s: %s" % (name, why))

    def _panel(self, a, name, rows=None, cols=None, dtype=None):
        """(address, row stride, rows, columns) of a 2-d panel with contiguous rows."""
        dtype = dtype or self._dtype
        if not isinstance(a, torch.Tensor) or a.dtype is not dtype or a.get_device() != self._dev:
            self._refuse(a, name, (dtype,), "")
        if a.dim() != 2:
            self._refuse(a, name, (dtype,), "expected 2 dimensions, got %d" % a.dim())
        n, d = a.shape
        ld, step = a.stride()
        if (rows is not None and n != rows) or (cols is not None and d != cols):
            self._refuse(a, name, (dtype,), "expected %s x %s, got %d x %d" % ("any" if rows is None else rows, "any" if cols is None else cols, n, d))
        if step != 1 and d > 1:
            self._refuse(a, name, (dtype,), "the elements of a row are not side by side")
        return a.data_ptr(), ld if n > 1 or ld > d else d, n, d

    def _floats(self, a, name, shape):
        """Address of a contiguous float32 tensor of this shape."""
        if not isinstance(a, torch.Tensor) or a.dtype is not torch.float32 or a.get_device() != self._dev:
            self._refuse(a, name, (torch.float32,), "")
        if a.shape != shape:
            raise SparseError("%s: expected shape %s, got %s" % (name, tuple(shape), tuple(a.shape)))
        if not a.is_contiguous():
            raise SparseError("%s: not contiguous" % name)
        return a.data_ptr()

    def _ids(self, a, name):
        """(address, bits, count) of contiguous indices."""
        if not isinstance(a, torch.Tensor) or a.get_device() != self._dev:
            self._refuse(a, name, (torch.int64, torch.int32), "")
        bits = 64 if a.dtype is torch.int64 else 32 if a.dtype is torch.int32 else 0
        if not bits:
            self._refuse(a, name, (torch.int64, torch.int32), "")
        if not a.is_contiguous():
            raise SparseError("%s: not contiguous" % name)
        return a.data_ptr(), bits, a.numel()

    def _out(self, out, name, rows, cols, dtype=None):
        """The result's panel: `out`, checked, or a new one."""
        dtype = dtype or self._dtype
        if out is None:
            out = torch.empty((rows, cols), dtype=dtype, device=self._device)
            return out, out.data_ptr(), cols or 1
        p, ld, _, _ = self._panel(out, name, rows, cols, dtype)
        return out, p, ld

    def _sum_type(self, out, dtype):
        dtype = dtype if dtype is not None else out.dtype if out is not None else self._dtype
        if dtype not in (self._dtype, torch.float32):
            raise SparseError("a gradient is %s or torch.float32, not %s" % (self._dtype, dtype))
        return dtype, self._code if dtype == self._dtype else 0

    def _call(self, f, *args):
        h = self.ctx.h
        if not h:
            raise SparseError("the context is closed")
        if f(h, _current_stream(self._dev), *args):
            raise SparseError(self.ctx.error() or "entry point failed")

    def _scratch(self, size):
        """A workspace for one call, from torch's allocator: it is reused in stream order, and a graph's own while one is
        being captured."""
        if size == 0:
            return None, None
        w = torch.empty(size, dtype=torch.uint8, device=self._device)
        return w, w.data_ptr()

    @staticmethod
    def _as_rows(a, ids):
        """ids.shape + (D,) as the panel [ids.numel(), D]."""
        if isinstance(a, torch.Tensor) and ids.dim() != 1 and a.shape[:-1] == ids.shape and a.is_contiguous():
            return a.view(ids.numel(), a.shape[-1])
        return a

    # ---- one entry per row
    def lookup(self, E, ids, vals=None, scale=1.0, out=None):
        """y[i] = scale * vals[i] * E[ids[i]], shape ids.shape + (D,): rows of the table E[V, D].  vals: float32, one per
        id, or None (ones).  `out`: a panel [ids.numel(), D] to write instead of a new tensor (returned as it is)."""
        e, lde, V, D = self._panel(E, "E")
        i, bits, n = self._ids(ids, "ids")
        f = self._floats(vals, "vals", ids.shape) if vals is not None else None
        y, p, ldy = self._out(out, "out", n, D)
        self._call(self._c_lookup, self._code, p, ldy, e, V, D, lde, i, bits, n, f, scale)
        return y if out is not None or ids.dim() == 1 else y.view(*ids.shape, D)

    def lookup_grad(self, dy, ids, V, vals=None, scale=1.0, out=None, accumulate=False, dtype=None):
        """lookup's gradient by the table: dE[v] = the sum of scale * vals[i] * dy[i] over the i with ids[i] = v, added in
        32 bits in an order that the ids, their number, the type and D decide.  dy: [ids.numel(), D] (or ids.shape + (D,), contiguous).  accumulate: added to
        `out` instead of written over it; rows no id names are then not touched.  dtype (without `out`): the module's
        element type or torch.float32."""
        V = int(V)
        if V < 0 or V > _MAX_ROWS:
            raise SparseError("lookup_grad: %d rows (0 to %d are offered)" % (V, _MAX_ROWS))
        i, bits, n = self._ids(ids, "ids")
        g, ldg, _, D = self._panel(self._as_rows(dy, ids), "dy", rows=n)
        f = self._floats(vals, "vals", ids.shape) if vals is not None else None
        if accumulate and out is None:
            raise SparseError("lookup_grad: accumulate needs `out`")
        dtype, code = self._sum_type(out, dtype)
        dE, p, lde = self._out(out, "out", V, D, dtype)
        size = self._c_grad_work(self._code, n, V, D)
        w, wp = self._scratch(size)
        self._call(self._c_lookup_grad, self._code, code, int(accumulate), p, V, D, lde, g, ldg, i, bits, n, f, scale, wp, size)
        return dE

    def lookup_vals_grad(self, dy, E, ids, scale=1.0):
        """lookup's gradient by vals: scale * <dy[i], E[ids[i]]>, float32, shape of ids."""
        i, bits, n = self._ids(ids, "ids")
        e, lde, V, D = self._panel(E, "E")
        g, ldg, _, _ = self._panel(self._as_rows(dy, ids), "dy", rows=n, cols=D)
        d = torch.empty(ids.shape, dtype=torch.float32, device=ids.device)
        self._call(self._c_lookup_dots, self._code, d.data_ptr(), g, ldg, e, V, D, lde, i, bits, n, scale)
        return d

    # ---- K entries per row
    def route(self, chosen, X):
        """Places for the experts that each token chose: chosen[tokens, K], 0 .. X-1 (anything else: no place)."""
        if isinstance(chosen, torch.Tensor) and chosen.dim() != 2:
            raise SparseError("chosen: expected 2 dimensions, got %d" % chosen.dim())
        X = int(X)
        if X < 1 or X > _MAX_EXPERTS:
            raise SparseError("route: %d experts (1 to %d are offered)" % (X, _MAX_EXPERTS))
        c, bits, n = self._ids(chosen, "chosen")
        buf = torch.empty(2 * n + X + 1, dtype=torch.int32, device=self._device)
        size = self._c_route_work(n, X)
        w, wp = self._scratch(size)
        p = buf.data_ptr()
        self._call(self._c_route, c, bits, n, X, p, p + 4 * n, p + 8 * n, wp, size)
        tokens, K = chosen.shape
        return Routing(buf, p, tokens, K, X)

    def _routing(self, r):
        if not isinstance(r, Routing):
            raise SparseError("expected a Routing (the result of route)")
        if r._on != self._dev:
            raise SparseError("the routing: expected one on cuda:%d" % self._dev)
        return r

    def _weights(self, w, r):
        return self._floats(w, "weights", (r.tokens, r.K)) if w is not None else None

    def dispatch(self, x, r, weights=None, out=None):
        """xs[pos[t, j]] = weights[t, j] * x[t]: [slots, D], rows in the order of their experts."""
        r = self._routing(r)
        a, lda, n, D = self._panel(x, "x", rows=r.tokens)
        xs, p, ld = self._out(out, "out", r.slots, D)
        self._call(self._c_dispatch, self._code, p, ld, r.slots, a, lda, n, D, r.K, r._pos, self._weights(weights, r))
        return xs

    def combine(self, ys, r, weights=None, out=None):
        """y[t] = sum over j of weights[t, j] * ys[pos[t, j]]: [tokens, D]."""
        r = self._routing(r)
        a, lda, _, D = self._panel(ys, "ys", rows=r.slots)
        y, p, ld = self._out(out, "out", r.tokens, D)
        self._call(self._c_combine, self._code, p, ld, a, lda, r.slots, r.tokens, D, r.K, r._pos, self._weights(weights, r))
        return y

    def dispatch_grad(self, dxs, r, weights=None, out=None):
        """dispatch's gradient by x: the sum of a token's rows of dxs (times its weights), which is combine."""
        return self.combine(dxs, r, weights, out)

    def combine_grad(self, dy, ys, r, weights, out=None):
        """combine's gradients: (dys, dweights), dys[pos[t, j]] = weights[t, j] * dy[t] and dweights[t, j] =
        <dy[t], ys[pos[t, j]]> in float32.  `out`: where dys goes.  Without weights: dispatch(dy, r)."""
        r = self._routing(r)
        g, ldg, n, D = self._panel(dy, "dy", rows=r.tokens)
        a, lda, _, _ = self._panel(ys, "ys", rows=r.slots, cols=D)
        if weights is None:
            raise SparseError("combine_grad: no weights (their absence makes the gradient dispatch(dy, r))")
        w = self._weights(weights, r)
        dys, p, ld = self._out(out, "out", r.slots, D)
        dw = torch.empty((r.tokens, r.K), dtype=torch.float32, device=self._device)
        self._call(self._c_combine_grad, self._code, p, ld, dw.data_ptr(), g, ldg, a, lda, r.slots, n, D, r.K, r._pos, w)
        return dys, dw

    # ---- one dense block per expert
    def _blocks(self, W, name, X, dtype=None):
        """(address, F, D, row stride, block stride) of [X, F, D] with contiguous rows."""
        dtype = dtype or self._dtype
        if not isinstance(W, torch.Tensor) or W.dtype is not dtype or W.get_device() != self._dev:
            self._refuse(W, name, (dtype,), "")
        if W.dim() != 3:
            self._refuse(W, name, (dtype,), "expected 3 dimensions, got %d" % W.dim())
        x, F, D = W.shape
        if x != X:
            raise SparseError("%s: %d blocks for %d experts" % (name, x, X))
        block, ld, step = W.stride()
        if step != 1 and D > 1:
            raise SparseError("%s: the elements of a row are not side by side" % name)
        return W.data_ptr(), F, D, ld if F > 1 or ld > D else D, block

    def experts(self, xs, W, r, out=None):
        """ys[p] = W[e] xs[p] for every expert e's places p: [slots, F] from xs[slots, D], W[X, F, D].  A row's last bits may
        depend on the other rows of the batch, not on the call."""
        r = self._routing(r)
        w, F, D, ldw, block = self._blocks(W, "W", r.X)
        a, lda, n, _ = self._panel(xs, "xs", rows=r.slots, cols=D)
        ys, p, ld = self._out(out, "out", n, F)
        self._call(self._c_experts, self._code, p, ld, a, lda, n, w, r.X, F, D, ldw, block, r._offsets)
        return ys

    def experts_grad_x(self, dys, W, r, out=None):
        """experts' gradient by xs: dxs[p] = W[e]^T dys[p]: [slots, D]."""
        r = self._routing(r)
        w, F, D, ldw, block = self._blocks(W, "W", r.X)
        a, lda, n, _ = self._panel(dys, "dys", rows=r.slots, cols=F)
        dxs, p, ld = self._out(out, "out", n, D)
        self._call(self._c_experts_grad_x, self._code, p, ld, a, lda, n, w, r.X, F, D, ldw, block, r._offsets)
        return dxs

    def experts_grad_w(self, dys, xs, r, out=None, accumulate=False, dtype=None):
        """experts' gradient by W: dW[e] = the sum of dys[p] xs[p]^T over e's places, [X, F, D]; accumulate and dtype as
        in lookup_grad."""
        r = self._routing(r)
        g, ldg, n, F = self._panel(dys, "dys", rows=r.slots)
        a, lda, _, D = self._panel(xs, "xs", rows=r.slots)
        if accumulate and out is None:
            raise SparseError("experts_grad_w: accumulate needs `out`")
        dtype, code = self._sum_type(out, dtype)
        if out is None:
            out = torch.empty((r.X, F, D), dtype=dtype, device=self._device)
        w, f, d, ldw, block = self._blocks(out, "out", r.X, dtype)
        if (f, d) != (F, D):
            raise SparseError("out: expected blocks of %d x %d, got %d x %d" % (F, D, f, d))
        self._call(self._c_experts_grad_w, self._code, code, int(accumulate), w, r.X, F, D, ldw, block, g, ldg, a, lda, n, r._offsets)
        return out
