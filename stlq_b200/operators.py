"""Routed 8-bit operators over libstlq_b200.so: rows quantised to 8 bits, products in 8-bit integers with a scale for each
row and channel, rows sorted by the expert (or root codeword) they were assigned to and back with weights applied, and the
gradient of that exchange.

Everything takes and returns CUDA tensors on the handle's device and runs on the current stream without synchronising;
what it allocates comes from torch's allocator on that stream.  Matrices are row-major; their rows may be strided, the
elements of a row may not.  Wrong shapes, types, layouts or devices raise ValueError before anything is launched.

    k = stlq_b200.Kernels(device=0)
    wq, ws = k.quantize_rows(weights)                 # once, at load
    q, s = k.quantize_rows(x)
    y = k.matmul_i8(q, s, wq, ws, out_dtype=x.dtype)

    r = k.sort_by_expert(ids, experts)                # ids (tokens, topk)
    q, s = k.dispatch_i8(x, r)
    y = k.matmul_i8_grouped(q, s, wq, ws, r.offsets)  # wq (experts, n, cols)
    out = k.combine(y, mix, r)
"""
from __future__ import annotations

import ctypes

from .encoder import F32, StlqB200Error, load_library

BF16, F16, I32, I64 = 2, 3, 4, 5

MAX_TOPK, MAX_SORT_EXPERTS, MAX_EXPERTS, MAX_I8_K = 64, 65536, 1024, 131071

_READY = None


def _ready():
    """The library with the operators' signatures, torch, and torch's types by code."""
    global _READY
    if _READY is None:
        import torch

        lib = load_library()
        i, l, z, v = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p
        lib.stlq_b200_kernels_create.argtypes = [i, ctypes.POINTER(v)]
        lib.stlq_b200_kernels_destroy.argtypes = [v]
        lib.stlq_b200_kernels_sync.argtypes = [v, v]
        lib.stlq_b200_quantize_rows.argtypes = [v, v, i, l, l, i, v, l, v, v]
        lib.stlq_b200_matmul_i8.argtypes = [v, v, l, v, v, l, v, v, l, i, i, v, i, l, v]
        lib.stlq_b200_matmul_i8_grouped.argtypes = [v, v, l, v, v, l, v, v, v, i, l, i, i, v, i, l, v]
        lib.stlq_b200_sort_by_expert_workspace.argtypes = [l, i, i, ctypes.POINTER(z)]
        lib.stlq_b200_sort_by_expert.argtypes = [v, v, i, l, i, i, v, v, v, v, z, v]
        lib.stlq_b200_dispatch.argtypes = [v, v, i, l, l, i, i, v, v, i, v, l, v]
        lib.stlq_b200_dispatch_i8.argtypes = [v, v, i, l, l, i, i, v, v, i, v, l, v, v]
        lib.stlq_b200_combine.argtypes = [v, v, i, l, l, i, i, v, i, v, v, i, v, l, v]
        lib.stlq_b200_combine_backward.argtypes = [v, v, i, l, v, l, l, i, i, v, i, v, v, i, v, l, v, v]
        floats = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
        _READY = lib, torch, floats, {torch.int32: I32, torch.int64: I64}
    return _READY


class Routing:
    """Where every choice of every row went: ``order`` (tokens * topk,) is the pairs t * topk + j in sorted order,
    ``position`` (tokens, topk) the sorted row of each pair, ``offsets`` (experts + 1,) the first row of each expert and,
    last, the rows kept; all int32.  ``Kernels.sort_by_expert`` makes one; one made from such arrays works as well."""

    __slots__ = ("order", "position", "offsets", "tokens", "topk", "experts")

    def __init__(self, order, position, offsets):
        import torch

        if position.dim() != 2 or offsets.dim() != 1 or order.dim() != 1:
            raise ValueError("order, position and offsets must have 1, 2 and 1 dimensions")
        self.order, self.position, self.offsets = order, position, offsets
        self.tokens, self.topk = position.shape
        self.experts = offsets.shape[0] - 1
        if order.shape[0] != self.tokens * self.topk:
            raise ValueError(f"order must have tokens * topk = {self.tokens * self.topk} elements, got {order.shape[0]}")
        if not 1 <= self.topk <= MAX_TOPK:
            raise ValueError(f"topk must be in [1, {MAX_TOPK}], got {self.topk}")
        if not 1 <= self.experts <= MAX_SORT_EXPERTS:
            raise ValueError(f"experts must be in [1, {MAX_SORT_EXPERTS}], got {self.experts}")
        for t in (order, position, offsets):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError("order, position and offsets must be contiguous int32")

    def __repr__(self):
        return f"Routing(tokens={self.tokens}, topk={self.topk}, experts={self.experts})"


class Kernels:
    """The kernel-provider handle on one GPU (``stlq_b200_kernels``).  One host thread at a time may use it."""

    def __init__(self, device: int = 0):
        self._lib, self._torch, self._floats, self._ints = _ready()
        self.device = self._torch.device("cuda", int(device))
        self.handle = None
        h = ctypes.c_void_p()
        self._check(self._lib.stlq_b200_kernels_create(int(device), ctypes.byref(h)), "stlq_b200_kernels_create")
        self.handle = h

    def close(self):
        if getattr(self, "handle", None) is not None:
            self._lib.stlq_b200_kernels_destroy(self.handle)
        self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- checks ----------------------------------------------------------------------------
    def _check(self, rc: int, what: str) -> None:
        if rc != 0:
            raise StlqB200Error(f"{what} failed ({rc}): {self._lib.stlq_b200_last_error().decode()}")

    def _stream(self):
        return self._torch.cuda.current_stream(self.device).cuda_stream

    def _on(self, name, t):
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}")

    def _rows(self, name, t, kinds):
        """A matrix of one of `kinds` with contiguous rows on the device; its leading dimension."""
        if t.dim() != 2 or t.dtype not in kinds:
            raise ValueError(f"{name} must be a matrix of {' or '.join(str(k)[6:] for k in kinds)}, got {tuple(t.shape)} {t.dtype}")
        self._on(name, t)
        rows, cols = t.shape
        ld = t.stride(0) if rows > 1 else max(cols, 1)
        if (cols > 1 and t.stride(1) != 1) or ld < cols:
            raise ValueError(f"the rows of {name} must be contiguous and not overlap, got strides {t.stride()}")
        return ld

    def _vector(self, name, t, n, kinds=None):
        if t.dim() != 1 or t.shape[0] != n or t.dtype not in (kinds or (self._torch.float32,)) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 of shape ({n},), got {tuple(t.shape)} {t.dtype}")
        self._on(name, t)

    def _routing(self, r, tokens=None):
        if not isinstance(r, Routing):
            raise ValueError("a Routing is needed (Kernels.sort_by_expert makes one)")
        if tokens is not None and r.tokens != tokens:
            raise ValueError(f"the routing has {r.tokens} rows, the matrix {tokens}")
        self._on("the routing", r.position)
        self._on("the routing", r.offsets)

    def _mix(self, w, r):
        if tuple(w.shape) != (r.tokens, r.topk) or w.dtype not in self._floats or not w.is_contiguous():
            raise ValueError(f"weights must be contiguous floats of shape ({r.tokens}, {r.topk}), got {tuple(w.shape)} {w.dtype}")
        self._on("weights", w)

    def _empty8(self, rows, cols):
        """int8 rows on 16-byte boundaries, as the products read them."""
        return self._torch.empty((rows, (cols + 15) & ~15), dtype=self._torch.int8, device=self.device)[:, :cols]

    def _operand(self, name, t):
        """`t` as a product reads it: on 16-byte boundaries, copied there if it is not.  (tensor, leading dimension)"""
        ld = self._rows(name, t, (self._torch.int8,))
        if t.shape[0] == 1:
            ld = (ld + 15) & ~15  # one row: its stride is not used, and bytes past its end are not read
        if ld % 16 == 0 and t.data_ptr() % 16 == 0:
            return t, ld
        out = self._empty8(*t.shape)
        out.copy_(t)
        return out, out.stride(0)

    # ---- operators -------------------------------------------------------------------------
    def quantize_rows(self, x):
        """(q int8 with x's shape, scale float32 (rows,)): scale = max |x| / 127 of a row, q = 127 x / max |x| rounded to
        the nearest integer, ties to even.  A row with an infinity or NaN has scale NaN."""
        ldx = self._rows("x", x, self._floats)
        rows, cols = x.shape
        q = self._empty8(rows, cols)
        scale = self._torch.empty(rows, dtype=self._torch.float32, device=self.device)
        self._check(self._lib.stlq_b200_quantize_rows(self.handle, x.data_ptr(), self._floats[x.dtype], ldx, rows, cols,
                                                      q.data_ptr(), (cols + 15) & ~15, scale.data_ptr(), self._stream()),
                    "stlq_b200_quantize_rows")
        return q, scale

    def _product(self, q, q_scale, w, w_scale, bias, offsets, experts, n, out_dtype, out):
        out_dtype = (out.dtype if out is not None else self._torch.bfloat16) if out_dtype is None else out_dtype
        rows, kdim = q.shape
        self._vector("q_scale", q_scale, rows)
        if w.shape[1] != kdim:
            raise ValueError(f"w has {w.shape[1]} columns, q {kdim}")
        if kdim > MAX_I8_K:
            raise ValueError(f"at most {MAX_I8_K} columns, got {kdim}")
        if out_dtype not in self._floats:
            raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
        if out is None:
            out = self._torch.empty((rows, n), dtype=out_dtype, device=self.device)
        elif tuple(out.shape) != (rows, n) or out.dtype != out_dtype:
            raise ValueError(f"out must be {out_dtype} of shape ({rows}, {n}), got {tuple(out.shape)} {out.dtype}")
        ldo = self._rows("out", out, (out_dtype,))
        q, ldq = self._operand("q", q)
        w, ldw = self._operand("w", w)
        b = bias.data_ptr() if bias is not None else None
        if offsets is None:
            rc = self._lib.stlq_b200_matmul_i8(self.handle, q.data_ptr(), ldq, q_scale.data_ptr(), w.data_ptr(), ldw,
                                               w_scale.data_ptr(), b, rows, n, kdim, out.data_ptr(),
                                               self._floats[out_dtype], ldo, self._stream())
            self._check(rc, "stlq_b200_matmul_i8")
        else:
            rc = self._lib.stlq_b200_matmul_i8_grouped(self.handle, q.data_ptr(), ldq, q_scale.data_ptr(), w.data_ptr(),
                                                       ldw, w_scale.data_ptr(), b, offsets.data_ptr(), experts, rows, n,
                                                       kdim, out.data_ptr(), self._floats[out_dtype], ldo, self._stream())
            self._check(rc, "stlq_b200_matmul_i8_grouped")
        return out

    def matmul_i8(self, q, q_scale, w, w_scale, bias=None, out_dtype=None, out=None):
        """q (rows, cols) times w (n, cols) transposed, both int8: (q w^T) q_scale[:, None] w_scale + bias, the sum exact,
        rounded once to ``out_dtype`` (bfloat16 unless said otherwise).  Rows of w that do not begin on 16-byte boundaries
        are copied on every call: quantize_rows lays them out once."""
        if q.dim() != 2 or w.dim() != 2:
            raise ValueError("q and w must be matrices")
        n = w.shape[0]
        self._vector("w_scale", w_scale, n)
        if bias is not None:
            self._vector("bias", bias, n)
        return self._product(q, q_scale, w, w_scale, bias, None, 1, n, out_dtype, out)

    def matmul_i8_grouped(self, q, q_scale, w, w_scale, offsets, bias=None, out_dtype=None, out=None):
        """matmul_i8 with the matrix w[e] (n, cols) of the expert whose rows offsets[e] .. offsets[e + 1] - 1 are; w
        (experts, n, cols), w_scale and bias (experts, n), offsets (experts + 1,) int32.  Rows from offsets[-1] on are
        zeros."""
        torch = self._torch
        if q.dim() != 2 or w.dim() != 3:
            raise ValueError("q must be a matrix and w have three dimensions (experts, n, cols)")
        experts, n, cols = w.shape
        if not 1 <= experts <= MAX_EXPERTS:
            raise ValueError(f"experts must be in [1, {MAX_EXPERTS}], got {experts}")
        self._vector("offsets", offsets, experts + 1, (torch.int32,))
        if tuple(w_scale.shape) != (experts, n) or (bias is not None and tuple(bias.shape) != (experts, n)):
            raise ValueError(f"w_scale and bias must have shape ({experts}, {n})")
        if experts > 1 and n > 0 and w.stride(0) != n * w.stride(1):
            w = w.contiguous()  # the experts' rows follow one another
        w = w.as_strided((experts * n, cols), (w.stride(1) if n > 1 or experts > 1 else max(cols, 1), w.stride(2) if cols > 1 else 1))
        w_scale = w_scale.reshape(-1)
        self._vector("w_scale", w_scale, experts * n)
        if bias is not None:
            bias = bias.reshape(-1)
            self._vector("bias", bias, experts * n)
        return self._product(q, q_scale, w, w_scale, bias, offsets, experts, n, out_dtype, out)

    def sort_by_expert(self, ids, experts: int) -> Routing:
        """The choices ids (tokens, topk) or (tokens,), int32 or int64, sorted by expert, those of an expert in order of
        t * topk + j; an id outside [0, experts) is a dropped choice, and dropped ones come last."""
        torch = self._torch
        if ids.dim() == 1:
            ids = ids[:, None]
        if ids.dim() != 2 or ids.dtype not in self._ints or not ids.is_contiguous():
            raise ValueError(f"ids must be contiguous int32 or int64 of shape (tokens, topk), got {tuple(ids.shape)} {ids.dtype}")
        self._on("ids", ids)
        tokens, topk = ids.shape
        experts = int(experts)
        need = ctypes.c_size_t()
        if self._lib.stlq_b200_sort_by_expert_workspace(tokens, topk, experts, ctypes.byref(need)) != 0:
            raise ValueError(self._lib.stlq_b200_last_error().decode())
        order = torch.empty(tokens * topk, dtype=torch.int32, device=self.device)
        position = torch.empty((tokens, topk), dtype=torch.int32, device=self.device)
        offsets = torch.empty(experts + 1, dtype=torch.int32, device=self.device)
        space = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._check(self._lib.stlq_b200_sort_by_expert(self.handle, ids.data_ptr(), self._ints[ids.dtype], tokens, topk,
                                                       experts, order.data_ptr(), position.data_ptr(), offsets.data_ptr(),
                                                       space.data_ptr(), need.value, self._stream()),
                    "stlq_b200_sort_by_expert")
        return Routing(order, position, offsets)

    def dispatch(self, x, routing: Routing):
        """x's rows in the order of their experts: (tokens * topk, cols), zeros for dropped choices.  Elements of 1, 2 or 4
        bytes.  Differentiable where x requires a gradient."""
        if self._torch.is_grad_enabled() and x.requires_grad:
            return _functions()[0].apply(x, self, routing)
        return self._dispatch(x, routing)

    def _dispatch(self, x, r):
        if x.dim() != 2 or x.element_size() not in (1, 2, 4):
            raise ValueError(f"x must be a matrix with elements of 1, 2 or 4 bytes, got {tuple(x.shape)} {x.dtype}")
        ldx = self._rows("x", x, (x.dtype,))
        self._routing(r, x.shape[0])
        cols = x.shape[1]
        out = self._torch.empty((r.tokens * r.topk, cols), dtype=x.dtype, device=self.device)
        self._check(self._lib.stlq_b200_dispatch(self.handle, x.data_ptr(), x.element_size(), ldx, r.tokens, cols, r.topk,
                                                 r.position.data_ptr(), r.offsets.data_ptr(), r.experts, out.data_ptr(),
                                                 max(cols, 1), self._stream()), "stlq_b200_dispatch")
        return out

    def dispatch_i8(self, x, routing: Routing):
        """dispatch(quantize_rows(x)) in one pass: (q (tokens * topk, cols) int8, scale (tokens * topk,)); zeros and scale
        0 for dropped choices."""
        ldx = self._rows("x", x, self._floats)
        r = routing
        self._routing(r, x.shape[0])
        cols = x.shape[1]
        q = self._empty8(r.tokens * r.topk, cols)
        scale = self._torch.empty(r.tokens * r.topk, dtype=self._torch.float32, device=self.device)
        self._check(self._lib.stlq_b200_dispatch_i8(self.handle, x.data_ptr(), self._floats[x.dtype], ldx, r.tokens, cols,
                                                    r.topk, r.position.data_ptr(), r.offsets.data_ptr(), r.experts,
                                                    q.data_ptr(), (cols + 15) & ~15, scale.data_ptr(), self._stream()),
                    "stlq_b200_dispatch_i8")
        return q, scale

    def dispatch_backward(self, dxs, routing: Routing):
        """The gradient of dispatch for its input: dx[t] = the sum of dxs over t's kept choices."""
        return self._combine(dxs, None, routing)

    def combine(self, y, weights, routing: Routing):
        """out[t] = sum over t's kept choices of weights[t, j] y[position[t, j]], in 32 bits, rounded once to y's type.
        weights (tokens, topk) in float32, bfloat16 or float16, or None for ones.  Differentiable where y or weights require
        a gradient."""
        if self._torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
            return _functions()[1].apply(y, weights, self, routing)
        return self._combine(y, weights, routing)

    def _combine(self, y, weights, r):
        ldy = self._rows("y", y, self._floats)
        self._routing(r)
        if y.shape[0] != r.tokens * r.topk:
            raise ValueError(f"y must have tokens * topk = {r.tokens * r.topk} rows, got {y.shape[0]}")
        if weights is not None:
            self._mix(weights, r)
        cols = y.shape[1]
        out = self._torch.empty((r.tokens, cols), dtype=y.dtype, device=self.device)
        self._check(self._lib.stlq_b200_combine(self.handle, y.data_ptr(), self._floats[y.dtype], ldy, r.tokens, cols, r.topk,
                                                weights.data_ptr() if weights is not None else None,
                                                self._floats[weights.dtype] if weights is not None else F32,
                                                r.position.data_ptr(), r.offsets.data_ptr(), r.experts, out.data_ptr(),
                                                max(cols, 1), self._stream()), "stlq_b200_combine")
        return out

    def combine_backward(self, dout, y, weights, routing: Routing):
        """The gradient of combine: (dy, dweights) for the gradient dout (tokens, cols) of its result; dy and dweights have
        the types of y and weights, and are zero for dropped choices."""
        r = routing
        self._routing(r)
        ldd = self._rows("dout", dout, self._floats)
        ldy = self._rows("y", y, (dout.dtype,))
        if dout.shape[0] != r.tokens or y.shape[0] != r.tokens * r.topk or dout.shape[1] != y.shape[1]:
            raise ValueError(f"dout and y must have {r.tokens} and {r.tokens * r.topk} rows of one length, got {tuple(dout.shape)} and {tuple(y.shape)}")
        self._mix(weights, r)
        cols = y.shape[1]
        dy = self._torch.empty((y.shape[0], cols), dtype=y.dtype, device=self.device)
        dweights = self._torch.empty((r.tokens, r.topk), dtype=weights.dtype, device=self.device)
        self._check(self._lib.stlq_b200_combine_backward(
            self.handle, dout.data_ptr(), self._floats[dout.dtype], ldd, y.data_ptr(), ldy, r.tokens, cols, r.topk,
            weights.data_ptr(), self._floats[weights.dtype], r.position.data_ptr(), r.offsets.data_ptr(), r.experts,
            dy.data_ptr(), max(cols, 1), dweights.data_ptr(), self._stream()), "stlq_b200_combine_backward")
        return dy, dweights

    def sync(self):
        """Waits for the current stream; raises if a kernel of this handle reported an error."""
        self._check(self._lib.stlq_b200_kernels_sync(self.handle, self._stream()), "stlq_b200_kernels_sync")


_FUNCTIONS = None


def _functions():
    """(dispatch, combine) for torch's autograd; made at the first use, since importing this module needs no torch."""
    global _FUNCTIONS
    if _FUNCTIONS is None:
        import torch
        from torch.autograd.function import once_differentiable

        class Dispatch(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, kernels, routing):
                if not x.is_floating_point():
                    raise ValueError("only floating rows have a gradient")
                ctx.kernels, ctx.routing = kernels, routing
                return kernels._dispatch(x, routing)

            @staticmethod
            @once_differentiable
            def backward(ctx, dxs):
                return ctx.kernels.dispatch_backward(dxs.contiguous(), ctx.routing), None, None

        class Combine(torch.autograd.Function):
            @staticmethod
            def forward(ctx, y, weights, kernels, routing):
                ctx.kernels, ctx.routing, ctx.ones = kernels, routing, weights is None
                ctx.save_for_backward(*((y,) if weights is None else (y, weights)))
                return kernels._combine(y, weights, routing)

            @staticmethod
            @once_differentiable
            def backward(ctx, dout):
                dout, k, r = dout.contiguous(), ctx.kernels, ctx.routing
                if ctx.ones:
                    return k._dispatch(dout, r), None, None, None
                y, weights = ctx.saved_tensors
                dy, dweights = k.combine_backward(dout, y, weights, r)
                return dy, dweights, None, None

        _FUNCTIONS = Dispatch, Combine
    return _FUNCTIONS
