"""Routed 8-bit operators over libstlq_b200.so: rows quantised to 8 bits, products in 8-bit integers with a scale for each
row and channel, rows sorted by the expert (or root codeword) they were assigned to and back with weights applied, and the
gradient of that exchange.

Everything takes and returns CUDA tensors on the handle's device and runs on the current stream without synchronising;
what it allocates comes from torch's allocator on that stream.  Matrices are row-major; their rows may be strided, the
elements of a row may not.  Wrong shapes, types, layouts or devices raise ValueError before anything is launched.

``dispatch`` and ``combine`` have gradients.  The others have none and their results carry none, whatever their arguments
require: they serve trained weights.  Forward-mode tangents are refused everywhere.

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

from .encoder import StlqB200Error, load_library

_READY = None


def _ready():
    """(the library, the binding), loaded at the first use; raises StlqB200Error where one is missing."""
    global _READY
    if _READY is None:
        import importlib

        import torch  # noqa: F401  (the binding needs its libraries)

        from . import build

        lib = load_library()
        try:
            ops = importlib.import_module("stlq_b200._operators")
        except ImportError as e:
            raise StlqB200Error(f"stlq_b200/_operators.so cannot be loaded ({e}): build it with `python -m stlq_b200.build`") from e
        built, here = getattr(ops, "BUILT_FOR", "another version"), build.built_for()
        if built != here:
            raise StlqB200Error(f"stlq_b200/_operators.so was built for {built} and this is {here}: build it with `python -m stlq_b200.build`")
        v = ctypes.c_void_p
        lib.stlq_b200_kernels_create.argtypes = [ctypes.c_int, ctypes.POINTER(v)]
        lib.stlq_b200_kernels_destroy.argtypes = [v]
        lib.stlq_b200_kernels_sync.argtypes = [v, v]
        names = ("last_error", "quantize_rows", "matmul_i8", "matmul_i8_grouped", "sort_by_expert_workspace", "sort_by_expert",
                 "dispatch", "dispatch_i8", "combine", "combine_backward")
        ops.give(StlqB200Error, *(ctypes.cast(getattr(lib, "stlq_b200_" + n), v).value for n in names))
        _READY = lib, ops
    return _READY


class Routing:
    """Where every choice of every row went: ``order`` (tokens * topk,) is the pairs t * topk + j in sorted order,
    ``position`` (tokens, topk) the sorted row of each pair, ``offsets`` (experts + 1,) the first row of each expert and,
    last, the rows kept; all int32.  ``Kernels.sort_by_expert`` makes one; one made from such arrays works as well."""

    __slots__ = ("order", "position", "offsets", "tokens", "topk", "experts")

    def __init__(self, order, position, offsets):
        self.tokens, self.topk, self.experts = _ready()[1].check_routing(order, position, offsets)
        self.order, self.position, self.offsets = order, position, offsets

    def __repr__(self):
        return f"Routing(tokens={self.tokens}, topk={self.topk}, experts={self.experts})"


class Kernels:
    """The kernel-provider handle on one GPU (``stlq_b200_kernels``).  One host thread at a time may use it."""

    def __init__(self, device: int = 0):
        self._h = 0
        self._lib, self._ops = _ready()
        self._d = int(device)
        h = ctypes.c_void_p()
        self._check(self._lib.stlq_b200_kernels_create(self._d, ctypes.byref(h)), "stlq_b200_kernels_create")
        self._h = h.value

    @property
    def handle(self):
        """The C handle, or None once closed."""
        return ctypes.c_void_p(self._h) if self._h else None

    def close(self):
        h, self._h = getattr(self, "_h", 0), 0
        if h:
            self._lib.stlq_b200_kernels_destroy(ctypes.c_void_p(h))

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int, what: str) -> None:
        if rc != 0:
            raise StlqB200Error(f"{what} failed ({rc}): {self._lib.stlq_b200_last_error().decode()}")

    def quantize_rows(self, x):
        """(q int8 with x's shape, scale float32 (rows,)): scale = max |x| / 127 of a row, q = 127 x / max |x| rounded to
        the nearest integer, ties to even.  A row with an infinity or NaN has scale NaN.  q's rows begin on 16-byte
        boundaries."""
        return self._ops.quantize_rows(self._h, self._d, x)

    def matmul_i8(self, q, q_scale, w, w_scale, bias=None, out_dtype=None, out=None):
        """q (rows, cols) times w (n, cols) transposed, both int8: (q w^T) q_scale[:, None] w_scale + bias, the sum exact,
        rounded once to ``out_dtype`` (out's type, else bfloat16, unless said otherwise).  ``out`` is written in place; it may
        not require a gradient.  Operands whose rows do not begin
        on 16-byte boundaries are copied on every call: quantize_rows lays them out once."""
        return self._ops.matmul_i8(self._h, self._d, q, q_scale, w, w_scale, bias, out_dtype, out)

    def matmul_i8_grouped(self, q, q_scale, w, w_scale, offsets, bias=None, out_dtype=None, out=None):
        """matmul_i8 with the matrix w[e] (n, cols) of the expert whose rows offsets[e] .. offsets[e + 1] - 1 are; w
        (experts, n, cols), w_scale and bias (experts, n), offsets (experts + 1,) int32.  Rows before offsets[0] and from
        offsets[-1] on are zeros.  At most 1,024 experts."""
        return self._ops.matmul_i8_grouped(self._h, self._d, q, q_scale, w, w_scale, offsets, bias, out_dtype, out)

    def sort_by_expert(self, ids, experts: int) -> Routing:
        """The choices ids (tokens, topk) or (tokens,), int32 or int64, sorted by expert, those of an expert in order of
        t * topk + j; an id outside [0, experts) is a dropped choice, and dropped ones come last."""
        r = Routing.__new__(Routing)
        r.order, r.position, r.offsets = self._ops.sort_by_expert(self._h, self._d, ids, experts)
        r.tokens, r.topk = r.position.shape
        r.experts = experts
        return r

    def dispatch(self, x, routing: Routing):
        """x's rows in the order of their experts: (tokens * topk, cols), zeros for dropped choices.  Elements of 1, 2 or 4
        bytes.  Differentiable where x requires a gradient."""
        if x.requires_grad:
            return _functions()[0].apply(x, self, routing)
        return self._ops.dispatch(self._h, self._d, x, routing.position, routing.offsets)

    def dispatch_i8(self, x, routing: Routing):
        """dispatch(quantize_rows(x)) in one pass: (q (tokens * topk, cols) int8, scale (tokens * topk,)); zeros and scale
        0 for dropped choices."""
        return self._ops.dispatch_i8(self._h, self._d, x, routing.position, routing.offsets)

    def dispatch_backward(self, dxs, routing: Routing):
        """The gradient of dispatch for its input: dx[t] = the sum of dxs over t's kept choices."""
        return self._ops.combine(self._h, self._d, dxs, None, routing.position, routing.offsets)

    def combine(self, y, weights, routing: Routing):
        """out[t] = sum over t's kept choices of weights[t, j] y[position[t, j]], in 32 bits, rounded once to y's type.
        weights (tokens, topk) in float32, bfloat16 or float16, or None for ones.  Differentiable where y or weights require
        a gradient."""
        if y.requires_grad or (weights is not None and weights.requires_grad):
            return _functions()[1].apply(y, weights, self, routing)
        return self._ops.combine(self._h, self._d, y, weights, routing.position, routing.offsets)

    def combine_backward(self, dout, y, weights, routing: Routing):
        """The gradient of combine: (dy, dweights) for the gradient dout (tokens, cols) of its result; dy and dweights have
        the types of y and weights, and are zero for dropped choices."""
        return self._ops.combine_backward(self._h, self._d, dout, y, weights, routing.position, routing.offsets)

    def sync(self):
        """Waits for the current stream; raises if a kernel of this handle, on any stream, reported an error since the last call:
        a product whose bounded waits ran out, which nothing else reports and whose result is not valid."""
        import torch

        self._check(self._lib.stlq_b200_kernels_sync(ctypes.c_void_p(self._h), torch.cuda.current_stream(self._d).cuda_stream),
                    "stlq_b200_kernels_sync")


_FUNCTIONS = None


def _functions():
    """(dispatch, combine) for torch's autograd; made at the first use, since importing this module needs no torch."""
    global _FUNCTIONS
    if _FUNCTIONS is None:
        import torch
        from torch.autograd.function import once_differentiable

        def save(ctx, kernels, routing, *tensors):
            """Keeps the routing's arrays as saved tensors, so that a change to them before the backward pass is an error.
            Arrays that were made in inference mode cannot be saved so, nor their changes be seen."""
            arrays = (routing.position, routing.offsets)
            ctx.kernels, ctx.untracked = kernels, arrays if any(t.is_inference() for t in arrays) else None
            ctx.save_for_backward(*tensors, *(() if ctx.untracked else arrays))

        def saved(ctx):
            return ctx.kernels._ops, (ctx.kernels._h, ctx.kernels._d), (*ctx.saved_tensors, *(ctx.untracked or ()))

        class Dispatch(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, kernels, routing):
                if not x.is_floating_point():
                    raise ValueError("only floating rows have a gradient")
                save(ctx, kernels, routing)
                return kernels.dispatch(x.detach(), routing)

            @staticmethod
            @once_differentiable
            def backward(ctx, dxs):
                ops, handle, arrays = saved(ctx)
                return ops.combine(*handle, dxs.contiguous(), None, *arrays), None, None

        class Combine(torch.autograd.Function):
            @staticmethod
            def forward(ctx, y, weights, kernels, routing):
                ctx.ones = weights is None
                save(ctx, kernels, routing, *(() if ctx.ones else (y, weights)))
                return kernels.combine(y.detach(), None if ctx.ones else weights.detach(), routing)

            @staticmethod
            @once_differentiable
            def backward(ctx, dout):
                ops, handle, held = saved(ctx)
                if ctx.ones:
                    return ops.dispatch(*handle, dout.contiguous(), *held), None, None, None
                dy, dweights = ops.combine_backward(*handle, dout.contiguous(), *held)
                return dy, dweights, None, None

        _FUNCTIONS = Dispatch, Combine
    return _FUNCTIONS
