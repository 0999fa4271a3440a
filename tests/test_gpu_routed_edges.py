"""GPU: the routed 8-bit operators where they meet torch and each other: sizes, streams, captures, errors and derivatives."""
import pytest

from conftest import have_cuda

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def k():
    if not have_cuda():
        pytest.skip("no CUDA device")
    import stlq_b200

    return stlq_b200.Kernels(0)


def test_rows_that_are_too_long(k):
    r = k.sort_by_expert(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), 1)
    x = torch.empty(1, 2**31 - 4095, dtype=torch.int8, device="cuda")
    h = torch.empty(1, 2**31 - 4095, dtype=torch.float16, device="cuda")
    w = torch.ones(1, 1, device="cuda")
    for call in (lambda: k.dispatch(x, r), lambda: k.dispatch_i8(h, r), lambda: k.quantize_rows(h), lambda: k.combine(h, w, r), lambda: k.combine_backward(h, h, w, r)):
        with pytest.raises(ValueError, match="2\\^31 - 4096"):
            call()


# ---- segments ----------------------------------------------------------------------------------

@pytest.mark.parametrize("kdim", [64, 0, 2048])
@pytest.mark.parametrize("rows,n,first,last", [(25, 40, 3, 10), (25, 40, 25, 25), (700, 40, 300, 690), (3000, 600, 100, 2999)])
def test_rows_before_the_first_segment_are_zeros(k, rows, n, first, last, kdim):
    """An offset above 0 leaves rows without an expert in front, as the last one does behind: zeros in an output that held others."""
    g = torch.Generator().manual_seed(rows + kdim)
    q = torch.randint(-128, 128, (rows, kdim), generator=g).to(torch.int8)
    w = torch.randint(-128, 128, (2, n, kdim), generator=g).to(torch.int8)
    bias = torch.randint(1, 100, (2, n), generator=g).float()
    out = torch.full((rows, n), 7.0, device="cuda")
    middle = (first + last) // 2
    offsets = torch.tensor([first, middle, last], dtype=torch.int32, device="cuda")
    one = torch.ones(rows, device="cuda")
    k.matmul_i8_grouped(q.cuda(), one, w.cuda(), torch.ones(2, n, device="cuda"), offsets, bias=bias.cuda(), out=out)
    k.sync()
    want = torch.zeros(rows, n, dtype=torch.float64)
    for e, (a, b) in enumerate(((first, middle), (middle, last))):
        want[a:b] = q[a:b].double() @ w[e].double().t() + bias[e]
    # Whole numbers: in 32 bits the sum, which is at most |want| + 100, and the addition of the bias each round by 2^-24 at most.
    assert ((out.double().cpu() - want).abs() <= 2.0**-23 * (want.abs() + 100)).all()
    assert (out[:first] == 0).all() and (out[last:] == 0).all()


@pytest.mark.parametrize("kdim", [64, 0])
def test_offsets_out_of_order_give_the_same_segments_without_terms(k, kdim):
    q, w = torch.zeros(50, kdim, dtype=torch.int8, device="cuda"), torch.zeros(4, 10, kdim, dtype=torch.int8, device="cuda")
    bias = torch.arange(1.0, 5.0, device="cuda")[:, None].expand(4, 10).contiguous()
    offsets = torch.tensor([-5, 30, 20, 2_000_000_000, 40], dtype=torch.int32, device="cuda")
    y = k.matmul_i8_grouped(q, torch.ones(50, device="cuda"), w, torch.ones(4, 10, device="cuda"), offsets, bias=bias, out_dtype=torch.float32)
    assert (y[:30] == 1).all() and (y[30:] == 3).all()


# ---- the handle --------------------------------------------------------------------------------

def test_a_new_handle_waits_for_no_work():
    if not have_cuda():
        pytest.skip("no CUDA device")
    import stlq_b200

    stlq_b200.Kernels(0).close()
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    torch.cuda._sleep(2_000_000_000)  # a second or so on the default stream
    done.record()
    h = stlq_b200.Kernels(0)
    assert not done.query()
    h.close()
    torch.cuda.synchronize()


def test_a_handle_made_and_closed_during_a_capture(k):
    import stlq_b200

    x = torch.ones(4, device="cuda")
    x + 1  # loaded before the capture
    other = stlq_b200.Kernels(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = stlq_b200.Kernels(0)
        other.close()
        y = x + 1
    graph.replay()
    assert (y == 2).all()
    q, s = h.quantize_rows(torch.ones(3, 16, device="cuda"))
    assert (h.matmul_i8(q, s, q, s, out_dtype=torch.float32) - 16).abs().max() < 1e-4
    h.sync()
    h.close()


# ---- torch's autograd --------------------------------------------------------------------------

@pytest.mark.parametrize("grouped", [False, True])
def test_out_counts_as_changed(k, grouped):
    """A tensor that a backward pass saved and a product then overwrote is an error, not a wrong gradient."""
    q, s = k.quantize_rows(torch.ones(4, 16, device="cuda"))
    a = torch.ones(4, 4, device="cuda", requires_grad=True)
    whole = torch.ones(4, 12, device="cuda")

    def product(out):
        if grouped:
            return k.matmul_i8_grouped(q, s, q[None], s[None], torch.tensor([0, 4], dtype=torch.int32, device="cuda"), out=out)
        return k.matmul_i8(q, s, q, s, out=out)

    for out in (whole[:, :4], torch.ones(4, 4, device="cuda")):
        loss = (a * out).sum()
        assert product(out) is not None and out._version == 1
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():
        held = torch.ones(4, 4, device="cuda")
        product(held)
    product(held)
    assert (held - 16).abs().max() < 1e-4
    assert product(None)._version == 0


def test_out_that_requires_a_gradient(k):
    q, s = k.quantize_rows(torch.ones(4, 16, device="cuda"))
    out = torch.ones(4, 4, device="cuda", requires_grad=True)
    for bad in (out, out * 1):
        with pytest.raises(ValueError, match="requires a gradient"):
            k.matmul_i8(q, s, q, s, out=bad)
    with torch.no_grad():
        k.matmul_i8(q, s, q, s, out=out)
    assert (out.detach() - 16).abs().max() < 1e-4


@pytest.mark.parametrize("which", ["position", "offsets"])
@pytest.mark.parametrize("op", ["dispatch", "combine", "ones"])
def test_a_routing_changed_before_the_backward_pass(k, op, which):
    """The gradient goes along the arrays that the forward pass used; where they changed, it is an error, not a wrong gradient."""
    ids, other = torch.tensor([[0], [1], [1]], device="cuda"), torch.tensor([[1], [-1], [0]], device="cuda")
    r = k.sort_by_expert(ids, 2)
    x = torch.ones(3, 4, device="cuda", requires_grad=True)

    def forward():
        if op == "dispatch":
            return k.dispatch(x, r).sum()
        return k.combine(x, torch.full((3, 1), 2.0, device="cuda") if op == "combine" else None, r).sum()

    forward().backward()
    assert (x.grad == (2 if op == "combine" else 1)).all()
    loss = forward()
    getattr(r, which).copy_(getattr(k.sort_by_expert(other, 2), which))
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    # Another array in its place is not a change to the one that was used.
    x.grad = None
    r = k.sort_by_expert(ids, 2)
    loss = forward()
    setattr(r, which, getattr(k.sort_by_expert(other, 2), which))
    loss.backward()
    assert (x.grad == (2 if op == "combine" else 1)).all()


@pytest.mark.parametrize("op", ["dispatch", "combine"])
def test_a_routing_made_in_inference_mode(k, op):
    with torch.inference_mode():
        r = k.sort_by_expert(torch.tensor([[0], [1], [-1]], device="cuda"), 2)
    x = torch.ones(3, 4, device="cuda", requires_grad=True)
    w = torch.ones(3, 1, device="cuda", requires_grad=True)
    (k.dispatch(x, r) if op == "dispatch" else k.combine(x, w, r)).sum().backward()
    assert x.grad.sum(1).tolist() == [4, 4, 0] and (op == "dispatch" or w.grad[:, 0].tolist() == [4, 4, 0])


def test_forward_mode_is_refused(k):
    """No operator has a forward-mode derivative; a tangent must not be lost silently."""
    import torch.autograd.forward_ad as fwd

    r = k.sort_by_expert(torch.tensor([[0], [1]], device="cuda"), 2)
    x, one = torch.ones(2, 16, device="cuda"), torch.ones(2, device="cuda")
    q, s = k.quantize_rows(x)
    with fwd.dual_level():
        d, v, w = fwd.make_dual(x, x), fwd.make_dual(one, one), fwd.make_dual(one[:, None], one[:, None])
        for call in (lambda: k.dispatch(d, r), lambda: k.combine(d, None, r), lambda: k.combine(x, w, r), lambda: k.quantize_rows(d),
                     lambda: k.dispatch_i8(d, r), lambda: k.matmul_i8(q, v, q, s), lambda: k.matmul_i8(q, s, q, s, bias=v),
                     lambda: k.dispatch_backward(d, r), lambda: k.combine_backward(d, x, one[:, None], r)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        # A tensor that requires a gradient too goes to the autograd functions, which have no such rule either.
        with pytest.raises((ValueError, RuntimeError)):
            k.dispatch(fwd.make_dual(x.clone().requires_grad_(), x), r)
        assert torch.equal(k.dispatch(x, r), x)  # ordinary tensors at a dual level
    for transform in (lambda: torch.func.jvp(lambda t: k.dispatch(t, r), (x,), (x,)), lambda: torch.func.grad(lambda t: k.dispatch(t, r).sum())(x),
                      lambda: torch.vmap(lambda t: k.dispatch(t, r))(x[None])):
        with pytest.raises((ValueError, RuntimeError)):
            transform()
    assert torch.equal(k.dispatch(x, r), x)


# ---- outputs inside a wider matrix -------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n,kdim,experts", [(40, 1, 32, 0), (40, 3, 32, 0), (300, 33, 32, 0), (300, 130, 48, 0), (1000, 255, 64, 0), (3000, 1001, 1490, 0),
                                                 (300, 130, 48, 3), (9000, 130, 1500, 24), (3000, 513, 2500, 24)])
def test_a_product_writes_its_own_channels_alone(k, dtype, rows, n, kdim, experts):
    """The output's rows lie on 16-byte boundaries and end inside 16 bytes: what follows them in the matrix stays.  The rows of
    both products (one form each of a CTA's own tiles and of pairs) are ones, so the values are exact."""
    whole = torch.full((rows, (n + 7) // 8 * 8 + 8), 7.0, dtype=dtype, device="cuda")
    out = whole[:, :n]
    q, one = torch.ones(rows, kdim, dtype=torch.int8, device="cuda"), torch.ones(rows, device="cuda")
    if experts:
        w, ws = torch.ones(experts, n, kdim, dtype=torch.int8, device="cuda"), torch.full((experts, n), 1 / kdim, device="cuda")
        offsets = torch.linspace(0, rows - 5, experts + 1).int().cuda()
        k.matmul_i8_grouped(q, one, w, ws, offsets, out=out)
        assert (out[-5:] == 0).all()
        out = out[:-5]
    else:
        k.matmul_i8(q, one, torch.ones(n, kdim, dtype=torch.int8, device="cuda"), torch.full((n,), 1 / kdim, device="cuda"), out=out)
    k.sync()
    # kdim * (1 / kdim), two roundings in 32 bits: one in the quotient, one in the product.
    assert ((out.double() - 1).abs() <= (2.0**-22 if dtype == torch.float32 else 2.0**-11 if dtype == torch.float16 else 2.0**-8)).all()
    assert (whole[:, n:] == 7).all()


def test_bytes_past_the_terms_are_not_used(k):
    """Rows of 16-byte multiples whose last bytes are no terms: they hold anything."""
    g = torch.Generator().manual_seed(3)
    for rows, n, kdim in ((70, 90, 17), (300, 200, 129), (1500, 2000, 1490), (130, 130, 2501), (5, 5, 1)):
        wide = (kdim + 15) // 16 * 16
        q, w = (torch.randint(-128, 128, (m, wide), generator=g).to(torch.int8) for m in (rows, n))
        y = k.matmul_i8(q.cuda()[:, :kdim], torch.ones(rows, device="cuda"), w.cuda()[:, :kdim], torch.ones(n, device="cuda"), out_dtype=torch.float32)
        want = q[:, :kdim].double() @ w[:, :kdim].double().t()
        assert ((y.double().cpu() - want).abs() <= 2.0**-24 * want.abs()).all()
