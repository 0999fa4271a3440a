"""GPU: the routed 8-bit operators (stlq_b200.Kernels) against their definitions in 64 bits on the CPU.

Bounds, with u = 2^-24 (a 32-bit rounding) and v the rounding of the result's type (2^-24, 2^-8 for bfloat16, 2^-11 for
float16, plus half its smallest number):
  quantise   16-bit rows: equal.  127 x is exact in 32 bits and a quotient that is no tie is further from one (v 2^-19
             relative) than its rounding (2^-24).  32-bit rows: two roundings of a number up to 127, so |q - 127 x / amax|
             <= 1/2 + 127 * 2u.  Scale: one rounding.
  product    the sum is exact; to float, two products and an addition: 4u (|sum s w| + |bias|), then v |y|.
  combine    k products and additions: (k + 1) u sum |w y|, then v.
  gradient   dy: one product (u), then v.  dweights: (cols + 1) u sum |dout y|, then v.
"""
import numpy as np
import pytest

from conftest import have_cuda

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0**-24
ROUND = {torch.float32: (U, 2.0**-150), torch.bfloat16: (2.0**-8, 2.0**-134), torch.float16: (2.0**-11, 2.0**-25)}
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def k():
    if not have_cuda():
        pytest.skip("no CUDA device")
    import stlq_b200

    return stlq_b200.Kernels(0)


def rng_for(*seed):
    g = torch.Generator()
    g.manual_seed(hash(seed) & 0x7FFFFFFF)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def randq(g, *shape):
    """int8 with every value, -128 too."""
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int32).to(torch.int8)


def close(got, want, slack, dtype):
    """|got - want| <= slack + the rounding of dtype, element by element; NaN where want is."""
    assert got.dtype == dtype
    got, rel = got.double().cpu(), ROUND[dtype]
    bad = ~((got - want).abs() <= slack + rel[0] * (want.abs() + slack) + rel[1])
    bad &= ~((got == want) | (torch.isnan(got) & torch.isnan(want)))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the bound, first at {bad.nonzero()[0].tolist()}"


def quantised(x):
    x = x.double()
    top = x.abs().amax(1) if x.shape[1] else torch.zeros(x.shape[0], dtype=torch.float64)
    fine = torch.isfinite(top)
    some = fine & (top > 0)
    v = torch.where(some[:, None], 127 * x / torch.where(some, top, 1.0)[:, None], 0.0)
    return v, torch.where(fine, top / 127, float("nan"))


def check_quantised(q, s, x):
    v, scale = quantised(x)
    q = q.cpu()
    if x.dtype == torch.float32:
        assert ((q.double() - v).abs() <= 0.5 + 127 * 2 * U).all()
    else:
        assert torch.equal(q, torch.round(v).to(torch.int8))
    close(s, scale, torch.zeros(()), torch.float32)


def route(ids, experts):
    flat = ids.reshape(-1).cpu().numpy().astype(object)
    key = np.array([int(i) if 0 <= i < experts else experts for i in flat], dtype=np.int64)
    order = np.argsort(key, kind="stable")
    position = np.empty_like(order)
    position[order] = np.arange(len(order))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=experts + 1))])[: experts + 1]
    return torch.from_numpy(order), torch.from_numpy(position).view(ids.shape), torch.from_numpy(offsets)


def check_route(r, ids, experts):
    order, position, offsets = route(ids, experts)
    assert torch.equal(r.order.cpu().long(), order)
    assert torch.equal(r.position.cpu().long(), position)
    assert torch.equal(r.offsets.cpu().long(), offsets)


def random_ids(g, tokens, topk, experts, drop=0.2, dtype=torch.int32):
    ids = torch.randint(0, experts, (tokens, topk), generator=g)
    return torch.where(torch.rand(tokens, topk, generator=g) < drop, -1, ids).to(dtype)


# ---- quantisation ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 30), (9, 96), (33, 128), (2, 1000), (7, 960), (3, 4096), (2, 8200), (1, 20001), (9, 20), (5, 1004), (3, 2044), (700, 2047), (900, 254), (4, 2300)])
def test_quantize_rows(k, dtype, rows, cols):
    x = randn(rng_for(1, rows, cols), rows, cols, dtype=dtype)
    q, s = k.quantize_rows(x.cuda())
    assert q.shape == x.shape and q.stride(0) % 16 == 0
    check_quantised(q, s, x)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_ties_zeros_and_infinities(k, dtype):
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal / 4
    x = torch.zeros(8, 37)
    x[1, :3] = torch.tensor([254.0, 1.0, 3.0])  # 0.5 and 1.5: to even
    x[2, 5] = -big
    x[2, 6] = big / 2
    x[3, 0], x[3, 1] = tiny, -tiny / 2
    x[4, 36] = float("inf")
    x[5, 0] = float("nan")
    x[6] = -2.0
    x[7, 3], x[7, 4] = float("-inf"), float("nan")
    x = x.to(dtype)
    q, s = k.quantize_rows(x.cuda())
    check_quantised(q, s, x)
    assert torch.isnan(s[[4, 5, 7]]).all() and (q[[0, 4, 5, 7]] == 0).all() and s[0] == 0
    assert q[1, :3].tolist() == [127, 0, 2]


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 7), (torch.float16, 10)])
def test_quantize_every_16_bit_quotient(k, dtype, bits):
    """Every mantissa of a row's largest value against every value down to 2^-9 of it: all the quotients that 16-bit rows can have, ties
    among them (the largest value's mantissa a multiple of 127, and half the largest value)."""
    one = 1 << bits
    top = torch.arange(one, 2 * one, dtype=torch.float64)  # the largest value's significand
    below = torch.cat([torch.arange(one, 2 * one, dtype=torch.float64) * 2.0**-s for s in range(10)])
    x = torch.where(below[None] <= top[:, None], below[None], -0.5 * below[None])
    x = torch.cat([top[:, None], x], 1) / 64  # exact in both types
    assert torch.equal(x.to(dtype).double(), x)
    q, s = k.quantize_rows(x.to(dtype).cuda())
    want = torch.round(127 * x / (top[:, None] / 64)).to(torch.int8)
    assert torch.equal(q.cpu(), want)


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_strided_and_unaligned(k, dtype):
    x = randn(rng_for(2), 11, 203, dtype=dtype)
    g = x.cuda()
    for view, want in ((g[:, 1:100], x[:, 1:100]), (g[::2, :96], x[::2, :96]), (g[3:4, 5:], x[3:4, 5:])):
        check_quantised(*k.quantize_rows(view), want)


def test_no_rows_and_no_columns(k):
    q, s = k.quantize_rows(torch.empty(0, 5, device="cuda"))
    assert q.shape == (0, 5) and s.shape == (0,)
    q, s = k.quantize_rows(torch.empty(4, 0, device="cuda"))
    assert q.shape == (4, 0) and (s == 0).all()
    w, ws = k.quantize_rows(torch.ones(6, 0, device="cuda"))
    y = k.matmul_i8(q, s, w, ws, bias=torch.arange(6.0, device="cuda"), out_dtype=torch.float32)
    assert torch.equal(y.cpu(), torch.arange(6.0).expand(4, 6))
    assert k.matmul_i8(q, s, w[:0], ws[:0]).shape == (4, 0)
    assert k.matmul_i8(q[:0], s[:0], w, ws).shape == (0, 6)
    r = k.sort_by_expert(torch.empty(0, 3, dtype=torch.int64, device="cuda"), 2000)
    assert r.order.numel() == 0 and (r.offsets == 0).all() and r.offsets.numel() == 2001
    x = torch.empty(0, 8, device="cuda")
    assert k.dispatch(x, r).shape == (0, 8) and k.combine(x, None, r).shape == (0, 8)
    assert k.dispatch_i8(x, r)[0].shape == (0, 8)


# ---- products ----------------------------------------------------------------------------------

def check_product(y, q, s, w, ws, bias, dtype):
    """y against rows q (CPU) times w."""
    terms = (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()[None]
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.double()
    close(y, terms + b, 4 * U * (terms.abs() + b.abs()), dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,n,kdim", [(1, 1, 1), (1, 130, 17), (2, 128, 128), (5, 300, 96), (16, 129, 960), (17, 64, 129), (31, 257, 256),
                                         (33, 40, 1000), (64, 128, 4096), (65, 500, 33), (127, 128, 640), (129, 1000, 300), (255, 130, 128),
                                         (256, 256, 512), (257, 129, 130), (700, 385, 1100), (1, 4096, 4096), (3, 1000, 5000), (1300, 2100, 257),
                                         (300, 8, 64), (20, 16, 128), (130, 24, 40), (2000, 32, 70), (100, 136, 8000), (5, 64, 2000), (1100, 4096, 96), (4000, 3000, 260)])
def test_matmul_i8(k, dtype, rows, n, kdim):
    g = rng_for(3, rows, n, kdim)
    q, w = randq(g, rows, kdim), randq(g, n, kdim)
    s, ws = torch.rand(rows, generator=g) + 0.01, (torch.rand(n, generator=g) + 0.01) / 128 / kdim
    bias = randn(g, n) if (rows + n) % 2 else None
    y = k.matmul_i8(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), None if bias is None else bias.cuda(), out_dtype=dtype)
    k.sync()
    check_product(y, q, s, w, ws, bias, dtype)


@pytest.mark.parametrize("dtype,rows,n,kdim", [(torch.float32, 7147, 2000, 52), (torch.float32, 3467, 1724, 208), (torch.bfloat16, 9000, 1944, 64), (torch.bfloat16, 5000, 4200, 300)])
def test_matmul_i8_every_time(k, dtype, rows, n, kdim):
    """Many tiles a block, with the last channels' tile partly past the end: forty calls give the same bits, and the right ones."""
    g = rng_for(17, rows, n)
    q, w = randq(g, rows, kdim), randq(g, n, kdim)
    s, ws, bias = torch.rand(rows, generator=g), torch.rand(n, generator=g) / 128 / kdim, randn(g, n)
    args = [t.cuda() for t in (q, s, w, ws, bias)]
    first = k.matmul_i8(*args, out_dtype=dtype)
    check_product(first, q, s, w, ws, bias, dtype)
    for _ in range(40):
        assert torch.equal(k.matmul_i8(*args, out_dtype=dtype), first)


def test_matmul_i8_longest_sum(k):
    """131,071 terms of (-128)^2 are 2^31 - 2^14: the sum stays below the end of 32 bits."""
    kdim = 131071
    q = torch.full((2, kdim), -128, dtype=torch.int8)
    w = torch.full((3, kdim), -128, dtype=torch.int8)
    w[1] = 127
    one = torch.ones(3)
    y = k.matmul_i8(q.cuda(), one[:2].cuda(), w.cuda(), one.cuda(), out_dtype=torch.float32)
    assert y[0].tolist() == [float(np.float32(16384 * kdim)), float(np.float32(-128 * 127 * kdim)), float(np.float32(16384 * kdim))]


def test_matmul_i8_layouts(k):
    """Operands off 16-byte boundaries, with strides, and an output that is part of a larger matrix."""
    g = rng_for(4)
    Q, W = randq(g, 70, 333), randq(g, 90, 400)
    s, ws = torch.rand(70, generator=g), torch.rand(90, generator=g) / 1e4
    for q, w, a, b in ((Q[:, 3:150], W[:, 5:152], s, ws), (Q[::2, :300], W[10:, 50:350], s[::2].contiguous(), ws[10:]), (Q[7:8, 9:], W[1:2, 1:325], s[7:8], ws[1:2])):
        qc, wc = Q.cuda(), W.cuda()
        qg = qc.as_strided(q.shape, q.stride(), q.storage_offset())
        wg = wc.as_strided(w.shape, w.stride(), w.storage_offset())
        whole = torch.full((q.shape[0], w.shape[0] + 9), 7.0, device="cuda")
        out = whole[:, 2:2 + w.shape[0]]
        y = k.matmul_i8(qg, a.cuda(), wg, b.cuda(), out=out)
        assert y.data_ptr() == out.data_ptr()
        check_product(y, q, a, w, b, None, torch.float32)
        assert (whole[:, :2] == 7).all() and (whole[:, 2 + w.shape[0]:] == 7).all()


def test_matmul_i8_bad_rows_stay_rows(k):
    """A NaN or infinite row, scale or bias reaches its own row or channel alone."""
    g = rng_for(5)
    x = randn(g, 40, 200)
    x[3, 9], x[30, 0] = float("inf"), float("nan")
    w, ws = randq(g, 50, 200), torch.rand(50, generator=g)
    ws[7] = float("nan")
    q, s = k.quantize_rows(x.cuda())
    y = k.matmul_i8(q, s, w.cuda(), ws.cuda(), out_dtype=torch.float32).cpu()
    bad = torch.isnan(y)
    want = torch.zeros_like(bad)
    want[[3, 30]] = True
    want[:, 7] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("tokens,topk,experts,n,kdim,drop", [
    (1, 1, 1, 5, 16, 0.0), (1, 2, 7, 130, 100, 0.0), (8, 8, 64, 200, 257, 0.1), (40, 2, 3, 128, 128, 0.3), (200, 4, 5, 129, 96, 0.2),
    (600, 2, 33, 100, 130, 0.0), (900, 1, 2, 256, 300, 0.9), (50, 3, 1024, 17, 48, 0.5), (20, 4, 6, 64, 64, 1.0), (3000, 1, 4, 140, 64, 0.05)])
def test_matmul_i8_grouped(k, dtype, tokens, topk, experts, n, kdim, drop):
    g = rng_for(6, tokens, topk, experts)
    ids = random_ids(g, tokens, topk, experts, drop)
    r = k.sort_by_expert(ids.cuda(), experts)
    x = randn(g, tokens, kdim)
    w, ws = randq(g, experts, n, kdim), torch.rand(experts, n, generator=g) / kdim
    bias = randn(g, experts, n) if topk % 2 else None
    q, s = k.dispatch_i8(x.cuda(), r)
    y = k.matmul_i8_grouped(q, s, w.cuda(), ws.cuda(), r.offsets, None if bias is None else bias.cuda(), out_dtype=dtype)
    k.sync()
    offsets = r.offsets.cpu().tolist()
    q, s, y = q.cpu(), s.cpu(), y.cpu()
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        if b > a:
            check_product(y[a:b], q[a:b], s[a:b], w[e], ws[e], None if bias is None else bias[e], dtype)
    assert (y[offsets[-1]:] == 0).all()


def test_matmul_i8_grouped_one_expert_has_all(k):
    g = rng_for(7)
    tokens, experts, n, kdim = 700, 40, 150, 200
    ids = torch.full((tokens, 1), 17)
    r = k.sort_by_expert(ids.cuda(), experts)
    q, w = randq(g, tokens, kdim), randq(g, experts, n, kdim)
    s, ws = torch.rand(tokens, generator=g), torch.rand(experts, n, generator=g)
    y = k.matmul_i8_grouped(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), r.offsets, out_dtype=torch.float32)
    check_product(y, q, s, w[17], ws[17], None, torch.float32)


def test_matmul_i8_grouped_offsets_out_of_order(k):
    """Offsets that no sort made are brought into order and into the rows: nothing is read or written elsewhere."""
    g = rng_for(8)
    q, w = randq(g, 50, 64), randq(g, 4, 10, 64)
    s, ws = torch.ones(50), torch.ones(4, 10) / 64
    offsets = torch.tensor([-5, 30, 20, 2_000_000_000, 40], dtype=torch.int32)
    y = k.matmul_i8_grouped(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), offsets.cuda(), out_dtype=torch.float32).cpu()
    check_product(y[:30], q[:30], s[:30], w[0], ws[0], None, torch.float32)
    check_product(y[30:], q[30:], s[30:], w[2], ws[2], None, torch.float32)


# ---- sort --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,topk,experts", [(1, 1, 1), (1, 8, 64), (5, 2, 3), (33, 1, 10), (1000, 4, 256), (512, 8, 1024), (4097, 1, 1025), (300, 64, 2000),
                                                 (20000, 2, 128), (70000, 1, 16384), (9000, 1, 65536), (100, 1, 65536),
                                                 (16384, 1, 100), (16385, 1, 100), (303104, 1, 3000), (303105, 1, 500), (151553, 2, 1024), (400000, 1, 1025),
                                                 (1024, 1, 65536), (1025, 1, 65536), (512, 2, 1025), (31, 1, 1025), (200, 4, 5000), (1, 2, 30000), (777, 1, 16384),
                                                 (4096, 1, 300), (4097, 1, 300), (500, 8, 1024), (2000, 2, 64)])
def test_sort_by_expert(k, dtype, tokens, topk, experts):
    ids = random_ids(rng_for(9, tokens, topk, experts), tokens, topk, experts, 0.1, dtype)
    check_route(k.sort_by_expert(ids.cuda(), experts), ids, experts)


@pytest.mark.parametrize("n", [10000, 4000, 1000])
@pytest.mark.parametrize("experts", [1, 300, 5000])
def test_sort_extreme_choices(k, experts, n):
    for fill in (0, experts - 1, experts, -1):
        ids = torch.full((n, 1), fill)
        check_route(k.sort_by_expert(ids.cuda(), experts), ids, experts)
    ids = torch.arange(n).view(-1, 1) % (experts + 1)
    check_route(k.sort_by_expert(ids.flip(0).contiguous().cuda(), experts), ids.flip(0), experts)
    ids = torch.tensor([[0, 2**32, -2**32, 2**63 - 1, -2**63, experts - 1]])
    check_route(k.sort_by_expert(ids.cuda(), experts), ids, experts)
    assert k.sort_by_expert(torch.zeros(4, dtype=torch.int64, device="cuda"), experts).position.shape == (4, 1)


# ---- exchange ----------------------------------------------------------------------------------

EXCHANGE = [(1, 1, 1, 1, 0.0), (3, 2, 4, 30, 0.3), (50, 8, 16, 96, 0.1), (33, 4, 7, 200, 0.0), (20, 64, 100, 17, 0.2), (9, 2, 3, 1030, 0.5),
            (130, 6, 8, 2048, 0.1), (5, 3, 2, 4104, 0.2), (40, 2, 5, 64, 1.0), (40, 3, 6, 1004, 0.1), (21, 2, 4, 20, 0.2), (7, 5, 3, 2302, 0.1)]


def setup_exchange(k, seed, tokens, topk, experts, cols, drop, dtype, wtype):
    g = rng_for(seed, tokens, topk, experts, cols)
    ids = random_ids(g, tokens, topk, experts, drop)
    r = k.sort_by_expert(ids.cuda(), experts)
    order, position, offsets = route(ids, experts)
    kept = int(offsets[-1])
    y = randn(g, tokens * topk, cols, dtype=dtype)
    y[kept:] = float("nan")  # never read
    return g, r, order, position, kept, y, randn(g, tokens, topk, dtype=wtype)


@pytest.mark.parametrize("dtype", FLOATS + [torch.int8, torch.uint8, torch.int32])
@pytest.mark.parametrize("tokens,topk,experts,cols,drop", EXCHANGE)
def test_dispatch(k, dtype, tokens, topk, experts, cols, drop):
    g, r, order, position, kept, _, _ = setup_exchange(k, 10, tokens, topk, experts, cols, drop, torch.float32, torch.float32)
    x = randn(g, tokens, cols, dtype=dtype) if dtype.is_floating_point else randq(g, tokens, cols).to(dtype)
    want = x[order // topk]
    want[kept:] = 0
    assert torch.equal(k.dispatch(x.cuda(), r).cpu(), want)
    wide = torch.zeros(tokens, cols + 3, dtype=dtype)
    wide[:, 1:1 + cols] = x
    assert torch.equal(k.dispatch(wide.cuda()[:, 1:1 + cols], r).cpu(), want)
    if dtype.is_floating_point:
        q, s = k.dispatch_i8(x.cuda(), r)
        check_quantised(q[:kept], s[:kept], want[:kept])
        assert (q[kept:] == 0).all() and (s[kept:] == 0).all()
        q1, s1 = k.quantize_rows(x.cuda())
        assert torch.equal(q[:kept].cpu(), q1.cpu()[order[:kept] // topk]) and torch.equal(s[:kept].cpu(), s1.cpu()[order[:kept] // topk])


def combined(y, w, position, kept):
    """(the sum, the sum of its terms' sizes) in 64 bits."""
    rows = y.double()[position.clamp(max=max(kept - 1, 0))]
    rows = torch.where((position < kept)[..., None], rows * w.double()[..., None], 0.0)
    return rows.sum(1), rows.abs().sum(1)


@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("tokens,topk,experts,cols,drop", EXCHANGE)
def test_combine_and_gradient(k, dtype, wtype, tokens, topk, experts, cols, drop):
    g, r, order, position, kept, y, w = setup_exchange(k, 11, tokens, topk, experts, cols, drop, dtype, wtype)
    want, size = combined(y, w, position, kept)
    close(k.combine(y.cuda(), w.cuda(), r), want, (topk + 1) * U * size, dtype)
    want, size = combined(y, torch.ones_like(w), position, kept)
    close(k.combine(y.cuda(), None, r), want, (topk + 1) * U * size, dtype)
    close(k.dispatch_backward(y.cuda(), r), want, (topk + 1) * U * size, dtype)

    dout = randn(g, tokens, cols, dtype=dtype)
    dy, dw = k.combine_backward(dout.cuda(), y.cuda(), w.cuda(), r)
    want = dout.double()[order // topk] * w.double().reshape(-1)[order][:, None]
    want[kept:] = 0
    close(dy, want, U * want.abs(), dtype)
    terms = torch.where((position < kept)[..., None], y.double()[position.clamp(max=max(kept - 1, 0))] * dout.double()[:, None], 0.0)
    close(dw, terms.sum(-1), (cols + 1) * U * terms.abs().sum(-1), wtype)


def test_exchange_strided_rows(k):
    g, r, order, position, kept, y, w = setup_exchange(k, 12, 30, 3, 5, 70, 0.2, torch.bfloat16, torch.float32)
    wide = torch.full((90, 100), float("nan"), dtype=torch.bfloat16)
    wide[:, 11:81] = y
    want, size = combined(y, w, position, kept)
    close(k.combine(wide.cuda()[:, 11:81], w.cuda(), r), want, 4 * U * size, torch.bfloat16)
    dout = randn(g, 30, 70, dtype=torch.bfloat16)
    dwide = torch.zeros(30, 77, dtype=torch.bfloat16)
    dwide[:, 5:75] = dout
    a = k.combine_backward(dout.cuda(), y.cuda(), w.cuda(), r)
    b = k.combine_backward(dwide.cuda()[:, 5:75], wide.cuda()[:, 11:81], w.cuda(), r)
    assert torch.equal(a[0], b[0])
    terms = torch.where((position < kept)[..., None], y.double()[position.clamp(max=kept - 1)] * dout.double()[:, None], 0.0)
    close(b[1], terms.sum(-1), 71 * U * terms.abs().sum(-1), torch.float32)


def test_no_choice_and_infinities(k):
    """A token without a choice gives zeros; an infinity or NaN of a kept row stays in its token and column."""
    ids = torch.tensor([[-1, -1], [0, 5], [1, 0]])
    r = k.sort_by_expert(ids.cuda(), 2)
    y = torch.ones(6, 40)
    y[r.position[1, 0].item(), 3] = float("inf")
    y[r.position[2, 1].item(), 5] = float("nan")
    y[3:] = float("nan")
    out = k.combine(y.cuda(), torch.ones(3, 2, device="cuda"), r).cpu()
    assert (out[0] == 0).all() and out[1, 3] == float("inf") and torch.isnan(out[2, 5])
    assert int((~torch.isfinite(out)).sum()) == 2
    dy, dw = k.combine_backward(torch.ones(3, 40, device="cuda"), y.cuda(), torch.full((3, 2), 2.0, device="cuda"), r)
    assert (dy[:3] == 2).all() and (dy[3:] == 0).all() and (dw[0] == 0).all() and dw[1, 1] == 0 and dw[2, 0] == 40


def test_positions_outside_the_rows_are_dropped(k):
    """Arrays that no sort made lead nowhere: positions outside [0, tokens * topk) count as dropped."""
    import stlq_b200

    position = torch.tensor([[0, -7], [2_000_000_000, 1], [3, -2**31]], dtype=torch.int32, device="cuda")
    for last in (4, 2**31 - 1, -5):
        offsets = torch.tensor([0, last], dtype=torch.int32, device="cuda")
        r = stlq_b200.Routing(torch.zeros(6, dtype=torch.int32, device="cuda"), position, offsets)
        y = torch.arange(6.0, device="cuda")[:, None].expand(6, 9).contiguous()
        out = k.combine(y, None, r)
        want = [0.0, 1.0, 3.0] if last > 0 else [0.0, 0.0, 0.0]
        assert out[:, 4].tolist() == want
        xs = k.dispatch(torch.ones(3, 9, device="cuda"), r)
        assert xs[[0, 1, 3]].eq(1.0 if last > 0 else 0.0).all()
        _, dw = k.combine_backward(torch.ones(3, 9, device="cuda"), y, torch.ones(3, 2, device="cuda"), r)
        assert dw.reshape(-1).tolist() == [9 * v for v in (0.0, 0.0, 0.0, want[1], want[2], 0.0)]


def test_autograd_against_the_formula_and_differences(k):
    """The exchange is linear in its rows and in its weights, so a central difference with a step of 1 is its derivative up to
    rounding: both values carry at most 2 (topk + 2) u times the sum of the sizes of their terms."""
    tokens, topk, experts, cols = 23, 3, 6, 18
    g = rng_for(13)
    ids = random_ids(g, tokens, topk, experts, 0.3).cuda()
    r = k.sort_by_expert(ids, experts)
    x = randn(g, tokens, cols).cuda().requires_grad_()
    w = randn(g, tokens, topk).cuda().requires_grad_()
    gate, dout = randn(g, tokens * topk, cols).cuda(), randn(g, tokens, cols).cuda()

    def loss(x, w):
        return (k.combine(k.dispatch(x, r) * gate, w, r).double() * dout.double()).sum()

    loss(x, w).backward()
    position, kept = r.position.cpu().long(), int(r.offsets[-1])
    hold = (position < kept)[..., None]
    rows = torch.where(hold, gate.double().cpu()[position.clamp(max=kept - 1)], 0.0)  # (tokens, topk, cols)
    parts = rows * w.detach().double().cpu()[..., None] * dout.double().cpu()[:, None]
    assert ((x.grad.double().cpu() - parts.sum(1)).abs() <= (topk + 4) * U * parts.abs().sum(1)).all()
    terms = rows * x.detach().double().cpu()[:, None] * dout.double().cpu()[:, None]
    assert ((w.grad.double().cpu() - terms.sum(-1)).abs() <= (cols + 4) * U * terms.abs().sum(-1)).all()
    with torch.no_grad():
        size = float((rows * (x.double().cpu().abs() + 1)[:, None] * (w.double().cpu().abs() + 1)[..., None] * dout.double().cpu()[:, None]).abs().sum())
        slack = 4 * (topk + 2) * U * size
        for t, c in ((0, 0), (5, 17), (22, 9)):
            for d, grad in ((x, x.grad), (w, w.grad)):
                at = (t, c % d.shape[1])
                up, down = d.clone(), d.clone()
                up[at] += 1
                down[at] -= 1
                args = ((up, w), (down, w)) if d is x else ((x, up), (x, down))
                slope = float(loss(*args[0]) - loss(*args[1])) / 2
                assert abs(slope - float(grad[at])) <= slack
    y = randn(g, tokens * topk, cols).cuda().requires_grad_()
    k.combine(y, None, r).backward(dout)
    want = k.dispatch(dout, r)
    assert torch.equal(y.grad, want)


# ---- the whole layer, streams, graphs, sizes ---------------------------------------------------

def test_routed_layer_on_another_stream_and_in_a_graph(k):
    g = rng_for(14)
    tokens, topk, experts, n, cols = 100, 4, 9, 136, 200
    w, ws = k.quantize_rows(randn(g, experts * n, cols).cuda())
    w, ws = w.unflatten(0, (experts, n)), ws.view(experts, n)
    x, mix = randn(g, tokens, cols, dtype=torch.bfloat16).cuda(), randn(g, tokens, topk).cuda()
    ids = random_ids(g, tokens, topk, experts).cuda()

    def layer():
        r = k.sort_by_expert(ids, experts)
        q, s = k.dispatch_i8(x, r)
        return k.combine(k.matmul_i8_grouped(q, s, w, ws, r.offsets, out_dtype=x.dtype), mix, r)

    want = layer()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [layer() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(y, want) for y in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    x.copy_(x.flip(0))
    ids.copy_(ids.flip(0))
    mix.copy_(mix.flip(0))
    graph.replay()
    assert torch.equal(out, want.flip(0))
    k.sync()


def test_offsets_past_32_bits(k):
    """Matrices of more than 2^31 elements: the last rows are as right as the first."""
    tokens, topk, cols = 36000, 2, 32768
    x = torch.randn(tokens, cols, device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(tokens, topk, dtype=torch.int32, device="cuda")
    r = k.sort_by_expert(ids, 1)
    xs = k.dispatch(x, r)
    assert xs.numel() > 2**31 and torch.equal(xs[-2:], x[-1:].expand(2, cols)) and torch.equal(xs[70000], x[35000])
    out = k.combine(xs, None, r)
    assert torch.equal(out[-1000:], (x[-1000:].float() * 2).bfloat16())
    dy, dw = k.combine_backward(x, xs, torch.full((tokens, topk), 0.5, device="cuda"), r)
    assert torch.equal(dy[-1], x[-1] * 0.5)
    size = float(x[-1].double().square().sum())
    assert abs(float(dw[-1, 1]) - size) <= (cols + 1) * U * size
    del xs, out, dy
    q, s = k.dispatch_i8(x, r)
    assert q.numel() > 2**31 and torch.equal(q[-1], k.quantize_rows(x[-1:])[0][0])
    del x
    w, ws = randq(rng_for(15), 300, cols), torch.ones(300) / cols
    y = k.matmul_i8(q, s, w.cuda(), ws.cuda(), out_dtype=torch.float32)
    check_product(y[-3:], q[-3:].cpu(), s[-3:].cpu(), w, ws, None, torch.float32)
    del y
    n = 65536
    w, ws = randq(rng_for(16), n, 16), torch.ones(n) / 16
    y = k.matmul_i8(q[:33000, :16].contiguous(), s[:33000].contiguous(), w.cuda(), ws.cuda(), out_dtype=torch.bfloat16)
    assert y.numel() > 2**31
    check_product(y[-2:], q[32998:33000, :16].cpu(), s[32998:33000].cpu(), w, ws, None, torch.bfloat16)


# ---- refusals ----------------------------------------------------------------------------------

def test_refusals(k):
    cuda = dict(device="cuda")
    x = torch.zeros(4, 8, **cuda)
    q, s = k.quantize_rows(x)
    r = k.sort_by_expert(torch.zeros(4, 2, dtype=torch.int64, **cuda), 3)
    y, w = torch.zeros(8, 8, **cuda), torch.zeros(4, 2, **cuda)
    W, WS = q.unflatten(0, (2, 2)), s.view(2, 2)
    bad = [
        lambda: k.quantize_rows(x.double()), lambda: k.quantize_rows(x[0]), lambda: k.quantize_rows(x.t()), lambda: k.quantize_rows(x.cpu()),
        lambda: k.quantize_rows(x[:1].expand(4, 8)),
        lambda: k.matmul_i8(q, s, q[:, :7], s), lambda: k.matmul_i8(q, s[:3], q, s), lambda: k.matmul_i8(q, s, q, s[:3]),
        lambda: k.matmul_i8(x, s, q, s), lambda: k.matmul_i8(q, s, q, s, bias=s[:2]), lambda: k.matmul_i8(q, s, q, s, out_dtype=torch.int32),
        lambda: k.matmul_i8(q, s.cpu(), q, s), lambda: k.matmul_i8(q, s, q, s, out=torch.zeros(4, 5, **cuda)),
        lambda: k.matmul_i8(q, s, q, s, out=torch.zeros(4, 8, **cuda)[:, ::2]), lambda: k.matmul_i8(q[0], s, q, s),
        lambda: k.matmul_i8(q, s, q.cpu(), s), lambda: k.matmul_i8(torch.zeros(1, 131072, dtype=torch.int8, **cuda), s[:1], torch.zeros(1, 131072, dtype=torch.int8, **cuda), s[:1]),
        lambda: k.matmul_i8_grouped(q, s, q, s, r.offsets), lambda: k.matmul_i8_grouped(q, s, W, WS, r.offsets),
        lambda: k.matmul_i8_grouped(q, s, W, WS[:1], r.offsets[:3]), lambda: k.matmul_i8_grouped(q, s, W, WS, r.offsets[:3].long()),
        lambda: k.matmul_i8_grouped(q, s, W, WS, r.offsets[:3].cpu()),
        lambda: k.sort_by_expert(torch.zeros(4, 2, **cuda), 3), lambda: k.sort_by_expert(r.position, 0), lambda: k.sort_by_expert(r.position, 65537),
        lambda: k.sort_by_expert(r.position.t(), 3), lambda: k.sort_by_expert(r.position.cpu(), 3), lambda: k.sort_by_expert(torch.zeros(2, 65, dtype=torch.int32, **cuda), 3),
        lambda: k.dispatch(x[:3], r), lambda: k.dispatch(x.double(), r), lambda: k.dispatch_i8(x[:2], r),
        lambda: k.dispatch_i8(q, r), lambda: k.combine(y[:7], w, r), lambda: k.combine(y, w[:3], r), lambda: k.combine(y, w.double(), r),
        lambda: k.combine(y.double(), w, r), lambda: k.combine(y, w.cpu(), r), lambda: k.combine(y, w.t().contiguous().t(), r),
        lambda: k.combine_backward(x, y.half(), w, r), lambda: k.combine_backward(x[:3], y, w, r), lambda: k.combine_backward(x, y[:, :4], w, r),
        lambda: k.combine_backward(x, y, w[:1], r),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")


def test_c_entries_refuse(k):
    """The library checks what the Python layer cannot be trusted to have checked, before anything is launched."""
    import ctypes

    lib, h = k._lib, k.handle
    i, l, z, v = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p
    lib.stlq_b200_quantize_rows.argtypes = [v, v, i, l, l, i, v, l, v, v]
    lib.stlq_b200_matmul_i8.argtypes = [v, v, l, v, v, l, v, v, l, i, i, v, i, l, v]
    lib.stlq_b200_matmul_i8_grouped.argtypes = [v, v, l, v, v, l, v, v, v, i, l, i, i, v, i, l, v]
    lib.stlq_b200_sort_by_expert.argtypes = [v, v, i, l, i, i, v, v, v, v, z, v]
    lib.stlq_b200_dispatch.argtypes = [v, v, i, l, l, i, i, v, v, i, v, l, v]
    lib.stlq_b200_combine.argtypes = [v, v, i, l, l, i, i, v, i, v, v, i, v, l, v]
    lib.stlq_b200_combine_backward.argtypes = [v, v, i, l, v, l, l, i, i, v, i, v, v, i, v, l, v, v]
    t = torch.zeros(4096, device="cuda")
    p = t.data_ptr()
    refused = [
        lib.stlq_b200_quantize_rows(h, p, 1, 8, 4, 8, p, 16, p, None), lib.stlq_b200_quantize_rows(h, p, 0, 7, 4, 8, p, 16, p, None),
        lib.stlq_b200_quantize_rows(h, p + 2, 0, 8, 4, 8, p, 16, p, None), lib.stlq_b200_quantize_rows(h, None, 0, 8, 4, 8, p, 16, p, None),
        lib.stlq_b200_quantize_rows(h, p, 0, 8, -1, 8, p, 16, p, None),
        lib.stlq_b200_matmul_i8(h, p + 8, 16, p, p, 16, p, None, 4, 4, 16, p, 0, 4, None), lib.stlq_b200_matmul_i8(h, p, 24, p, p, 16, p, None, 4, 4, 16, p, 0, 4, None),
        lib.stlq_b200_matmul_i8(h, p, 16, p, p, 16, p, None, 4, 4, 16, p, 5, 4, None), lib.stlq_b200_matmul_i8(h, p, 16, p, p, 16, p, None, 4, 4, 16, p, 0, 3, None),
        lib.stlq_b200_matmul_i8(h, p, 16, None, p, 16, p, None, 4, 4, 16, p, 0, 4, None), lib.stlq_b200_matmul_i8(h, p, 131072, p, p, 131072, p, None, 1, 1, 131072, p, 0, 1, None),
        lib.stlq_b200_matmul_i8_grouped(h, p, 16, p, p, 16, p, None, None, 2, 4, 4, 16, p, 0, 4, None),
        lib.stlq_b200_matmul_i8_grouped(h, p, 16, p, p, 16, p, None, p, 1025, 4, 4, 16, p, 0, 4, None),
        lib.stlq_b200_sort_by_expert(h, p, 0, 4, 2, 3, p, p, p, p, 4096, None), lib.stlq_b200_sort_by_expert(h, p, 4, 40000, 2, 3, p, p, p, p, 1, None),
        lib.stlq_b200_sort_by_expert(h, p, 4, 2**31, 1, 3, p, p, p, p, 4096, None),
        lib.stlq_b200_dispatch(h, p, 8, 8, 4, 8, 2, p, p, 3, p, 8, None), lib.stlq_b200_dispatch(h, p, 4, 8, 4, 8, 65, p, p, 3, p, 8, None),
        lib.stlq_b200_dispatch(h, p, 4, 8, 4, 8, 2, None, p, 3, p, 8, None),
        lib.stlq_b200_combine(h, p, 1, 8, 4, 8, 2, None, 0, p, p, 3, p, 8, None), lib.stlq_b200_combine(h, p, 0, 8, 4, 8, 2, p, 4, p, p, 3, p, 8, None),
        lib.stlq_b200_combine_backward(h, p, 0, 8, p, 8, 4, 8, 2, None, 0, p, p, 3, p, 8, p, None),
        lib.stlq_b200_combine_backward(h, p, 0, 4, p, 8, 4, 8, 2, p, 0, p, p, 3, p, 8, p, None),
    ]
    assert refused == [1] * len(refused)
    assert lib.stlq_b200_last_error()
    k.sync()


def test_example_routed_roots():
    """The example that runs the operators together.  An 8-bit row has at most 1/254 of its largest value's error in each element and
    so has the matrix; over 128 elements with a largest value some 2 to 4 times their root mean square, each gives about 1 %."""
    if not have_cuda():
        pytest.skip("no CUDA device")
    import importlib.util
    import os

    from conftest import ROOT

    spec = importlib.util.spec_from_file_location("routed_roots", os.path.join(ROOT, "examples", "routed_roots.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    error, before, after = m.main(vectors=3000, roots=20, dim=128, out_dim=48)
    assert error < 0.02 and after < before
