"""GPU: every form of the 8-bit products -- a CTA's own tiles, CTA pairs, clusters that divide the terms, each tile height -- for
one matrix and for segments of awkward lengths, every element against 64 bits.

The library picks the form from the sizes; each case's comment says which form that is on 148 multiprocessors.  Bounds as in
test_gpu_routed.py: the sum is exact, then 4u (|sum s w| + |bias|) and the rounding of the result's type."""
import pytest

from conftest import have_cuda
from test_gpu_routed import FLOATS, U, close, randn, randq, rng_for

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def k():
    if not have_cuda():
        pytest.skip("no CUDA device")
    import stlq_b200

    return stlq_b200.Kernels(0)


def terms8(g, *shape):
    """int8 rows on 16-byte boundaries, with other values after their terms."""
    return randq(g, *shape[:-1], (shape[-1] + 15) // 16 * 16).cuda()[..., :shape[-1]]


def lengths(rows, experts):
    """Rows of each expert: around the heights of tiles and boxes, none, and the rest (all but a few rows) over the last ones."""
    awkward = [1, 31, 0, 33, 127, 129, 0, 255, 257, 63, 16, 240, 15, 17]
    dropped = min(37, rows // 10)
    out, left = [], rows - dropped
    for e in range(experts):
        rest = experts - e
        out.append(left if rest == 1 else min(left // 2, awkward[e]) if e < len(awkward) and experts > 2 else left // rest)
        left -= out[-1]
    return out


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,n,kdim", [
    (5, 130, 48), (900, 300, 48), (600, 1000, 48), (5000, 130, 48), (600, 2000, 100),            # a CTA each, 16, 32, 64 and 128 high
    (5000, 500, 1500), (1500, 2000, 1500), (1493, 2001, 1500), (2999, 1000, 1490),                # pairs
    (130, 130, 2500), (5, 130, 2500), (400, 130, 4096), (20, 1000, 2500),                         # clusters: 16 high by 4 and 8, 32 by 4 and 8
    (1500, 130, 8000), (600, 130, 8000), (599, 129, 7999)])                                       # 64 high by 2 and 4
def test_one_matrix(k, dtype, rows, n, kdim):
    g = rng_for(21, rows, n, kdim)
    q, w = terms8(g, rows, kdim), terms8(g, n, kdim)
    s, ws = torch.rand(rows, generator=g) + 0.01, (torch.rand(n, generator=g) + 0.01) / 128 / kdim
    bias = randn(g, n) if rows % 2 else None
    whole = torch.full((rows, n + 16), 7.0, dtype=dtype, device="cuda")
    out = whole[:, 8:8 + n]
    k.matmul_i8(q, s.cuda(), w, ws.cuda(), None if bias is None else bias.cuda(), out=out)
    k.sync()
    terms = (q.double() @ w.double().t()).cpu() * s.double()[:, None] * ws.double()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.double()
    close(out, terms + b, 4 * U * (terms.abs() + b.abs()), dtype)
    assert (whole[:, :8] == 7).all() and (whole[:, 8 + n:] == 7).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows,n,kdim,experts", [
    (20, 100, 48, 4), (1500, 130, 48, 4), (600, 300, 48, 33), (3000, 130, 48, 3), (2000, 130, 48, 33), (5000, 130, 48, 4), (900, 700, 48, 24),  # a CTA each, 16 to 128 high
    (9000, 130, 1500, 24), (9000, 200, 1500, 33), (3000, 770, 1501, 12), (5000, 500, 1501, 16), (3000, 513, 2500, 24), (5000, 1000, 2500, 33),   # pairs
    (20, 130, 4096, 16), (5, 300, 2500, 6), (5, 100, 2500, 4), (130, 130, 8000, 24), (70, 130, 4096, 12), (20, 300, 2500, 3),                    # clusters: 16 high by 2, 4, 8; 32 by 2, 4, 8
    (400, 130, 8000, 24), (130, 130, 8000, 12), (200, 300, 8000, 16)])                                                                           # 64 high by 2 and 4
def test_segments(k, dtype, rows, n, kdim, experts):
    g = rng_for(22, rows, n, kdim, experts)
    each = lengths(rows, experts)
    offsets = torch.tensor([0] + each).cumsum(0)
    kept = int(offsets[-1])
    assert min(each) >= 0 and rows // 2 <= kept < rows or rows < 10
    q, w = terms8(g, rows, kdim), terms8(g, experts, n, kdim)
    s, ws = torch.rand(rows, generator=g) + 0.01, (torch.rand(experts, n, generator=g) + 0.01) / 128 / kdim
    bias = randn(g, experts, n) if experts % 2 == 0 else None
    # One output on 16-byte boundaries (stores by TMA) and one that is not (stores by the threads); both inside others' memory.
    for pad, at in ((-n % 8 + 8, 0), (3, 1)):
        whole = torch.full((rows, n + pad), 7.0, dtype=dtype, device="cuda")
        out = whole[:, at:at + n]
        k.matmul_i8_grouped(q, s.cuda(), w, ws.cuda(), offsets.int().cuda(), None if bias is None else bias.cuda(), out=out)
        k.sync()
        for e in range(experts):
            a, b = int(offsets[e]), int(offsets[e + 1])
            terms = (q[a:b].double() @ w[e].double().t()).cpu() * s[a:b].double()[:, None] * ws[e].double()
            plus = torch.zeros(n, dtype=torch.float64) if bias is None else bias[e].double()
            close(out[a:b], terms + plus, 4 * U * (terms.abs() + plus.abs()), dtype)
        assert (out[kept:] == 0).all()
        assert (whole[:, :at] == 7).all() and (whole[:, at + n:] == 7).all()
