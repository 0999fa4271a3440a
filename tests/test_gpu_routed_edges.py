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
