"""The routed 8-bit operators' entry points refuse bad calls on the host, without a GPU."""
import ctypes

import pytest

import stlq_b200
from stlq_b200 import operators

torch = pytest.importorskip("torch")


def test_c_entries_reject_a_null_handle():
    lib = operators._ready()[0]
    i, l, z, v = ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_void_p
    lib.stlq_b200_quantize_rows.argtypes = [v, v, i, l, l, i, v, l, v, v]
    lib.stlq_b200_matmul_i8.argtypes = [v, v, l, v, v, l, v, v, l, i, i, v, i, l, v]
    lib.stlq_b200_matmul_i8_grouped.argtypes = [v, v, l, v, v, l, v, v, v, i, l, i, i, v, i, l, v]
    lib.stlq_b200_sort_by_expert.argtypes = [v, v, i, l, i, i, v, v, v, v, z, v]
    lib.stlq_b200_dispatch.argtypes = [v, v, i, l, l, i, i, v, v, i, v, l, v]
    lib.stlq_b200_dispatch_i8.argtypes = [v, v, i, l, l, i, i, v, v, i, v, l, v, v]
    lib.stlq_b200_combine.argtypes = [v, v, i, l, l, i, i, v, i, v, v, i, v, l, v]
    lib.stlq_b200_combine_backward.argtypes = [v, v, i, l, v, l, l, i, i, v, i, v, v, i, v, l, v, v]
    calls = [
        lambda: lib.stlq_b200_quantize_rows(None, None, 0, 8, 4, 8, None, 16, None, None),
        lambda: lib.stlq_b200_matmul_i8(None, None, 16, None, None, 16, None, None, 4, 4, 16, None, 0, 4, None),
        lambda: lib.stlq_b200_matmul_i8_grouped(None, None, 16, None, None, 16, None, None, 4096, 2, 4, 4, 16, None, 0, 4, None),
        lambda: lib.stlq_b200_sort_by_expert(None, None, 4, 4, 2, 3, None, None, None, None, 0, None),
        lambda: lib.stlq_b200_dispatch(None, None, 4, 8, 4, 8, 2, None, None, 3, None, 8, None),
        lambda: lib.stlq_b200_dispatch_i8(None, None, 0, 8, 4, 8, 2, None, None, 3, None, 16, None, None),
        lambda: lib.stlq_b200_combine(None, None, 0, 8, 4, 8, 2, None, 0, None, None, 3, None, 8, None),
        lambda: lib.stlq_b200_combine_backward(None, None, 0, 8, None, 8, 4, 8, 2, None, 0, None, None, 3, None, 8, None, None),
        lambda: lib.stlq_b200_kernels_sync(None, None),
    ]
    for call in calls:
        assert call() == 1
        assert b"handle is null" in lib.stlq_b200_last_error()


@pytest.mark.parametrize("tokens,topk,experts,rc", [(0, 1, 1, 0), (1, 1, 1, 0), (1000, 8, 256, 0), (1 << 20, 1, 65536, 0), (1, 1, 0, 1), (1, 1, 65537, 1),
                                                    (1, 0, 4, 1), (1, 65, 4, 1), (-1, 1, 4, 1), (1 << 31, 1, 4, 1), (1 << 30, 2, 4, 1)])
def test_sort_workspace(tokens, topk, experts, rc):
    lib = operators._ready()[0]
    lib.stlq_b200_sort_by_expert_workspace.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_size_t)]
    size = ctypes.c_size_t(7)
    assert lib.stlq_b200_sort_by_expert_workspace(tokens, topk, experts, ctypes.byref(size)) == rc
    assert (size.value == 0) if rc or tokens == 0 else (size.value < (1 << 31))
    assert (size.value > 0) == (rc == 0 and tokens * topk > (4096 if experts <= 1024 else 1024))
    assert lib.stlq_b200_sort_by_expert_workspace(1, 1, 1, None) == 1


def test_routing_checks_its_arrays():
    def make(order=6, position=(3, 2), offsets=5, dtype=torch.int32):
        return stlq_b200.Routing(torch.zeros(order, dtype=dtype), torch.zeros(position, dtype=dtype), torch.zeros(offsets, dtype=dtype))

    r = make()
    assert (r.tokens, r.topk, r.experts) == (3, 2, 4) and "tokens=3" in repr(r)
    for bad in (dict(order=5), dict(offsets=1), dict(position=(3, 0), order=0), dict(dtype=torch.int64), dict(position=(6,)),
                dict(position=(2, 65), order=130), dict(offsets=65538)):
        with pytest.raises(ValueError):
            make(**bad)


def test_kernels_need_a_gpu_or_say_so():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(stlq_b200.StlqB200Error):
        stlq_b200.Kernels(0)
