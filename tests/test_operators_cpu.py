"""Query adapters and distillation where there is no GPU: what they refuse, and the 64-bit references of the GPU tests."""
import ctypes as C

import numpy as np
import pytest
import torch

from _operators import adapters_grad_ref, adapters_ref, distill_ref
from rag_system_amd import _lib, faiss_compat as faiss
from rag_system_amd.adapters import QueryAdapters


def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="GPU memory"):
        QueryAdapters(torch.zeros(4, 4), torch.zeros(1, 2, 4), torch.zeros(1, 4, 2))
    with pytest.raises(ValueError, match="GPU memory"):
        QueryAdapters(np.zeros((4, 4), np.float32), np.zeros((1, 2, 4)), np.zeros((1, 4, 2)))


class _Backend:
    def __init__(self, d, metric, *a):
        self.ntotal, self.d = 0, d


def test_distill_refuses_host_data_and_backends_without_it():
    faiss.set_backend_factory(_Backend)
    try:
        index = faiss.IndexFlatIP(4)
        with pytest.raises(NotImplementedError):
            index.distill(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))
        with pytest.raises(ValueError):
            index.distill(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), over="rows")
        index._b.distill = lambda *a: None
        with pytest.raises(ValueError, match="GPU memory"):
            index.distill(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))
        with pytest.raises(ValueError, match="GPU memory"):
            index.distill(np.zeros((2, 4), np.float32), np.zeros((2, 1), np.int64), np.zeros((2, 1), np.float32))
    finally:
        faiss.set_backend_factory(None)


def test_workspace_sizes_and_their_refusals():
    lib, out = _lib.load_library(), C.c_int64()
    assert lib.rag_adapter_ws_bytes(0, 64, 384, 384, 8, 16, 0, C.byref(out)) == 0
    small = out.value
    assert lib.rag_adapter_ws_bytes(1, 64, 384, 384, 8, 16, 1, C.byref(out)) == 0 and out.value > small > 0
    for bad in ((2, 1, 4, 4, 1, 1), (0, -1, 4, 4, 1, 1), (0, (1 << 24) + 1, 4, 4, 1, 1), (0, 1, 0, 4, 1, 1), (0, 1, 4, 8193, 1, 1),
                (0, 1, 4, 4, 0, 1), (0, 1, 4, 4, 4097, 1), (0, 1, 4, 4, 1, 0), (0, 1, 4, 4, 1, 129)):
        assert lib.rag_adapter_ws_bytes(*bad, 0, C.byref(out)) == _lib.RAG_ERR_INVALID_ARG, bad
    assert lib.rag_adapter_ws_bytes(0, 1, 4, 4, 1, 1, 0, None) == _lib.RAG_ERR_INVALID_ARG


def test_nothing_runs_before_init():
    lib = _lib.load_library()
    if lib.rag_device_count() > 0:
        pytest.skip("a GPU is visible")
    z = C.c_void_p(0)
    assert lib.rag_adapter_apply_dev(0, 1, 4, 4, 1, 1, z, 4, z, z, z, z, z, z, 4, z, 0, z) == _lib.RAG_ERR_NOT_INIT
    assert lib.rag_adapter_grad_dev(0, 1, 4, 4, 1, 1, z, 4, z, z, z, z, z, z, 4, z, 4, z, z, z, 0, z) == _lib.RAG_ERR_NOT_INIT
    assert lib.rag_flat_distill_dev(z, 1, z, 4, 1, z, z, 0.1, 1.0, 0, z, z, z, 4, z, 0, z) == _lib.RAG_ERR_NOT_INIT
    assert lib.rag_flat_distill_ws_bytes(z, 1, 1, 0, 1, C.byref(C.c_int64())) == _lib.RAG_ERR_NOT_INIT


@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("over", ["list", "index"])
def test_distill_reference_against_differences(metric, over):
    """The reference's own gradient, by central differences in 64 bits."""
    g = torch.Generator().manual_seed(1)
    q, X = torch.randn(3, 5, generator=g).double(), torch.randn(11, 5, generator=g).double()
    ids, z = torch.tensor([[0, 4, 4], [9, -1, 2], [-1, -1, -1]]), torch.randn(3, 3, generator=g)
    f = lambda t: distill_ref(t, X, ids, z, 0.7, 1.3, metric, over)    # noqa: E731
    _, dq, _, _ = f(q)
    for j in range(5):
        h = torch.zeros_like(q)
        h[:, j] = 1e-5
        diff = (f(q + h)[0] - f(q - h)[0]) / 2e-5
        assert float((diff - dq[:, j]).abs().max()) < 1e-8
    assert float(f(q)[0][2]) == 0 and not dq[2].any()


def test_adapter_reference_against_autograd():
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).double().requires_grad_()     # noqa: E731
    x, W, A, B, c, dy = r(6, 5), r(4, 5), r(3, 2, 5), r(3, 4, 2), r(3), torch.randn(6, 4, generator=g).double()
    slots = [0, -1, 2, 2, 1, 0]
    y = torch.stack([W @ x[t] + (c[s] * (B[s] @ (A[s] @ x[t])) if s >= 0 else 0) for t, s in enumerate(slots)])
    assert float((y - adapters_ref(x, W, A, B, c, slots)[0]).abs().max()) < 1e-12
    (y * dy).sum().backward()
    ref = adapters_grad_ref(x, W, A, B, c, slots, dy)
    for name, t in (("dx", x), ("dA", A), ("dB", B)):
        assert float((ref[name][0] - t.grad).abs().max()) < 1e-12


@pytest.mark.parametrize("dtype,d_in,d_out", [(1, 8191, 8), (0, 4095, 4), (1, 8190, 16)])
@pytest.mark.parametrize("n", [1 << 21, 1 << 22, (1 << 22) + 77, 1 << 23, 1 << 24])
def test_no_filled_up_copies_of_more_pieces_than_are_counted(n, dtype, d_in, d_out):
    """The copies' 16-byte pieces are counted in 32 bits: a backward whose x has 2^31 or more of them is served without copies (a
    workspace with no room for one of x)."""
    lib, out = _lib.load_library(), C.c_int64()
    e, size = (8, 2) if dtype == 1 else (4, 4)
    whole = (d_in + e - 1) // e * e
    pieces = n * (whole // e)
    assert lib.rag_adapter_ws_bytes(dtype, n, d_in, d_out, 2, 1, 1, C.byref(out)) == 0
    if pieces >= 1 << 31:
        assert out.value < n * whole * size
