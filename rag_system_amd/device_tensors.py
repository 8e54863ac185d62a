"""Checks of the torch tensors that the device entry points are called with.

torch is optional for searching (numpy in, numpy out); the entry points that work on data already in HBM
(IndexFlat.add / distill, adapters.QueryAdapters) take its tensors.  Work runs on torch's current stream of the
tensors' device, workspaces come from torch's allocator on that stream (so a captured graph owns its own), and
results are new tensors that carry no autograd history.

A call on one query is over in the time that Python needs for a handful of attribute look-ups, so the checks are
written for the tensor that passes them.
"""
from . import _lib

_torch = None
_raw_stream = None


def torch_module():
    global _torch, _raw_stream
    if _torch is None:
        import torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _torch = torch
    return _torch


def is_tensor(x):
    """A torch tensor in GPU memory (torch is not imported for the answer)."""
    return getattr(x, "is_cuda", False) is True and type(x).__module__.split(".")[0] == "torch"


def engine_for(t, name):
    """The library, initialised; `t` must be on the GPU it runs on (one process per GPU)."""
    if not is_tensor(t):
        raise ValueError("%s must be a torch tensor in GPU memory, got %s" % (name, type(t).__name__))
    lib = _lib.engine()
    if t.device.index != _lib.device():
        raise ValueError("%s is on %s, the engine runs on device %d (one process per GPU)" % (name, t.device, _lib.device()))
    return lib


def check(t, name, dtype, shape, index):
    """Raise ValueError unless `t` is a tensor of this type and shape (None: any size) on GPU `index`."""
    if not getattr(t, "is_cuda", False) is True:
        raise ValueError("%s must be a torch tensor in GPU memory, got %s" % (name, type(t).__name__))
    if t.dtype != dtype:
        raise ValueError("%s must be of type %s, got %s" % (name, dtype, t.dtype))
    s = t.shape
    if s != shape and (len(s) != len(shape) or any(w is not None and w != g for w, g in zip(shape, s))):
        raise ValueError("%s must have the shape (%s), got %s"
                         % (name, ", ".join("any" if w is None else str(w) for w in shape), tuple(s)))
    if t.get_device() != index:
        raise ValueError("%s is on %s, not on GPU %d" % (name, t.device, index))
    return t


def rows(t):
    """A matrix as the kernels read one: (tensor, distance between its rows in elements).  Rows may lie any distance
    apart; a matrix whose values within a row do, or whose rows overlap, is copied."""
    n, d = t.shape
    if t.is_contiguous():
        return t, d
    if (d > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < d):
        return t.contiguous(), d
    return t, (t.stride(0) if n > 1 else d)


def stream_of(t):
    """hipStream_t of torch's current stream on the tensor's device."""
    if _raw_stream is None:
        torch_module()
    return _raw_stream(t.get_device())


def workspace(n_bytes, like):
    torch = torch_module()
    return torch.empty(max(int(n_bytes), 1), dtype=torch.uint8, device=like.device)
