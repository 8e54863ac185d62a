"""Checks of the torch tensors that the device entry points are called with.

torch is optional for searching (numpy in, numpy out); the entry points that work on data already in HBM
(IndexFlat.add / distill, adapters.QueryAdapters) take its tensors.  Work runs on torch's current stream of the
tensors' device, workspaces come from torch's allocator on that stream (so a captured graph owns its own), and
results are new tensors that carry no autograd history.
"""
from . import _lib


def is_tensor(x):
    """A torch tensor in GPU memory (torch is not imported for the answer)."""
    return type(x).__module__.split(".")[0] == "torch" and getattr(x, "is_cuda", False)


def engine_for(t, name):
    """The library, initialised; `t` must be on the GPU it runs on (one process per GPU)."""
    if not is_tensor(t):
        raise ValueError("%s must be a torch tensor in GPU memory, got %s" % (name, type(t).__name__))
    lib = _lib.engine()
    if t.device.index != _lib.device():
        raise ValueError("%s is on %s, the engine runs on device %d (one process per GPU)" % (name, t.device, _lib.device()))
    return lib


def check(t, name, dtype, shape, like=None):
    """Raise ValueError unless `t` is a GPU tensor of this type and shape (None: any size), on `like`'s device."""
    if not is_tensor(t):
        raise ValueError("%s must be a torch tensor in GPU memory, got %s" % (name, type(t).__name__))
    if t.dtype != dtype:
        raise ValueError("%s must be of type %s, got %s" % (name, dtype, t.dtype))
    if t.dim() != len(shape) or any(s is not None and s != g for s, g in zip(shape, t.shape)):
        raise ValueError("%s must have the shape (%s), got %s"
                         % (name, ", ".join("any" if s is None else str(s) for s in shape), tuple(t.shape)))
    if like is not None and t.device != like.device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, like.device))
    return t


def rows(t):
    """A matrix as the kernels read one: (tensor, distance between its rows in elements).  Rows may lie any distance
    apart; a matrix whose values within a row do, or whose rows overlap, is copied."""
    n, d = t.shape
    if (d > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else d)


def stream_of(t):
    import torch
    return torch.cuda.current_stream(t.device).cuda_stream


def workspace(n_bytes, like):
    import torch
    return torch.empty(max(int(n_bytes), 1), dtype=torch.uint8, device=like.device)
