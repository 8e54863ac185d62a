"""Low-rank query adapters: one shared projection and a bank of small corrections, one slot per store, user or task.

The reference searches with the embedding model's vector as it is (search_engine.py:141); a QueryAdapters bank turns it
into the vector that its requester's adapter says, for many requesters in one call:

    y_t = W x_t + scale[s] B[s] (A[s] x_t),    s = slots[t]   (-1: no adapter)

    bank = QueryAdapters(W, A, B, scale)             # torch tensors in HBM, float32 or bfloat16
    y = bank.apply(x, slots)                          # n x d_out
    dx, dA, dB = bank.grad(x, slots, dy)              # gradients; W is frozen

SearchEngine(..., query_adapters=bank) applies it to its queries, and SearchEngine.distill_step trains it against the
cross-encoder (IndexFlat.distill).  The tensors stay the caller's: an optimiser that updates A and B in place is seen
by the next call.  Kernels: csrc/adapter.hip (rag_adapter_apply_dev, rag_adapter_grad_dev).
"""
import ctypes as C

import numpy as np

from . import _lib, device_tensors as dt

MAX_SLOTS = 4096
MAX_RANK = 128
MAX_REQUESTS = 1 << 24


class QueryAdapters:
    """weight: d_out x d_in.  A: slots x rank x d_in.  B: slots x d_out x rank.  All float32 or all bfloat16, contiguous,
    on the engine's GPU.  scale: slots float32 (None: ones), usually alpha / rank.  A slot of lower rank has zeros in
    its last rows of A and columns of B."""

    def __init__(self, weight, A, B, scale=None):
        torch = dt.torch_module()
        self._lib = dt.engine_for(weight, "weight")
        self._index = weight.get_device()
        if weight.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError("weight must be of type float32 or bfloat16, got %s" % weight.dtype)
        dt.check(weight, "weight", weight.dtype, (None, None), self._index)
        self.d_out, self.d_in = (int(v) for v in weight.shape)
        dt.check(A, "A", weight.dtype, (None, None, self.d_in), self._index)
        self.n_slots, self.rank = int(A.shape[0]), int(A.shape[1])
        if not 1 <= self.n_slots <= MAX_SLOTS or not 1 <= self.rank <= MAX_RANK:
            raise ValueError("%d slots of rank %d: 1 to %d slots of rank 1 to %d are served"
                             % (self.n_slots, self.rank, MAX_SLOTS, MAX_RANK))
        if not 1 <= self.d_in <= 8192 or not 1 <= self.d_out <= 8192:
            raise ValueError("d_in=%d, d_out=%d: widths of 1 to 8192 are served" % (self.d_in, self.d_out))
        if scale is None:
            scale = torch.ones(self.n_slots, dtype=torch.float32, device=weight.device)
        self.weight, self.A, self.B, self.scale = weight, A, B, scale
        self._code = _lib.DTYPE_BF16 if weight.dtype == torch.bfloat16 else _lib.DTYPE_F32
        self._dtype, self._f32, self._i64 = weight.dtype, torch.float32, torch.int64
        self._shapes = ((self.d_out, self.d_in), (self.n_slots, self.rank, self.d_in), (self.n_slots, self.d_out, self.rank),
                        (self.n_slots,))
        self._ws_bytes = {}
        self._weights()

    @property
    def dtype(self):
        return self._dtype

    @property
    def device(self):
        return self.weight.device

    def _weights(self):
        """Pointers of the bank as it is now (the tensors may have been replaced since)."""
        out = []
        for name, t, shape in zip(("weight", "A", "B", "scale"), (self.weight, self.A, self.B, self.scale), self._shapes):
            dt.check(t, name, self._f32 if name == "scale" else self._dtype, shape, self._index)
            if not t.is_contiguous():
                raise ValueError("%s must be contiguous" % name)
            out.append(t.data_ptr())
        return out

    def slots_tensor(self, slots, n):
        """slots as the kernels read them: int64, n of them, in HBM.  A sequence of integers (None: no adapter) is checked
        here; a tensor on the GPU is taken as it is (a request outside [-1, n_slots) gets NaN)."""
        torch = dt.torch_module()
        if dt.is_tensor(slots):
            if slots.dtype == torch.int32:
                slots = slots.to(torch.int64)
            dt.check(slots, "slots", self._i64, (n,), self._index)
            return slots if slots.is_contiguous() else slots.contiguous()
        host = np.array([-1 if s is None else s for s in np.asarray(slots, dtype=object).reshape(-1)], dtype=object)
        if len(host) != n:
            raise ValueError("%d slots for %d requests" % (len(host), n))
        if any(int(s) != s or not -1 <= s < self.n_slots for s in host):
            raise ValueError("slots must be integers in [-1, %d)" % self.n_slots)
        return torch.from_numpy(host.astype(np.int64)).to(self.device)

    def _input(self, t, name, width):
        dt.check(t, name, self._dtype, (None, width), self._index)
        if t.shape[0] > MAX_REQUESTS:
            raise ValueError("%s has %d rows: at most %d are served" % (name, t.shape[0], MAX_REQUESTS))
        return dt.rows(t.detach() if t.requires_grad else t)

    def _workspace(self, n, want_grad):
        need = self._ws_bytes.get((n, want_grad))
        if need is None:
            out = C.c_int64()
            _lib.check(self._lib.rag_adapter_ws_bytes(self._code, n, self.d_in, self.d_out, self.n_slots, self.rank, want_grad,
                                                      C.byref(out)), self._lib)
            if len(self._ws_bytes) > 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[(n, want_grad)] = out.value
        return dt.workspace(need, self.weight), need

    def apply(self, x, slots):
        """x: n x d_in, of the bank's type, in HBM.  Returns y, n x d_out, of the same type (rounded once from float32
        sums).  On torch's current stream; may be captured into a graph (with slots in HBM)."""
        x, ldx = self._input(x, "x", self.d_in)
        n = x.shape[0]
        slots = self.slots_tensor(slots, n)
        w, a, b, scale = self._weights()
        y = x.new_empty((n, self.d_out))
        ws, ws_bytes = self._workspace(n, 0)
        rc = self._lib.rag_adapter_apply_dev(self._code, n, self.d_in, self.d_out, self.n_slots, self.rank, x.data_ptr(), ldx, w, a, b,
                                             scale, slots.data_ptr(), y.data_ptr(), self.d_out, ws.data_ptr(), ws_bytes,
                                             dt.stream_of(x))
        if rc:
            _lib.check(rc, self._lib)
        return y

    def grad(self, x, slots, dy, input_grad=True):
        """Backward of apply(): (dx, dA, dB) for the gradient dy of y.  dx has the type of x (None with
        input_grad=False: embeddings of a frozen model need none); dA and dB are float32 and whole (zeros for slots
        that no request has).  Equal calls give equal bits."""
        x, ldx = self._input(x, "x", self.d_in)
        dy, lddy = self._input(dy, "dy", self.d_out)
        n = x.shape[0]
        if dy.shape[0] != n:
            raise ValueError("dy has %d rows, x has %d" % (dy.shape[0], n))
        slots = self.slots_tensor(slots, n)
        w, a, b, scale = self._weights()
        dx = x.new_empty((n, self.d_in)) if input_grad else None
        dA = x.new_empty(self._shapes[1], dtype=self._f32)
        dB = x.new_empty(self._shapes[2], dtype=self._f32)
        ws, ws_bytes = self._workspace(n, 1)
        rc = self._lib.rag_adapter_grad_dev(self._code, n, self.d_in, self.d_out, self.n_slots, self.rank, x.data_ptr(), ldx, w, a, b,
                                            scale, slots.data_ptr(), dy.data_ptr(), lddy, dx.data_ptr() if input_grad else None,
                                            self.d_in, dA.data_ptr(), dB.data_ptr(), ws.data_ptr(), ws_bytes, dt.stream_of(x))
        if rc:
            _lib.check(rc, self._lib)
        return dx, dA, dB

    def apply_host(self, x, slots):
        """apply() for a host array (n x d_in), as the embedding manager returns it: n x d_out float32 on the host."""
        torch = dt.torch_module()
        x = np.ascontiguousarray(x, dtype=np.float32).reshape(-1, self.d_in)
        return self.apply(torch.from_numpy(x).to(self.device).to(self.dtype), slots).float().cpu().numpy()
