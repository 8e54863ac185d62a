"""What the operators hold in 32 bits, seen where a rounding to fewer bits cannot hide behind long sums or the output's own
rounding: inputs whose products and sums are exact, and a result that cancels."""
import numpy as np
import pytest
import torch

from _operators import U32
from rag_system_amd import faiss_compat as faiss
from rag_system_amd.adapters import QueryAdapters

pytestmark = pytest.mark.gpu
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def _two_parts(w):
    """float32 values as the sum of two bfloat16 (each rounded to nearest): what such a pair keeps of them."""
    hi = w.bfloat16().float()
    return hi + (w - hi).bfloat16().float()


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("M", [1, 3, 8, 31, 60, 130])
@pytest.mark.parametrize("d", [40, 384, 768, 2050])
def test_weights_of_the_softmax_keep_32_bits(M, d, storage):
    """Student and teacher agree, so that the gradient is what the weights lose.

    Four rows (0, 1, 0 ...) and four (-1, 0, 1, 0 ...); query a (1, 0 ...), temperature 1/2: logits 0 and -2 a, both exact.  The
    teacher's two entries, a row of each kind, have the scores 0 and -2 a: the same softmax, w / (1 + w) for the second kind with
    w = exp(-2 a), and dq = 0.  The a are those bfloat16 values whose w two bfloat16 hold worst.
    Allowed, in units of U32 relative to a probability: an exponential 6 (its argument at most 2, rounded twice, and two
    units of the result) and the same for the teacher's; sums of eight weights and of eight weighted rows 8 each and 2 for the
    shares; the teacher's sum 1; divisions 2 and 2: 45 in all with the second order.  Times 1/temperature = 2 and p <= 1/2."""
    a = torch.arange(64, 129).float() / 128                      # bfloat16, 1/8 to 1 in all: w from 0.78 to 0.13
    a = torch.cat([a / 4, a / 2, a])
    w = torch.exp(-2 * a.double()).float()
    lost = ((w - _two_parts(w)).abs() / w)
    a = a[lost.argsort(descending=True)[:M]]
    if len(a) < M:
        a = a.repeat(-(-M // len(a)))[:M]
    X = torch.zeros(8, d)
    X[0::2, 1] = 1
    X[1::2, 0], X[1::2, 2] = -1, 1
    q = torch.zeros(M, d)
    q[:, 0] = a
    index = faiss.IndexFlat(d, 0, storage=storage)
    index.add(X.to(TYPE[storage]).cuda())
    ids = torch.tensor([[2, 5]]).repeat(M, 1).cuda()
    scores = torch.stack([torch.zeros(M), -2 * a], 1).cuda()
    _, dq = index.distill(q.to(TYPE[storage]).cuda(), ids, scores, 0.5, 1.0)
    assert float(dq.float().abs().max()) <= 45 * U32


def _worst_in_two_parts(k):
    """float32 values in [1, 2) that two bfloat16 hold worst."""
    v = 1 + torch.rand(4096, generator=torch.Generator().manual_seed(1))
    return v[((v - _two_parts(v)).abs() / v).argsort(descending=True)[:k]].tolist()


def _three_parts(v):
    a = torch.tensor(v).bfloat16().float()
    b = (v - a).bfloat16().float()
    return [float(a), float(b), float(v - a - b)]


def _cancelling(n, wide, R, S, c, dtype):
    """W, A, B, scale, slots and x (n x 8): W x = -c in every column, from three products that hold c's 24 bits, and an adapter that adds
    c (slot -1: nothing).  Every product and every sum, in any order, is exact in float32."""
    x = torch.zeros(n, 8)
    x[:, :3], x[:, 5] = 1, 1
    W = torch.zeros(wide, 8)
    W[:, :3] = -torch.tensor(_three_parts(c))
    A, B = torch.zeros(S, R, 8), torch.zeros(S, wide, R)
    A[:, R // 2, 5], B[:, :, R // 2] = 1, 1
    slots = torch.arange(n) % (S + 1) - 1 if S > 2 else torch.arange(n) * (S + 1) // n - 1
    slots = slots.clamp(min=0) if n == 1 else slots
    return (t.to(dtype).cuda() for t in (x, W, A, B)), torch.full((S,), c, device="cuda"), slots.cuda()


# one launch; two launches; tiles of few and of many slots, ranks of one step and of two; ranks that no tile keeps; no whole pieces
SHAPES = [(1, 16, 1, 1), (9, 40, 16, 2), (70, 65, 16, 1), (70, 130, 33, 40), (300, 96, 5, 2), (520, 1904, 16, 2), (520, 1904, 40, 2), (520, 1904, 32, 30),
          (2100, 2000, 100, 2), (4200, 1040, 13, 5)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,wide,R,S", SHAPES)
def test_low_rank_vectors_keep_32_bits(n, wide, R, S, dtype):
    """u = c x and v = c dy enter the products with B and A with all of their bits, whatever the weights' type: y and dx are zero."""
    for c in _worst_in_two_parts(3):
        (x, W, A, B), scale, slots = _cancelling(n, wide, R, S, c, TYPE[dtype])
        want = torch.where(slots >= 0, 0.0, -c).to(x.dtype)[:, None].expand(n, wide)
        assert torch.equal(QueryAdapters(W, A, B, scale).apply(x, slots), want)
        # the backward is the same with the matrices transposed
        bank = QueryAdapters(W.t().contiguous(), B.transpose(1, 2).contiguous(), A.transpose(1, 2).contiguous(), scale)
        dx, _, _ = bank.grad(torch.zeros(n, wide, dtype=x.dtype, device="cuda"), slots, x)
        assert torch.equal(dx, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,wide,R,S", SHAPES)
def test_low_rank_vectors_as_large_as_can_be(n, wide, R, S, dtype):
    """u next to the largest float32, which lies behind the largest bfloat16, and infinite: B u as the formula has it."""
    for c, b in ((3.4e38, 2.0 ** -20), (-3.4e38, 2.0 ** -20), (float("inf"), 0.5), (float("-inf"), 0.5)):
        (x, W, A, B), _, slots = _cancelling(n, wide, R, S, 1.0, TYPE[dtype])
        B *= b
        scale = torch.full((S,), c, device="cuda")
        B[B == 0] = b                            # (an infinity times zero is none)
        A[:, :, 5] = 1
        x2 = x.clone()
        x2[:, 5] = 1.0 / 128                     # (R of them are added; c / 128 stays in range, and is exact)
        if np.isfinite(c):
            A[:, :, 5], x2[:, 5], B[:, :, 1:] = 0, 1, 0
            A[:, 0, 5] = 1
            B[:, :, 0] = b
        low = c * b if np.isfinite(c) else c
        want = torch.where(slots >= 0, torch.tensor(low, dtype=torch.float64), -1.0).to(x.device)
        got = QueryAdapters(W, A, B, scale).apply(x2, slots).double()
        half = torch.finfo(x.dtype).eps / 2 + 8 * U32
        finite = torch.isfinite(want)
        assert torch.equal(torch.isfinite(got), finite[:, None].expand_as(got))
        assert torch.equal(got[~finite], want[~finite][:, None].expand(-1, wide))
        assert float(((got - want[:, None]).abs() / want[:, None].abs())[finite].max()) <= half if finite.any() else True
        bank = QueryAdapters(W.t().contiguous(), B.transpose(1, 2).contiguous(), A.transpose(1, 2).contiguous(), scale)
        dx = bank.grad(torch.zeros(n, wide, dtype=x.dtype, device="cuda"), slots, x2)[0]
        assert torch.equal(dx.double(), got)
