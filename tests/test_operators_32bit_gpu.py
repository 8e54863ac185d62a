"""What the operators hold in 32 bits, seen where a rounding to fewer bits cannot hide behind long sums or the output's own
rounding: inputs whose products and sums are exact, and a result that cancels."""
import numpy as np
import pytest
import torch

from _operators import U32
from rag_system_amd import faiss_compat as faiss

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
