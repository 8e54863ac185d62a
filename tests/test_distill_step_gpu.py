"""SearchEngine.distill_step trains the score that its strategies serve: the adapted query at unit length."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from _strategy_fakes import DIM, FakeEmbeddingManager
from rag_system_amd import faiss_compat as faiss
from rag_system_amd.adapters import QueryAdapters
from rag_system_amd.search_engine import SearchEngine

pytestmark = pytest.mark.gpu
QUERIES = ["alpha beta row", "merge score", "gamma delta page index", "query", "beta beta merge"]
SLOTS = [0, 1, None, 1, 2]


class _CrossEncoder:
    def __init__(self):
        self.asked = []

    def predict(self, pairs):
        self.asked.append([t for _, t in pairs])
        return np.array([2.0 * np.sin(7.0 * len(q) + 3.0 * int(t.split()[-1])) for q, t in pairs])


def _engine(width, metric, n=60, seed=1, spread=3.0):
    """An index of `width` columns beside a bank DIM -> width whose results are of many lengths (spread)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")     # noqa: E731
    bank = QueryAdapters(spread * r(width, DIM), r(3, 4, DIM), r(3, width, 4), torch.full((3,), 1.5, device="cuda"))
    X = torch.nn.functional.normalize(r(n, width), dim=1)
    index = faiss.IndexFlat(width, metric)
    index.add(X)
    store = SimpleNamespace(index=index, indices_present={"faiss"}, chunks_data=[{"chunk": "row %d" % i, "doc_id": "d%d" % i} for i in range(n)])
    return SearchEngine(store, FakeEmbeddingManager(), cross_encoder=_CrossEncoder(), query_adapters=bank), bank, X


def _served(bank, A, B):
    """The served queries in 64 bits, as a function of the adapters."""
    em = FakeEmbeddingManager()
    x = torch.from_numpy(np.stack([em.embed_query(q) for q in QUERIES])).double().cuda()
    y = []
    for t, s in enumerate(SLOTS):
        v = bank.weight.double() @ x[t]
        y.append(v if s is None else v + bank.scale[s].double() * (B[s] @ (A[s] @ x[t])))
    y = torch.stack(y)
    return y / y.norm(dim=1, keepdim=True)


@pytest.mark.parametrize("over", ["index", "list"])
@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("width", [DIM // 2, DIM, DIM + 8])
def test_gradient_of_the_served_score(width, metric, over):
    """Loss, dA and dB of the mean loss against autograd in 64 bits through the normalised query.  y is a sum of 16 + 4 products, off by
    2^-18 of its products' magnitudes, 2^-16 of its length; a logit (beta 2, at most 8 for the squared distance) by sqrt(24) 2^-16 2 and its own sum's
    (24 + 6) 2^-24 8, together below 2^-12.5; a probability by twice that, 2^-11.5; the gradient's parts by as much of what they are
    before they cancel, beta |x| = 2 and, at most, the largest value of each gradient times 2: allowed is 2^-10 of that."""
    se, bank, X = _engine(width, metric)
    tau, k = 0.5, 9
    loss, dA, dB = se.distill_step(QUERIES, SLOTS, top_k=k, temperature=tau, teacher_temperature=1.5, over=over)
    A, B = bank.A.double().requires_grad_(), bank.B.double().requires_grad_()
    q = _served(bank, A, B)
    s = q @ X.double().t() if metric == 0 else -((q[:, None] - X.double()[None]) ** 2).sum(2)
    # the teacher is asked about the list that is served
    ids = s.detach().topk(k, dim=1).indices
    asked = se.cross_encoder.asked[0]
    assert asked == ["row %d" % j for row in ids.tolist() for j in row]
    z = torch.tensor(se.cross_encoder.predict([(QUERIES[t], "row %d" % j) for t in range(len(QUERIES)) for j in ids[t].tolist()]),
                     device="cuda").reshape(len(QUERIES), k) / 1.5
    logp = torch.log_softmax(z, 1)
    mine = (s / tau).gather(1, ids)
    lse = torch.logsumexp(s / tau if over == "index" else mine, 1)
    want = (logp.exp() * (logp - mine)).sum(1) + lse
    want.mean().backward()
    for got, ref in ((loss, want.detach()), (dA, A.grad), (dB, B.grad)):
        assert float((got.double() - ref).abs().max()) < 2.0 ** -10 * float(ref.abs().max())


@pytest.mark.parametrize("over", ["index", "list"])
def test_gradient_against_differences(over):
    """Central differences of distill_step's own mean loss along directions of the bank (every row in the list, so that the list
    does not change).  Temperature 1: a loss is off by less than 2^-18 (logits of 24 products, at most 1), a step of 2^-6 leaves
    2^-12 of that; the unit query turns by at most |direction| <= 1, so the third derivative times 2^-12 / 6 is below 2^-11."""
    se, bank, X = _engine(24, 0)
    h = 2.0 ** -6
    step = lambda: se.distill_step(QUERIES, SLOTS, top_k=60, temperature=1.0, over=over)     # noqa: E731
    _, dA, dB = step()
    g = torch.Generator(device="cuda").manual_seed(5)
    for t, grad in ((bank.A, dA), (bank.B, dB)):
        for _ in range(4):
            v = torch.randn(t.shape, generator=g, device="cuda")
            v += 3 * grad * v.norm() / grad.norm()               # (mostly along the gradient: the change is one that shows)
            v /= v.norm()
            keep = t.clone()
            t.copy_(keep + h * v)
            up = step()[0].double().mean()
            t.copy_(keep - h * v)
            dn = step()[0].double().mean()
            t.copy_(keep)
            assert abs(float((up - dn) / (2 * h)) - float((grad.double() * v.double()).sum())) < 2.0 ** -10


def test_length_of_the_adapted_query_does_not_count():
    """A bank k times as long serves the same scores: the same loss, and 1/k of the gradients with respect to what is k times as
    large.  (k a power of two: every product and norm is scaled exactly.)"""
    se, bank, _ = _engine(24, 0)
    loss, dA, dB = se.distill_step(QUERIES, SLOTS, top_k=9, temperature=0.5)
    bank.weight.mul_(8)
    bank.B.mul_(8)
    loss8, dA8, dB8 = se.distill_step(QUERIES, SLOTS, top_k=9, temperature=0.5)
    assert torch.equal(loss, loss8) and torch.equal(dA, dA8) and torch.equal(dB, 8 * dB8)


def test_an_adapted_query_of_length_zero():
    """A norm below 1e-9 counts as 1, in the search and in its gradient: loss and gradients are finite."""
    se, bank, _ = _engine(24, 0)
    bank.weight.zero_()
    bank.B.zero_()
    loss, dA, dB = se.distill_step(QUERIES, SLOTS, top_k=9, temperature=0.5)
    assert torch.isfinite(loss).all() and torch.isfinite(dB).all() and bool(dB.any()) and not dA.any()


@pytest.mark.parametrize("bank_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_types_of_bank_and_index(storage, bank_type):
    """Every pair of types takes a step, close to the float32 one (bfloat16 holds 2^-8; the gradients are sums of some ten terms)."""
    se, bank, X = _engine(24, 0)
    want = se.distill_step(QUERIES, SLOTS, top_k=60, temperature=1.0)
    index = faiss.IndexFlat(24, 0, storage=storage)
    index.add(X)
    se.vector_storage.index = index
    se.query_adapters = QueryAdapters(*(t.to(bank_type) for t in (bank.weight, bank.A, bank.B)), bank.scale)
    got = se.distill_step(QUERIES, SLOTS, top_k=60, temperature=1.0)
    for a, b in zip(got, want):
        assert a.dtype == torch.float32 and float((a - b).abs().max()) <= 2.0 ** -3 * float(b.abs().max())


def test_queries_without_a_vector():
    """An embedding of NaN finds no row: the teacher is not asked about it, its loss is 0, and NaN reaches its own slot alone.  Where no
    query finds a row there is nothing to learn from, and the call says so."""
    se, bank, _ = _engine(24, 0)
    embed = se.embedding_manager.model.encode
    which = []

    class Model:
        def encode(self, texts):
            v = np.array(embed(texts))
            v[which] = np.nan
            return v
    se.embedding_manager.model = Model()
    want = se.distill_step(QUERIES, [0, 1, 2, 0, 0], top_k=9, temperature=0.5)
    which += [1]
    loss, dA, dB = se.distill_step(QUERIES, [0, 1, 2, 0, 0], top_k=9, temperature=0.5)
    assert len(se.cross_encoder.asked[1]) == 4 * 9 and float(loss[1]) == 0
    for t, w in ((loss[[0, 2, 3, 4]], want[0][[0, 2, 3, 4]]), (dA[[0, 2]], want[1][[0, 2]]), (dB[[0, 2]], want[2][[0, 2]])):
        assert torch.equal(t, w)
    which += [0, 2, 3, 4]
    with pytest.raises(ValueError, match="no query finds"):
        se.distill_step(QUERIES, [0, 1, 2, 0, 0], top_k=9, temperature=0.5)
    assert len(se.cross_encoder.asked) == 2
