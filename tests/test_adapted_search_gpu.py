"""Query adapters, search and distillation used together: the training step, its capture, and SearchEngine's calls."""
import numpy as np
import pytest
import torch

from _operators import adapters_grad_ref, adapters_ref, assert_within, distill_ref
from _strategy_fakes import DIM, FakeEmbeddingManager
from rag_system_amd import faiss_compat as faiss
from rag_system_amd.adapters import QueryAdapters
from rag_system_amd.search_engine import SearchEngine
from rag_system_amd.vector_storage import VectorStorage

pytestmark = pytest.mark.gpu


def _bank(S, R, d_in, d_out, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")     # noqa: E731
    return QueryAdapters((r(d_out, d_in) * d_in ** -0.5).to(dtype), (r(S, R, d_in) * d_in ** -0.5).to(dtype),
                         (0.3 * r(S, d_out, R) * R ** -0.5).to(dtype), torch.full((S,), 2.0, device="cuda"))


def _step(bank, index, x, slots, scores, k, over):
    y = bank.apply(x, slots)
    _, ids = index.search(y.float().cpu().numpy(), k)
    ids = torch.from_numpy(ids).cuda()
    loss, dy = index.distill(y, ids, scores, 0.1, 1.0, over)
    return y, ids, loss, dy, bank.grad(x, slots, dy)


@pytest.mark.parametrize("over", ["index", "list"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 6, 70])
def test_training_step(n, dtype, over):
    """Each stage against 64 bits on what the stage before it gave."""
    storage = "bf16" if dtype == torch.bfloat16 else "f32"
    bank = _bank(5, 8, 48, 64, dtype)
    X = torch.nn.functional.normalize(torch.randn(700, 64, device="cuda"), dim=1).to(dtype)
    index = faiss.IndexFlat(64, 0, storage=storage)
    index.add(X)
    x = torch.nn.functional.normalize(torch.randn(n, 48, device="cuda"), dim=1).to(dtype)
    slots = torch.randint(-1, 5, (n,), device="cuda")
    scores = torch.randn(n, 12, device="cuda")
    y, ids, loss, dy, (dx, dA, dB) = _step(bank, index, x, slots, scores, 12, over)
    w = (bank.weight, bank.A, bank.B, bank.scale, slots.tolist())
    assert_within(y, *adapters_ref(x, *w), "y")
    ref_loss, ref_dy, e_loss, e_dy = distill_ref(y, X, ids, scores, 0.1, 1.0, 0, over)
    assert_within(loss, ref_loss, e_loss, "loss")
    assert_within(dy, ref_dy, e_dy, "dy")
    g = adapters_grad_ref(x, *w, dy)
    for name, got in (("dx", dx), ("dA", dA), ("dB", dB)):
        assert_within(got, *g[name], name)


def test_whole_gradient_against_autograd():
    """dA, dB and dx of the mean loss of the whole chain, against torch's autograd through the same formulas in 64 bits.  A logit
    (at most 10, 40 columns) is off by (40 + 6) 2^-24 10 = 2^-15.2, a probability by that and its maximum's, 2^-14.2; what the
    products with the bank add (32 + 40 steps of 2^-24) is far below.  Allowed: 2^-14 of each gradient's largest value."""
    bank = _bank(3, 4, 32, 40, seed=3)
    X = torch.nn.functional.normalize(torch.randn(700, 40, device="cuda"), dim=1)
    index = faiss.IndexFlatIP(40)
    index.add(X)
    n, k, tau = 25, 9, 0.1
    x, slots, z = torch.randn(n, 32, device="cuda"), torch.randint(0, 3, (n,), device="cuda"), torch.randn(n, k, device="cuda")
    ids = torch.randint(0, 700, (n, k), device="cuda")
    y = bank.apply(x, slots)
    loss, dy = index.distill(y, ids, z, tau, 1.0, weights=torch.full((n,), 1.0 / n, device="cuda"))
    dx, dA, dB = bank.grad(x, slots, dy)
    W, A, B, c, xd, Xd = (t.double().clone().requires_grad_() for t in (bank.weight, bank.A, bank.B, bank.scale, x, X))
    yd = xd @ W.t() + c[slots][:, None] * torch.einsum("nor,nr->no", B[slots], torch.einsum("nri,ni->nr", A[slots], xd))
    logits = yd @ Xd.t() / tau
    logp = torch.log_softmax(z.double(), 1)
    want = (logp.exp() * (logp - torch.log_softmax(logits, 1).gather(1, ids))).sum(1)
    want.mean().backward()
    for got, ref in ((loss, want.detach()), (dx, xd.grad), (dA, A.grad), (dB, B.grad)):
        assert float((got.double() - ref).abs().max()) < 2.0 ** -14 * float(ref.abs().max())


def test_captured_training_step():
    """apply, distill and grad in one graph, the bank updated in place between replays, other work beside them."""
    bank = _bank(4, 8, 64, 64, seed=5)
    X = torch.nn.functional.normalize(torch.randn(3000, 64, device="cuda"), dim=1)
    index = faiss.IndexFlatL2(64)
    index.add(X)
    n, k = 40, 10
    x, slots, z = torch.randn(n, 64, device="cuda"), torch.randint(-1, 4, (n,), device="cuda"), torch.randn(n, k, device="cuda")
    ids = torch.randint(0, 3000, (n, k), device="cuda")

    def step():
        y = bank.apply(x, slots)
        loss, dy = index.distill(y, ids, z, 0.5, 1.0)
        return (loss,) + bank.grad(x, slots, dy, input_grad=False)[1:]
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for it in range(4):
        x.normal_()
        g.replay()
        index.search(x.cpu().numpy(), 3)
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), it
        bank.A.sub_(0.1 * out[1])
        bank.B.sub_(0.1 * out[2])


# ---- SearchEngine ---------------------------------------------------------------------------------------------------

class _CrossEncoder:
    def predict(self, pairs):
        return np.array([float(len(set(q.split()) & set(t.split()))) for q, t in pairs])


def _store(n=60):
    em = FakeEmbeddingManager()
    vs = VectorStorage(DIM)
    words = ["alpha", "beta", "gamma", "delta", "index", "query", "row", "page", "score", "merge"]
    rng = np.random.default_rng(4)
    for i in range(n):
        text = " ".join(rng.choice(words, 6)) + " %d" % i
        vs.add_vector(em.embed_query(text), "doc%d" % i, text, "src%d" % i)
    vs.rebuild_bm25_index()
    vs.rebuild_tfidf_index()
    return em, vs


QUERIES = ["alpha beta row", "merge score", "gamma delta page index", "query"]


def test_identity_bank_changes_nothing():
    em, vs = _store()
    eye = QueryAdapters(torch.eye(DIM, device="cuda"), torch.randn(3, 4, DIM, device="cuda"), torch.zeros(3, DIM, 4, device="cuda"))
    plain, adapted = SearchEngine(vs, em), SearchEngine(vs, em, query_adapters=eye)
    for strategy in ("faiss", "hybrid", "multi", "rrf"):
        for adapter in (None, 2):
            a = plain.search_with_strategy(QUERIES[0], strategy, top_k=5)
            b = adapted.search_with_strategy(QUERIES[0], strategy, top_k=5, adapter=adapter)
            assert [r["doc_id"] for r in a] == [r["doc_id"] for r in b]
            # (a product with the identity is exact, a norm of one is off by a few units in the last place)
            assert np.allclose([r["score"] for r in a], [r["score"] for r in b], rtol=0, atol=2e-6)


def test_each_request_gets_its_adapter():
    em, vs = _store()
    bank = _bank(3, 4, DIM, DIM, seed=8)
    se = SearchEngine(vs, em, query_adapters=bank)
    slots = [0, None, 2, 1]
    x = torch.from_numpy(np.stack([em.embed_query(q) for q in QUERIES]))
    y, _ = adapters_ref(x, bank.weight, bank.A, bank.B, bank.scale, [-1 if s is None else s for s in slots])
    y = (y / y.norm(dim=1, keepdim=True)).numpy()
    rows = vs.index.reconstruct_n(0, vs.index.ntotal).astype(np.float64)
    batch = se.search_faiss_batch(QUERIES, top_k=6, adapters=slots)
    for i, (q, s) in enumerate(zip(QUERIES, slots)):
        want = np.sort(rows @ y[i])[::-1][:6]
        for hits in (se.search_faiss(q, top_k=6, adapter=s), batch[i]):
            assert np.allclose([h["score"] for h in hits], want, rtol=0, atol=1e-5)
        for strategy in ("hybrid", "multi", "rrf"):
            assert se.search_with_strategy(q, strategy, top_k=4, adapter=s)
        mmr = se.search_with_strategy(q, "faiss", top_k=4, adapter=s, use_mmr=True, mmr_reuse_index_vectors=True)
        assert mmr[0]["doc_id"] == batch[i][0]["doc_id"]


def test_adapters_need_a_bank():
    em, vs = _store(8)
    se = SearchEngine(vs, em)
    with pytest.raises(ValueError):
        se.search_faiss(QUERIES[0], adapter=0)
    with pytest.raises(ValueError):
        se.search_faiss_batch(QUERIES, adapters=[0, 0, 0, 0])
    with pytest.raises(ValueError):
        se.distill_step(QUERIES)
    se = SearchEngine(vs, em, query_adapters=_bank(2, 2, DIM, DIM))
    for bad in ([0, 0, 0], [0, 1, 2, 0]):
        with pytest.raises(ValueError):
            se.search_faiss_batch(QUERIES, adapters=bad)
    with pytest.raises(ValueError):
        se.distill_step(QUERIES)                    # no cross-encoder


@pytest.mark.parametrize("over", ["index", "list"])
def test_distill_step(over):
    em, vs = _store()
    bank = _bank(2, 4, DIM, DIM, seed=9)
    se = SearchEngine(vs, em, cross_encoder=_CrossEncoder(), query_adapters=bank)
    slots = [0, 1, None, 1]
    loss, dA, dB = se.distill_step(QUERIES, slots, top_k=7, temperature=0.2, over=over)
    x = torch.from_numpy(np.stack([em.embed_query(q) for q in QUERIES])).cuda()
    y = bank.apply(x, slots)
    _, ids = vs.index.search(y.cpu().numpy(), 7)
    z = torch.from_numpy(np.array([se.cross_encoder.predict([(q, vs.chunks_data[j]["chunk"]) for j in row])
                                   for q, row in zip(QUERIES, ids)], dtype=np.float32)).cuda()
    want_loss, dy = vs.index.distill(y, torch.from_numpy(ids).cuda(), z, 0.2, 1.0, over, weights=torch.full((4,), 0.25, device="cuda"))
    _, wA, wB = bank.grad(x, slots, dy, input_grad=False)
    assert torch.equal(loss, want_loss) and torch.equal(dA, wA) and torch.equal(dB, wB)


def test_distill_step_refuses_an_empty_list():
    em, vs = _store(8)
    se = SearchEngine(vs, em, cross_encoder=_CrossEncoder(), query_adapters=_bank(2, 2, DIM, DIM))
    for k in (0, -1):
        with pytest.raises(ValueError, match="top_k"):
            se.distill_step(QUERIES, top_k=k)
