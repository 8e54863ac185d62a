"""IndexFlat.distill (rag_flat_distill_dev) against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from _operators import U32, assert_within, distill_ref
from rag_system_amd import _lib, faiss_compat as faiss

pytestmark = pytest.mark.gpu
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
PAD = -3.4028234663852886e38


def make(M, N, d, K, storage="f32", metric=0, seed=0, ragged=True, extra=0):
    """(index, X, q, ids, scores); rows of unit length, queries near a row, lists of several lengths (one of them empty)."""
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + 7 * M + 3 * N + d + K)
    X = torch.randn(N, d, generator=g, device="cuda")
    X = (X / X.norm(dim=1, keepdim=True).clamp(min=1e-6)).to(TYPE[storage])
    src = torch.randint(0, N, (M,), generator=g, device="cuda")
    q = X[src].float() + 0.5 * d ** -0.5 * torch.randn(M, d, generator=g, device="cuda")
    q = q.to(TYPE[storage])
    ids = torch.randint(0, N, (M, K), generator=g, device="cuda")     # the same row twice now and then
    if K:
        ids[:, 0] = src
    scores = 2 * torch.randn(M, K, generator=g, device="cuda")
    if ragged and M > 2 and K:
        end = torch.randint(0, K + 1, (M, 1), generator=g, device="cuda")
        end[M // 2], end[0] = 0, K
        behind = torch.arange(K, device="cuda")[None] >= end
        ids, scores = torch.where(behind, -1, ids), torch.where(behind, PAD, scores)
    index = faiss.IndexFlat(d, metric, storage=storage)
    index.add(X)
    assert index.ntotal == N
    return index, X, q, ids, scores


def check(index, X, q, ids, scores, over, metric, tau=0.1, tau_t=1.5, weights=None, grad=True, **kw):
    loss, dq = index.distill(q, ids, scores, tau, tau_t, over, weights, grad)
    ref_loss, ref_dq, e_loss, e_dq = distill_ref(q, X, ids, scores, tau, tau_t, metric, over, weights)
    assert_within(loss, ref_loss, e_loss, "loss")
    assert loss.dtype == torch.float32
    if grad:
        assert dq.dtype == q.dtype
        assert_within(dq, ref_dq, e_dq, "dq")
    else:
        assert dq is None
    return loss, dq


@pytest.mark.parametrize("over", ["list", "index"])
@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("M,N,d,K", [(1, 1, 1, 1), (1, 2, 3, 2), (1, 300, 384, 10), (3, 33, 64, 7), (5, 31, 100, 3),
                                     (16, 257, 128, 16), (17, 300, 387, 33), (33, 129, 770, 5), (64, 64, 32, 64),
                                     (65, 320, 384, 10), (130, 290, 96, 9), (260, 200, 40, 4), (7, 300, 1030, 8)])
def test_small(M, N, d, K, metric, storage, over):
    index, X, q, ids, scores = make(M, N, d, K, storage, metric)
    check(index, X, q, ids, scores, over, metric)


@pytest.mark.parametrize("storage,d", [("f32", 1536), ("f32", 1540), ("bf16", 2050), ("f32", 8192), ("bf16", 8192)])
def test_long_rows(storage, d):
    for over in ("list", "index"):
        for M in (1, 40):
            index, X, q, ids, scores = make(M, 70, d, 6, storage, 0)
            check(index, X, q, ids, scores, over, 0)


@pytest.mark.parametrize("M", [1, 2, 8, 31, 48, 100, 300])
@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_many_rows(M, storage):
    """Rows over all splits and tiles; every row's weight has to arrive (a row left out is 1/N of the mass, 60 times what
    is allowed)."""
    N = 5003
    index, X, q, ids, scores = make(M, N, 72, 12, storage, 0, seed=3)
    loss, dq = check(index, X, q, ids, scores, "index", 0)
    flat_q = torch.zeros_like(q)                # every logit 0: the softmax is 1/N for each row
    loss, dq = index.distill(flat_q, ids, scores, 0.1, 1.0, "index")
    live = (ids >= 0).any(1)
    p = torch.softmax(torch.where(ids >= 0, scores, -np.inf)[live].double(), 1)
    ent = torch.where(p > 0, p * torch.log(p), 0.0).sum(1)
    want = ent + np.log(N)
    assert float((loss[live].double() - want).abs().max()) < 64 * U32 * np.log(N)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("M", [1, 40])
def test_loss_alone_is_the_same_loss(storage, M):
    for over in ("list", "index"):
        for metric in (0, 1):
            index, X, q, ids, scores = make(M, 500, 100, 9, storage, metric, seed=5)
            a, _ = check(index, X, q, ids, scores, over, metric, grad=True)
            b, _ = check(index, X, q, ids, scores, over, metric, grad=False)
            # Each is within e of the formula's value: their logits are sums of the same 100 products, in orders of their own,
            # and a list of one near entry has a loss of nearly 0 = (-s) + s with |s| up to 30, where an ulp is 1.9e-6.  So
            # they differ by up to 2 e (a multiple of the loss' own size alone leaves the cancelled s out of account).
            _, _, e, _ = distill_ref(q, X, ids, scores, 0.1, 1.5, metric, over)
            assert_within(b, a.double().cpu(), 2 * e)


def test_weights_and_temperatures():
    index, X, q, ids, scores = make(37, 400, 48, 11, seed=6)
    w = torch.randn(37, device="cuda")
    for over in ("list", "index"):
        for tau, tau_t in ((0.02, 0.1), (1.0, 30.0), (50.0, 2.0)):
            check(index, X, q, ids, scores, over, 0, tau, tau_t, w)


def test_empty_lists_and_pads():
    index, X, q, ids, scores = make(4, 50, 64, 5, ragged=False)
    ids[1] = -1
    scores[1] = float("nan")                       # what stands beside a pad is not read
    scores[2] = -np.inf                            # entries the teacher gives nothing
    ids[3, 2:] = -1
    scores[3, 2:] = torch.tensor([np.inf, -np.inf, float("nan")])
    scores[0, 1] = -np.inf                         # an entry with p = 0: in the list's softmax, not in the teacher's
    for over in ("list", "index"):
        loss, dq = check(index, X, q, ids, scores, over, 0)
        assert loss[1] == 0 and loss[2] == 0 and not dq[1].any() and not dq[2].any()
        assert torch.isfinite(loss).all() and torch.isfinite(dq).all()
    no = torch.empty(4, 0, device="cuda")
    for over in ("list", "index"):                 # k = 0: every list is empty
        loss, dq = index.distill(q, no.long(), no, over=over)
        assert not loss.any() and not dq.any()


def test_rows_outside_the_index_are_not_read():
    index, X, q, ids, scores = make(6, 50, 64, 5, ragged=False)
    ids[1, 3], ids[2, 0], ids[4, 4] = 50, -2, 1 << 40
    for over in ("list", "index"):
        loss, dq = check(index, X, q, ids, scores, over, 0)
        assert torch.isnan(loss).tolist() == [False, True, True, False, True, False]


def test_nothing_to_do():
    index = faiss.IndexFlatIP(16)
    e = torch.empty(0, 16, device="cuda")
    loss, dq = index.distill(e, e[:, :3].long(), e[:, :3])
    assert loss.shape == (0,) and dq.shape == (0, 16)
    q = torch.ones(2, 16, device="cuda")               # an empty index: no row number is valid
    for over in ("list", "index"):
        loss, dq = index.distill(q, torch.tensor([[-1], [0]], device="cuda"), torch.ones(2, 1, device="cuda"), over=over)
        assert loss[0] == 0 and torch.isnan(loss[1]) and not dq[0].any() and torch.isnan(dq[1]).all()


def test_large_and_special_logits():
    """Logits far apart (the running maximum moves by thousands) and a row of NaN."""
    index, X, q, ids, scores = make(20, 700, 64, 6, ragged=False, seed=8)
    check(index, X, q * 30, ids, scores, "index", 0, tau=0.01)
    check(index, X, q * 30, ids, scores, "list", 0, tau=0.01)
    bad = X.clone()
    bad[345] = float("nan")
    idx = faiss.IndexFlatIP(64)
    idx.add(bad)
    loss, dq = idx.distill(q, ids, scores)
    assert torch.isnan(loss).all() and torch.isnan(dq).all()


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_strides_and_alignment(storage):
    index, X, q, ids, scores = make(21, 130, 99, 7, storage, 0, seed=9)
    want = {over: index.distill(q, ids, scores, over=over) for over in ("list", "index")}
    wide = torch.zeros(21, 205, dtype=q.dtype, device="cuda")
    wide[:, 3:102] = q
    forms = [wide[:, 3:102], q.t().contiguous().t(), torch.cat([q.flatten(), q.flatten()[:1]])[0:].as_strided((21, 99), (99, 1))]
    ids2, scores2 = ids.t().contiguous().t(), scores.repeat(1, 2)[:, :7]
    for form in forms:
        for over in ("list", "index"):
            loss, dq = index.distill(form, ids2, scores2, over=over)
            assert torch.equal(loss, want[over][0]) and torch.equal(dq, want[over][1])


def test_gradient_against_differences():
    """Central differences of the loss itself along random directions.  The float32 loss is off by about 2^-22; a step of
    2^-6 leaves that divided by 2^-5, and the third derivative (beta^3 by moments of unit rows) times 2^-12 / 6."""
    for metric in (0, 1):
        for over in ("list", "index"):
            index, X, q, ids, scores = make(12, 200, 32, 8, "f32", metric, ragged=False, seed=11)
            tau, h = 1.0, 2.0 ** -6
            g = torch.Generator(device="cuda").manual_seed(2)
            _, dq = index.distill(q, ids, scores, tau, 1.0, over)
            for _ in range(4):
                v = torch.randn(12, 32, generator=g, device="cuda")
                v /= v.norm(dim=1, keepdim=True)
                up, _ = index.distill(q + h * v, ids, scores, tau, 1.0, over, grad=False)
                dn, _ = index.distill(q - h * v, ids, scores, tau, 1.0, over, grad=False)
                diff = (up.double() - dn.double()) / (2 * h)
                allow = 2 * 8 * 2.0 ** -22 / (2 * h) + 8 * h * h / 6
                assert float((diff - (dq.double() * v.double()).sum(1)).abs().max()) < allow


def test_same_call_same_bits():
    for M, over in ((1, "index"), (40, "index"), (200, "index"), (40, "list")):
        index, X, q, ids, scores = make(M, 3000, 200, 20, seed=12)
        a, b = index.distill(q, ids, scores, over=over), index.distill(q, ids, scores, over=over)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_staged_rows_are_seen():
    """Rows added one by one wait on the host until something reads the index."""
    index, X, q, ids, scores = make(5, 40, 24, 4)
    extra = torch.nn.functional.normalize(torch.randn(3, 24), dim=1)
    for r in extra.numpy():
        index.add(r[None])
    X2 = torch.cat([X, extra.cuda()])
    ids[0, 0] = 42
    check(index, X2, q, ids, scores, "index", 0)
    check(index, X2, q, ids, scores, "list", 0)


@pytest.mark.parametrize("M", [1, 40])
def test_graph_replays(M):
    """Captured, replayed with other inputs, the eager call and a second graph between the replays."""
    index, X, q, ids, scores = make(M, 900, 96, 10, metric=1, seed=13)
    eager = lambda: index.distill(q, ids, scores)                        # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for over in ("index", "list"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = index.distill(q, ids, scores, over=over)
        graphs.append((g, out, over))
    for it in range(4):
        q.copy_(torch.nn.functional.normalize(torch.randn_like(q), dim=1))
        scores.add_(torch.randn_like(scores) * (scores > PAD))
        for g, _, _ in graphs:
            g.replay()
        for g, out, over in graphs:
            want = index.distill(q, ids, scores, over=over)
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), (it, over)
    index.add(torch.nn.functional.normalize(torch.randn(5000, 96, device="cuda"), dim=1))   # the arena moves
    junk = [torch.randn(5000, 96, device="cuda") for _ in range(8)]                          # noqa: F841
    want = distill_ref(q, X, ids, scores, 0.05, 1.0, 1, "index")
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert_within(graphs[0][1][0], want[0], want[2])       # the rows it was captured with


def test_capture_refuses_what_it_cannot_record():
    index, X, q, ids, scores = make(3, 60, 16, 4, metric=1, seed=14)
    refused = []
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep = q + 1                                                       # noqa: F841
        try:
            index.distill(q, ids, scores)                                  # norms not computed yet
        except _lib.EngineError as e:
            refused.append(str(e))
    assert len(refused) == 1 and "capture" in refused[0]
    check(index, X, q, ids, scores, "index", 1)


def test_other_streams_and_threads():
    import threading
    index, X, q, ids, scores = make(30, 4000, 128, 10, seed=15)
    want = index.distill(q, ids, scores)
    torch.cuda.synchronize()
    bad = []

    def work():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(10):
                got = index.distill(q, ids, scores)
                st.synchronize()
                if not (torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])):
                    bad.append(1)
    ts = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in ts]
    for _ in range(10):
        index.search(q.cpu().numpy(), 5)
    [t.join() for t in ts]
    assert not bad


def test_search_is_what_it_was():
    index, X, q, ids, scores = make(9, 2000, 64, 10, metric=1, seed=16)
    qn = q.cpu().numpy()
    D0, I0 = index.search(qn, 10)
    index.distill(q, ids, scores)
    D1, I1 = index.search(qn, 10)
    assert np.array_equal(D0, D1) and np.array_equal(I0, I1)


def test_refusals():
    index, X, q, ids, scores = make(4, 30, 16, 3)
    bad = [dict(q=q.double()), dict(q=q.bfloat16()), dict(q=q[:, :8]), dict(q=q.cpu()), dict(q=q.cpu().numpy()),
           dict(ids=ids.int()), dict(ids=ids[:3]), dict(scores=scores[:, :2]), dict(scores=scores.double()),
           dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e-45),
           dict(teacher_temperature=0.0), dict(teacher_temperature=float("inf")), dict(over="rows"),
           dict(weights=torch.ones(3, device="cuda")), dict(weights=torch.ones(4, device="cuda").double()),
           dict(ids=ids.cpu()),
           dict(ids=torch.zeros(4, 1025, dtype=torch.int64, device="cuda"), scores=torch.zeros(4, 1025, device="cuda"))]
    for kw in bad:
        with pytest.raises(ValueError):
            index.distill(**{**dict(q=q, ids=ids, scores=scores), **kw})
    check(index, X, q, ids, scores, "index", 0)


def test_c_refusals():
    """At the C entry: workspace too small or misaligned, strides below d, NULL buffers; nothing is launched."""
    import ctypes as C
    index, X, q, ids, scores = make(4, 30, 16, 3)
    lib, h = index._b._lib, index._b._h
    need = C.c_int64()
    assert lib.rag_flat_distill_ws_bytes(h, 4, 3, 0, 1, C.byref(need)) == 0 and need.value > 0
    ws = torch.empty(need.value + 256, dtype=torch.uint8, device="cuda")
    loss, dq = torch.full((4,), 7.0, device="cuda"), torch.full((4, 16), 7.0, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())      # noqa: E731

    def call(nq=4, ldq=16, k=3, over=0, qp=p(q), wsp=p(ws), n_ws=need.value, lddq=16, lossp=p(loss)):
        return lib.rag_flat_distill_dev(h, nq, qp, ldq, k, p(ids), p(scores), 0.1, 1.0, over, None, lossp, p(dq), lddq,
                                        wsp, n_ws, C.c_void_p(0))
    bad = [dict(n_ws=need.value - 1), dict(wsp=C.c_void_p(ws.data_ptr() + 16)), dict(wsp=C.c_void_p(None)), dict(ldq=15),
           dict(lddq=15), dict(qp=C.c_void_p(None)), dict(lossp=C.c_void_p(None)), dict(k=1025), dict(k=-1), dict(nq=-1),
           dict(nq=65536), dict(over=2)]
    for kw in bad:
        assert call(**kw) == _lib.RAG_ERR_INVALID_ARG, kw
    torch.cuda.synchronize()
    assert bool((loss == 7).all()) and bool((dq == 7).all())
    assert call() == 0


def rising(M, N, d, storage, metric, seed=0):
    """(index, X, q, ids, scores): every third query sees its logits (tau 0.1) rise by 40 from 32 rows to the next 32, eight
    times over, then again from the start; the others lie across that direction, and one is zero."""
    g = torch.Generator(device="cuda").manual_seed(seed + M + d)
    u = torch.nn.functional.normalize(torch.randn(d, generator=g, device="cuda"), dim=0)

    def across(n):
        r = torch.randn(n, d, generator=g, device="cuda")
        r -= (r @ u)[:, None] * u
        return r / r.norm(dim=1, keepdim=True)

    k = (torch.arange(N, device="cuda") // 32 % 8).float()
    far = (4.0 * 7) ** 0.5
    a = far - (4.0 * (7 - k)) ** 0.5 if metric == 1 else 4.0 * k
    X = (across(N) + a[:, None] * u).to(TYPE[storage])
    q = across(M)
    q[::3] = (far if metric == 1 else 1.0) * u + 0.05 * across(len(q[::3]))
    if M > 1:
        q[1] = 0
    q = q.to(TYPE[storage])
    ids = torch.randint(0, N, (M, 3), generator=g, device="cuda")
    scores = torch.randn(M, 3, generator=g, device="cuda")
    index = faiss.IndexFlat(d, metric, storage=storage)
    index.add(X)
    return index, X, q, ids, scores


@pytest.mark.parametrize("M,N,d", [(1, 70001, 64), (3, 70001, 64), (12, 70001, 64), (12, 20001, 700), (30, 40001, 100), (64, 40001, 40),
                                   (300, 70001, 32), (33000, 20001, 32), (20000, 33001, 72)])
@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("metric", [0, 1])
def test_rising_logits_and_long_shares(M, N, d, storage, metric):
    """The reference of a query's weights moves within a share (its logits rise by far more than its slack) while other
    queries' stay; the largest batches leave one or two shares of more than a hundred tiles."""
    index, X, q, ids, scores = rising(M, N, d, storage, metric)
    loss, dq = index.distill(q, ids, scores, 0.1, 1.0, "index")
    some = torch.unique(torch.tensor([0, 1, 2, 3, 15, 16, 17, 47, M // 2, M - 2, M - 1]).clamp(0, M - 1)).cuda()
    ref_loss, ref_dq, e_loss, e_dq = distill_ref(q[some], X, ids[some], scores[some], 0.1, 1.0, metric, "index")
    assert_within(loss[some], ref_loss, e_loss, "loss")
    assert_within(dq[some], ref_dq, e_dq, "dq")
    assert torch.isfinite(loss).all() and torch.isfinite(dq).all()
    alone, _ = index.distill(q, ids, scores, 0.1, 1.0, "index", grad=False)
    assert_within(alone[some], ref_loss, e_loss, "loss alone")


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_rows_replaced_while_a_call_is_under_way(storage):
    """reset() and add() behind a call that is still running: it has read the rows that were there."""
    index, X, q, ids, scores = make(512, 400000, 64, 5, storage, 1, seed=21)
    other = X[:300000].flip(0).float().cpu().numpy()
    want = index.distill(q, ids, scores)
    torch.cuda.synchronize()
    ids2 = ids.clamp(max=299999)
    got = index.distill(q, ids, scores)
    index.reset()
    index.add(other)
    new = index.distill(q, ids2, scores)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    fresh = faiss.IndexFlat(64, 1, storage=storage)
    fresh.add(other)
    again = fresh.distill(q, ids2, scores)
    assert torch.equal(new[0], again[0]) and torch.equal(new[1], again[1])


@pytest.mark.parametrize("storage,d", [("f32", 40), ("f32", 1024), ("bf16", 770), ("f32", 8192)])
@pytest.mark.parametrize("M", [1, 6, 70])
def test_longest_lists(M, d, storage):
    index, X, q, ids, scores = make(M, 900, d, 1024, storage, 0, seed=22)
    for over in ("list", "index"):
        check(index, X, q, ids, scores, over, 0)


@pytest.mark.parametrize("d", [64, 99])
@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_added_from_hbm_are_those_added_from_the_host(d, storage, dtype):
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(1500, 2 * d, generator=g, device="cuda").to(TYPE[dtype])
    a, b = (faiss.IndexFlat(d, 0, storage=storage) for _ in range(2))
    for part in (x[:700, :d], x[700:701, d:], x[:0, :d], x[701:, :d]):      # rows apart from each other, one, none
        a.add(part)
        b.add(part.float().cpu().numpy())
    assert a.ntotal == b.ntotal == 1500
    assert np.array_equal(a.reconstruct_n(0, 1500), b.reconstruct_n(0, 1500))
    q = np.random.default_rng(0).standard_normal((3, d)).astype(np.float32)
    for u, v in zip(a.search(q, 5), b.search(q, 5)):
        assert np.array_equal(u, v)
    if storage == "f32":
        assert a._b._lib.rag_flat_add_bf16_dev(a._b._h, 1, x.data_ptr(), None) == _lib.RAG_ERR_INVALID_ARG
    for bad in (x[:, :d - 1], x[:, :d].double(), x[0, :d]):
        with pytest.raises(ValueError):
            a.add(bad)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("M", [3, 20, 70, 130])
def test_bad_queries_stay_alone(M, storage):
    """A query of NaN or infinities gives NaN, and not a bit of the others changes (each is a lane of its own in every product)."""
    index, X, q, ids, scores = make(M, 3000, 64, 6, storage, 0, seed=23, ragged=False)
    for over in ("list", "index"):
        for grad in (True, False):
            want = index.distill(q, ids, scores, over=over, grad=grad)
            bad = q.clone()
            bad[1], bad[M - 1] = float("nan"), float("inf")
            got = index.distill(bad, ids, scores, over=over, grad=grad)
            keep = [i for i in range(M) if i not in (1, M - 1)]
            assert torch.isnan(got[0][[1, M - 1]]).all()
            assert torch.equal(got[0][keep], want[0][keep])
            if grad:
                assert torch.isnan(got[1][[1, M - 1]]).all() and torch.equal(got[1][keep], want[1][keep])
