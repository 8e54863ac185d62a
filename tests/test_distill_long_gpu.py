"""IndexFlat.distill over long shares of the rows, and rows wider than the matrix forms hold: sums that many rows go into."""
import pytest
import torch

from _operators import U32, assert_within, distill_ref
from rag_system_amd import faiss_compat as faiss
from test_distill_gpu import TYPE, check, make, rising

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("M,d", [(1, 72), (3, 400), (12, 72), (40, 72), (300, 72), (2100, 72), (2048, 1544)])
def test_rows_that_are_all_the_same(M, d, storage):
    """Every logit is 0 and every row the teacher's: dq is what the sum of 300000 equal values loses.  A sum of 4096 rows at most
    (64 tiles of 64), then the sums' own, 147 of 2048 rows or fewer, and the shares': (4096 + 147 + 16) U32 of the value at most.  Adding up all
    rows in one float32 loses up to 2^-9 of it."""
    N, tau = 300000, 0.5
    v = (0.05 + 0.15 * torch.rand(d, generator=torch.Generator().manual_seed(d))).to(TYPE[storage]).cuda()
    index = faiss.IndexFlat(d, 0, storage=storage)
    index.add(v.expand(N, d).contiguous())
    q = torch.zeros(M, d, dtype=TYPE[storage], device="cuda")
    loss, dq = index.distill(q, torch.full((M, 1), 7, device="cuda"), torch.zeros(M, 1, device="cuda"), tau, 1.0)
    allow = (4096 + 147 + 16) * U32 * v.float() / tau
    assert bool((dq.float().abs() <= allow).all()), float((dq.float().abs() / v.float()).max())
    assert float((loss.double() - torch.tensor(float(N)).double().log()).abs().max()) < 8 * U32 * 13


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("M,N,d", [(300, 5003, 2050), (2, 40001, 1540), (2050, 2500, 1600)])
def test_wide_rows_with_rising_logits(M, N, d, metric, storage):
    """Many steps a share, whose logits rise by 40 from one to the next, at widths that the matrix forms do not hold."""
    index, X, q, ids, scores = rising(M, N, d, storage, metric)
    loss, dq = index.distill(q, ids, scores, 0.1, 1.0, "index")
    some = torch.unique(torch.tensor([0, 1, 2, 3, 47, M // 2, M - 2, M - 1]).clamp(0, M - 1)).cuda()
    ref_loss, ref_dq, e_loss, e_dq = distill_ref(q[some], X, ids[some], scores[some], 0.1, 1.0, metric, "index")
    assert_within(loss[some], ref_loss, e_loss, "loss")
    assert_within(dq[some], ref_dq, e_dq, "dq")
    assert torch.isfinite(loss).all() and torch.isfinite(dq).all()
    alone, _ = index.distill(q, ids, scores, 0.1, 1.0, "index", grad=False)
    assert_within(alone[some], ref_loss, e_loss, "loss alone")


@pytest.mark.parametrize("storage", ["f32", "bf16"])
@pytest.mark.parametrize("metric", [0, 1])
@pytest.mark.parametrize("M,d", [(1, 1544), (5, 1544), (40, 2050), (3, 8192)])
def test_wide_rows(M, d, metric, storage):
    index, X, q, ids, scores = make(M, 1300, d, 9, storage, metric, seed=31)
    check(index, X, q, ids, scores, "index", metric)
    check(index, X, q, ids, scores, "index", metric, grad=False)


@pytest.mark.parametrize("storage", ["f32", "bf16"])
def test_wide_rows_with_bad_values(storage):
    """A row of NaN among many, and a query of NaN: NaN in every query, and in that query alone."""
    index, X, q, ids, scores = make(9, 700, 2050, 4, storage, 0, seed=32, ragged=False)
    want = index.distill(q, ids, scores)
    bad = q.clone()
    bad[4] = float("nan")
    loss, dq = index.distill(bad, ids, scores)
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.isnan(loss[4]) and torch.isnan(dq[4]).all()
    assert torch.equal(loss[keep], want[0][keep]) and torch.equal(dq[keep], want[1][keep])
    X = X.clone()
    X[555] = float("nan")
    other = faiss.IndexFlat(2050, 0, storage=storage)
    other.add(X)
    loss, dq = other.distill(q, ids, scores)
    assert torch.isnan(loss).all() and torch.isnan(dq).all()
