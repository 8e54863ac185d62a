"""Query adapters and distillation in 64 bits, with the error that 32-bit sums are allowed.

U32 is half a step of float32 relative to the value.  A sum of n products in float32, in any order, is off by at most
(n + 1) U32 times the sum of the products' magnitudes (to first order); that is what the `allow` results hold, with a
few more steps for the scalings and exponentials on the way."""
import numpy as np
import torch

U32 = torch.finfo(torch.float32).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def split_rest(dtype):
    """What a float32 factor of a product with bfloat16 weights may lose: it is multiplied as its bfloat16 h, off by up to half
    a step (2^-8 of the value), and the bfloat16 of the difference, off by half a step of that: 2^-8 * 2^-8 of the value.  (Where
    the sums are long, their own allowance hides it: 768 products 2^-13.4; it is more than that of 5 products, 2^-19.8.)"""
    return half_step(dtype) ** 2 if dtype == torch.bfloat16 else 0.0


def adapters_ref(x, W, A, B, scale, slots):
    """(y, allow) in 64 bits; slots: list of ints, -1 = none."""
    rest = split_rest(x.dtype)
    x, W, A, B, scale = (t.detach().cpu().double() for t in (x, W, A, B, scale))
    y, mag = x @ W.t(), x.abs() @ W.abs().t()
    low = torch.zeros_like(mag)                 # of the adapters alone
    for t, s in enumerate(slots):
        if s >= 0:
            y[t] += scale[s] * (B[s] @ (A[s] @ x[t]))
            low[t] = scale[s].abs() * (B[s].abs() @ (A[s].abs() @ x[t].abs()))
    # a product of A passes its own sum over d_in, the scaling, the product with B and the sum over d_in + rank
    return y, (2 * W.shape[1] + A.shape[1] + 6) * U32 * (mag + low) + rest * low


def adapters_grad_ref(x, W, A, B, scale, slots, dy):
    """{dx, dA, dB: (value, allow)}"""
    rest = split_rest(x.dtype)
    x, W, A, B, scale, dy = (t.detach().cpu().double() for t in (x, W, A, B, scale, dy))
    n, (d_out, d_in), (S, R, _) = x.shape[0], W.shape, A.shape
    out = {}
    for sign in (False, True):
        f = torch.abs if sign else (lambda t: t)
        dx, dA, dB = f(dy) @ f(W), torch.zeros_like(A), torch.zeros_like(B)
        low = torch.zeros_like(dx)
        for t, s in enumerate(slots):
            if s < 0:
                continue
            u = f(scale[s]) * (f(A[s]) @ f(x[t]))
            v = f(scale[s]) * (f(B[s]).t() @ f(dy[t]))
            low[t] = f(A[s]).t() @ v
            dx[t] += low[t]
            dA[s] += torch.outer(v, f(x[t]))
            dB[s] += torch.outer(f(dy[t]), u)
        for k, t in (("dx", dx), ("dA", dA), ("dB", dB)):
            out.setdefault(k, []).append(t)
    steps = {"dx": 2 * d_out + R + 6, "dA": d_out + n + 6, "dB": d_in + n + 6}
    return {k: (v, steps[k] * U32 * m + (rest * low if k == "dx" else 0.0)) for k, (v, m) in out.items()}


def distill_ref(q, X, ids, scores, tau, tau_t, metric, over, weights=None):
    """loss, dq and what each may be off by, all in 64 bits.  metric 0: inner product, 1: L2."""
    q, X, z = (t.detach().cpu().double() for t in (q, X, scores))
    ids = ids.cpu()
    M, d = q.shape
    N, K = X.shape[0], ids.shape[1]
    w = torch.ones(M, dtype=torch.float64) if weights is None else weights.cpu().double()
    loss, dq = torch.zeros(M, dtype=torch.float64), torch.zeros(M, d, dtype=torch.float64)
    e_loss, e_dq = torch.zeros_like(loss), torch.zeros_like(dq)
    qX = q @ X.t()
    mag = (q.abs() @ X.abs().t()) / tau
    s_all = qX / tau
    if metric == 1:
        xx, qq = (X * X).sum(1), (q * q).sum(1)
        s_all = -(qq[:, None] + xx[None, :] - 2 * qX) / tau
        mag = (2 * q.abs() @ X.abs().t() + xx[None, :] + qq[:, None]) / tau
    g = 2.0 if metric == 1 else 1.0
    for i in range(M):
        at = [(int(t), float(v)) for t, v in zip(ids[i], z[i]) if int(t) != -1]
        if any(t < -1 or t >= N for t, _ in at):
            loss[i], dq[i] = np.nan, np.nan
            continue
        if not any(v != -np.inf for _, v in at):
            continue
        t = torch.tensor([a for a, _ in at])
        zi = torch.tensor([v for _, v in at], dtype=torch.float64) / tau_t
        p = torch.softmax(zi, 0)
        rows = X[t]
        s = -((q[i] - rows) ** 2).sum(1) / tau if metric == 1 else rows @ q[i] / tau
        sup, sup_rows, m_sup = (s, rows, mag[i, t]) if over == "list" else (s_all[i], X, mag[i])
        lse = torch.logsumexp(sup, 0)
        P = torch.exp(sup - lse)
        kl = torch.where(p > 0, p * (torch.log(p) - s), 0.0)
        loss[i] = kl.sum() + lse
        dq[i] = w[i] * g / tau * (P @ sup_rows - p @ rows)
        # a logit is off by its sum of d products and three scalings; a probability by its logit, the logit of the
        # maximum, the exponential of their difference and the sum they are divided by
        e_s = (d + 6) * U32 * m_sup.max()
        e_z = 4 * U32 * zi[zi > -1e30].abs().max()
        spread = float((lse - sup).clamp(max=100).max())
        e_P = 2 * e_s + (spread + len(sup) + 8) * U32
        e_p = 2 * e_z + (min(float(zi.max() - zi.min()), 100.0) + K + 8) * U32
        e_loss[i] = e_P + e_s + (e_p + (K + 8) * U32) * (p * (torch.log(p.clamp(min=1e-300)).abs() + s.abs())).sum() \
            + 4 * U32 * (lse.abs() + loss[i].abs())
        e_dq[i] = w[i].abs() * g / tau * ((e_P + (len(sup) + 8) * U32) * (P @ sup_rows.abs())
                                          + (e_p + (K + 8) * U32) * (p @ rows.abs())) + 4 * U32 * dq[i].abs()
    return loss, dq, e_loss, e_dq


def assert_within(got, want, allow, what=""):
    """Elementwise |got - want| <= allow + half a step of got's type; NaN where (and only where) want is NaN."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    g = got.detach().cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(g), nan), "%s: NaN in other places" % what
    off = (g - want).abs() - (allow + half_step(got.dtype) * want.abs() + torch.finfo(got.dtype).tiny)
    off = torch.where(nan, torch.zeros_like(off), off)
    assert off.numel() == 0 or float(off.max()) <= 0, "%s: off by %.3g where %.3g is allowed" % (
        what, float((g - want).abs().flatten()[off.argmax()]), float((allow + half_step(got.dtype) * want.abs()).flatten()[off.argmax()]))
