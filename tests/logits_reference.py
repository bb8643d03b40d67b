"""The class-logit operators in 64 bits, written from their definitions (NumPy, one row at a time), and the error bounds the
kernels are held to.

Bounds.  u = 2^-24 is half a step of float32.  With t = (x - m) log2(e) / T a kernel makes three roundings and one of the
constant (4 u |t| absolute), 2^t adds 2 u relative, a sum of n terms in a tree or in runs at most `adds` u relative, log2 2 u of
its result.  So a log-probability is off by at most  u (4 |t| + 4 + adds + 4 l2)  in absolute terms, l2 = log2 of the sum; a
probability by as much relatively.  A rounding to the gradient's type adds half a step of it, and where float16 goes
subnormal at most 2^-25."""
import numpy as np
import torch

U = 2.0 ** -24
EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def adds(C):
    """Additions one running sum sees at most: 64 lanes or more share a long row, four or more a short one."""
    return 64 + (C / 64 if C > 256 else C / 4)


class Row:
    """Softmax statistics of one row of logits (float64 values of the stored numbers)."""

    def __init__(self, x, T):
        self.x, self.T = np.asarray(x, np.float64), T
        self.bad = bool(np.isnan(self.x).any() or (self.x == np.inf).any())
        self.m = np.nan if self.bad else self.x.max()
        self.empty = not self.bad and self.m == -np.inf
        if self.bad or self.empty:
            fill = np.nan if self.bad else -np.inf
            self.logp = np.full(len(self.x), fill)
            self.p = np.full(len(self.x), np.nan if self.bad else 0.0)
            self.entropy = np.nan if self.bad else 0.0
            self.err = np.full(len(self.x), np.inf)
            return
        with np.errstate(over='ignore'):
            z = (self.x - self.m) / T
        e = np.exp(z)
        s = e.sum()
        self.logp = z - np.log(s)
        self.p = e / s
        pl = self.p * np.where(self.p > 0, self.logp, 0.0)
        self.entropy = -pl.sum()
        t = np.where(np.isinf(z), 0.0, -z) * 1.4427
        l2 = np.log2(s)
        self.err = U * (4 * t + 4 + adds(len(self.x)) + 4 * l2)      # of log p_i, absolute
        self.p_err = self.p * np.expm1(np.minimum(self.err, 1.0)) + 1e-37
        mean_t = (self.p * t).sum()
        # entropy = l2 - (sum e t) / s: l2's own error and that of the mean of t
        self.entropy_err = U * ((adds(len(self.x)) + 16) * (2 + mean_t + l2) + 4 * (self.p * t * t).sum())


def top(x, k):
    """Ids of the k largest values: NaN first, then value descending; ties to the lowest id."""
    x = np.asarray(x, np.float64)
    nan = np.isnan(x)
    return np.lexsort((np.arange(len(x)), np.where(nan, 0.0, -x), ~nan))[:k].tolist()


def score_grad(row, label, g_lp, g_ent, ids, g_top):
    """d/dx of g_lp log p[label] + g_ent H + sum g_top log p[ids], and a bound on a float32 evaluation."""
    n = len(row.x)
    if row.empty:
        return np.zeros(n), np.zeros(n)
    hits, total, size = np.zeros(n), 0.0, 0.0
    for i, g in [(label, g_lp)] + list(zip(ids, g_top)):
        if 0 <= i < n:
            hits[i] += g
            total += g
            size += abs(g)
    logp = np.where(np.isinf(row.logp), 0.0, row.logp)
    inner = total + g_ent * (logp + row.entropy)
    grad = (hits - row.p * inner) / row.T
    inner_err = U * (len(ids) + 8) * size + abs(g_ent) * (row.err + row.entropy_err + 4 * U * (np.abs(logp) + row.entropy))
    err = (row.p_err * np.abs(inner) + row.p * (inner_err + 4 * U * np.abs(inner)) + U * (len(ids) + 8) * np.abs(hits)
           + 4 * U * np.abs(grad) * row.T) / row.T
    return grad, err


def distill(row, tl, ids, bucket, w):
    """Loss and gradient of one row, with bounds on float32 evaluations of both."""
    n, T = len(row.x), row.T
    if w == 0 or row.empty:
        return 0.0, np.zeros(n), 0.0, np.zeros(n)
    use = [(i, t) for i, t in zip(ids, tl) if 0 <= i < n]
    k = len(use)
    t = np.array([t for _, t in use], np.float64)
    at = np.array([i for i, _ in use], np.int64)
    q0 = 0.0
    if bucket:
        q, logq = np.exp(t), t
        q0 = max(0.0, 1.0 - q.sum())
    elif k and t.max() > -np.inf:
        z = t - t.max()
        logq = z - np.log(np.exp(z).sum())
        q = np.exp(logq)
    else:
        q, logq = np.zeros(k), np.full(k, -np.inf)
    on = q > 0
    terms = q[on] * (logq[on] - row.logp[at[on]])
    loss = terms.sum()
    # float32: q to (k + 8 + 4 |log q|) u relative, log q and log p absolute
    q_rel = U * (k + 8 + 4 * np.abs(np.where(on, logq, 0.0)))
    err = (q[on] * (q_rel[on] * np.abs(logq[on] - row.logp[at[on]]) + row.err[at[on]] + q_rel[on]
                    + 4 * U * (np.abs(logq[on]) + np.abs(row.logp[at[on]])))).sum() + U * (k + 8) * np.abs(terms).sum()
    mass = q.sum()
    hits, hits_err = np.zeros(n), np.zeros(n)
    for j in range(k):
        hits[at[j]] += q[j]
        hits_err[at[j]] += q[j] * (q_rel[j] + U * k)
    off = np.ones(n, bool)
    off[at] = False
    p0 = row.p[off].sum()
    factor = np.ones(n)
    if bucket and p0 > 0:
        mass += q0
        r0 = 8 * U + (row.err[off] * row.p[off]).sum() / p0 + U * adds(n)       # relative, of p0
        if q0 > 0:
            d = np.log(q0) - np.log(p0)
            loss += q0 * d
            err += 4 * U * (abs(d) + 1) + q0 * (r0 + 4 * U * (abs(np.log(q0)) + abs(np.log(p0)))) + 8 * U * abs(q0 * d)
        grad = np.where(off, row.p * (mass - q0 / p0), row.p * mass - hits)
        gerr = np.where(off, row.p_err * abs(mass) + row.p / p0 * (p0 * (r0 + 4 * U) + q0 * (8 * U + r0) + 4 * U),
                        row.p_err * mass + hits_err + 8 * U * row.p)
    else:
        grad = row.p * mass - hits
        gerr = row.p_err * mass + hits_err + (k + 8) * U * row.p
    f = w * T
    return (w * T * T * loss, f * grad, abs(w) * T * T * err + 8 * U * abs(w * T * T * loss),
            abs(f) * gerr + 8 * U * np.abs(f * grad))


def within(got, want, err, what):
    got, want, err = np.asarray(got, np.float64), np.asarray(want, np.float64), np.asarray(err, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    want = np.where(np.abs(want) > np.finfo(np.float32).max, np.copysign(np.inf, want), want)   # outputs are float32: no larger values
    same = (np.isnan(got) & np.isnan(want)) | (got == want)
    with np.errstate(invalid='ignore'):
        ok = same | (np.isfinite(got) & np.isfinite(want) & (np.abs(got - want) <= err))
    if not ok.all():
        at = tuple(np.argwhere(~ok)[0])
        raise AssertionError('%s: %d of %d outside, first at %r: got %r, want %r, bound %r'
                             % (what, (~ok).sum(), ok.size, at, got[at], want[at], np.broadcast_to(err, want.shape)[at]))
