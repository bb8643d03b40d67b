"""GPU tests of metric.distill_loss where a result lives on a small difference, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import logits_reference as R
from object_detection_amd import metric as M

pytestmark = pytest.mark.gpu
F32 = torch.float32
RESTS = (3e-2, 1e-4, 1e-5, 1e-6, 1e-7)          # the teacher's mass off the list
SHARES = (0.5, 2.0)                             # the student's, over that


def _nearly_everything_listed(rows, C, K, T):
    """Student logits, teacher values and classes: row i's list leaves RESTS[i % 5] to the other classes, the student about half or twice that."""
    gen = torch.Generator().manual_seed(C + K)
    rest = torch.tensor(RESTS, dtype=torch.float64)[torch.arange(rows) % len(RESTS)]
    p0 = rest * torch.tensor(SHARES, dtype=torch.float64)[torch.arange(rows) // len(RESTS) % 2]
    ids = torch.stack([torch.randperm(C, generator=gen)[:K] for _ in range(min(rows, 20))])[torch.arange(rows) % 20]
    logq = torch.log_softmax(torch.randn(rows, K, generator=gen, dtype=torch.float64), 1) + torch.log1p(-rest)[:, None]
    off = torch.log_softmax(0.5 * torch.randn(rows, C - K, generator=gen, dtype=torch.float64), 1) + torch.log(p0)[:, None]
    listed = torch.log_softmax(logq + 0.01 * torch.randn(rows, K, generator=gen, dtype=torch.float64), 1) + torch.log1p(-p0)[:, None]
    at_off = torch.ones(rows, C, dtype=torch.bool).scatter_(1, ids, False)
    x = torch.empty(rows, C, dtype=torch.float64)
    x[at_off] = off.flatten()
    x.scatter_(1, ids, listed)
    return (T * x).float().cuda(), logq.float().cuda(), ids.int().cuda()


@pytest.mark.parametrize('rows,C,K', [(20, 90, 1), (20, 90, 20), (20, 1400, 4), (20, 5000, 20), (520, 2100, 1), (520, 9000, 20), (4, 70001, 128), (10, 131075, 1)])
@pytest.mark.parametrize('T', [1.0, 2.0])
def test_bucket_where_the_list_holds_nearly_everything(rows, C, K, T):
    """Off the list the gradient is T r_i (p0 (sum q + q0) - q0) of two small masses, r the softmax over those classes.

    Bound.  With e = Row.err's largest, a sum's relative error: p0 = off / (on + off) is off by 2 e + 4 U relative and its product with
    sum q + q0 (three roundings and its own) by 4 U more; q0 is a difference of 64-bit numbers, K exponentials to 2 steps and K additions
    off by (K + 4) 2^-51, and rounds once to 32 bits.  Each r_i is off by e and the two products by U each, relative."""
    x, tl, ids = _nearly_everything_listed(rows, C, K, T)
    kw = dict(temperature=T, rest='bucket', reduction=None)
    loss, grad = M.distill_loss(x, tl, ids, return_grad=True, **kw)
    leaf = x.clone().requires_grad_()
    again, = torch.autograd.grad(M.distill_loss(leaf, tl, ids, **kw).sum(), leaf)
    xs, t, n = x.double().cpu().numpy(), tl.double().cpu().numpy(), ids.cpu().numpy()
    for i in range(rows) if rows <= 20 else list(range(20)) + [rows // 2, rows - 1]:
        row = R.Row(xs[i], T)
        want, wg, le, ge = R.distill(row, t[i], n[i], True, 1.0)
        off = np.ones(C, bool)
        off[n[i]] = False
        q0, p0, e, U = 1.0 - np.exp(t[i]).sum(), row.p[off].sum(), row.err.max(), R.U
        dense = p0 * (2 * e + 8 * U) + max(q0, 0.0) * U + (K + 4) * 2.0 ** -51
        bound = ge + 4 * U * np.abs(wg) + R.TINY[F32]
        bound[off] = T * row.p[off] / p0 * dense + (e + 8 * U) * np.abs(wg[off]) + R.TINY[F32]
        R.within(float(loss[i]), want, le, 'loss of row %d' % i)
        for got in (grad, again):
            R.within(got[i].double().cpu().numpy(), wg, bound, 'gradient of row %d' % i)


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('rows,C,K,pad', [(530, 2100, 128, 0), (600, 3001, 7, 5), (520, 9000, 33, 0), (530, 16001, 64, 2), (520, 33333, 5, 0),
                                          (515, 65537, 20, 0), (515, 131073, 9, 0), (40, 80, 8, 0), (40, 1500, 30, 3)])
def test_bucket_gradient_of_every_class_of_every_row(rows, C, K, pad, dtype):
    """Against the formula in 64 bits on the device, with a bound that scales with each class's own gradient off the list.

    Bound, with e, p0, q0 as above: p0 (sum q + q0) - q0 is off by p0 (2 e + 8 U) + q0 U, and where p0 > 1/2, as sum q less the
    listed classes' mass, by that mass's (2 e + 4 U) and 2 U sum q; r_i and its products by (e + 8 U) relative; the result is rounded to its type.
    At a listed class p and q are off by (2 e + 8 U) and (K + 8 + 4 |log q|) U relative."""
    gen = torch.Generator().manual_seed(C)
    x = torch.randn(rows, C + pad, generator=gen) * 2.0
    x.scatter_add_(1, torch.randint(0, C, (rows, 6), generator=gen), torch.full((rows, 6), 6.0))
    x = x.to(dtype).cuda()[:, :C]
    teacher = x.float() + torch.randn(rows, C, generator=gen).cuda()
    r = M.label_logprobs(teacher, top_k=K)
    tl, ids = r.top_logprobs, r.top_labels
    w = torch.rand(rows, generator=gen).cuda() + 0.5
    if dtype == torch.float16:
        w *= 2.0 ** 13                                          # as a step that scales its loss: keeps the gradients in float16's range
    w[1::5] = 0.0
    _, grad = M.distill_loss(x, tl, ids, rest='bucket', row_weights=w, reduction=None, return_grad=True)
    leaf = x.detach().requires_grad_()
    again, = torch.autograd.grad(M.distill_loss(leaf, tl, ids, rest='bucket', row_weights=w, reduction=None).sum(), leaf)

    z = x.double()
    z = z - z.amax(1, keepdim=True)
    s = z.exp().sum(1, keepdim=True)
    p = z.exp() / s
    at = ids.long()
    off = torch.ones_like(p, dtype=torch.bool).scatter_(1, at, False)
    q = tl.double().exp()
    q0, p0 = (1.0 - q.sum(1, keepdim=True)).clamp(min=0), torch.where(off, p, 0.0).sum(1, keepdim=True)
    p_on = 1.0 - p0
    weight = w.double()[:, None]
    want = (p / p0 * (p0 - q0)).scatter(1, at, p.gather(1, at) - q) * weight
    U = R.U
    e = U * (4 * 1.4427 * -z.amin(1, keepdim=True) + 4 + R.adds(C) + 4 * s.log2())
    dense = torch.where(p0 > 0.5, p_on * (2 * e + 4 * U) + 2 * U * q.sum(1, keepdim=True), p0 * (2 * e + 8 * U) + q0 * U) + (K + 4) * 2.0 ** -51
    listed = p.gather(1, at) * (2 * e + 8 * U) + q * U * (K + 8 + 4 * tl.double().abs())
    bound = (p / p0 * dense).scatter(1, at, listed) * weight + (e + 8 * U + R.EPS[dtype]) * want.abs() + R.TINY[dtype]
    # the bound tells a class's gradient from 0 (which a vector left out would hold) nearly everywhere
    seen = off & (weight > 0)
    assert (bound[seen] < 0.5 * want[seen].abs()).double().mean() > 0.9
    for g in (grad, again):
        wrong = (g.double() - want).abs() > bound
        assert not wrong.any(), (int(wrong.sum()), wrong.nonzero()[:4].tolist())
        assert (g[1::5] == 0).all()
