"""GPU tests of metric.label_logprobs and metric.distill_loss against their definitions in 64 bits (logits_reference.py, which
also derives every tolerance)."""
import numpy as np
import pytest
import torch

import logits_reference as R
from object_detection_amd import _lib
from object_detection_amd import metric as M

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float('inf')


def _make(seed, rows, C, dtype, pad=0, sigma=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C + pad, generator=gen) * sigma
    at = torch.randint(0, C, (rows, min(6, C)), generator=gen)
    x[torch.arange(rows)[:, None], at] += 6.0
    return x.to(dtype).cuda()[:, :C]


def _np(t):
    return t.detach().double().cpu().numpy()


def check_scores(x, labels, k, T, r):
    xs = _np(x)
    for i in range(len(xs)):
        row = R.Row(xs[i], T)
        R.within(_np(r.entropy)[i], row.entropy, 0.0 if row.bad or row.empty else row.entropy_err, 'entropy of row %d' % i)
        if labels is not None:
            lab = int(labels[i])
            if 0 <= lab < len(xs[i]):
                R.within(_np(r.logprobs)[i], row.logp[lab], row.err[lab], 'logprob of row %d' % i)
            else:
                assert float(r.logprobs[i]) == 0.0
        if k:
            ids = R.top(xs[i], k)
            assert r.top_labels[i].tolist() == ids, i
            R.within(_np(r.top_logprobs)[i], row.logp[ids], row.err[ids], 'top logprobs of row %d' % i)


SHAPES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (33, 20, 5), (21, 33, 4), (40, 150, 9), (11, 301, 6), (9, 600, 16), (5, 1300, 8), (3, 1900, 3), (9, 64, 64), (70, 80, 5), (6, 90, 17), (17, 255, 128), (4, 1000, 10), (3, 2049, 20),
          (5, 4097, 100), (2, 50021, 64), (1, 131075, 8), (2, 262144, 128)]


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,C,k', SHAPES)
def test_scores(rows, C, k, dtype):
    x = _make(rows * 1000 + C, rows, C, dtype)
    labels = torch.randint(0, C, (rows,), generator=torch.Generator().manual_seed(C)).int()
    labels[rows // 2] = -1 if rows > 2 else labels[rows // 2]
    for T in (1.0, 0.7):
        check_scores(x, labels, k, T, M.label_logprobs(x, labels.cuda(), top_k=k, temperature=T))


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,C', [(1, 1), (9, 90), (5, 700), (7, 2500), (5, 4099), (3, 8009), (1030, 9001), (2, 100003)])
def test_scores_without_alternatives(rows, C, dtype):
    x = _make(C, rows, C, dtype)
    labels = (torch.arange(rows) * 31) % C
    at = _sample(rows) if rows > 20 else list(range(rows))
    r = M.label_logprobs(x, labels.cuda(), temperature=1.3)
    assert r.top_labels is None and r.top_logprobs is None
    check_scores(x[at], labels[at], 0, 1.3, M.LabelLogprobs(r.logprobs[at], r.entropy[at], None, None))


@pytest.mark.parametrize('C', [5, 80, 3001, 70001])
def test_scores_of_rows_that_lie_apart_transposed_or_once(C):
    x = _make(C, 6, C, BF16, pad=13)
    assert x.stride(0) == C + 13
    labels = torch.arange(6) % C
    check_scores(x, labels, 4, 1.0, M.label_logprobs(x, labels.cuda(), top_k=4))
    y = x.t().contiguous().t()                                  # classes apart: copied
    check_scores(y, labels, 4, 1.0, M.label_logprobs(y, labels.cuda(), top_k=4))
    z = x[2:3].expand(6, C)                                     # one row read six times
    check_scores(z, labels, 4, 1.0, M.label_logprobs(z, labels.cuda(), top_k=4))
    w = x.reshape(2, 3, C)
    r = M.label_logprobs(w, labels.reshape(2, 3).cuda(), top_k=4)
    assert r.logprobs.shape == (2, 3) and r.entropy.shape == (2, 3) and r.top_labels.shape == (2, 3, 4)
    one = M.label_logprobs(x[1], torch.tensor(1).cuda(), top_k=2)
    assert one.logprobs.shape == () and torch.equal(one.entropy, r.entropy[0, 1]) and one.top_labels.shape == (2,)


@pytest.mark.parametrize('rows', [1, 40])
@pytest.mark.parametrize('C', [6, 80, 1500, 40000])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_scores_under_masks_ties_and_extremes(dtype, C, rows):
    low = torch.finfo(dtype).min
    k = min(C, 9)
    gen = torch.Generator().manual_seed(C)
    cases = {}
    x = torch.randn(C, generator=gen)
    cases['forbidden'] = torch.where(torch.rand(C, generator=gen) < 0.6, torch.full_like(x, -INF), x)
    cases['lowest'] = torch.where(torch.rand(C, generator=gen) < 0.6, torch.full_like(x, low), x)
    cases['all forbidden'] = torch.full((C,), -INF)
    cases['all lowest'] = torch.full((C,), low)
    cases['lowest and forbidden'] = torch.where(torch.arange(C) % 3 == 0, torch.tensor(low), torch.tensor(-INF))
    cases['one allowed'] = torch.full((C,), -INF).index_fill(0, torch.tensor(C - 1), 1.5)
    cases['equal'] = torch.full((C,), 2.5)
    cases['zeros of both signs'] = torch.where(torch.arange(C) % 2 == 0, 0.0, -0.0)
    cases['few values'] = torch.randint(-2, 3, (C,), generator=gen).float()
    cases['ascending'] = torch.arange(C) / 64.0
    cases['shifted'] = x + (1000.0 if dtype != F32 else 100000.0)
    cases['highest'] = torch.full((C,), torch.finfo(dtype).max)
    cases['far apart'] = torch.where(torch.arange(C) == C // 2, torch.finfo(dtype).max, low)
    cases['nan'] = x.clone().index_fill(0, torch.tensor(C // 2), float('nan'))
    cases['inf'] = x.clone().index_fill(0, torch.tensor(C // 3), INF)
    for name, v in cases.items():
        v = v.to(dtype)
        x = v[None].repeat(rows, 1).cuda()
        labels = torch.full((rows,), C // 2)
        for T in (1.0, 0.1):
            r = M.label_logprobs(x, labels.cuda(), top_k=k, temperature=T)
            for t in r:                                          # equal rows give equal results, NaN included
                assert torch.equal(torch.nan_to_num(t, nan=7.0), torch.nan_to_num(t[:1], nan=7.0).expand_as(t)), name
            try:
                check_scores(x[:1], labels[:1], k, T, r)
            except AssertionError as e:
                raise AssertionError('%s, T %s: %s' % (name, T, e))


def check_score_grad(x, labels, k, T, g_lp, g_ent, g_top, ids, grad):
    assert grad.dtype == x.dtype and grad.shape == x.shape
    xs, gs = _np(x), _np(grad)
    for i in range(len(xs)):
        row = R.Row(xs[i], T)
        want, err = R.score_grad(row, int(labels[i]), g_lp[i], g_ent[i], ids[i][:k], g_top[i][:k])
        R.within(gs[i], want, err + R.EPS[x.dtype] * np.abs(want) + R.TINY[x.dtype], 'gradient of row %d' % i)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,C,k', [(1, 1, 1), (4, 5, 3), (70, 80, 5), (20, 150, 2), (9, 333, 1), (6, 700, 3), (4, 1301, 9), (3, 1001, 40), (2, 5000, 128), (3, 70003, 7), (1, 200000, 2)])
def test_score_gradients(rows, C, k, dtype):
    T = 0.8
    x = _make(C, rows, C, dtype, pad=3).requires_grad_()
    gen = torch.Generator().manual_seed(1)
    labels = torch.randint(0, C, (rows,), generator=gen)
    if rows > 1:
        labels[1] = -1
    r = M.label_logprobs(x, labels.cuda(), top_k=k, temperature=T)
    labels[0] = int(r.top_labels[0, 0])                          # the label is an alternative too
    r = M.label_logprobs(x, labels.cuda(), top_k=k, temperature=T)
    g_lp, g_ent, g_top = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen), torch.randn(rows, k, generator=gen)
    ids = r.top_labels.tolist()
    for a, b, c in ((g_lp, g_ent, g_top), (g_lp, None, None), (None, g_ent, None), (None, None, g_top)):
        outs = [(o, g) for o, g in ((r.logprobs, a), (r.entropy, b), (r.top_logprobs, c)) if g is not None]
        grad, = torch.autograd.grad([o for o, _ in outs], x, [g.cuda() for _, g in outs], retain_graph=True)
        check_score_grad(x, labels, k, T, np.zeros(rows) if a is None else a.double().numpy(), np.zeros(rows) if b is None else b.double().numpy(),
                         np.zeros((rows, k)) if c is None else c.double().numpy(), ids, grad)


def test_score_gradients_under_masks_and_in_empty_rows():
    C = 300
    x = torch.randn(5, C, generator=torch.Generator().manual_seed(2)).cuda()
    x[0, 10:200] = -INF
    x[1] = -INF
    x[2, :] = -INF
    x[2, 7] = 0.0
    x[3, 100:] = torch.finfo(F32).min
    labels = torch.tensor([5, 5, 7, 3, 9])
    xg = x.clone().requires_grad_()
    r = M.label_logprobs(xg, labels.cuda(), top_k=3)
    g = torch.tensor([1.0, 2.0, -3.0, 0.5, 1.0], dtype=torch.float64)
    grad, = torch.autograd.grad([r.logprobs, r.entropy], xg, [g.float().cuda(), torch.ones(5).cuda()])
    check_score_grad(x, labels, 0, 1.0, g.numpy(), np.ones(5), np.zeros((5, 3)), r.top_labels.tolist(), grad)
    assert (grad[1] == 0).all()


def test_score_gradient_against_differences():
    """Central differences of the forward kernel, h = 2^-5: the third derivatives of log p and H are below 4 / T^3, the
    difference of two outputs off by 2e-6 each is divided by 2 h."""
    C, h, T = 12, 2.0 ** -5, 1.5
    x = torch.randn(1, C, generator=torch.Generator().manual_seed(3)).cuda()
    lab = torch.tensor([4]).cuda()

    def f(v):
        r = M.label_logprobs(v, lab.expand(len(v)), temperature=T)
        return (1.3 * r.logprobs - 0.7 * r.entropy).double()
    step = h * torch.eye(C, device='cuda')
    want = (f(x + step) - f(x - step)) / (2 * h)
    xg = x.clone().requires_grad_()
    r = M.label_logprobs(xg, lab, temperature=T)
    grad, = torch.autograd.grad((1.3 * r.logprobs - 0.7 * r.entropy).sum(), xg)
    assert (grad[0] - want).abs().max() < 2 * h * h / 6 * 4 / T ** 3 + 4 * 2e-6 / (2 * h)


# ---------------------------------------------------------------------------------------------- distillation
def _list(seed, x, K, T, noise=1.0):
    teacher = x.float() + noise * torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).to(x.device)
    r = M.label_logprobs(teacher, top_k=K, temperature=T)
    return r.top_logprobs, r.top_labels


def check_distill(x, tl, ids, T, rest, w, losses=None, grad=None, scale=1.0, up=None):
    xs, t, n = _np(x), _np(tl), ids.cpu().numpy()
    ws = np.ones(len(xs)) if w is None else _np(w)
    gs = None if grad is None else _np(grad)
    total_err = 0.0
    for i in range(len(xs)):
        loss, g, le, ge = R.distill(R.Row(xs[i], T), t[i], n[i], rest == 'bucket', ws[i])
        total_err += le
        if losses is not None:
            R.within(_np(losses)[i], loss, le, 'loss of row %d' % i)
        if grad is not None:
            f = scale * (1.0 if up is None else float(up[i]))
            R.within(gs[i], f * g, abs(f) * (ge + 4 * R.U * np.abs(g)) + R.EPS[x.dtype] * np.abs(f * g) + R.TINY[x.dtype],
                     'gradient of row %d' % i)
    return total_err


@pytest.mark.parametrize('rest', ['renormalise', 'bucket'])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,C,K', [(1, 1, 1), (5, 3, 3), (4, 20, 1), (70, 80, 8), (9, 90, 33), (12, 150, 128), (9, 333, 5), (7, 701, 60), (5, 1300, 9), (3, 128, 128), (16, 1000, 10), (5, 2050, 128),
                                      (3, 30011, 32), (2, 131075, 64), (1, 262144, 20)])
def test_distill(rows, C, K, dtype, rest):
    T = 2.0 if K % 2 else 1.0
    x = _make(C + K, rows, C, dtype, pad=K % 5)
    tl, ids = _list(C, x, K, T)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(5)).cuda() + 0.5
    if rows > 1:
        w[1] = 0.0
        ids[0, K // 2:] = -1
    kw = dict(temperature=T, rest=rest, row_weights=w)
    losses, grad = M.distill_loss(x, tl, ids, reduction=None, return_grad=True, **kw)
    assert losses.shape == (rows,) and losses.dtype == F32 and grad.dtype == dtype and grad.is_contiguous()
    err = check_distill(x, tl, ids, T, rest, w, losses, grad)
    # without the gradient another kernel adds the row up in another order: within the same bound of the exact loss
    check_distill(x, tl, ids, T, rest, w, M.distill_loss(x, tl, ids, reduction=None, **kw))
    # autograd: one value a row, then reduced
    xg = x.detach().requires_grad_()
    up = torch.randn(rows, generator=torch.Generator().manual_seed(6))
    g, = torch.autograd.grad(M.distill_loss(xg, tl, ids, reduction=None, **kw), xg, up.cuda())
    check_distill(x, tl, ids, T, rest, w, None, g, up=up.double().numpy())
    total = losses.double().sum().item()
    size = losses.double().abs().sum().item()
    for reduction, scale in (('sum', 1.0), ('mean', 1.0 / rows)):
        loss, g1 = M.distill_loss(x, tl, ids, reduction=reduction, return_grad=True, **kw)
        assert abs(loss.item() - total * scale) <= 4 * R.U * abs(total * scale) + 1e-14 * size
        check_distill(x, tl, ids, T, rest, w, None, g1, scale=scale)
        xg = x.detach().requires_grad_()
        l2 = M.distill_loss(xg, tl, ids, reduction=reduction, **kw)
        # both sums lie within err (the rows' bounds added) of the exact one, and each rounds once
        assert abs(l2.item() - loss.item()) <= scale * 2 * err + 2 * R.U * abs(loss.item())
        g2, = torch.autograd.grad(3.0 * l2, xg)
        check_distill(x, tl, ids, T, rest, w, None, g2, scale=3.0 * scale)


@pytest.mark.parametrize('rest', ['renormalise', 'bucket'])
@pytest.mark.parametrize('C', [40, 900, 20000])
def test_distill_lists_with_gaps_duplicates_and_odd_values(C, rest):
    rows, K = 12, 7
    x = _make(C, rows, C, F32)
    tl, ids = _list(1, x, K, 1.0)
    ids[0] = -1                                                 # nothing listed
    ids[1, 1:] = -1
    ids[2, 3] = ids[2, 0]                                       # the same class twice, three times
    ids[3, 2] = ids[3, 4] = ids[3, 6]
    ids[4, 0] = C                                               # outside
    ids[4, 1] = 2 ** 31 - 1
    ids[4, 2] = -2 ** 31
    tl[5, 2:] = -INF                                            # listed without probability
    tl[6] = -INF
    x[7, ids[7, 1].item()] = -INF                               # the student forbids a class the teacher uses: infinite
    x[8] = -INF                                                 # an empty row
    x[9, C // 4:] = torch.finfo(F32).min
    off = torch.ones(C, dtype=torch.bool)
    off[ids[10].long().cpu()] = False
    x[10, off.cuda()] = -INF                                    # the student has nothing off the list
    x[11, off.cuda()] = -200.0                                  # next to nothing (some of the listed classes differ: fine)
    losses, grad = M.distill_loss(x, tl, ids, rest=rest, reduction=None, return_grad=True)
    check_distill(x, tl, ids, 1.0, rest, None, losses, grad)
    assert losses[7].item() == INF and losses[8].item() == 0 and (grad[8] == 0).all()
    if rest == 'renormalise':
        assert losses[0].item() == 0 and (grad[0] == 0).all()


def test_distill_ignored_rows_are_not_read_and_bad_rows_are_nan():
    x = _make(1, 6, 500, BF16)
    tl, ids = _list(2, x, 4, 1.0)
    w = torch.tensor([1.0, 0.0, 2.0, 0.0, 1.0, 1.0]).cuda()
    x[1] = float('nan')
    x[3] = INF
    x[5, 3] = float('nan')
    losses, grad = M.distill_loss(x, tl, ids, row_weights=w, reduction=None, return_grad=True)
    assert losses[1].item() == 0 and losses[3].item() == 0 and (grad[1] == 0).all() and (grad[3] == 0).all()
    assert torch.isnan(losses[5]) and torch.isnan(grad[5].float()).all()
    assert torch.isfinite(losses[[0, 2, 4]]).all() and torch.isfinite(grad[[0, 2, 4]].float()).all()
    xg = x.detach().requires_grad_()
    g, = torch.autograd.grad(M.distill_loss(xg, tl, ids, row_weights=w, reduction=None)[:5].sum(), xg)
    assert (g[1] == 0).all() and (g[3] == 0).all() and torch.isfinite(g[:5].float()).all()


@pytest.mark.parametrize('rest', ['renormalise', 'bucket'])
def test_distill_gradient_against_differences(rest):
    """Central differences of the forward kernel, h = 2^-5: the loss's third derivative is below 4 T^2 / T^3; the difference of
    two losses off by 4e-6 each is divided by 2 h."""
    C, K, h, T = 14, 5, 2.0 ** -5, 1.5
    x = _make(3, 1, C, F32, sigma=1.0)
    tl, ids = _list(4, x, K, T)
    step = h * torch.eye(C, device='cuda')

    def f(v):
        return M.distill_loss(v, tl.expand(C, K), ids.expand(C, K), temperature=T, rest=rest, reduction=None).double()
    want = (f(x + step) - f(x - step)) / (2 * h)
    _, grad = M.distill_loss(x, tl, ids, temperature=T, rest=rest, return_grad=True)
    assert (grad[0] - want).abs().max() < 2 * h * h / 6 * 4 / T + 4 * 4e-6 / (2 * h)


@pytest.mark.parametrize('C', [90, 1400, 11921, 60001])
@pytest.mark.parametrize('T', [1.0, 4.0])
def test_bucket_where_student_and_teacher_hardly_differ(C, T):
    """The list holds little and both masses off it are near 1: the loss is a small difference, and has to come from what is listed.

    Bound.  e = U (4 t + 4 + adds(C) + 4 l2) is a sum's relative error (Row.err over all classes at most `spread`, its largest).  on / off is off
    by 2 e relative, so log p0 = -log(1 + on / off) by p_on (2 e + 4 U); q by (K + 8 + 4 |log q|) U relative, log q0 by as much of sum q / q0.
    A listed term by q (q_rel |d| + e + q_rel + 4 U (|log q| + |log p|)), and every product and sum by a few U of its own size."""
    rows, K = 24, 3
    g = torch.Generator().manual_seed(C)
    teacher = torch.randn(rows, C, generator=g).cuda()
    x = teacher + 0.05 * torch.randn(rows, C, generator=g).cuda()
    r = M.label_logprobs(teacher, top_k=K, temperature=T)
    tl, ids = r.top_logprobs, r.top_labels
    loss, grad = M.distill_loss(x, tl, ids, temperature=T, rest='bucket', reduction=None, return_grad=True)
    leaf = x.clone().requires_grad_()
    again, = torch.autograd.grad(M.distill_loss(leaf, tl, ids, temperature=T, rest='bucket'), leaf)
    xs, t, n = _np(x), _np(tl), ids.cpu().numpy()
    for i in range(rows):
        row = R.Row(xs[i], T)
        want, wg, _, _ = R.distill(row, t[i], n[i], True, 1.0)
        q, lp = np.exp(t[i]), row.logp[n[i]]
        q0, p_on, e, U = 1 - q.sum(), row.p[n[i]].sum(), row.err.max(), R.U
        q_rel = U * (K + 8 + 4 * np.abs(t[i]))
        mass_err = (q * q_rel).sum() + 2 * U * q.sum()
        err = (q * (q_rel * np.abs(t[i] - lp) + e + q_rel + 4 * U * (np.abs(t[i]) + np.abs(lp)))).sum()
        err += p_on * (2 * e + 4 * U) + mass_err / q0 + 8 * U * (abs(np.log(q0)) + abs(np.log(1 - p_on)) + np.abs(q * (t[i] - lp)).sum())
        R.within(float(loss[i]), want, T * T * err + 4 * U * want, 'loss of row %d' % i)
        # off the list: T r_i (sum q - p_on)
        off = np.ones(C, bool)
        off[n[i]] = False
        dense = p_on * (2 * e + 4 * U) + mass_err
        bound = T * row.p[off] / (1 - p_on) * dense + (2 * e + 16 * U) * np.abs(wg[off]) + R.TINY[F32]
        for got in (grad, again):
            R.within(_np(got[i])[off], wg[off], bound, 'gradient of row %d' % i)


def test_renormalised_list_does_not_see_a_shift_of_the_teacher():
    x = _make(5, 8, 200, F32)
    t = torch.randn(8, 10, generator=torch.Generator().manual_seed(1)).cuda()
    t = (t * 64).round() / 64                                   # so that adding 16 is exact
    ids = torch.stack([torch.randperm(200, generator=torch.Generator().manual_seed(i))[:10] for i in range(8)]).int().cuda()
    a = M.distill_loss(x, t, ids, reduction=None)
    assert torch.equal(a, M.distill_loss(x, t + 16.0, ids, reduction=None))


# ---------------------------------------------------------------------------------------------- as a program uses them
def test_teacher_to_student_step():
    """The teacher's scores feed the student's loss; the student's own scores (a policy term) and the dense focal loss on the
    same logits join it; one backward."""
    B, N, C, K, T = 2, 150, 80, 6, 2.0
    gen = torch.Generator().manual_seed(9)
    feats = torch.randn(B, N, 16, generator=gen).cuda()
    wt = torch.randn(16, C, generator=gen).cuda()
    ws = torch.randn(16, C, generator=gen).cuda().requires_grad_()
    r = M.label_logprobs(feats @ wt, top_k=K, temperature=T)
    labels = r.top_labels[..., 0].clone()
    labels[:, ::3] = -1
    mask = (labels >= 0).float()
    y_true = torch.nn.functional.one_hot(labels.clamp(min=0).long(), C).float()

    def step():
        logits = feats @ ws
        s = M.label_logprobs(logits, labels)
        return (M.distill_loss(logits, r.top_logprobs, r.top_labels, temperature=T, row_weights=mask, reduction='mean')
                - 0.1 * s.logprobs.sum() - 0.01 * s.entropy.mean() + 0.01 * M.focal_loss(y_true, logits, from_logits=True))

    loss = step()
    grad, = torch.autograd.grad(loss, ws)
    # the same in float64 on the host, focal's own gradient taken from its operator
    w64 = ws.detach().double().cpu().requires_grad_()
    z = feats.double().cpu() @ w64
    tl, ti, lab, mk = r.top_logprobs.double().cpu(), r.top_labels.long().cpu(), labels.long().cpu(), mask.double().cpu()
    q = torch.softmax(tl, -1)
    rows = T * T * mk * (q * (q.log() - torch.log_softmax(z / T, -1).gather(-1, ti))).sum(-1)
    lp = torch.log_softmax(z, -1)
    given = torch.where(lab >= 0, lp.gather(-1, lab.clamp(min=0)[..., None])[..., 0], 0.0)
    ent = -(lp.exp() * lp).sum(-1)
    want, = torch.autograd.grad(rows.mean() - 0.1 * given.sum() - 0.01 * ent.mean(), w64)
    ones, = torch.autograd.grad(0.01 * M.focal_loss(y_true, feats @ ws, from_logits=True), ws)
    want = want + ones.double().cpu()
    # 300 rows of gradients (1e-6 relative each), a float32 product of 300 terms
    assert (grad.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()
    with torch.no_grad():
        ws -= 1e-3 * grad
    assert torch.isfinite(step())


def _sample(rows):
    """A few rows of many: the first, the last and some between."""
    return sorted({0, 1, rows // 3, rows // 2, rows - 2, rows - 1})


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,C,k', [(1030, 1500, 33), (1100, 4100, 128), (1030, 9001, 5), (1100, 16390, 64), (1030, 40003, 20), (1030, 70001, 128)])
def test_many_long_rows_with_top_classes(rows, C, k, dtype):
    """Whole rows a block (few rows are split instead): some against the definition, all classes against the split kernel's."""
    x = _make(C, rows, C, dtype)
    labels = torch.arange(rows) % C
    labels[3::7] = -1
    r = M.label_logprobs(x, labels.cuda(), top_k=k)
    at = _sample(rows)
    check_scores(x[at], labels[at], k, 1.0, M.LabelLogprobs(r.logprobs[at], r.entropy[at], r.top_logprobs[at], r.top_labels[at]))
    few = M.label_logprobs(x[:200], labels[:200].cuda(), top_k=k)
    assert torch.equal(r.top_labels[:200], few.top_labels)


@pytest.mark.parametrize('rest', ['renormalise', 'bucket'])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('rows,C,K,pad', [(530, 2100, 128, 0), (600, 3001, 7, 5), (520, 9000, 33, 0), (530, 16001, 64, 2), (520, 33333, 5, 0),
                                          (515, 65537, 20, 0), (515, 131073, 9, 0)])
def test_many_long_rows_with_their_gradient(rows, C, K, pad, dtype, rest):
    """The one-read kernel and, where a row does not fit a block's registers, the kernels beside it; masked rows among them."""
    x = _make(C, rows, C, dtype, pad=pad)
    tl, ids = _list(C, x, K, 1.0)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(5)).cuda() + 0.5
    w[1::5] = 0.0
    x[rows // 2] = -INF
    x[rows // 3, : C // 2] = torch.finfo(dtype).min
    ids[rows - 1, 1:3] = ids[rows - 1, 0]
    ids[0, -1] = -1
    losses, grad = M.distill_loss(x, tl, ids, rest=rest, row_weights=w, reduction=None, return_grad=True)
    at = _sample(rows)
    check_distill(x[at], tl[at], ids[at], 1.0, rest, w[at], losses[at], grad[at])
    assert (losses[1::5] == 0).all() and (grad[1::5] == 0).all() and losses[rows // 2].item() == 0 and (grad[rows // 2] == 0).all()
    xg = x.detach().requires_grad_()
    l2 = M.distill_loss(xg, tl, ids, rest=rest, row_weights=w, reduction=None)
    g2, = torch.autograd.grad(l2.sum(), xg)
    check_distill(x[at], tl[at], ids[at], 1.0, rest, w[at], l2[at], g2[at])
    # Every row both ways.  A probability is off by at most u (4 |t| + 4 + adds + 4 l2) relative, |t| < 120 and l2 < 17 here, and a
    # gradient by half a step of its type.  Off a renormalised list the gradient is a product with p; elsewhere it is a
    # difference of probabilities (at most w), so that the same error counts absolutely.
    rel = 2 * R.U * (4 * 120 + 4 + R.adds(C) + 4 * 17)
    a, b = grad.double(), g2.double()
    differences = torch.zeros_like(a)
    if rest == 'bucket':
        differences += w[:, None]
    else:
        differences.scatter_(1, ids.clamp(min=0).long(), w.double()[:, None].expand(-1, K).contiguous())
    assert ((a - b).abs() <= (2 * R.EPS[dtype] + rel) * a.abs() + rel * differences + 2 * R.TINY[dtype]).all()


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_millions_of_classes(dtype):
    rows, C = 2, 3000001
    x = _make(7, rows, C, dtype)
    labels = torch.tensor([C - 1, 5])
    r = M.label_logprobs(x, labels.cuda(), top_k=128)
    check_scores(x, labels, 128, 1.0, r)
    tl, ids = r.top_logprobs - 0.5, r.top_labels.clone()
    ids[1, 3] = C - 1
    for rest in ('renormalise', 'bucket'):
        losses, grad = M.distill_loss(x, tl, ids, rest=rest, reduction=None, return_grad=True)
        check_distill(x, tl, ids, 1.0, rest, None, losses, grad)


@pytest.mark.parametrize('rest', ['renormalise', 'bucket'])
def test_more_logits_than_the_caches_hold(rest):
    rows, C = 1100, 131075                                       # 288 MB, rows at odd addresses
    x = _make(1, 11, C, BF16)[torch.arange(rows).cuda() % 11]
    labels = (torch.arange(rows) * 119) % C
    at = _sample(rows)
    r = M.label_logprobs(x, labels.cuda())
    check_scores(x[at], labels[at], 0, 1.0, M.LabelLogprobs(r.logprobs[at], r.entropy[at], None, None))
    tl, ids = _list(2, x[:11], 16, 1.0)
    pick = torch.arange(rows).cuda() % 11
    losses = M.distill_loss(x, tl[pick], ids[pick], rest=rest, reduction=None)
    check_distill(x[at], tl[pick][at], ids[pick][at], 1.0, rest, None, losses[at])
    assert torch.equal(losses[:88], losses[88:176])              # the same rows on the same boundaries (8 rows of 131075 apart)
    xg = x.detach().requires_grad_()
    g, = torch.autograd.grad(M.label_logprobs(xg, labels.cuda()).logprobs.sum(), xg)
    check_score_grad(x[at], labels[at], 0, 1.0, np.ones(len(at)), np.zeros(len(at)), np.zeros((len(at), 1)), [[0]] * len(at), g[at])


@pytest.mark.parametrize('rest', ['renormalise', 'bucket'])
def test_gradient_of_more_logits_than_the_caches_hold(rest):
    """A gradient has the bits that its rows give in a smaller call."""
    rows, C, part = 82000, 4100, 2048                           # 672 MB
    x = _make(5, part, C, BF16).repeat(41, 1)[:rows]
    tl, ids = _list(5, x[:part], 5, 1.0)
    tl, ids = tl.repeat(41, 1)[:rows], ids.repeat(41, 1)[:rows]

    def grad(n):
        leaf = x[:n].requires_grad_()
        loss = M.distill_loss(leaf, tl[:n], ids[:n], rest=rest, reduction=None)
        return loss, torch.autograd.grad(loss.sum(), leaf)[0]
    l0, g0 = grad(part)
    l, g = grad(rows)
    for r in range(0, rows, part):
        n = min(part, rows - r)
        assert torch.equal(l[r:r + n], l0[:n]) and torch.equal(g[r:r + n], g0[:n]), r


def test_results_do_not_change_from_call_to_call():
    x = _make(1, 40, 30011, BF16)
    x = (x.float() * 4).round().div(4).to(BF16)                 # many ties
    tl, ids = _list(1, x, 64, 1.0)
    labels = torch.arange(40).cuda()
    a = M.label_logprobs(x, labels, top_k=64)
    la, ga = M.distill_loss(x, tl, ids, rest='bucket', reduction='mean', return_grad=True)
    for _ in range(4):
        b = M.label_logprobs(x, labels, top_k=64)
        lb, gb = M.distill_loss(x, tl, ids, rest='bucket', reduction='mean', return_grad=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(la, lb) and torch.equal(ga, gb)


def test_many_row_losses_are_summed_in_double():
    rows = 70001
    x = _make(2, rows, 9, F32)
    tl, ids = _list(2, x, 3, 1.0)
    losses = M.distill_loss(x, tl, ids, reduction=None)
    for reduction, n in (('sum', 1), ('mean', rows)):
        got = M.distill_loss(x, tl, ids, reduction=reduction).item()
        want = losses.double().sum().item() / n
        assert abs(got - want) <= 4 * R.U * abs(want) + 1e-12


def test_empty_batches():
    x = torch.zeros(0, 50, device='cuda', requires_grad=True)
    r = M.label_logprobs(x, torch.zeros(0, dtype=torch.int32), top_k=3)
    assert r.logprobs.shape == (0,) and r.top_labels.shape == (0, 3)
    g, = torch.autograd.grad([r.logprobs, r.top_logprobs], x, [torch.zeros(0).cuda(), torch.zeros(0, 3).cuda()])
    assert g.shape == (0, 50)
    for reduction in ('sum', 'mean', None):
        loss = M.distill_loss(x, torch.zeros(0, 4), torch.zeros(0, 4, dtype=torch.int32), reduction=reduction)
        assert loss.sum().item() == 0 and loss.shape == ((0,) if reduction is None else ())
        g, = torch.autograd.grad(loss.sum(), x)
        assert g.shape == (0, 50)
    assert M.label_logprobs(torch.zeros(2, 0, 50)).entropy.shape == (2, 0)


def test_rows_beyond_32_bit_offsets():
    C, apart = 5003, 2 ** 31 + 64
    buf = torch.empty(2 * apart + C, dtype=BF16, device='cuda')
    x = buf.as_strided((3, C), (apart, 1))
    x.copy_(_make(8, 3, C, BF16))
    labels = torch.tensor([1, 2, 5000])
    check_scores(x, labels, 5, 1.0, M.label_logprobs(x, labels.cuda(), top_k=5))
    tl, ids = _list(3, x, 5, 1.0)
    losses, grad = M.distill_loss(x, tl, ids, reduction=None, return_grad=True)
    check_distill(x, tl, ids, 1.0, 'renormalise', None, losses, grad)
    xg = x.detach().requires_grad_()
    g, = torch.autograd.grad(M.label_logprobs(xg, labels.cuda()).logprobs.sum(), xg)
    check_score_grad(x, labels, 0, 1.0, np.ones(3), np.zeros(3), np.zeros((3, 1)), [[0]] * 3, g)
    del buf, x, xg, g, grad


def test_gradients_beyond_32_bit_offsets():
    rows, C = 17000, 131072                                     # 2.2e9 elements
    x = _make(1, 5, C, BF16)
    pick = torch.arange(rows) % 5
    few = x.expand(1, 5, C)[0]
    big = few[pick.cuda()]
    tl, ids = _list(3, few, 4, 1.0)
    w = torch.zeros(rows, device='cuda')
    w[[0, 1, 8000, rows - 2, rows - 1]] = 1.0
    at = [0, 1, 8000, rows - 2, rows - 1]
    losses, grad = M.distill_loss(big, tl[pick], ids[pick], row_weights=w, reduction=None, return_grad=True)
    check_distill(big[at], tl[pick][at], ids[pick][at], 1.0, 'renormalise', None, losses[at], grad[at])
    assert int((grad[7990:8000] != 0).sum()) == 0
    del big, grad


@pytest.mark.parametrize('C', [80, 40000])
def test_another_stream_and_host_inputs(C):
    x = _make(C, 20, C, F32)
    tl, ids = _list(C, x, 4, 1.0)
    labels = torch.arange(20)
    want = M.label_logprobs(x, labels.cuda(), top_k=4)
    lw, gw = M.distill_loss(x, tl, ids, return_grad=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = torch.empty_like(x).copy_(x)
        got = M.label_logprobs(y, labels.cuda(), top_k=4)
        lg, gg = M.distill_loss(y, tl, ids, return_grad=True)
        yg = y.detach().requires_grad_()
        ga, = torch.autograd.grad(M.distill_loss(yg, tl, ids), yg)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and torch.equal(lw, lg) and torch.equal(gw, gg)
    check_distill(x, tl, ids, 1.0, 'renormalise', None, None, ga)
    host = M.label_logprobs(x.cpu().numpy(), labels.numpy(), top_k=4)
    assert host.entropy.is_cuda and all(torch.equal(a, b) for a, b in zip(want, host))


@pytest.mark.parametrize('rows,C', [(3, 60001), (300, 80), (40, 9001)])
def test_replay_from_a_hip_graph(rows, C):
    """Forward, loss with gradient and an autograd step captured once and replayed on fresh inputs, eager work between."""
    K, T = 6, 1.0
    x = _make(1, rows, C, BF16)
    tl, ids = _list(1, x, K, T)
    labels = (torch.arange(rows) % C).int().cuda()

    def work(src):
        r = M.label_logprobs(src, labels, top_k=K)
        loss, grad = M.distill_loss(src, tl, ids, rest='bucket', reduction='mean', return_grad=True)
        leaf = src.detach().requires_grad_()
        s = M.label_logprobs(leaf, labels)
        g, = torch.autograd.grad([M.distill_loss(leaf, tl, ids), s.entropy], leaf, [torch.ones((), device='cuda'), labels.float()])
        return list(r) + [loss, grad, g]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(x)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                          # two graphs, neither may disturb the other's scratch memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(work(x))
        graphs.append(g)
    for seed in range(2, 6):
        x.copy_(_make(seed, rows, C, BF16))
        new = _list(seed, x, K, T)
        tl.copy_(new[0]), ids.copy_(new[1])
        for o in outs[0] + outs[1]:
            o.fill_(3)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        eager = work(x)
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, eager)), seed


def test_two_threads_on_two_streams():
    import threading
    x = [_make(i, 64, 20011, BF16) for i in range(2)]
    lists = [_list(i, x[i], 16, 1.0) for i in range(2)]
    want = [(M.label_logprobs(x[i], top_k=16), M.distill_loss(x[i], *lists[i], return_grad=True)) for i in range(2)]
    torch.cuda.synchronize()
    bad = []

    def go(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                r = M.label_logprobs(x[i], top_k=16)
                l, g = M.distill_loss(x[i], *lists[i], return_grad=True)
                s.synchronize()
                if not (torch.equal(r.top_labels, want[i][0].top_labels) and torch.equal(r.entropy, want[i][0].entropy)
                        and torch.equal(l, want[i][1][0]) and torch.equal(g, want[i][1][1])):
                    bad.append(i)
    ts = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_gradient_of_a_broadcast_row():
    x = _make(1, 1, 300, F32).requires_grad_()
    labels = torch.arange(8).cuda()
    g, = torch.autograd.grad(M.label_logprobs(x.expand(8, 300), labels).logprobs.sum(), x)
    each = [torch.autograd.grad(M.label_logprobs(x, labels[i:i + 1]).logprobs.sum(), x)[0] for i in range(8)]
    torch.testing.assert_close(g, torch.stack(each).sum(0), rtol=0, atol=16 * R.U)


@pytest.mark.parametrize('C', [90, 5000])
def test_gradients_without_labels_and_of_some_outputs(C):
    x = _make(C, 6, C, F32).requires_grad_()
    r = M.label_logprobs(x, top_k=2)
    assert r.logprobs is None and r.entropy.requires_grad and r.top_logprobs.requires_grad and not r.top_labels.requires_grad
    g, = torch.autograd.grad(r.top_logprobs[:, 1].sum(), x, retain_graph=True)
    up = np.zeros((6, 2))
    up[:, 1] = 1
    check_score_grad(x, torch.full((6,), -1), 2, 1.0, np.zeros(6), np.zeros(6), up, r.top_labels.tolist(), g)
    g2, = torch.autograd.grad(r.top_logprobs[:, 1].sum(), x)     # the same graph once more
    assert torch.equal(g, g2)
    with torch.no_grad():
        assert not M.label_logprobs(x).entropy.requires_grad
    y = torch.randn(3, C, device='cuda', dtype=torch.float64, requires_grad=True)
    g, = torch.autograd.grad(M.label_logprobs(y, torch.zeros(3, dtype=torch.int64)).logprobs.sum(), y)
    assert g.dtype == torch.float64 and g.shape == y.shape


def test_inputs_changed_before_the_backward_pass_are_noticed():
    x = _make(1, 4, 50, F32).requires_grad_()
    tl, ids = _list(1, x.detach(), 3, 1.0)
    loss = M.distill_loss(x, tl, ids)
    ids.zero_()
    with pytest.raises(RuntimeError):
        loss.backward()


def test_ids_wider_than_int32():
    x = _make(2, 4, 50, F32)
    wide = torch.tensor([7, (1 << 32) + 7, -(1 << 63), 1 << 40])
    fits = torch.tensor([7, -1, -1, -1])
    a, b = M.label_logprobs(x, wide), M.label_logprobs(x, fits.int().cuda())
    assert torch.equal(a.logprobs, b.logprobs) and (a.logprobs[1:] == 0).all() and a.logprobs[0] < 0
    tl = torch.full((4, 2), -1.0)
    la, lb = (M.distill_loss(x, tl, torch.stack([torch.arange(4), i], -1).cuda(), reduction=None) for i in (wide, fits))
    assert torch.equal(la, lb)
    for bad in (torch.zeros(4), torch.zeros(4, device='cuda', dtype=F16)):
        with pytest.raises(ValueError):
            M.label_logprobs(x, bad)


def test_python_refusals():
    x = torch.zeros(4, 10, device='cuda')
    ids = torch.zeros(4, 3, dtype=torch.int32)
    tl = torch.zeros(4, 3)
    for kw in (dict(top_k=11), dict(top_k=-1), dict(temperature=0.0), dict(temperature=float('nan')), dict(temperature=1e7),
               dict(labels=torch.zeros(5, dtype=torch.int32)), dict(labels=torch.zeros(4, 1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            M.label_logprobs(x, **kw)
    with pytest.raises(ValueError):
        M.label_logprobs(torch.zeros(4, 1000, device='cuda'), top_k=129)
    for bad in (torch.zeros(4, 0, device='cuda'), torch.zeros((), device='cuda')):
        with pytest.raises(ValueError):
            M.label_logprobs(bad)
    for a, kw in (((tl, ids[:, :0]), {}), ((tl[:, :2], ids), {}), ((tl, ids[:3]), {}), ((tl, ids), dict(rest='tail')),
                  ((tl, ids), dict(temperature=-1.0)), ((tl, ids), dict(row_weights=torch.ones(3))),
                  ((torch.zeros(4, 129), torch.zeros(4, 129, dtype=torch.int32)), {})):
        with pytest.raises(ValueError):
            M.distill_loss(x, *a, **kw)
    xg = x.clone().requires_grad_()
    g, = torch.autograd.grad(M.distill_loss(xg, tl, ids), xg, create_graph=True)
    with pytest.raises(RuntimeError):                           # no second derivative, and it says so
        torch.autograd.grad(g.sum(), xg)
    assert M.MAX_TOP == 128 and _lib.load() is not None
