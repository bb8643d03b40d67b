"""Refusals of the class-logit entry points, decided on the host before any GPU work, and the drop-in signatures; and the 64-bit
reference of their GPU tests against known answers."""
import ctypes
import inspect
import math

import numpy as np
import pytest
import torch

import logits_reference as R
from object_detection_amd import _lib, build, metric


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _lib.load()


def test_bad_arguments_are_refused(lib):
    buf = (ctypes.c_float * 64)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    if p.value % 16:
        p = ctypes.c_void_p(p.value + 16 - p.value % 16)
    odd = ctypes.c_void_p(p.value + 4)
    byte = ctypes.c_void_p(p.value + 1)
    big = 1 << 20
    score = dict(logits=p, dtype=0, rows=2, C=10, stride=10, labels=p, k=2, t=1.0, lp=p, ent=p, tlp=p, tid=p, stats=p, ws=p, n=big, s=None)
    score_b = dict(logits=p, dtype=0, rows=2, C=10, stride=10, labels=p, k=2, tid=p, t=1.0, stats=p, ulp=p, uent=p, utop=p, grad=p, s=None)
    dist = dict(logits=p, dtype=0, rows=2, C=10, stride=10, tl=p, ids=p, K=2, t=1.0, rest=0, w=p, scale=1.0, rows_=p, loss=p, stats=p, grad=p,
                ws=p, n=big, s=None)
    dist_b = dict(logits=p, dtype=0, rows=2, C=10, stride=10, tl=p, ids=p, K=2, t=1.0, rest=0, w=p, scale=1.0, stats=p, up=p, upr=0, grad=p, s=None)
    common = [dict(logits=None), dict(dtype=3), dict(dtype=-1), dict(C=0), dict(C=(1 << 24) + 1), dict(t=0.0), dict(t=-1.0), dict(t=math.nan),
              dict(t=math.inf), dict(logits=byte), dict(rows=1 << 41), dict(stride=1 << 41), dict(stats=odd)]
    for name, base, more in (
            ('odbox_label_logprobs', score, [dict(k=11), dict(k=-1), dict(k=129, C=200), dict(labels=None), dict(tlp=None), dict(tid=None)]),
            ('odbox_label_logprobs_backward', score_b, [dict(k=11), dict(stats=None), dict(grad=None), dict(labels=None), dict(tid=None),
                                                        dict(grad=byte)]),
            ('odbox_distill_loss', dist, [dict(K=0), dict(K=129), dict(rest=2), dict(tl=None), dict(ids=None), dict(rows_=None, loss=None),
                                          dict(ws=odd), dict(ws=None), dict(grad=byte)]),
            ('odbox_distill_loss_backward', dist_b, [dict(K=0), dict(rest=-1), dict(up=None), dict(stats=None), dict(grad=None), dict(grad=byte)])):
        for change in common + more:
            rc = getattr(lib, name)(*dict(base, **change).values())
            assert rc == -1, (name, change, rc, lib.odbox_last_error())
            assert name.encode() in lib.odbox_last_error(), (name, change)
    assert lib.odbox_distill_loss(*dict(dist, n=8).values()) == -3 and b'odbox_distill_loss' in lib.odbox_last_error()
    # nothing to do is a success, decided before a pointer is looked at
    assert lib.odbox_label_logprobs(*dict(score, rows=0, logits=None).values()) == 0
    assert lib.odbox_label_logprobs_backward(*dict(score_b, rows=0, logits=None).values()) == 0
    assert lib.odbox_distill_loss(*dict(dist, rows=0, logits=None, loss=None).values()) == 0
    assert lib.odbox_distill_loss_backward(*dict(dist_b, rows=0, logits=None).values()) == 0


def test_workspace_queries(lib):
    for rows in (0, 1, 7, 4096, 1 << 40):
        for C in (1, 80, 4097, 131072, 1 << 24):
            assert lib.odbox_label_logprobs_workspace(rows, C, 1) >= lib.odbox_label_logprobs_workspace(rows, C, 0) >= 0
            assert lib.odbox_distill_loss_workspace(rows, C, 128) >= 4 * rows
    for C in (0, -5):
        assert lib.odbox_label_logprobs_workspace(4, C, 1) == 0 and lib.odbox_distill_loss_workspace(4, C, 1) == 0
    assert lib.odbox_label_logprobs_workspace(4, 100, -1) == 0


def test_signatures():
    def params(f):
        return list(inspect.signature(f).parameters)
    assert params(metric.label_logprobs) == ['logits', 'labels', 'top_k', 'temperature']
    assert params(metric.distill_loss) == ['logits', 'teacher_logprobs', 'teacher_labels', 'temperature', 'rest', 'row_weights', 'reduction',
                                           'return_grad']
    assert metric.LabelLogprobs._fields == ('logprobs', 'entropy', 'top_logprobs', 'top_labels')


@pytest.mark.skipif(torch.cuda.is_available(), reason='checks the no-GPU behaviour')
def test_no_cpu_fallback():
    with pytest.raises(_lib.OdboxError):
        metric.label_logprobs(np.zeros((2, 3), np.float32))
    with pytest.raises(_lib.OdboxError):
        metric.distill_loss(np.zeros((2, 3), np.float32), np.zeros((2, 1)), np.zeros((2, 1)))


def test_rows_view_reads_in_place_what_can_be():
    x = torch.zeros(6, 20)
    assert metric._rows_view(x)[1:] == (6, 20, 20)
    v = metric._rows_view(x[:, :13])
    assert v[1:] == (6, 13, 20) and v[0].data_ptr() == x.data_ptr()
    assert metric._rows_view(x[:, :13].reshape(2, 3, 13))[1:] == (6, 13, 20)
    assert metric._rows_view(x.view(2, 3, 20)[..., :7])[1:] == (6, 7, 20)
    assert metric._rows_view(x[::2])[1:] == (3, 20, 40)
    assert metric._rows_view(x[:1].expand(5, 20))[1:] == (5, 20, 0)
    assert metric._rows_view(x.t())[1:] == (20, 6, 6) and metric._rows_view(x.t())[0].data_ptr() != x.data_ptr()
    assert metric._rows_view(x[0])[1:] == (1, 20, 20) and metric._rows_view(x[0, :1])[1:] == (1, 1, 1)
    assert metric._rows_view(torch.zeros(0, 4))[1:] == (0, 4, 4)
    assert metric._rows_view(x.view(2, 3, 20).transpose(0, 1))[1:] == (6, 20, 20)


def test_reference_known_answers():
    row = R.Row([0.0, math.log(2.0), math.log(5.0), -np.inf], 1.0)
    np.testing.assert_allclose(row.p, [0.125, 0.25, 0.625, 0.0], rtol=1e-15)
    assert abs(row.entropy - (0.125 * math.log(8) + 0.25 * math.log(4) + 0.625 * math.log(1.6))) < 1e-15
    assert R.top([1.0, 3.0, 3.0, float('nan'), -np.inf], 5) == [3, 1, 2, 0, 4]
    # teacher 0.5 / 0.25 on classes 1 and 2
    loss, grad, _, _ = R.distill(row, [math.log(0.5), math.log(0.25)], [1, 2], False, 1.0)
    q = np.array([2 / 3, 1 / 3])
    assert abs(loss - (q[0] * math.log(q[0] / 0.25) + q[1] * math.log(q[1] / 0.625))) < 1e-15
    np.testing.assert_allclose(grad, [0.125, 0.25 - q[0], 0.625 - q[1], 0.0], atol=1e-15)
    loss, grad, _, _ = R.distill(row, [math.log(0.5), math.log(0.25)], [1, 2], True, 2.0)
    assert abs(loss - 2 * (0.5 * math.log(2) + 0.25 * math.log(0.4) + 0.25 * math.log(2))) < 1e-15
    np.testing.assert_allclose(grad, 2 * np.array([0.125 - 0.25, 0.25 - 0.5, 0.625 - 0.25, 0.0]), atol=1e-15)


@pytest.mark.parametrize('bucket', [False, True])
def test_reference_gradients_against_autograd(bucket):
    gen = torch.Generator().manual_seed(1)
    C, T = 9, 1.7
    x = torch.randn(C, generator=gen, dtype=torch.float64, requires_grad=True)
    logp = torch.log_softmax(x / T, 0)
    ids, tl = [2, 5, 2, -1], torch.log(torch.tensor([0.3, 0.2, 0.1, 0.5], dtype=torch.float64))
    use = torch.tensor([2, 5, 2])
    q = tl[:3].exp() if bucket else torch.softmax(tl[:3], 0)
    loss = (q * (q.log() - logp[use])).sum()
    if bucket:
        off = torch.ones(C, dtype=torch.bool)
        off[use] = False
        q0 = 1 - q.sum()
        loss = loss + q0 * (q0.log() - torch.logsumexp(logp[off], 0))
    grad, = torch.autograd.grad(T * T * loss, x, retain_graph=True)
    row = R.Row(x.detach().numpy(), T)
    got, g, _, _ = R.distill(row, tl.numpy(), ids, bucket, 1.0)
    assert abs(got - T * T * loss.item()) < 1e-13
    np.testing.assert_allclose(g, grad.numpy(), atol=1e-13)
    ent = -(logp.exp() * logp).sum()
    grad, = torch.autograd.grad(0.5 * logp[3] + 2.0 * ent - logp[3] + 0.25 * logp[0], x)
    g, _ = R.score_grad(row, 3, 0.5, 2.0, [3, 0], [-1.0, 0.25])
    np.testing.assert_allclose(g, grad.numpy(), atol=1e-13)


def test_class_ids_that_int32_cannot_hold_are_outside_the_classes():
    wide = [3, -1, 10, -100, (1 << 32) + 3, -(1 << 63), (1 << 63) - 1, -(1 << 32)]
    got = metric._class_ids(torch.tensor(wide), 10, torch.device('cpu'), torch.Size([8]), 'labels')
    assert got.dtype == torch.int32 and got[0] == 3
    assert all(not 0 <= v < 10 for v in got[1:].tolist()), got
    assert metric._class_ids(torch.tensor([200], dtype=torch.uint8), 300, torch.device('cpu'), torch.Size([1]), 'labels').tolist() == [200]
    for bad in (torch.tensor([1.0]), torch.tensor([1.0], dtype=torch.float16)):
        with pytest.raises(ValueError):
            metric._class_ids(bad, 10, torch.device('cpu'), torch.Size([1]), 'labels')
