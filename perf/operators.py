"""The class-logit operators of object_detection_amd.metric as measured: log-probabilities of given labels with
entropy and top alternatives (`label_logprobs`), and distillation from a teacher's top classes (`distill_loss`).

`listed()` holds the cases, `prepare` makes what a program has in hand before the call, `run` is one pass: in elementary
torch operations in 32 bits (64 where 32 lose what matters) while `own` is false, through the package's entry points
while it is true.  `exact` is the same from the definition in 64 bits."""
import math

import torch

own = False

_DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_MAX_ELEMENTS = 4096 * 131072           # the largest listed case's logits; a drawn case stays below
_ROWS_AT_A_TIME = 1 << 27               # elements the plain selection of top classes ranks at once


def listed():
    return [
        # one token of one sequence: the score of the sampled id and eight alternatives, latency counts
        dict(name='score-one', op='score', rows=1, classes=131072, dtype='bf16', top=8, temperature=1.0, labels=True,
             masked=0.0, grad=False),
        # a decode batch under a grammar mask (three classes in five forbidden), float32 logits, a temperature
        dict(name='score-decode-48', op='score', rows=48, classes=65537, dtype='f32', top=20, temperature=0.7, labels=True,
             masked=0.6, grad=False),
        # a prompt's scores: log-probability and entropy of every position, padded positions labelled -1
        dict(name='score-prompt', op='score', rows=2048, classes=131072, dtype='bf16', top=0, temperature=1.0, labels=True,
             masked=0.0, grad=False),
        # a teacher's pass that stores its 64 best classes a row
        dict(name='score-teacher', op='score', rows=4096, classes=32768, dtype='bf16', top=64, temperature=2.0, labels=False,
             masked=0.0, grad=False),
        # five alternatives for every anchor of a batch of 8 images of 512 x 512 with 80 classes
        dict(name='score-anchors', op='score', rows=8 * 49104, classes=80, dtype='f32', top=5, temperature=1.0, labels=True,
             masked=0.0, grad=False),
        # a policy-gradient step: weighted log-probabilities and an entropy bonus, forward and backward, odd sizes
        dict(name='score-step', op='score', rows=1021, classes=100003, dtype='f16', top=0, temperature=1.0, labels=True,
             masked=0.0, grad=True),
        # a whole-image head of 1000 classes, small batch: loss and gradient
        dict(name='distill-images', op='distill', rows=16, classes=1000, dtype='f32', top=10, temperature=4.0,
             rest='renormalise', mode='grad', ragged=False, pad=0),
        # the class head of 8 images' anchors in half precision, autograd, a quarter of the rows weighted 0
        dict(name='distill-anchors', op='distill', rows=8 * 49104, classes=80, dtype='f16', top=8, temperature=2.0,
             rest='renormalise', mode='autograd', ragged=False, pad=0),
        # odd rows and classes, the teacher's remaining mass as one more class, lists of unequal length
        dict(name='distill-odd', op='distill', rows=777, classes=50021, dtype='f32', top=32, temperature=1.0,
             rest='bucket', mode='grad', ragged=True, pad=0),
        # evaluation of a student: the losses alone
        dict(name='distill-eval', op='distill', rows=2048, classes=32768, dtype='f32', top=20, temperature=1.0,
             rest='renormalise', mode='forward', ragged=False, pad=0),
        # a training step through autograd, rows of a padded vocabulary
        dict(name='distill-autograd', op='distill', rows=2048, classes=131072, dtype='bf16', top=64, temperature=1.0,
             rest='bucket', mode='autograd', ragged=False, pad=128),
        # the largest: a training step that takes loss and gradient from one call
        dict(name='distill-step', op='distill', rows=4096, classes=131072, dtype='bf16', top=64, temperature=2.0,
             rest='renormalise', mode='grad', ragged=True, pad=0),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(['score', 'distill'])
    classes = spread(8, 262144)
    rows = spread(1 if op == 'score' else 4, min(8 * 49104, _MAX_ELEMENTS // (2 * classes)))
    if rng.random() < 0.5:
        classes |= 1
    case = dict(op=op, rows=rows, classes=classes, dtype=rng.choice(['f32', 'f16', 'bf16']),
                temperature=rng.choice([0.7, 1.0, 2.0, 4.0]))
    if op == 'score':
        grad = rng.random() < 0.35
        case.update(top=0 if grad else rng.choice([0, min(spread(1, 128), classes)]), labels=grad or rng.random() < 0.8,
                    masked=0.0 if grad else rng.choice([0.0, 0.4]), grad=grad)
    else:
        case.update(top=min(spread(1, 128), classes), rest=rng.choice(['renormalise', 'bucket']),
                    mode=rng.choice(['forward', 'grad', 'autograd']), ragged=rng.random() < 0.5, pad=rng.choice([0, 0, 8, 37]))
    return case


def _weighted(rows):
    """How many of the rows carry a weight: a quarter of an anchor batch is ignored, one row in 16 of a longer one."""
    return rows - (rows // 4 if rows >= 65536 else rows // 16)


def _loss_scale(case):
    """What a half-precision step multiplies its mean loss with, so that gradients stay in float16's range."""
    return float(2 ** math.ceil(math.log2(case['rows']))) if case['dtype'] == 'f16' else 1.0


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    R, C, K, dt = case['rows'], case['classes'], case['top'], _DTYPES[case['dtype']]

    def logits():
        # a broad background and a few classes that stand out, as a trained head gives
        x = torch.randn(R, C, generator=gen, device=dev) * 2.0 - 3.0
        few = min(12, C)
        at = torch.randint(0, C, (R, 1), generator=gen, device=dev) + torch.arange(few, device=dev) * (C // few)
        at %= C
        up = torch.rand(R, few, generator=gen, device=dev) * 4.0 + 2.0 + 0.6 * math.log(max(C, 12) / 12)
        return x.scatter_(1, at, up)

    x = logits()
    state = dict(case=case)
    if case['op'] == 'score':
        lab = torch.randint(0, C, (R,), generator=gen, device=dev)
        if case['masked']:
            off = torch.rand(R, C, generator=gen, device=dev) < case['masked']
            off.scatter_(1, lab[:, None], False)               # a sampled label is never a forbidden one
            x = x.masked_fill_(off, -math.inf)
        if R >= 16:
            lab[torch.randperm(R, generator=gen, device=dev)[:R // 16]] = -1
        state['labels'] = lab.to(torch.int32) if case['labels'] else None
        if case['grad']:
            scale = _loss_scale(case) / R
            state['up_logprobs'] = torch.randn(R, generator=gen, device=dev) * scale
            state['up_entropy'] = torch.full((R,), 0.01 * scale, device=dev)
        state['logits'] = x.to(dt)
        return state
    # the teacher sees the same rows a little differently; its list is what its own scores rank best
    step = max(1, _ROWS_AT_A_TIME // C)
    ids = torch.empty(R, K, dtype=torch.int32, device=dev)
    lps = torch.empty(R, K, device=dev)
    for r in range(0, R, step):
        t = (x[r:r + step] + 1.5 * torch.randn(min(step, R - r), C, generator=gen, device=dev)) / case['temperature']
        order = torch.argsort(t, dim=1, descending=True, stable=True)[:, :K]
        ids[r:r + step] = order.to(torch.int32)
        lps[r:r + step] = (t.gather(1, order).double() - torch.logsumexp(t.double(), 1, keepdim=True)).float()
    if case['ragged']:
        n = torch.randint(1, K + 1, (R, 1), generator=gen, device=dev)
        ids = torch.where(torch.arange(K, device=dev)[None] < n, ids, -1)
    w = torch.rand(R, generator=gen, device=dev) + 0.5
    w[torch.randperm(R, generator=gen, device=dev)[:R - _weighted(R)]] = 0.0
    if case['mode'] == 'grad':
        w *= _loss_scale(case)
    elif case['mode'] == 'autograd':
        state['up_loss'] = torch.full((), _loss_scale(case), device=dev)
    if case['pad']:
        buf = torch.zeros(R, C + case['pad'], dtype=dt, device=dev)
        buf[:, :C] = x
        x = buf[:, :C]
    state.update(logits=x.to(dt), teacher_logprobs=lps, teacher_labels=ids.contiguous(), row_weights=w)
    return state


# ---------------------------------------------------------------------------------------------- the plain forms
def _softmax_parts(x):
    """x - max, exp of it and the sum; a class at -inf has probability 0."""
    z = x - x.amax(1, keepdim=True)
    e = torch.exp(z)
    return z, e, e.sum(1, keepdim=True)


def _plain_top(x, k):
    """The k largest of each row by (value, then lowest index): one 64-bit key an element, so nothing ties."""
    C = x.shape[1]
    step = max(1, _ROWS_AT_A_TIME // C)
    low = C - 1 - torch.arange(C, device=x.device, dtype=torch.int64)
    out = []
    for r in range(0, x.shape[0], step):
        bits = (x[r:r + step] + 0.0).contiguous().view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).to(torch.int64)
        out.append(C - 1 - (torch.topk((order << 24) | low, k, dim=1).values & 0xffffff))
    return torch.cat(out)


def _plain_score(s, c):
    x32 = s['logits'].float()
    x = x32 / c['temperature']
    z, e, total = _softmax_parts(x)
    log_total = torch.log(total)
    p = e / total
    entropy = (log_total - (p * z.masked_fill(z == -math.inf, 0.0)).sum(1, keepdim=True))[:, 0]
    out = {'entropy': entropy}
    if s['labels'] is not None:
        lab = s['labels'].long()
        given = lab >= 0
        lp = (z.gather(1, lab.clamp(min=0)[:, None]) - log_total)[:, 0]
        out['logprobs'] = torch.where(given, lp, 0.0)
    if c['top']:
        top = _plain_top(x32, c['top'])
        out['top_logprobs'] = z.gather(1, top) - log_total
        out['top_labels'] = top.to(torch.int32)
    if c['grad']:
        up = torch.where(given, s['up_logprobs'], 0.0)[:, None]
        g = -p * (up + s['up_entropy'][:, None] * (z - log_total + entropy[:, None]))
        g.scatter_add_(1, lab.clamp(min=0)[:, None], up)
        out['grad'] = (g / c['temperature']).to(s['logits'].dtype)
    return out


def _plain_distill(s, c):
    T = c['temperature']
    z, e, total = _softmax_parts(s['logits'].float() / T)
    log_total = torch.log(total)
    ids = s['teacher_labels'].long()
    valid = ids >= 0
    first = ids[:, :1]                                          # the lists hold at least one class
    ids = torch.where(valid, ids, first)
    tl = s['teacher_logprobs'].masked_fill(~valid, -math.inf)
    w = s['row_weights'][:, None]
    lp = z.gather(1, ids) - log_total
    if c['rest'] == 'renormalise':
        tz, te, tt = _softmax_parts(tl)
        q, logq = te / tt, tz - torch.log(tt)
    else:
        q, logq = torch.exp(tl), tl
    loss = (q * (logq.masked_fill(~valid, 0.0) - lp)).sum(1, keepdim=True)
    if c['rest'] == 'bucket':
        q0 = (1.0 - torch.exp(tl.double()).sum(1, keepdim=True)).clamp(min=0.0).float()
        zr = z.scatter(1, ids, -math.inf)                       # the classes off the list, with a maximum of their own
        top = zr.amax(1, keepdim=True)
        there = top > -math.inf
        top = torch.where(there, top, 0.0)
        er = torch.exp(zr - top)
        tr = torch.where(there, er.sum(1, keepdim=True), 1.0)
        log_p0 = top + torch.log(tr) - log_total
        loss = loss + torch.where((q0 > 0) & there, q0 * (torch.log(q0) - log_p0), 0.0)
    rows = torch.where(w != 0, w * (T * T) * loss, 0.0)
    mean = rows.sum() / rows.shape[0]
    if c['mode'] == 'forward':
        return {'loss': rows[:, 0]}
    p = e / total
    if c['rest'] == 'bucket':
        g = er * (torch.where(there, torch.exp(log_p0) - q0, 0.0) / tr)
        g.scatter_(1, ids, p.gather(1, ids))
    else:
        g = p
    g.scatter_add_(1, ids, -q)
    g *= w * (T / rows.shape[0])
    if c['mode'] == 'autograd':
        g *= s['up_loss']
    return {'loss': mean, 'grad': g.to(s['logits'].dtype)}


def run(state):
    s, c = state, state['case']
    if not own:
        return _plain_score(s, c) if c['op'] == 'score' else _plain_distill(s, c)
    from object_detection_amd import metric
    if c['op'] == 'score':
        x = s['logits'].detach().requires_grad_() if c['grad'] else s['logits']
        r = metric.label_logprobs(x, s['labels'], top_k=c['top'], temperature=c['temperature'])
        out = {'entropy': r.entropy}
        if s['labels'] is not None:
            out['logprobs'] = r.logprobs
        if c['top']:
            out['top_logprobs'] = r.top_logprobs
            out['top_labels'] = r.top_labels
        if c['grad']:
            out['grad'], = torch.autograd.grad([r.logprobs, r.entropy], [x], [s['up_logprobs'], s['up_entropy']])
            out['entropy'], out['logprobs'] = r.entropy.detach(), r.logprobs.detach()
        return out
    a = (s['teacher_logprobs'], s['teacher_labels'])
    kw = dict(temperature=c['temperature'], rest=c['rest'], row_weights=s['row_weights'])
    if c['mode'] == 'forward':
        return {'loss': metric.distill_loss(s['logits'], *a, reduction='none', **kw)}
    if c['mode'] == 'grad':
        loss, grad = metric.distill_loss(s['logits'], *a, reduction='mean', return_grad=True, **kw)
        return {'loss': loss, 'grad': grad}
    x = s['logits'].detach().requires_grad_()
    loss = metric.distill_loss(x, *a, reduction='mean', **kw)
    grad, = torch.autograd.grad(loss, x, s['up_loss'])
    return {'loss': loss.detach(), 'grad': grad}


def work(case):
    R, C, K = case['rows'], case['classes'], case['top']
    size = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'score':
        n = R * C
        move = n * size * (2 if case['grad'] else 1) + R * (4 + (8 if case['labels'] else 0) + 8 * K + (8 if case['grad'] else 0))
        return {'bytes': move, 'flops': n * (6 + (6 if case['grad'] else 0))}
    live = _weighted(R)
    grads = case['mode'] != 'forward'
    move = live * C * size + (R * C * size + 4 if grads else 4 * R) + live * 8 * K + 4 * R
    return {'bytes': move, 'flops': live * C * (4 + (4 if grads else 0)) + live * K * 10}


# ---------------------------------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    x = s['logits'].double()
    T = case['temperature']
    if case['op'] == 'score':
        if case['grad']:
            x.requires_grad_()
        logp = torch.log_softmax(x / T, 1)
        entropy = torch.special.entr(logp.exp()).sum(1)
        out = {'entropy': entropy.detach()}
        if s['labels'] is not None:
            lab = s['labels'].long()
            lp = torch.where(lab < 0, 0.0, logp[torch.arange(len(lab), device=lab.device), lab.clamp(min=0)])
            out['logprobs'] = lp.detach()
        if case['top']:
            tops = []
            step = max(1, _ROWS_AT_A_TIME // case['classes'])
            for r in range(0, case['rows'], step):
                tops.append(torch.sort(x[r:r + step], dim=1, descending=True, stable=True).indices[:, :case['top']])
            top = torch.cat(tops)
            out['top_logprobs'] = logp.gather(1, top)
            out['top_labels'] = top.to(torch.int32)
        if case['grad']:
            total = (lp * s['up_logprobs'].double()).sum() + (entropy * s['up_entropy'].double()).sum()
            out['grad'], = torch.autograd.grad(total, x)
        return out
    x.requires_grad_(case['mode'] != 'forward')
    logp = torch.log_softmax(x / T, 1)
    tl, ids = s['teacher_logprobs'].double(), s['teacher_labels'].long()
    listed_ = ids >= 0
    if case['rest'] == 'renormalise':
        logq = torch.log_softmax(tl.masked_fill(~listed_, -math.inf), 1)
    else:
        logq = tl.masked_fill(~listed_, -math.inf)
    q = logq.exp()
    cross = torch.where(listed_, q * (torch.where(listed_, logq, 0.0) - logp.gather(1, ids.clamp(min=0))), 0.0).sum(1)
    if case['rest'] == 'bucket':
        q0 = (1.0 - q.sum(1)).clamp(min=0.0)
        hidden = torch.zeros_like(logp, dtype=torch.bool)
        rows = torch.arange(case['rows'], device=ids.device)[:, None].expand_as(ids)[listed_]
        hidden[rows, ids[listed_]] = True
        some = (~hidden).any(1) & (q0 > 0)
        left = torch.logsumexp(logp.masked_fill(hidden, -1e300), 1)
        cross = cross + torch.where(some, q0 * (torch.log(torch.where(some, q0, 1.0)) - left), 0.0)
    w = s['row_weights'].double()
    rows_ = T * T * w * cross
    if case['mode'] == 'forward':
        return {'loss': rows_}
    loss = rows_.mean()
    grad, = torch.autograd.grad(loss, x, s['up_loss'].double() if case['mode'] == 'autograd' else None)
    return {'loss': loss.detach(), 'grad': grad}
