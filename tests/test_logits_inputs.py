"""What metric.label_logprobs and metric.distill_loss make of tensors that autograd or the host still has a claim on."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from object_detection_amd import metric as M


@pytest.mark.parametrize('requires_grad', [False, True])
def test_forward_mode_tangents_are_refused(requires_grad):
    """A dual tensor need not require a gradient; its tangent may not get lost without a word.  Decided before any GPU work."""
    x = torch.zeros(3, 7, requires_grad=requires_grad)
    tl, ids = torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones(3, 7))
        for call in (lambda: M.label_logprobs(d), lambda: M.distill_loss(d, tl, ids), lambda: M.distill_loss(d, tl, ids, return_grad=True)):
            with pytest.raises(NotImplementedError, match='forward-mode'):
                call()
            with pytest.raises(NotImplementedError, match='forward-mode'), torch.no_grad():
                call()
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(lambda v: M.label_logprobs(v).entropy, (x.detach(),), (torch.ones(3, 7),))


@pytest.mark.gpu
def test_pinned_inputs_may_be_written_after_the_call():
    """The stream is busy when the calls are made, so that a copy that nobody waits for would read what is written afterwards."""
    rows, C, K = 600, 5000, 8
    gen = torch.Generator().manual_seed(1)
    host = dict(x=torch.randn(rows, C, generator=gen), labels=torch.randint(0, C, (rows,), generator=gen).int(), tl=torch.randn(rows, K, generator=gen),
                ids=torch.randint(0, C, (rows, K), generator=gen).int(), w=torch.rand(rows, generator=gen))
    dev = {k: v.cuda() for k, v in host.items()}
    pinned = {k: v.pin_memory() for k, v in host.items()}

    def calls(t):
        return [M.label_logprobs(t['x'], t['labels'], top_k=3), M.distill_loss(t['x'], t['tl'], t['ids'], row_weights=t['w'], reduction=None, return_grad=True)]
    want = calls(dev)
    a = torch.randn(4096, 4096, device='cuda')
    torch.cuda.synchronize()
    for _ in range(40):
        b = a @ a
    got = calls(pinned)
    for v in pinned.values():
        v.fill_(3)
    for p, q in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(p, q))
    assert b.shape == a.shape


@pytest.mark.gpu
@pytest.mark.parametrize('pin', [False, True])
def test_host_inputs_in_a_capture(pin):
    x = torch.randn(20, 5000, generator=torch.Generator().manual_seed(2)).cuda()
    labels = torch.arange(20).int()
    labels = labels.pin_memory() if pin else labels
    want = M.label_logprobs(x, labels.cuda()).logprobs
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        M.label_logprobs(x, labels)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        r = M.label_logprobs(x, labels)
    for _ in range(3):
        r.logprobs.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.logprobs, want)
