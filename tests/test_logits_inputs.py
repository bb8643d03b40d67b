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
