"""The loss in a training step's other forms: changed in place, soft targets, gradients that add up."""
import pytest
import torch as ch

from test_gpu_cross_entropy import TYPES, check, formula, make, probabilities

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_a_loss_is_changed_in_place(reduction):
    """``loss /= steps``, as in accumulation: the gradient is that of the changed loss."""
    from ffcv_b200.training import MixupCrossEntropy
    logits, labels, mixed, _ = make(24, 100, ch.float32, 3)
    for target in (labels, mixed):
        x, y = logits.clone().requires_grad_(), logits.clone().requires_grad_()
        loss = MixupCrossEntropy(0.1, reduction=reduction)(x, target)
        want = MixupCrossEntropy(0.1, reduction=reduction)(y, target) / 4
        loss /= 4
        assert ch.equal(loss, want) and not loss._is_view()
        loss += 1.0
        loss.sum().backward()
        want.sum().backward()
        assert ch.equal(x.grad, y.grad)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('classes', [10, 1000, 30001])
@pytest.mark.parametrize('smoothing', [0.0, 0.1])
def test_probabilities(classes, dtype, smoothing):
    """Targets given as probabilities, of 32 bits and of the logits' type, that need not add up to one."""
    from ffcv_b200.training import cross_entropy
    logits, _, _, gen = make(12, classes, dtype, 7)
    soft = ch.softmax(ch.randn((12, classes), generator=gen, device='cuda'), 1)
    soft[3] *= 0.25
    soft[5] = 0.0
    for given in (soft, soft.to(dtype)):
        t = probabilities(classes, soft=given, smoothing=smoothing)
        want_loss, want_grad = formula(logits, t)
        x = logits.clone().requires_grad_()
        loss = cross_entropy(x, soft=given, label_smoothing=smoothing)
        loss.backward()
        check(loss.detach(), x.grad, logits, t, want_loss, want_grad, 12)
