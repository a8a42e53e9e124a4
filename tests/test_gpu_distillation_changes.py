"""Distillation beside masked classes, against the formulas in 64 bits."""
import math

import pytest

torch = pytest.importorskip('torch')
from test_gpu_distillation import BF16, F16, F32, formula, make  # noqa: E402

pytestmark = pytest.mark.gpu


def in_half_steps(got, want, both, dtype, more=0.0):
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    room = torch.finfo(dtype).eps / 2 * want.abs() + 1e-5 * both + step + more  # as in test_gpu_distillation
    return bool(((got.double() - want).abs() <= room).all())


@pytest.mark.parametrize('n,classes,kept', [(6, 3, 1), (24, 40, 6), (24, 3001, 64), (9, 50000, 64), (5, 130001, 40)])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('smoothing,tau', [(0.1, 2.0), (1.0, 3.5), (0.1, 1.0)])
@pytest.mark.parametrize('lowest', [True, False])
def test_smoothing_beside_masked_classes(n, classes, kept, dtype, smoothing, tau, lowest):
    """Masked classes have a share of a smoothed target: with -inf the loss has no end, with the type's lowest value it is as large as the formula has it.  The terms of
    the loss against labels are of one sign, and each is off by 2^-24 of itself for a difference, a product and the share's own rounding; so that loss is right to
    2^-24 (classes / 32 + 100) of itself, which allows an addition for each of 32 classes that a thread has and those of all trees.  The other one
    is off by 2e-6 of its sizes."""
    from ffcv_b200.training import distillation, distillation_with_grad
    value = torch.finfo(dtype).min if lowest else -math.inf
    gen = torch.Generator('cuda').manual_seed(classes)
    for target in ('labels', 'mixed'):
        x, t, where, how = make(n, classes, kept, dtype, target=target)
        masked = torch.rand((n, classes), generator=gen, device='cuda') < 0.5
        masked[3] = False
        x[3] = 1.0
        masked.scatter_(1, where.clamp(min=0).long(), False)  # (what the teacher knows, and labels, are not masked)
        for labels in [how['labels']] if target == 'labels' else [how['mixed'][:, 0].long(), how['mixed'][:, 1].long()]:
            masked.scatter_(1, labels[:, None], False)
        x.masked_fill_(masked, value)
        loss, grad = distillation_with_grad(x, t, where, temperature=tau, hard_weight=0.5, label_smoothing=smoothing, reduction='none', **how)
        want, grad_want, both, size = formula(x, t, where, tau=tau, hard=0.5, smoothing=smoothing, reduction='none', **how)
        endless = want == math.inf
        assert bool((endless == (masked.any(1) & (not lowest))).all()) and torch.equal(loss[endless], want[endless].float())
        room = 2e-6 * size + 1e-7 + 2.0 ** -24 * (classes / 32 + 100) * want.abs()
        assert bool(((loss.double() - want).abs() <= room)[~endless].all()), float(((loss.double() - want).abs() / room)[~endless].max())
        assert bool(want[~endless].float().isfinite().all()) and in_half_steps(grad, grad_want, both, dtype)
        leaf = x.detach().requires_grad_()
        again = distillation(leaf, t, where, temperature=tau, hard_weight=0.5, label_smoothing=smoothing, reduction='none', **how).detach()
        assert torch.equal(again[endless], loss[endless]) and bool(((again.double() - want).abs() <= room)[~endless].all())


@pytest.mark.parametrize('n,classes,kept', [(24, 40, 6), (24, 3001, 64), (5, 130001, 40)])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('tau', [0.25, 0.5, 1.0])
def test_the_lowest_value_at_temperatures_below_1(n, classes, kept, dtype, tau):
    """A teacher's row of the type's lowest value alone is uniform over its entries, beside others it is no part; a class of the teacher that is masked with it for the student costs
    tau q times as much, at any temperature.  Tolerances as in test_gpu_distillation, and what q is off by: its exponent e = (t - top) / tau is a difference, divided by tau
    and multiplied by log2(e) with a factor that has two roundings itself, so it is off by 4 roundings of 2^-24 of e, and the exponential by 2^-22 of itself (the sum of them by no
    more): 2^-22 (1 + |e|) of q, which here is multiplied by up to 3.4e38; a q below 2^-126 is 0.  A p of the gradient is off by as much, with e = (x - top) / tau, where it is not
    below 2^-126 (|e| < 88); below it is 0."""
    from ffcv_b200.training import distillation_with_grad
    lowest = torch.finfo(dtype).min
    x, t, where, _ = make(n, classes, kept, dtype, target='none', teacher_dtype=dtype, ragged=False)
    t[1] = lowest
    t[2, : kept // 2] = lowest
    x[torch.arange(n) % 2 == 1] = x[torch.arange(n) % 2 == 1].scatter(1, where[1::2, :1].long(), lowest)
    x[1] = 0.0
    loss, grad = distillation_with_grad(x, t, where, temperature=tau, reduction='none')
    even = t.clone()
    even[1] = 0.0  # (64 bits lose the logarithm of their number beside the lowest value of 32)
    want, grad_want, both, size = formula(x, even, where, tau=tau, reduction='none')
    q = torch.softmax(even.double() / tau, 1)
    apart = (even.double() - even.double().amax(1, keepdim=True)).abs() / tau
    far = x.double().amax(1, keepdim=True) - x.double().gather(1, where.long())
    room = 2e-6 * size + 1e-7 + tau * torch.where(q > 0, 2.0 ** -22 * (1 + apart) * q * far, 0.0).sum(1) + tau * torch.where(q < 2.0 ** -125, q * far, 0.0).sum(1)
    assert bool(want.float().isfinite().all()) and bool(((loss.double() - want).abs() <= room).all()), (loss, want)
    short = (x.double().amax(1, keepdim=True) - x.double()).div(tau).clamp(max=88)
    more = 2.0 ** -126 + 2.0 ** -22 * (1 + short) * both + torch.zeros_like(both).scatter_add_(1, where.long(), 2.0 ** -22 * (1 + apart.clamp(max=88)) * tau * q)
    assert in_half_steps(grad, grad_want, both, dtype, more)
