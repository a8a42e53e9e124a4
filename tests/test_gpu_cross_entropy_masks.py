"""Losses of masked logits and of logits far from zero, against the formula in 64 bits.

A loss is S log(sum exp(x - top)) + sum T (top - x), terms of one sign.  Each difference and each product is off by 2^-24 of itself, T by
four times that, a sum by 2^-24 per addition that a thread makes (classes / 32 here, at most) and per level of a tree, and so is the sum
of exponentials, whose terms are off by 2^-24 (3 X + 4) with X the distance of those that count from the largest (25 is more than enough:
exp(-25) is less than the sum's last bit).  So a loss is right to 2^-24 (classes / 32 + 100) of itself and of S, and S 2^-24 * 75 more."""
import math

import pytest
import torch as ch

pytestmark = pytest.mark.gpu

TYPES = [ch.float32, ch.bfloat16, ch.float16]


def targets_of(n, classes, gen):
    labels = ch.randint(classes, (n,), generator=gen, device='cuda')
    mixed = ch.stack([labels.float(), labels.roll(1).float(), ch.rand(n, generator=gen, device='cuda')], 1)
    soft = ch.softmax(2 * ch.randn((n, classes), generator=gen, device='cuda'), 1)
    return labels, mixed, soft


def probabilities(classes, target, smoothing):
    c = ch.arange(classes, device='cuda')
    if 'labels' in target:
        p = (c == target['labels'][:, None]).double()
    elif 'mixed' in target:
        m = target['mixed'].double()
        p = m[:, 2:] * (c == m[:, :1]) + (1 - m[:, 2:]) * (c == m[:, 1:2])
    else:
        p = target['soft'].double()
    return (1 - smoothing) * p + smoothing / classes


def losses(x, t):
    x = x.double()
    top = x.amax(1, keepdim=True)
    empty = (top == -math.inf)[:, 0]
    top = ch.where(top == -math.inf, 0.0, top)
    loss = t.sum(1) * ch.exp(x - top).sum(1).log() + ch.where(t > 0, t * (top - x), 0.0).sum(1)
    return ch.where(empty, 0.0, loss)


def check(x, target, smoothing):
    from ffcv_b200.training import cross_entropy, cross_entropy_with_grad
    classes = x.shape[1]
    t = probabilities(classes, target, smoothing)
    want, mass = losses(x, t), t.sum(1)
    unit = 2.0 ** -24
    room = unit * (classes / 32 + 100) * (want + mass) + unit * 75 * mass
    with_grad, grad = cross_entropy_with_grad(x, label_smoothing=smoothing, reduction='none', **target)
    leaf = x.detach().requires_grad_()
    for got in (with_grad, cross_entropy(leaf, label_smoothing=smoothing, reduction='none', **target)):
        endless = want == math.inf
        assert ch.equal(got[endless], want[endless].float())
        off = (got.detach().double() - want).abs()[~endless]
        assert bool((off <= room[~endless]).all()), float((off / room[~endless]).max())
    if not bool(endless.any()):
        mean = cross_entropy_with_grad(x, label_smoothing=smoothing, **target)[0]
        assert abs(float(mean) - float(want.mean())) <= float(room.mean()) + unit * float(want.mean())
    assert bool(ch.isfinite(grad).all())


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('classes', [2, 40, 3001, 50000])
@pytest.mark.parametrize('smoothing', [0.0, 0.1, 1.0])
def test_masks(classes, dtype, smoothing):
    """Classes masked with -inf or with the type's lowest value: some, all, all but the labels'; rows at even and odd places."""
    from ffcv_b200.training import cross_entropy_with_grad  # noqa: F401
    gen = ch.Generator('cuda').manual_seed(classes)
    n = 12
    labels, mixed, soft = targets_of(n, classes, gen)
    for value in (-math.inf, ch.finfo(dtype).min):
        for room in (0, 3):  # (with columns left over, rows lie otherwise than the gradient's)
            x = (3 * ch.randn((n, classes + room), generator=gen, device='cuda')).to(dtype)[:, :classes]
            masked = ch.rand((n, classes), generator=gen, device='cuda') < 0.5
            masked[7] = False
            x.masked_fill_(masked, value)
            x[4] = value
            x[5] = value
            x[ch.arange(n) != 4, labels[ch.arange(n) != 4]] = 1.0
            x[ch.arange(n) != 4, labels.roll(1)[ch.arange(n) != 4]] = 0.5
            allowed = ch.where(x > value, soft, 0.0)
            for target in (dict(labels=labels), dict(mixed=mixed), dict(soft=allowed), dict(soft=soft), dict(soft=soft.to(dtype))):
                check(x, target, smoothing)


@pytest.mark.parametrize('classes', [2, 40, 3001, 50000])
@pytest.mark.parametrize('smoothing', [0.0, 0.1])
@pytest.mark.parametrize('offset', [1e4, -3e5])
def test_logits_far_from_zero(classes, smoothing, offset):
    """What all logits of a row share does not change a loss, nor its digits."""
    gen = ch.Generator('cuda').manual_seed(classes)
    labels, mixed, soft = targets_of(9, classes, gen)
    x = 3 * ch.randn((9, classes), generator=gen, device='cuda') + offset
    for target in (dict(labels=labels), dict(mixed=mixed), dict(soft=soft)):
        check(x, target, smoothing)


def test_a_masked_row_leaves_the_mean_a_number():
    """The usual mask, the lowest value of 32 bits, with smoothing: a row of it has the loss of a uniform one."""
    from ffcv_b200.training import cross_entropy
    x = ch.randn(8, 40, device='cuda')
    x[3] = ch.finfo(ch.float32).min
    y = ch.arange(8, device='cuda')
    rows = cross_entropy(x, y, label_smoothing=0.1, reduction='none')
    assert abs(float(rows[3]) - math.log(40)) < 1e-5
    keep = ch.arange(8, device='cuda') != 3
    want = ch.nn.functional.cross_entropy(x[keep].double(), y[keep], label_smoothing=0.1, reduction='sum')
    mean = cross_entropy(x, y, label_smoothing=0.1)
    assert abs(float(mean) - (float(want) + math.log(40)) / 8) < 1e-5
