"""Cross entropy and its gradient against the formula in 64 bits, and against differences.

Tolerances: with |x| <= X the exponent of 2 that stands for exp(x - max) is off by at most 2^-24 * 2 * 1.45 X, the
exponential itself by 2^-22, the sum over the classes by 2^-24 per addition a thread makes (at most 64 here) and per level of
the tree (10): a probability is off by RELATIVE(X) = 2^-24 (3 X + 80) of itself, a loss by that and by 2^-23 of the terms it
is the difference of.  What is rounded to 16 bits is off by half a unit in the last place more."""
import math

import pytest
import torch as ch

pytestmark = pytest.mark.gpu

TYPES = [ch.float32, ch.bfloat16, ch.float16]
UNIT = {t: ch.finfo(t).eps / 2 for t in TYPES}
TINY = {ch.float32: 2.0 ** -126, ch.bfloat16: 2.0 ** -126, ch.float16: 2.0 ** -25}  # (subnormal results are flushed or rounded)


def probabilities(classes, labels=None, mixed=None, soft=None, smoothing=0.0):
    if labels is not None:
        p = (ch.arange(classes, device=labels.device) == labels[:, None]).double()
    elif mixed is not None:
        c = ch.arange(classes, device=mixed.device)
        lam = mixed[:, 2:].double()
        p = lam * (c == mixed[:, :1]) + (1 - lam) * (c == mixed[:, 1:2])
    else:
        p = soft.double()
    return (1 - smoothing) * p + smoothing / classes


def formula(logits, t, counted=None):
    """Losses of the rows, and the gradient of their sum."""
    x = logits.double()
    empty = (x == -math.inf).all(1)
    x = ch.where(empty[:, None], 0.0, x)
    lse = ch.logsumexp(x, 1)
    loss = t.sum(1) * lse - ch.where(t > 0, t * x, 0.0).sum(1)
    grad = t.sum(1, keepdim=True) * ch.exp(x - lse[:, None]) - t
    off = empty if counted is None else empty | ~counted
    return ch.where(off, 0.0, loss), ch.where(off[:, None], 0.0, grad)


def check(loss, grad, logits, t, want_loss, want_grad, rows, k=1.0):
    finite = ch.where(ch.isfinite(logits), logits, 0.0).double()
    big = float(finite.abs().max())
    rel = 2.0 ** -24 * (3 * big + 80)
    mass = float(t.sum(1).max())
    room = mass * (rel + 2.0 ** -23 * (2 * big + math.log(logits.shape[1])))
    assert abs(float(loss) - float(want_loss.sum()) / rows) <= room + 2.0 ** -22 * abs(float(want_loss.sum()) / rows)
    want = want_grad * (k / rows)
    bound = UNIT[grad.dtype] * want.abs() + TINY[grad.dtype] + (want + t * (k / rows)).abs() * (rel + 2.0 ** -22) + 2.0 ** -22 * t * (k / rows)
    off = (grad.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


def make(n, classes, dtype, seed=0, scale=3.0):
    gen = ch.Generator('cuda').manual_seed(seed)
    logits = (ch.randn((n, classes), generator=gen, device='cuda') * scale).to(dtype)
    labels = ch.randint(classes, (n,), generator=gen, device='cuda')
    lam = ch.rand(n, generator=gen, device='cuda')
    return logits, labels, ch.stack([labels.float(), labels.roll(1).float(), lam], 1), gen


SHAPES = [(1, 1), (1, 2), (3, 7), (512, 10), (5, 33), (64, 1000), (17, 1001), (9, 4096), (7, 21841), (3, 65537), (2, 130001)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('n, classes', SHAPES)
def test_targets(n, classes, dtype):
    from ffcv_b200.training import cross_entropy_with_grad
    logits, labels, mixed, gen = make(n, classes, dtype)
    soft = ch.softmax(ch.randn((n, classes), generator=gen, device='cuda'), 1)
    for target in (dict(labels=labels), dict(mixed=mixed), dict(soft=soft), dict(soft=soft.to(dtype))):
        for smoothing in (0.0, 0.1):
            t = probabilities(classes, smoothing=smoothing, **target)
            want_loss, want_grad = formula(logits, t)
            loss, grad = cross_entropy_with_grad(logits, label_smoothing=smoothing, **target)
            assert loss.dtype == ch.float32 and grad.dtype == dtype and grad.shape == logits.shape
            check(loss, grad, logits, t, want_loss, want_grad, n)


def test_int32_labels_and_grad_scale():
    from ffcv_b200.training import cross_entropy_with_grad
    logits, labels, _, _ = make(64, 100, ch.float16)
    t = probabilities(100, labels)
    want_loss, want_grad = formula(logits, t)
    loss, grad = cross_entropy_with_grad(logits, labels.int(), grad_scale=1024.0)
    check(loss, grad, logits, t, want_loss, want_grad, 64, 1024.0)


@pytest.mark.parametrize('classes', [10, 1000, 4099, 70001])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_strides(classes, dtype):
    """Rows cut out of a wider matrix, rows that begin at odd places, columns that do not lie together."""
    from ffcv_b200.training import cross_entropy_with_grad
    wide = (ch.randn((6, classes + 13), generator=ch.Generator('cuda').manual_seed(1), device='cuda') * 3).to(dtype)
    labels = ch.tensor([0, classes - 1, 1, 2, 3, classes // 2], device='cuda') % classes
    t = probabilities(classes, labels)
    for logits in (wide[:, :classes], wide[:, 5:5 + classes], wide[:, 8:8 + classes], wide[:, :classes].t().contiguous().t()):
        want_loss, want_grad = formula(logits, t)
        loss, grad = cross_entropy_with_grad(logits, labels)
        check(loss, grad, logits, t, want_loss, want_grad, 6)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('classes', [40, 3001, 50000])
def test_masks(classes, dtype):
    """Masked classes (-inf, or the type's lowest value), a row with none left, ignored rows."""
    from ffcv_b200.training import cross_entropy_with_grad
    logits, labels, _, gen = make(12, classes, dtype, 3)
    for value in (-math.inf, ch.finfo(dtype).min):
        x = logits.masked_fill(ch.rand(logits.shape, generator=gen, device='cuda') < 0.5, value)
        x[ch.arange(12), labels] = 1.0
        x[4] = value
        y = labels.clone()
        y[[0, 7]] = -100
        counted = y != -100
        t = probabilities(classes, y)
        want_loss, want_grad = formula(x, t, counted)
        loss, grad = cross_entropy_with_grad(x, y, ignore_index=-100)
        if value == -math.inf:
            assert not grad[4].any()
            check(loss, grad, x, t, want_loss, want_grad, 10)
        else:  # a row of lowest values is uniform; its logits swallow what is added to them
            keep = ch.arange(12, device='cuda') != 4
            p = (grad[4].double() * 10 + t[4]).clamp(max=1)
            assert float((p - 1 / classes).abs().max()) < 2 * UNIT[dtype] + 1e-6
            check(0.0, grad[keep], ch.where(x > value, x, 0.0)[keep], t[keep], want_loss[keep] * 0, want_grad[keep], 10)


def test_nothing_counted_and_no_rows():
    from ffcv_b200.training import cross_entropy, cross_entropy_with_grad
    x = ch.randn(5, 9, device='cuda')
    loss, grad = cross_entropy_with_grad(x, ch.full((5,), -1, device='cuda'), ignore_index=-1)
    assert float(loss) == 0.0 and not grad.any()
    loss, grad = cross_entropy_with_grad(x[:0], ch.zeros(0, dtype=ch.long, device='cuda'), reduction='sum')
    assert float(loss) == 0.0 and grad.shape == (0, 9)
    assert float(cross_entropy_with_grad(x[:0], ch.zeros(0, dtype=ch.long, device='cuda'))[0]) == 0.0
    x.requires_grad_()
    cross_entropy(x, ch.full((5,), -1, device='cuda'), ignore_index=-1).backward()
    assert not x.grad.any()


@pytest.mark.parametrize('classes', [10, 2000, 40001])
def test_what_is_no_number_stays_in_its_row(classes):
    from ffcv_b200.training import cross_entropy_with_grad
    logits, labels, mixed, _ = make(8, classes, ch.float32, 5)
    x = logits.clone()
    x[1, classes // 2] = math.nan
    x[2, 1] = math.inf
    y = labels.clone()
    y[3], y[4] = classes, -3
    loss, grad = cross_entropy_with_grad(x, y, reduction='none')
    assert bool(ch.isnan(loss[1:5]).all()) and bool(ch.isnan(grad[1:5]).all())
    t = probabilities(classes, labels)
    want_loss, want_grad = formula(logits, t)
    good = ch.tensor([0, 5, 6, 7], device='cuda')
    for i in good.tolist():
        check(loss[i], grad[i:i + 1], logits[i:i + 1], t[i:i + 1], want_loss[i:i + 1], want_grad[i:i + 1], 1)
    mixed[5, 1] = math.nan
    assert ch.isnan(cross_entropy_with_grad(logits, mixed=mixed, reduction='none')[0]).nonzero().flatten().tolist() == [5]


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('classes', [10, 1000, 30001])
def test_autograd(classes, dtype, reduction):
    from ffcv_b200.training import cross_entropy
    n = 24
    logits, labels, mixed, gen = make(n, classes, dtype, 7)
    up = ch.rand(n, generator=gen, device='cuda') * 8 if reduction == 'none' else ch.tensor(1024.0, device='cuda')
    labels[3] = 5
    for target, counted in ((dict(labels=labels, ignore_index=5), labels != 5), (dict(mixed=mixed), None)):
        t = probabilities(classes, labels=target.get('labels'), mixed=target.get('mixed'))
        want_loss, want_grad = formula(logits, t, counted)
        rows = n if counted is None else int(counted.sum())
        x = logits.clone().requires_grad_()
        loss = cross_entropy(x, reduction=reduction, **target)
        loss.backward(up)
        if reduction == 'none':
            assert loss.shape == (n,)
            for i in range(n):
                check(loss[i], x.grad[i:i + 1], logits[i:i + 1], t[i:i + 1], want_loss[i:i + 1], want_grad[i:i + 1], 1, float(up[i]))
        else:
            k = 1 if reduction == 'sum' else rows
            # (where all rows are added up the room for a loss is that of each of them)
            check(loss / (n if reduction == 'sum' else 1), x.grad, logits, t * (1 if counted is None else counted[:, None]),
                  want_loss / (n if reduction == 'sum' else 1), want_grad, k, 1024.0)


def test_gradient_against_differences():
    """(f(x + e d) - f(x - e d)) / 2e: the loss's third derivative along d is below 1 here, so e = 2^-6 is good for 2^-12 / 6 and
    the rounding of two losses of about 5 for 2^-22 * 5 / 2^-5."""
    from ffcv_b200.training import cross_entropy_with_grad
    logits, _, mixed, gen = make(4, 300, ch.float32, 9)
    d = ch.randn(logits.shape, generator=gen, device='cuda')
    d /= d.norm()
    f = lambda x: float(cross_entropy_with_grad(x, mixed=mixed, label_smoothing=0.1, reduction='sum')[0])  # noqa: E731
    grad = cross_entropy_with_grad(logits, mixed=mixed, label_smoothing=0.1, reduction='sum')[1]
    e = 2.0 ** -6
    assert abs((f(logits + e * d) - f(logits - e * d)) / (2 * e) - float((grad * d).sum())) < 2.0 ** -12 / 6 + 4 * 2.0 ** -17 * 5


def test_the_same_bits_every_time_and_on_another_stream():
    from ffcv_b200.training import cross_entropy_with_grad
    logits, labels, _, _ = make(4096, 999, ch.bfloat16, 11)
    loss, grad = cross_entropy_with_grad(logits, labels, ignore_index=3)
    side = ch.cuda.Stream()
    side.wait_stream(ch.cuda.current_stream())
    with ch.cuda.stream(side):
        again = cross_entropy_with_grad(logits, labels, ignore_index=3)
    side.synchronize()
    assert ch.equal(again[0], loss) and ch.equal(again[1], grad)


def test_module_takes_what_the_label_pipeline_makes():
    from ffcv_b200.training import MixupCrossEntropy, cross_entropy
    logits, labels, mixed, _ = make(32, 10, ch.float32, 13)
    assert ch.equal(MixupCrossEntropy(0.1)(logits, mixed), cross_entropy(logits, mixed=mixed, label_smoothing=0.1))
    assert ch.equal(MixupCrossEntropy()(logits, labels), cross_entropy(logits, labels))


def test_refusals():
    from ffcv_b200.training import cross_entropy, cross_entropy_with_grad
    x, y = ch.randn(4, 5, device='cuda'), ch.zeros(4, dtype=ch.long, device='cuda')
    for bad, kind in ((dict(), ValueError), (dict(labels=y, mixed=ch.zeros(4, 3, device='cuda')), ValueError), (dict(labels=y[:3]), ValueError),
                      (dict(labels=y.float()), TypeError), (dict(labels=y.cpu()), ValueError), (dict(mixed=ch.zeros(4, 2, device='cuda')), ValueError),
                      (dict(soft=ch.zeros(4, 4, device='cuda')), ValueError), (dict(soft=ch.zeros(4, 5, device='cuda', requires_grad=True)), ValueError),
                      (dict(labels=y, label_smoothing=1.5), ValueError), (dict(labels=y, reduction='max'), ValueError),
                      (dict(mixed=ch.zeros(4, 3, device='cuda'), ignore_index=0), ValueError)):
        for call in (cross_entropy, cross_entropy_with_grad):
            with pytest.raises(kind):
                call(x, **bad)
    with pytest.raises(TypeError):
        cross_entropy(x.cpu(), y)
    with pytest.raises(TypeError):
        cross_entropy(x.double(), y)
    with pytest.raises(ValueError):
        cross_entropy(x[0], y)
