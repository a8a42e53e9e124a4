"""Distillation from a teacher's largest logits against the formulas in 64 bits.

Tolerances.  Sums of exponentials and shares are made in 32 bits: p = exp((x - lse) / tau) is off by 2^-22 of itself for the exponential, by 2^-24 of its
exponent's size, at most 100 here, for the difference and the product before it (together 8e-6), and q as much; so a gradient, a difference of two such
numbers, is off by 1e-5 of what their sizes add up to, and by half a step of its type.  A row's loss is a sum of differences of logarithms: 1e-6 of the
sizes of q log q, q x / tau and log sum, times tau^2.
"""
import math

import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(n, classes, kept, dtype, target='labels', seed=0, teacher_dtype=F16, index=torch.int32, ragged=True):
    gen = torch.Generator('cuda').manual_seed(seed)
    x = (torch.randn(n, classes, generator=gen, device='cuda') * 3).to(dtype)
    t = (torch.randn(n, kept, generator=gen, device='cuda') * 4).to(teacher_dtype)
    where = torch.rand(n, classes, generator=gen, device='cuda').argsort(1)[:, :kept].to(index)
    if ragged and kept > 1:
        where[::3, kept // 2:] = -1
        where[1::5] = -7
        t[2::4, 0] = -math.inf
    label = torch.randint(classes, (n,), generator=gen, device='cuda')
    label[::2] = where[::2, 0].clamp(min=0).long()  # often a class that the teacher has too
    if target == 'mixed':
        return x, t, where, dict(mixed=torch.stack([label.float(), label.roll(1).float(), torch.rand(n, generator=gen, device='cuda')], 1))
    return x, t, where, dict(labels=label) if target == 'labels' else {}


def formula(x, t, where, labels=None, mixed=None, tau=1.0, hard=0.0, smoothing=0.0, ignore=None, reduction='mean', upstream=None):
    """Loss, gradient, and the sizes that their errors go by."""
    z, (n, classes) = x.double(), x.shape
    top = z.amax(1, keepdim=True)  # (taken off first: beside the type's lowest value 64 bits lose a logarithm of the number of classes too)
    z = z - torch.where(top.abs() == math.inf, 0.0, top)
    t = (t.double() / tau).masked_fill(where < 0, -math.inf)
    q = torch.softmax(t, 1).masked_fill((t == -math.inf).all(1, keepdim=True), 0.0)
    at = where.long().clamp(min=0)
    there = (q.sum(1, keepdim=True) > 0).double()
    log_q = torch.log(torch.where(q > 0, q, 1.0))
    lse = torch.logsumexp(z / tau, 1, keepdim=True)
    log_p = z.gather(1, at) / tau - lse
    rows = tau * tau * torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    size = tau * tau * torch.where(q > 0, q * (log_q.abs() + (z.gather(1, at) / tau).abs() + lse.abs() + 1), 0.0).sum(1)
    p = torch.exp(z / tau - lse)
    dense_q = torch.zeros_like(z).scatter_add_(1, at, q)
    grad, both = tau * (there * p - dense_q), tau * (there * p + dense_q)
    counts = torch.ones(n, dtype=torch.bool, device='cuda')
    if labels is not None or mixed is not None:
        column = torch.arange(classes, device='cuda')
        if labels is not None:
            target = (column == labels[:, None]).double()
            counts = counts if ignore is None else labels != ignore
        else:
            lam = mixed[:, 2:].double()
            target = lam * (column == mixed[:, :1]) + (1 - lam) * (column == mixed[:, 1:2])
        target = target * (1 - smoothing) + smoothing / classes
        lse = torch.logsumexp(z, 1, keepdim=True)
        total = target.sum(1, keepdim=True)
        more = total[:, 0] * lse[:, 0] - torch.where(target > 0, target * z, 0.0).sum(1)
        p = total * torch.exp(z - lse)
        if hard:
            rows, grad, both = (rows * (1 - hard) if hard < 1 else 0) + hard * more, (1 - hard) * grad + hard * (p - target), (1 - hard) * both + hard * (p + target)
            size = size + lse[:, 0].abs() + torch.where(target > 0, target * z, 0.0).abs().sum(1)
    dead = ~counts | (z == -math.inf).all(1)
    rows, grad, both, size = (v.masked_fill(dead if v.dim() == 1 else dead[:, None], 0.0) for v in (rows, grad, both, size))
    k = torch.full((n, 1), 1.0 / max(1, int(counts.sum())) if reduction == 'mean' else 1.0, dtype=torch.float64, device='cuda')
    if upstream is not None:
        grad, both = grad * upstream.double().view(-1, 1), both * upstream.double().abs().view(-1, 1)
    if reduction == 'none':
        return rows, grad * k, both * k, size
    over = k[0, 0] if n else 1.0
    return rows.sum() * over, grad * k, both * k, size.sum() * over


def near(loss, grad, want, dtype):
    loss_want, grad_want, both, size = want
    assert ((loss.double() - loss_want).abs() <= 2e-6 * size + 1e-7).all() or torch.equal(loss.double(), loss_want), (loss, loss_want)
    assert grad.dtype == dtype
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    room = torch.finfo(dtype).eps / 2 * grad_want.abs() + 1e-5 * both + step
    off = (grad.double() - grad_want).abs()
    assert (off <= room).all(), float((off / room).max())


def check(x, t, where, target, tau=1.0, hard=0.0, smoothing=0.0, ignore=None, reduction='mean', scale=1.0):
    from ffcv_b200.training import distillation_with_grad
    loss, grad = distillation_with_grad(x, t, where, temperature=tau, hard_weight=hard, label_smoothing=smoothing, ignore_index=ignore, reduction=reduction,
                                        grad_scale=scale, **target)
    loss_want, *rest, size = formula(x, t, where, tau=tau, hard=hard, smoothing=smoothing, ignore=ignore, reduction=reduction, **target)
    near(loss, grad, (loss_want, *(v * scale for v in rest), size), x.dtype)
    return loss, grad


SIZES = [(1, 1, 1), (3, 2, 2), (70, 10, 3), (33, 100, 32), (33, 100, 33), (20, 700, 30), (300, 1000, 10), (17, 1001, 64), (9, 5000, 100), (5, 21841, 64), (3, 50021, 200),
         (2, 130001, 1024), (40, 2048, 1024), (200, 40000, 7)]


@pytest.mark.parametrize('n,classes,kept', SIZES)
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_teacher_alone(n, classes, kept, dtype):
    x, t, where, target = make(n, classes, kept, dtype, target='none')
    check(x, t, where, target, tau=2.0, scale=64.0)


@pytest.mark.parametrize('n,classes,kept', SIZES)
@pytest.mark.parametrize('dtype,target,smoothing,tau', [(F32, 'mixed', 0.1, 1.0), (BF16, 'labels', 0.0, 3.5), (F16, 'mixed', 0.0, 4.0), (BF16, 'labels', 0.1, 0.5)])
def test_with_labels(n, classes, kept, dtype, target, smoothing, tau):
    x, t, where, target = make(n, classes, kept, dtype, target=target, index=torch.int64, teacher_dtype=dtype)
    check(x, t, where, target, tau=tau, hard=0.3, smoothing=smoothing, reduction='sum')


@pytest.mark.parametrize('n,classes,kept', [(50, 30, 12), (30, 300, 200), (6, 30000, 40), (20, 3, 500), (4, 130001, 1000)])
@pytest.mark.parametrize('hard', [0.0, 0.5, 1.0])
def test_the_same_class_twice(n, classes, kept, hard):
    x, t, where, target = make(n, max(classes, kept), kept, F32, target='mixed')
    where = (where % min(classes, 20)).int()
    where[::4, 1:] = where[::4, :1]  # one class alone
    check(x, t, where, target, tau=2.0, hard=hard)


@pytest.mark.parametrize('classes,kept', [(100, 5), (3000, 64), (130001, 64)])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('hard', [0.0, 0.4])
def test_ignored_samples_masks_and_infinities(classes, kept, reduction, hard):
    n = 24
    x, t, where, target = make(n, classes, kept, BF16, ragged=False)
    keep = torch.rand(n, classes, device='cuda') < 0.5
    keep.scatter_(1, where.long(), True).scatter_(1, target['labels'][:, None], True)
    x = x.masked_fill(~keep, -math.inf)
    x[3] = -math.inf                    # nothing is left
    x[5, :] = torch.finfo(BF16).min     # a uniform row
    t[7] = -math.inf                    # a teacher that says nothing
    t[8] = torch.finfo(F16).min
    where[9] = -1
    t[9] = math.nan                     # (not read as anything)
    target['labels'][10:14] = -100
    x[11] = math.nan
    from ffcv_b200.training import distillation_with_grad
    loss, grad = distillation_with_grad(x, t, where, temperature=2.0, hard_weight=hard, ignore_index=-100, reduction=reduction, **target)
    clean, t2 = x.clone(), t.clone()
    clean[11], t2[9] = 0.0, 0.0
    labels = target['labels']
    want = formula(clean, t2, where, labels=labels, tau=2.0, hard=hard, ignore=-100, reduction=reduction)
    near(loss, grad, want, BF16)
    assert not grad[3].any() and not grad[10:14].any()


def test_what_is_no_class_or_number():
    from ffcv_b200.training import distillation_with_grad
    for kept in (5, 40):
        for bad in (500, 1 << 40):
            x, t, where, target = make(20, 500, kept, BF16, index=torch.int64, ragged=False)
            where[6, kept - 1] = bad
            rows, grad = distillation_with_grad(x, t, where, reduction='none')
            assert rows.isnan().nonzero().flatten().tolist() == [6] and grad.isnan().any(1).nonzero().flatten().tolist() == [6] and grad[6].isnan().all()
        for value in (math.nan, math.inf):
            x, t, where, target = make(20, 500, kept, F32, ragged=False)
            t[4, 1], x[9, 100] = value, value
            rows, grad = distillation_with_grad(x, t, where, reduction='none')
            assert rows.isnan().nonzero().flatten().tolist() == [4, 9] and grad[4].isnan().any() and grad[9].isnan().all()
        x, t, where, target = make(20, 500, kept, F32, ragged=False)
        target['labels'][2] = 500
        rows, grad = distillation_with_grad(x, t, where, hard_weight=0.5, reduction='none', **target)
        assert rows.isnan().nonzero().flatten().tolist() == [2] and grad[2].isnan().all()
        rows, grad = distillation_with_grad(x, t, where, hard_weight=0.0, reduction='none', **target)
        assert not rows.isnan().any() and not grad.isnan().any()
        x[5, int(where[5, 0])] = -math.inf  # a class that the teacher knows and the student cannot have
        rows, grad = distillation_with_grad(x, t, where, reduction='none')
        assert float(rows[5]) == math.inf and grad.isfinite().all()


@pytest.mark.parametrize('n,classes,kept', [(200, 10, 4), (50, 1000, 64), (6, 130001, 300)])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
@pytest.mark.parametrize('hard', [0.0, 0.3])
def test_autograd(n, classes, kept, reduction, hard):
    from ffcv_b200.training import Distillation, distillation
    x, t, where, target = make(n, classes, kept, F32, target='mixed')
    x.requires_grad_()
    upstream = torch.randn(n, device='cuda') if reduction == 'none' else torch.tensor(3.0, device='cuda')
    loss = distillation(x, t, where, temperature=2.0, hard_weight=hard, label_smoothing=0.1, reduction=reduction, **target)
    grad, = torch.autograd.grad(loss, x, upstream)
    with torch.no_grad():
        near(loss, grad, formula(x, t, where, tau=2.0, hard=hard, smoothing=0.1, reduction=reduction, upstream=upstream, **target), F32)
    module = Distillation(2.0, hard, 0.1, reduction=reduction)
    assert torch.equal(module(x, t, where, target['mixed']), loss)


def test_gradient_against_differences():
    from ffcv_b200.training import distillation, distillation_with_grad
    x, t, where, target = make(40, 60, 8, F32, target='mixed')
    _, grad = distillation_with_grad(x, t, where, temperature=2.0, hard_weight=0.4, reduction='sum', **target)
    way = torch.randn_like(x)
    step = 2.0 ** -6
    up, down = (float(distillation(x + s * step * way, t, where, temperature=2.0, hard_weight=0.4, reduction='sum', **target)) for s in (1, -1))
    want = float((grad * way).sum())
    assert abs((up - down) / (2 * step) - want) <= 0.01 * abs(want) + 0.01


@pytest.mark.parametrize('how', ['columns', 'odd', 'transposed', 'expanded'])
@pytest.mark.parametrize('classes,kept', [(40, 6), (3001, 70)])
def test_strides(how, classes, kept):
    x, t, where, target = make(30, classes, kept, BF16)
    if how == 'columns':
        x, t, where = (torch.cat([v, v], 1)[:, :v.shape[1]] for v in (x, t, where))
    elif how == 'odd':
        x, t, where = (torch.cat([v[:, :1], v], 1)[:, 1:] for v in (x, t, where))
    elif how == 'transposed':
        x, t, where = (v.t().contiguous().t() for v in (x, t, where))
    else:
        x, t, where = (v[:1].expand_as(v) for v in (x, t, where))
    target['labels'] = torch.stack([target['labels']] * 2, 1)[:, 0]
    check(x, t, where, target, tau=2.0, hard=0.5)


def test_no_samples_the_same_bits_and_graphs():
    from ffcv_b200.training import distillation_with_grad
    x, t, where, target = make(500, 2000, 64, BF16)
    loss, grad = distillation_with_grad(x[:0], t[:0], where[:0])
    assert float(loss) == 0 and grad.shape == (0, 2000)
    call = lambda: distillation_with_grad(x, t, where, temperature=2.0, hard_weight=0.5, ignore_index=3, **target)  # noqa: E731
    first = [v.clone() for v in call()]
    for _ in range(3):
        assert all(torch.equal(a, f) for a, f in zip(call(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, f) for a, f in zip(other, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    x2, t2, where2, target2 = make(500, 2000, 64, BF16, seed=5)
    x.copy_(x2), t.copy_(t2), where.copy_(where2), target['labels'].copy_(target2['labels'])
    graph.replay()
    assert all(torch.equal(a, f) for a, f in zip(out, call())) and not torch.equal(out[1], first[1])
