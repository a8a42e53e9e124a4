"""Cross entropy of a linear layer: upstream gradients that are no numbers or very large, smoothing beside masked classes, against the formulas in 64 bits and with
the tolerances of test_gpu_linear_cross_entropy."""
import math

import pytest

torch = pytest.importorskip('torch')
from test_gpu_linear_cross_entropy import BF16, F16, formula, make, near  # noqa: E402

pytestmark = pytest.mark.gpu


def rows_and_grads(x, w, b, target, upstream, ignore=None):
    from ffcv_b200.training import linear_cross_entropy
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
    loss = linear_cross_entropy(leaves[0], leaves[1], bias=leaves[2], reduction='none', ignore_index=ignore, **target)
    return loss.detach(), torch.autograd.grad(loss, leaves, upstream)


@pytest.mark.parametrize('value', [math.inf, -math.inf, math.nan, 1e30])
@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('n,classes,width', [(40, 50, 32), (700, 3001, 136)])
def test_upstream_of_ignored_rows_counts_for_nothing(n, classes, width, dtype, value):
    """G is held relative to the largest upstream gradient of a row that counts, in steps of 2^-38 of that in fp16."""
    x, w, b, target = make(n, classes, width, dtype, True, 'labels')
    gone = torch.randperm(n, generator=torch.Generator().manual_seed(n))[:n // 3].cuda()
    target['labels'][gone] = -100
    clean = x.clone()
    x[gone] = math.nan
    upstream = torch.rand(n, device='cuda') + 0.5
    quiet = upstream.clone()
    upstream[gone], quiet[gone] = value, 0.0
    loss, grads = rows_and_grads(x, w, b, target, upstream, ignore=-100)
    want, grads_want, sizes, z = formula(clean, w, b, ignore=-100, reduction='none', upstream=quiet, **target)
    assert not loss[gone].any() and not grads[0][gone].any()
    least = 2.0 ** -38 * 1.5
    sizes = [(s + least * more, both) for (s, both), more in zip(sizes, (w.double().abs().sum(0), clean.double().abs().sum(0), float(n)))]
    near(grads, grads_want, sizes, dtype)


@pytest.mark.parametrize('value', [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize('others', [1.0, 0.0])
@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('n,classes,width', [(40, 50, 32), (700, 3001, 136)])
def test_an_upstream_that_is_no_number_is_its_own_rows(n, classes, width, dtype, others, value):
    """Hidden values' gradients of other rows do not know of it; those of weights and bias are sums over all rows."""
    x, w, b, target = make(n, classes, width, dtype, True, 'labels')
    upstream = (torch.rand(n, device='cuda') + 0.5) * others
    quiet = upstream.clone()
    upstream[17], quiet[17] = value, 0.0
    _, (dx, dw, db) = rows_and_grads(x, w, b, target, upstream)
    assert dx.isnan().any(1).nonzero().flatten().tolist() == [17] and not dw.isfinite().any() and not db.isfinite().any()
    want, (dx_want, *_), (sizes, *_), z = formula(x, w, b, reduction='none', upstream=quiet, **target)
    dx[17] = 0.0
    near([dx], [dx_want], [(sizes[0] + 2.0 ** -38 * 1.5 * w.double().abs().sum(0), sizes[1])], dtype)


@pytest.mark.parametrize('masked', [-math.inf, torch.finfo(BF16).min])
@pytest.mark.parametrize('smoothing', [0.1, 1.0])
@pytest.mark.parametrize('target', ['labels', 'mixed'])
@pytest.mark.parametrize('n,classes,width', [(3, 2, 8), (40, 50, 32), (150, 700, 64), (300, 20000, 72)])
def test_smoothing_beside_masked_classes(n, classes, width, target, smoothing, masked):
    """Classes masked by their bias have a share of a smoothed target: with -inf the loss has no end, with the type's lowest value it is as large as the formula has it.
    Such a loss is a sum of terms of one sign, each off by 2^-24 of itself for a difference, a product and the share's own rounding; so it is
    right to 2^-24 (classes / 32 + 100) of itself, which allows an addition for each of 32 classes that a thread has and those of all trees."""
    from ffcv_b200.training import linear_cross_entropy, linear_cross_entropy_with_grad
    x, w, b, how = make(n, classes, width, BF16, True, target)
    b[1::2] = masked
    b[:classes // 3] = masked
    b[classes // 2 // 2 * 2] = 0.5
    b[0] = 0.25
    if target == 'labels':
        how['labels'] = torch.where(torch.arange(n, device='cuda') % 2 == 0, 0, classes // 2 // 2 * 2)
    else:
        how['mixed'][:, 0], how['mixed'][:, 1] = 0, classes // 2 // 2 * 2
    rows, dx, dw, db = linear_cross_entropy_with_grad(x, w, bias=b, label_smoothing=smoothing, reduction='none', **how)
    again = linear_cross_entropy(x, w, bias=b, label_smoothing=smoothing, reduction='none', **how)
    want, grads_want, sizes, z = formula(x, w, b, smoothing=smoothing, reduction='none', **how)
    assert torch.equal(rows, again)
    if masked == -math.inf:
        assert bool((want == math.inf).all()) and torch.equal(rows, want.float())
    else:
        assert bool(want.float().isfinite().all())
        assert bool(((rows.double() - want).abs() <= 2.0 ** -24 * (classes / 32 + 100) * want).all()), ((rows.double() - want) / want).abs().max()
    near((dx, dw, db), grads_want, sizes, BF16)


def test_rows_of_the_lowest_value_are_uniform():
    """Nothing but masked classes: a uniform row, as where logits are kept."""
    from ffcv_b200.training import linear_cross_entropy
    for n, classes, width in ((40, 50, 32), (300, 20000, 72)):
        x, w, b, target = make(n, classes, width, BF16, True, 'labels')
        b[:] = torch.finfo(BF16).min
        rows = linear_cross_entropy(x, w, bias=b, label_smoothing=0.1, reduction='none', **target)
        assert bool(((rows - math.log(classes)).abs() < 1e-5).all())


@pytest.mark.parametrize('n,classes,width', [(1, 5, 8), (3, 130, 16), (40, 1000, 64), (129, 257, 72), (300, 20000, 72), (1021, 3001, 200)])
@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('target', ['labels', 'mixed'])
def test_gradient_of_the_bias_is_rounded_once(n, classes, width, dtype, target):
    """It is a sum of 32-bit values: off by 4e-6 of what is added up, as the logits' gradients are, and by half a step of itself."""
    x, w, b, how = make(n, classes, width, dtype, True, target)
    from ffcv_b200.training import linear_cross_entropy_with_grad
    scale = 256.0  # (fp16's smallest numbers have few digits)
    db = linear_cross_entropy_with_grad(x, w, bias=b, label_smoothing=0.05, grad_scale=scale, **how)[3].double()
    want, sizes = (v[2] for v in formula(x, w, b, smoothing=0.05, **how)[1:3])
    small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    room = torch.finfo(dtype).eps / 2 * (want * scale).abs() + 4e-6 * sizes[1] * scale + small
    assert bool(((db - want * scale).abs() <= room).all()), float(((db - want * scale).abs() / room).max())
