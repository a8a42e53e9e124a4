"""Cross entropy of a linear layer: upstream gradients that are no numbers or very large, against the formulas in 64 bits and with the
tolerances of test_gpu_linear_cross_entropy."""
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
