"""Cross entropy of a linear layer without its logits against the formulas in 64 bits.

Tolerances.  Logits have sums of 32 bits of exact products: an error of about 1e-6 of the sizes added up, and losses of the rows as much.  The
gradient of the logits is rounded to 16 bits (half a step, eps / 2, of each), multiplied and summed in 32 bits, and the sum is rounded
once more: relative to what the products' sizes add up to (|G| |w|, computed in 64 bits) an element is off by eps / 2 for the one, and by
eps / 2 of itself for the other.  Before that rounding it is a difference S p - T of two numbers of 32 bits: p = exp(z - lse) is off by the error of z and by
that of the exponential, S and T by a few roundings of 2^-24, all relative to the two numbers and not to their difference, which may be 0 (one class:
p = 1, T = S).  So 4e-6 of (S p + T) |w| comes on top.  A row's shares below the smallest normal number are held in fp16 times 2^15 and lose nothing that counts.
"""
import math

import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(n, classes, width, dtype, bias, target, seed=0):
    gen = torch.Generator('cuda').manual_seed(seed)
    x = torch.randn(n, width, generator=gen, device='cuda').to(dtype)
    w = (torch.randn(classes, width, generator=gen, device='cuda') * (2 / math.sqrt(width))).to(dtype)
    b = (torch.randn(classes, generator=gen, device='cuda') * 0.5).to(dtype) if bias else None
    labels = torch.randint(classes, (n,), generator=gen, device='cuda')
    if target == 'mixed':
        return x, w, b, dict(mixed=torch.stack([labels.float(), labels.roll(1).float(), torch.rand(n, generator=gen, device='cuda')], 1))
    return x, w, b, dict(labels=labels)


def formula(x, w, b, labels=None, mixed=None, smoothing=0.0, ignore=None, reduction='mean', upstream=None):
    """Loss per row, loss, gradients, and what the sizes of the gradients' products add up to."""
    x, w = x.double(), w.double()
    z = x @ w.t() + (0 if b is None else b.double())
    n, classes = z.shape
    column = torch.arange(classes, device='cuda')
    if labels is not None:
        target = (column == labels[:, None]).double()
        counts = torch.ones(n, dtype=torch.bool, device='cuda') if ignore is None else labels != ignore
    else:
        lam = mixed[:, 2:].double()
        target = lam * (column == mixed[:, :1]) + (1 - lam) * (column == mixed[:, 1:2])
        counts = torch.ones(n, dtype=torch.bool, device='cuda')
    target = target * (1 - smoothing) + smoothing / classes
    lse = torch.logsumexp(z, 1)
    nothing = lse == -math.inf
    rows = target.sum(1) * lse - torch.where(target > 0, target * z, 0.0).sum(1)
    grad = target.sum(1, keepdim=True) * torch.exp(z - lse[:, None]) - target
    dead = ~counts | nothing
    rows, grad, x = rows.masked_fill(dead, 0.0), grad.masked_fill(dead[:, None], 0.0), x.masked_fill(~counts[:, None], 0.0)
    k = torch.full((n, 1), 1.0 / max(1, int(counts.sum())) if reduction == 'mean' else 1.0, dtype=torch.float64, device='cuda')
    if upstream is not None:
        k = k * upstream.double().view(-1, 1)
    grad = grad * k
    grads = [grad @ w, grad.t() @ x, grad.sum(0)]
    both = (target.sum(1, keepdim=True) * torch.exp(z - lse[:, None]) + target).masked_fill(dead[:, None], 0.0) * k.abs()  # S p + T
    sizes = [(grad.abs() @ w.abs(), both @ w.abs()), (grad.abs().t() @ x.abs(), both.t() @ x.abs()), (grad.abs().sum(0), both.sum(0))]
    loss = rows if reduction == 'none' else rows.sum() * (1.0 / max(1, int(counts.sum())) if reduction == 'mean' else 1.0)
    return loss, grads, sizes, z


def near(got, want, sizes, dtype):
    half = torch.finfo(dtype).eps / 2
    for name, g, f, (s, both) in zip(('hidden', 'weight', 'bias'), got, want, sizes):
        if g is None:
            continue
        assert g.dtype == dtype and g.shape == f.shape, name
        small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # (a step of the smallest numbers)
        room = half * s * 1.01 + half * f.abs() + 4e-6 * both + small
        off = ((g.double() - f).abs() - room).max()
        assert off <= 0, (name, float(off), float(((g.double() - f).abs() / room).max()))


def near_loss(got, want, z):
    room = 4e-6 * (1 + z.abs().max())
    assert torch.allclose(got.double(), want, rtol=2e-6, atol=float(room)), (got, want)


def check(x, w, b, target, smoothing=0.0, ignore=None, reduction='mean', scale=1.0):
    from ffcv_b200.training import linear_cross_entropy_with_grad
    loss, *grads = linear_cross_entropy_with_grad(x, w, bias=b, label_smoothing=smoothing, ignore_index=ignore, reduction=reduction, grad_scale=scale, **target)
    want, grads_want, sizes, z = formula(x, w, b, smoothing=smoothing, ignore=ignore, reduction=reduction, **target)
    near_loss(loss, want, z)
    near(grads, [g * scale for g in grads_want], [(s * abs(scale), both * abs(scale)) for s, both in sizes], x.dtype)
    assert (grads[2] is None) == (b is None)
    return loss, grads


SIZES = [(1, 1, 1), (1, 2, 8), (2, 10, 16), (128, 128, 64), (129, 257, 72), (64, 1000, 384), (300, 511, 130), (7, 21841, 96), (1021, 3001, 200), (2500, 130, 768), (127, 127, 1)]


@pytest.mark.parametrize('n,classes,width', SIZES)
@pytest.mark.parametrize('dtype', [BF16, F16])
def test_labels(n, classes, width, dtype):
    x, w, b, target = make(n, classes, width, dtype, True, 'labels')
    check(x, w, b, target, scale=64.0)


@pytest.mark.parametrize('n,classes,width', SIZES)
def test_mixed_and_smoothed_without_bias(n, classes, width):
    x, w, b, target = make(n, classes, width, BF16, False, 'mixed')
    check(x, w, None, target, smoothing=0.1, reduction='sum')


@pytest.mark.parametrize('n,classes,width,ignored', [(1, 5, 8, 0), (1, 5, 8, 1), (130, 300, 72, 65), (1000, 777, 264, 600), (3000, 50, 64, 2999), (257, 1000, 130, 257)])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_ignored_rows_are_not_read(n, classes, width, ignored, reduction):
    x, w, b, target = make(n, classes, width, BF16, True, 'labels')
    gone = torch.randperm(n, device='cuda')[:ignored]
    target['labels'][gone] = -100
    clean = x.clone()
    x[gone] = math.nan
    from ffcv_b200.training import linear_cross_entropy_with_grad
    loss, *grads = linear_cross_entropy_with_grad(x, w, bias=b, ignore_index=-100, reduction=reduction, **target)
    want, grads_want, sizes, z = formula(clean, w, b, ignore=-100, reduction=reduction, **target)
    near_loss(loss, want, z)
    near(grads, grads_want, sizes, BF16)
    assert (grads[0][gone] == 0).all()


@pytest.mark.parametrize('masked', [-math.inf, torch.finfo(BF16).min])
@pytest.mark.parametrize('smoothing', [0.0])
def test_classes_masked_by_their_bias(masked, smoothing):
    x, w, b, target = make(150, 700, 64, BF16, True, 'labels')
    b[::3] = masked
    b[-200:] = masked
    target['labels'] = torch.randint(0, 166, (150,), device='cuda') * 3 + 1
    check(x, w, b, target)
    b[:] = -math.inf  # no class is left: rows of no loss
    loss, grads = check(x, w, b, target)
    assert float(loss) == 0 and all(not bool(g.any()) for g in grads)


def test_labels_outside_the_classes():
    from ffcv_b200.training import linear_cross_entropy_with_grad
    for bad in (-1, 50, 1 << 40, -(1 << 40)):
        x, w, b, target = make(40, 50, 32, BF16, True, 'labels')
        target['labels'][7] = bad
        rows, dx, dw, db = linear_cross_entropy_with_grad(x, w, bias=b, reduction='none', **target)
        assert rows.isnan().nonzero().flatten().tolist() == [7] and dx.isnan().any(1).nonzero().flatten().tolist() == [7]
        assert dw.isnan().all() and db.isnan().all()


def test_values_that_are_no_numbers_show():
    from ffcv_b200.training import linear_cross_entropy_with_grad
    for value in (math.nan, math.inf):
        x, w, b, target = make(200, 300, 64, F16, True, 'labels')
        x[150, 3] = value
        rows, dx, _, _ = linear_cross_entropy_with_grad(x, w, bias=b, reduction='none', **target)
        assert rows.isnan().nonzero().flatten().tolist() == [150] and dx.isnan().all(1).nonzero().flatten().tolist() == [150]


@pytest.mark.parametrize('n,classes,width', [(300, 1000, 96), (1, 7, 8), (1000, 2050, 130)])
@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
def test_autograd(n, classes, width, dtype, reduction):
    from ffcv_b200.training import linear_cross_entropy
    x, w, b, target = make(n, classes, width, dtype, True, 'mixed')
    leaves = [t.requires_grad_() for t in (x, w, b)]
    upstream = torch.randn(n, device='cuda') * 3e4 if reduction == 'none' else torch.tensor(1024.0, device='cuda')
    loss = linear_cross_entropy(x, w, bias=b, reduction=reduction, label_smoothing=0.05, **target)
    grads = torch.autograd.grad(loss, leaves, upstream)
    scale = 2.0 ** -15 if dtype == F16 and reduction == 'none' else 1.0
    if scale != 1.0:  # (whole sums of such gradients do not fit fp16)
        grads = torch.autograd.grad(linear_cross_entropy(x, w, bias=b, reduction=reduction, label_smoothing=0.05, **target), leaves, upstream * scale)
    with torch.no_grad():
        want, grads_want, sizes, z = formula(x, w, b, smoothing=0.05, reduction=reduction, upstream=upstream * scale, **target)
        near_loss(loss, want, z)
        most = float(upstream.abs().max()) * scale  # G is held relative to the largest upstream: its smallest steps are of that
        if reduction == 'none':
            least = 2.0 ** -40 * most
            sizes = [(s + least * other, both) for (s, both), other in zip(sizes, (w.double().abs().sum(0), x.double().abs().sum(0), float(n)))]
        near(grads, grads_want, sizes, dtype)


def test_gradients_that_are_not_wanted():
    from ffcv_b200.training import linear_cross_entropy
    x, w, b, target = make(200, 1000, 96, BF16, True, 'labels')
    leaves = [x, w, b]
    whole = [t.clone().requires_grad_() for t in leaves]
    linear_cross_entropy(whole[0], whole[1], bias=whole[2], **target).backward()
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2), (0, 1)):
        some = [t.clone().requires_grad_(k in wanted) for k, t in enumerate(leaves)]
        linear_cross_entropy(some[0], some[1], bias=some[2], **target).backward()
        for k, (s, f) in enumerate(zip(some, whole)):
            assert (s.grad is None) == (k not in wanted)
            if k in wanted:
                assert torch.allclose(s.grad.float(), f.grad.float(), rtol=2 ** -7, atol=1e-6)  # (sums may be cut into other parts)


def test_gradient_against_differences():
    from ffcv_b200.training import linear_cross_entropy, linear_cross_entropy_with_grad
    x, w, b, target = make(64, 200, 32, F16, True, 'mixed')
    _, dx, dw, db = linear_cross_entropy_with_grad(x, w, bias=b, reduction='sum', **target)
    step = 2.0 ** -5  # losses have 1e-5 of noise; the third derivative brings step^2
    for t, g in ((x, dx), (w, dw), (b, db)):
        way = torch.randn_like(t.float()).sign()
        up, down = ((t.float() + s * step * way).to(F16) for s in (1, -1))
        moved = up.double() - down.double()
        args = lambda v: [v if t is o else o for o in (x, w, b)]  # noqa: E731
        losses = []
        for v in (up, down):
            a = args(v)
            losses.append(float(linear_cross_entropy(a[0], a[1], bias=a[2], reduction='sum', **target)))
        want = float((g.double() * moved).sum())
        assert abs(losses[0] - losses[1] - want) <= 0.05 * abs(want) + 0.05, (losses, want)


@pytest.mark.parametrize('how', ['columns', 'offset', 'padded', 'expanded', 'transposed'])
def test_strides(how):
    x, w, b, target = make(260, 500, 80, BF16, True, 'labels')
    if how == 'columns':
        x, w = (torch.cat([t, t], 1)[:, :80] for t in (x, w))
    elif how == 'offset':  # rows that begin between 16-byte boundaries
        x, w = (torch.cat([t[:, :1], t], 1).contiguous()[:, 1:] for t in (x, w))
    elif how == 'padded':
        x, w = (torch.nn.functional.pad(t, (0, 8))[:, :80] for t in (x, w))
    elif how == 'expanded':
        x = x[:1].expand(260, 80)
        b = b[:1].expand(500)
    else:
        x, w = (t.t().contiguous().t() for t in (x, w))
    target['labels'] = torch.stack([target['labels']] * 2, 1)[:, 0]
    check(x, w, b, target)


def test_pieces_of_the_classes():
    """More rows times classes than the workspace holds gradients of at once: sums of hidden's gradient go on from piece to piece."""
    from ffcv_b200.training import linear_cross_entropy_with_grad
    torch.cuda.empty_cache()
    x, w, b, target = make(5000, 60001, 72, BF16, True, 'labels')
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss, *grads = linear_cross_entropy_with_grad(x, w, bias=b, **target)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 5000 * 60001 * 2  # the logits in 16 bits
    want, grads_want, sizes, z = formula(x, w, b, **target)
    near_loss(loss, want, z)
    near(grads, grads_want, sizes, BF16)


def test_the_same_bits_every_time():
    from ffcv_b200.training import linear_cross_entropy_with_grad
    x, w, b, target = make(1021, 5000, 200, BF16, True, 'labels')
    first = linear_cross_entropy_with_grad(x, w, bias=b, **target)
    for _ in range(3):
        again = linear_cross_entropy_with_grad(x, w, bias=b, **target)
        assert all(torch.equal(a, f) for a, f in zip(again, first))


def test_no_samples():
    from ffcv_b200.training import linear_cross_entropy_with_grad
    x, w, b, _ = make(0, 20, 16, BF16, True, 'labels')
    labels = torch.zeros(0, dtype=torch.long, device='cuda')
    loss, dx, dw, db = linear_cross_entropy_with_grad(x, w, labels, bias=b)
    assert float(loss) == 0 and dx.shape == (0, 16) and not dw.any() and not db.any()
    assert linear_cross_entropy_with_grad(x, w, labels, bias=b, reduction='none')[0].shape == (0,)


def test_module():
    from ffcv_b200.training import LinearCrossEntropy
    layer = LinearCrossEntropy(64, 100, label_smoothing=0.1, device='cuda', dtype=BF16)
    assert sorted(layer.state_dict()) == ['bias', 'weight']
    x, _, _, target = make(50, 100, 64, BF16, False, 'mixed')
    x.requires_grad_()
    loss = layer(x, target['mixed'])
    loss.backward()
    want, grads, sizes, z = formula(x.detach(), layer.weight.detach(), layer.bias.detach(), smoothing=0.1, **target)
    near_loss(loss.detach(), want, z)
    near([x.grad, layer.weight.grad, layer.bias.grad], grads, sizes, BF16)
    assert layer.logits(x).shape == (50, 100)
    labels = target['mixed'][:, 0].long()
    near_loss(layer(x, labels).detach(), formula(x.detach(), layer.weight.detach(), layer.bias.detach(), smoothing=0.1, labels=labels)[0], z)


def test_in_a_graph_and_on_another_stream():
    from ffcv_b200.training import linear_cross_entropy_with_grad
    x, w, b, target = make(700, 3000, 128, BF16, True, 'labels')
    target['labels'][:200] = -100
    call = lambda: linear_cross_entropy_with_grad(x, w, bias=b, ignore_index=-100, **target)  # noqa: E731
    first = [t.clone() for t in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, f) for a, f in zip(other, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = call()
    x2, w2, b2, target2 = make(700, 3000, 128, BF16, True, 'labels', seed=1)
    x.copy_(x2), w.copy_(w2), b.copy_(b2), target['labels'].copy_(target2['labels'])
    target['labels'][500:] = -100
    graph.replay()
    again = call()
    assert all(torch.equal(a, f) for a, f in zip(kept, again)) and not torch.equal(again[1], first[1])
