"""Group norm with an activation against the formulas in 64 bits.

Tolerances.  x is exact; mean and 1 / deviation have 32 bits, joined from parts in some ten steps: 4e-6 of the sizes (|x| + |mean|) r |w| + |b| that make up
a covers them and the activation's exponential and division (2^-21), whose slope is at most 1.13.  A gradient is a sum of numbers made so: 2e-5 of the
sizes of its parts, in which dy stands for da, whose error is that of a times a second derivative of at most 1.  Each result is rounded once: half a step.
"""
import math

import pytest

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ACTS = {None: lambda a: a, 'relu': torch.relu, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}


def make(samples, channels, sides, dtype, seed=0, params=None, level=1.0):
    gen = torch.Generator('cuda').manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen, device='cuda')  # noqa: E731
    last = lambda t: t.movedim(-1, 1)  # noqa: E731
    x = last((rand(samples, *sides, channels) * torch.exp(0.5 * rand(channels)) + level * rand(samples, *([1] * len(sides)), channels)).to(dtype))
    dy = last(rand(samples, *sides, channels).to(dtype))
    params = dtype if params is None else params
    return x, dy, (1 + 0.3 * rand(channels)).to(params), (0.3 * rand(channels)).to(params)


def formula(x, dy, groups, w, b, act, eps=1e-5):
    """y, dx, dw, db and the sizes that their errors go by."""
    samples, channels = x.shape[:2]
    flat = lambda t: t.double().reshape(samples, groups, channels // groups, -1)  # noqa: E731
    param = lambda p, other: (torch.full((channels,), other, dtype=torch.float64, device='cuda') if p is None else p.double()).view(1, groups, -1, 1)  # noqa: E731
    v, d, w, b = flat(x), flat(dy), param(w, 1.0), param(b, 0.0)
    mean = v.mean((2, 3), keepdim=True)
    rate = 1 / torch.sqrt(((v - mean) ** 2).mean((2, 3), keepdim=True) + eps)
    hat = (v - mean) * rate
    a = (hat * w + b).requires_grad_()
    with torch.enable_grad():
        y = ACTS[act](a)
        da, = torch.autograd.grad(y, a, d)
    a, y = a.detach(), y.detach()
    size_hat = (v.abs() + mean.abs()) * rate
    size = size_hat * w.abs() + b.abs()
    over = lambda t: t.mean((2, 3), keepdim=True)  # noqa: E731
    dx = rate * (da * w - over(da * w) - hat * over(da * w * hat))
    part = d.abs() * (1 + size)
    if act == 'relu':  # an a that rounding may bring to the other side of 0 says nothing
        part = part + torch.where(a.abs() < 4e-6 * size, 1e5 * d.abs(), 0.0)
    size_dx = rate * (part * w.abs() + over(part * w.abs()) + size_hat * over(part * w.abs() * size_hat))
    back = lambda t: t.reshape(x.shape)  # noqa: E731
    of = lambda t: t.sum((0, 3)).view(-1)  # noqa: E731
    return {'y': (back(y), back(size)), 'x': (back(dx), back(size_dx)), 'weight': (of(da * hat), of(part * size_hat)), 'bias': (of(da), of(part))}


def near(got, want, rate):
    value, size = want
    step = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    room = torch.finfo(got.dtype).eps / 2 * value.abs() * 1.0001 + rate * size + step
    off = (got.double() - value).abs()
    assert (off <= room).all(), (float((off / room).max()), got.shape)


def check(x, dy, groups, w, b, act, eps=1e-5):
    from ffcv_b200.training import group_norm_act_backward, group_norm_act_forward
    how = dict(weight=w, bias=b, activation=act, eps=eps)
    y, stats = group_norm_act_forward(x, groups, **how)
    grads = group_norm_act_backward(dy, x, stats, groups, **how)
    want = formula(x, dy, groups, w, b, act, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.movedim(1, -1).is_contiguous()
    near(y, want['y'], 4e-6)
    assert sorted(grads) == sorted(['x'] + ['weight'] * (w is not None) + ['bias'] * (b is not None))
    for name, g in grads.items():
        assert g.dtype == (x.dtype if name == 'x' else w.dtype if w is not None else b.dtype)
        near(g, want[name], 2e-5)
    return y, stats, grads


SHAPES = [(2, 512, (7, 7), 32), (1, 1, (2, 3), 1), (3, 6, (5, 4), 3), (2, 30, (9,), 2), (2, 480, (28, 30), 16), (1, 64, (100, 120), 8), (1, 32, (300, 301), 4),
          (2, 4096, (3,), 1), (5, 20, (), 4), (300, 8, (2, 2), 8), (2, 16, (1000,), 2), (4, 96, (14, 15), 1), (2, 2048, (7, 5, 2), 32), (3, 24, (61, 67), 2), (1, 264, (40, 41), 11),
          (1, 3, (401, 501), 1), (1, 1032, (1, 70), 1)]


@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype,act', [(F32, 'silu'), (BF16, 'relu'), (F16, 'gelu'), (F32, None), (BF16, 'gelu')])
def test_shapes(shape, dtype, act):
    samples, channels, sides, groups = shape
    x, dy, w, b = make(samples, channels, sides, dtype)
    check(x, dy, groups, w, b, act)


@pytest.mark.parametrize('weight', [True, False])
@pytest.mark.parametrize('bias', [True, False])
@pytest.mark.parametrize('dtype,params', [(BF16, F32), (F32, F16), (F16, BF16)])
@pytest.mark.parametrize('sides', [(6, 7), (170, 171)])
def test_parameters_of_another_type_or_none(weight, bias, dtype, params, sides):
    x, dy, w, b = make(2, 64, sides, dtype, params=params)
    check(x, dy, 4, w if weight else None, b if bias else None, 'silu')


@pytest.mark.parametrize('sides', [(13, 9), (150, 151)])
@pytest.mark.parametrize('how', ['nchw', 'channels', 'rows', 'columns', 'offset', 'samples', 'expanded', 'strided weight'])
def test_strides(how, sides):
    x, dy, w, b = make(3, 48, sides, F16)
    other = make(3, 48, sides, F16, seed=1)[0]
    if how == 'nchw':
        x, dy = x.contiguous(), dy.contiguous()
    elif how == 'channels':  # every position has other channels too
        x, dy = torch.cat([x, other], 1)[:, :48], torch.cat([other, dy], 1)[:, 48:]
    elif how == 'rows':
        x, dy = torch.cat([x, other], 2)[:, :, 3:3 + sides[0]], torch.cat([dy, other], 2)[:, :, :sides[0]]
    elif how == 'columns':
        x, dy = torch.cat([x, other], 3)[..., 2:2 + sides[1]], torch.cat([dy, other], 3)[..., :sides[1]]
    elif how == 'offset':  # values that begin between 16-byte boundaries
        shift = lambda t: torch.cat([t[:1, :1].reshape(-1)[:1], t.movedim(1, -1).reshape(-1)])[1:].view(3, *sides, 48).movedim(-1, 1)  # noqa: E731
        x, dy = shift(x), shift(dy)
    elif how == 'samples':
        x, dy = torch.cat([x, other])[::2], torch.cat([other, dy])[::2]
    elif how == 'expanded':
        x, dy = x[:1].expand_as(x), dy[:, :1, :1, :1].expand_as(dy)
    else:
        w, b = torch.stack([w, b], 1).unbind(1)
    check(x, dy, 6, w, b, 'gelu')


@pytest.mark.parametrize('sides', [(10, 10), (170, 200)])
def test_large_means_and_single_values(sides):
    x, dy, w, b = make(2, 32, sides, F32)
    x += 1000.0
    x[0, :, 0, 0] = 0.0  # the first position is not like the others
    y, stats, _ = check(x, dy, 4, w, b, None)
    exact = x.double().reshape(2, 4, -1)
    assert torch.allclose(stats[..., 0].double(), exact.mean(2), rtol=2e-7)
    assert torch.allclose(stats[..., 1].double(), 1 / torch.sqrt(exact.var(2, correction=0) + 1e-5), rtol=2e-5)


def test_constant_groups():
    """A deviation of 0: only eps is left of it, and nothing of x."""
    x, dy, w, b = make(2, 32, (8, 8), F32)
    x[:] = 5.0
    y, stats, grads = check(x, dy, 4, w, b, None)
    assert torch.equal(y, b.view(1, 32, 1, 1).expand_as(y)) and (stats[..., 1] - 1e-5 ** -0.5).abs().max() < 0.01


@pytest.mark.parametrize('sides', [(6, 6), (170, 200)])
def test_what_is_no_number_stays_in_its_group(sides):
    from ffcv_b200.training import group_norm_act_backward, group_norm_act_forward
    for value in (math.nan, math.inf):
        x, dy, w, b = make(2, 32, sides, BF16)
        x[1, 9, 3, 3] = value
        for act in ACTS:
            y, stats = group_norm_act_forward(x, 4, weight=w, bias=b, activation=act)
            bad = y.isnan().flatten(2).any(2)
            assert not bad[0].any() and bad[1].nonzero().flatten().tolist() == list(range(8, 16))
            dx = group_norm_act_backward(dy, x, stats, 4, weight=w, bias=b, activation=act)['x']
            assert not dx[0].isnan().any() and not dx[1, 16:].isnan().any() and not dx[1, :8].isnan().any()


@pytest.mark.parametrize('sides', [(6, 7), (170, 171)])
@pytest.mark.parametrize('act', list(ACTS))
def test_autograd(sides, act):
    from ffcv_b200.training import GroupNormAct, group_norm_act
    x, dy, w, b = make(3, 32, sides, F32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = group_norm_act(*[x, 4, w, b], activation=act)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        want = formula(x, dy, 4, w, b, act)
        for g, name in zip((y, *grads), ('y', 'x', 'weight', 'bias')):
            near(g, want[name], 2e-5)
    module = GroupNormAct(4, 32, act, device='cuda')
    module.load_state_dict({'weight': w.detach(), 'bias': b.detach()})
    assert torch.equal(module(x), y)
    torch.nn.GroupNorm(4, 32).load_state_dict(module.state_dict())
    for wanted in range(3):  # one gradient alone
        some = [t.detach().requires_grad_(k == wanted) for k, t in enumerate(leaves)]
        g, = torch.autograd.grad(group_norm_act(some[0], 4, some[1], some[2], activation=act), some[wanted], dy)
        assert torch.equal(g, grads[wanted])


def test_gradient_against_differences():
    from ffcv_b200.training import group_norm_act
    x, dy, w, b = make(2, 16, (5, 6), F32)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(group_norm_act(x, 2, w, b, activation='gelu'), leaves, dy)
    step = 2.0 ** -7
    for k, g in enumerate(grads):
        way = torch.randn_like(g)
        ends = []
        for sign in (1, -1):
            args = [t.detach() + (sign * step * way if i == k else 0) for i, t in enumerate(leaves)]
            ends.append(float((group_norm_act(args[0], 2, args[1], args[2], activation='gelu').double() * dy).sum()))
        want = float((g.double() * way).sum())
        assert abs((ends[0] - ends[1]) / (2 * step) - want) <= 0.01 * abs(want) + 0.02


def test_nothing_to_norm():
    from ffcv_b200.training import group_norm_act
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3), (2, 8, 0)):
        x = torch.zeros(shape, device='cuda', requires_grad=True)
        w, b = (torch.ones(8, device='cuda', requires_grad=True) for _ in range(2))
        y = group_norm_act(x, 2, w, b, activation='silu')
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize('sides', [(20, 21), (170, 171)])
def test_the_same_bits_streams_and_graphs(sides):
    from ffcv_b200.training import group_norm_act_backward, group_norm_act_forward
    x, dy, w, b = make(3, 64, sides, BF16)

    def call():
        y, stats = group_norm_act_forward(x, 4, weight=w, bias=b, activation='silu')
        return [y, stats, *group_norm_act_backward(dy, x, stats, 4, weight=w, bias=b, activation='silu').values()]

    first = [t.clone() for t in call()]
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
    x2, dy2, w2, b2 = make(3, 64, sides, BF16, seed=3)
    x.copy_(x2), dy.copy_(dy2), w.copy_(w2), b.copy_(b2)
    graph.replay()
    assert all(torch.equal(a, f) for a, f in zip(out, call())) and not torch.equal(out[0], first[0])
