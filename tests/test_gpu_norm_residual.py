"""The seam between two blocks, forward and backward, against the formulas in 64 bits and against differences.

Tolerances.  A row's sums are made of at most 16 additions per thread and 10 levels of a tree, so a mean is off by
K 2^-24 of its terms' size, K = 32; a normalised value therefore by K 2^-24 (1 + r max|y|), r being 1 / deviation; what is
made of them is bounded by the same factor times the largest terms of the row.  Column sums add up `rows` terms: rows 2^-24 of
the sum of their sizes, and the terms' own errors.  What is rounded to 16 bits is off by half a unit in its last place more."""
import itertools

import pytest
import torch as ch

pytestmark = pytest.mark.gpu

TYPES = [ch.float32, ch.bfloat16, ch.float16]
UNIT = {t: ch.finfo(t).eps / 2 for t in TYPES}
TINY = {ch.float32: 0.0, ch.bfloat16: 0.0, ch.float16: 2.0 ** -25}
K = 32 * 2.0 ** -24
EPS = 1e-6


def make(shape, dtype, norm, post, gate, scale, bias=True, param=ch.float32, seed=0):
    gen = ch.Generator('cuda').manual_seed(seed)
    r = lambda *s: ch.randn(s, generator=gen, device='cuda')  # noqa: E731
    d = shape[-1]
    v = dict(x=(r(*shape) * 2 + 0.5).to(dtype), h=(r(*shape) * 0.7).to(dtype))
    if norm:
        v['weight'] = (1 + 0.3 * r(d)).to(param)
        if bias:
            v['bias'] = (0.2 * r(d)).to(param)
    if post:
        v['post_weight'] = (1 + 0.3 * r(d)).to(param)
        if bias:
            v['post_bias'] = (0.2 * r(d)).to(param)
    if gate == 'token':
        v['gate'] = r(*shape).to(dtype)
    elif gate == 'sample':
        v['gate'] = r(*shape[:-2], 1, d).to(dtype)
    if scale:
        v['scale'] = (0.3 + 0.1 * r(d)).to(param)
    return v, r(*shape).to(dtype), r(*shape).to(dtype)


def reference(v, dy, dz, norm, post, number=1.0):
    """Results, gradients, and per result how large the numbers were that it is made of."""
    v = {k: t.double().requires_grad_() for k, t in v.items()}

    def normed(a, kind):
        mean = a.mean(-1, keepdim=True) if kind == 'layer' else 0.0 * a.mean(-1, keepdim=True)
        r = ((a - mean) ** 2).mean(-1, keepdim=True).add(EPS).rsqrt()
        return (a - mean) * r, r

    x = v['x']
    big = lambda t: t.detach().abs().amax(-1, keepdim=True)  # noqa: E731
    size = {}
    one = ch.ones((), dtype=ch.float64, device=x.device)
    w, pw = v.get('weight', one), v.get('post_weight', one)
    y = x
    if 'h' in v:
        inner, r_in = normed(v['h'], post) if post else (v['h'], one)
        err_in = (1 + r_in * big(v['h'])).detach() if post else one  # of inner, times K
        u = inner * pw + v.get('post_bias', 0 * one)
        f = number * v.get('gate', one) * v.get('scale', one)
        y = x + f * u
        big_f, size_u = big(f * one.expand(x.shape[-1])), big(u) + err_in * big(pw)
        size['y'] = big(x) + big_f * size_u
    out, outputs, ups = {}, [], []
    if 'h' in v:
        out['y'] = y
        outputs.append(y)
        ups.append(dy.double())
    if norm:
        outer, r_out = normed(y, norm)
        z = outer * w + v.get('bias', 0 * one)
        out['z'] = z
        outputs.append(z)
        ups.append(dz.double())
        size['outer'] = (1 + r_out * (size['y'] if 'h' in v else big(x))).detach()
        size['z'] = size['outer'] * big(w) + big(v.get('bias', one))
    names = [k for k in v]
    grads = dict(zip(names, ch.autograd.grad(outputs, [v[k] for k in names], ups)))
    if 'h' not in v and dy is not None:
        grads['x'] = grads['x'] + dy.double()
    # sizes of the gradients' terms
    t = big(dy.double())
    if norm:
        g = big(dz.double() * w)
        t = t + r_out.detach() * g * (1 + big(outer)) * (1 + big(outer) + size['outer'])
        size['dweight'] = (dz.double().abs() * size['outer']), (dz.double() * outer).abs().detach()
        size['dbias'] = 0 * dz.double(), dz.double().abs()
    size['dx'] = t
    if 'h' in v:
        dx = grads['x'].abs()
        size['dh'] = t * big_f
        e_u = size_u
        size['dscale'] = (t * big(v.get('gate', one) * one.expand(x.shape[-1])) * e_u * abs(number)).expand(x.shape), dx * (number * v.get('gate', one) * u).abs().detach()
        size['dgate'] = (t * big(v.get('scale', one) * one.expand(x.shape[-1])) * e_u * abs(number)).expand(x.shape), dx * (number * v.get('scale', one) * u).abs().detach()
        if post:
            gi = t * big_f * big(pw)
            size['dpost_weight'] = (t * big_f * (big(inner) + err_in)).expand(x.shape), dx * (f * inner).abs().detach()
            size['dpost_bias'] = (t * big_f).expand(x.shape), dx * f.abs().detach()
            size['dh'] = r_in.detach() * gi * (1 + big(inner)) * (1 + big(inner) + err_in)
    return {k: t.detach() for k, t in out.items()}, grads, size


def near(name, got, want, bound):
    off = (got.double() - want).abs()
    room = bound + UNIT[got.dtype] * want.abs() + TINY[got.dtype]
    assert got.shape == want.shape, name
    assert bool((off <= room).all()), (name, float((off / room.clamp(min=1e-300)).max()))


def check(v, dy, dz, norm, post, number=1.0, got=None):
    from ffcv_b200.training import norm_residual_backward, norm_residual_forward
    how = {k: t for k, t in v.items() if k not in ('x', 'h')}
    how.update(norm=norm, post_norm=post, eps=EPS)
    if 'scale' not in v and number != 1.0:
        how['scale'] = number
    if got is None:
        y, z, stats = norm_residual_forward(v['x'], v.get('h'), **how)
        grads = norm_residual_backward(dy, dz if norm else None, v['x'], v.get('h'), stats, **how)
        assert set(grads) == set(v)
    else:
        y, z, grads = got
    out, want, size = reference(v, dy, dz, norm, post, number)
    width = v['x'].shape[-1]
    if 'y' in out:
        near('y', y, out['y'], K * size['y'])
    else:
        assert y is None or y is v['x']
    if norm:
        near('z', z, out['z'], K * size['z'])
    else:
        assert z is None
    near('dx', grads['x'], want['x'], K * size['dx'])
    if 'h' in v:
        near('dh', grads['h'], want['h'], K * size['dh'])
    rows = v['x'].numel() // width
    for name in ('weight', 'bias', 'post_weight', 'post_bias', 'scale', 'gate'):
        if name not in v:
            continue
        own, terms = (s.reshape(rows, width) for s in size['d' + name])
        if name == 'gate' and v['gate'].shape == v['x'].shape:
            near(name, grads[name], want[name], (K * own).view(v['x'].shape))
        elif name == 'gate':
            samples = v['gate'].numel() // width
            per = lambda s: s.view(samples, -1, width).sum(1).view(v['gate'].shape)  # noqa: E731
            near(name, grads[name], want[name], per(K * own) + rows // samples * 2.0 ** -24 * per(terms))
        else:
            near(name, grads[name], want[name], (K * own + rows * 2.0 ** -24 * terms).sum(0))


@pytest.mark.parametrize('norm, post, gate, scale', itertools.product(['layer', 'rms', None], [None, 'layer', 'rms'], [None, 'sample', 'token'], [False, True]))
@pytest.mark.parametrize('dtype, shape', [(ch.float32, (3, 5, 40)), (ch.bfloat16, (2, 7, 1024)), (ch.float16, (4, 3, 333))], ids=str)
def test_forms(shape, dtype, norm, post, gate, scale):
    v, dy, dz = make(shape, dtype, norm, post, gate, scale)
    check(v, dy, dz, norm, post)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('width', [1, 2, 7, 8, 32, 100, 192, 255, 256, 264, 776, 1000, 1025, 2048, 4097, 6000, 8200, 9001, 12288, 16383, 16384])
def test_widths(width, dtype):
    v, dy, dz = make((2, 3, width), dtype, 'layer', 'rms', 'sample', True, seed=width)
    check(v, dy, dz, 'layer', 'rms')
    v, dy, dz = make((1, 2, width), dtype, 'rms', None, None, False, seed=width)
    check(v, dy, dz, 'rms', None)


@pytest.mark.parametrize('shape', [(1, 1, 64), (1, 1000, 64), (1000, 1, 64), (333, 3, 72), (7, 513, 128), (2, 4000, 96), (5000, 64), (40,), (2, 2, 3, 5, 24)], ids=str)
@pytest.mark.parametrize('gate', [None, 'sample', 'token'])
def test_rows(shape, gate):
    if gate == 'sample' and len(shape) < 3:
        gate = None
    for dtype in (ch.float32, ch.bfloat16):
        v, dy, dz = make(shape, dtype, 'layer', 'layer', gate, True)
        check(v, dy, dz, 'layer', 'layer')


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_number_parameters_of_16_bits_and_missing_ones(dtype):
    v, dy, dz = make((2, 9, 200), dtype, 'layer', 'layer', 'token', False)
    check(v, dy, dz, 'layer', 'layer', number=-0.25)
    if dtype != ch.float32:
        v, dy, dz = make((2, 9, 200), dtype, 'layer', 'layer', 'sample', True, param=dtype)
        check(v, dy, dz, 'layer', 'layer')
    v, dy, dz = make((2, 9, 200), dtype, 'layer', 'rms', None, True, bias=False)
    check({k: t for k, t in v.items() if k != 'weight'}, dy, dz, 'layer', 'rms')
    v, dy, dz = make((2, 9, 200), dtype, 'rms', None, None, False)
    del v['h']
    check(v, dy, dz, 'rms', None)


def test_gate_shapes():
    from ffcv_b200.training import norm_residual, norm_residual_forward
    v, dy, dz = make((3, 4, 48), ch.float32, 'layer', None, 'sample', False)
    base = dict(weight=v['weight'], bias=v['bias'])
    want = norm_residual_forward(v['x'], v['h'], gate=v['gate'], **base)[1]
    assert ch.equal(want, norm_residual_forward(v['x'], v['h'], gate=v['gate'][:, 0], **base)[1])
    one = norm_residual_forward(v['x'], v['h'], gate=v['gate'][0, 0], **base)[1]
    assert ch.equal(one, norm_residual_forward(v['x'], v['h'], gate=v['gate'][:1].expand(3, 4, 48).contiguous(), **base)[1])
    narrow = ch.randn(3, 4, 1, device='cuda', requires_grad=True)  # broadcast over the channels: expanded first
    y, z = norm_residual(v['x'], v['h'], gate=narrow, **base)
    g, = ch.autograd.grad([y, z], narrow, [dy, dz])
    full = narrow.detach().expand(3, 4, 48).contiguous().requires_grad_()
    y, z = norm_residual(v['x'], v['h'], gate=full, **base)
    assert ch.equal(g, ch.autograd.grad([y, z], full, [dy, dz])[0].sum(-1, keepdim=True))


def test_strides_and_alignment():
    """Rows with gaps, rows that begin at odd places, transposed batches, gradients that are expanded numbers."""
    for dtype in TYPES:
        v, dy, dz = make((4, 6, 64), dtype, 'layer', 'rms', 'token', True)
        big = ch.randn(4, 6, 3 * 64 + 1, device='cuda').to(dtype)
        for cut in (big[..., 64:128], big[..., 1:65], big[..., :64]):
            v['h'] = cut
            check(v, dy, dz, 'layer', 'rms')
        v['h'] = ch.randn(6, 4, 64, device='cuda').to(dtype).transpose(0, 1)
        v['gate'] = ch.randn(4, 6, 64, device='cuda').to(dtype).transpose(1, 2).contiguous().transpose(1, 2)
        check(v, ch.ones((), dtype=dtype, device='cuda').expand(4, 6, 64), dz.flip(0).flip(0), 'layer', 'rms')


def test_rows_of_one_value_and_large_offsets():
    """Variance 0, and a mean far larger than the deviation: the deviation is taken of what is left."""
    v, dy, dz = make((2, 8, 512), ch.float32, 'layer', 'layer', None, True)
    v['x'][0, 0], v['h'][0, 0], v['h'][1, 1] = 3.0, -2.0, 0.0
    v['h'][1, 2] += 1000.0
    v['x'][1, 3] += 1000.0
    check(v, dy, dz, 'layer', 'layer')


def test_autograd_and_parts():
    """Only what is asked for; y or z unused; the same gradients as the direct call."""
    from ffcv_b200.training import NormResidual, norm_residual
    for dtype in (ch.float32, ch.bfloat16):
        v, dy, dz = make((3, 50, 96), dtype, 'layer', 'rms', 'sample', True)
        leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
        y, z = norm_residual(**leaves, norm='layer', post_norm='rms', eps=EPS)
        grads = dict(zip(leaves, ch.autograd.grad([y, z], list(leaves.values()), [dy, dz], retain_graph=True)))
        check(v, dy, dz, 'layer', 'rms', got=(y, z, grads))
        none = ch.zeros_like(dz)
        got = ch.autograd.grad(y, [leaves['x'], leaves['h'], leaves['gate']], dy, retain_graph=True)
        _, want, size = reference(v, dy, none, 'layer', 'rms')
        near('dh', got[1], want['h'], K * size['dh'])
        got, = ch.autograd.grad(z, leaves['weight'], dz)
        _, want, size = reference(v, none, dz, 'layer', 'rms')
        near('dweight', got, want['weight'], (K * size['dweight'][0] + 150 * 2.0 ** -24 * size['dweight'][1]).reshape(-1, 96).sum(0))
    module = NormResidual(96, 'layer', 'rms', scale=0.1).cuda()
    x, h = (ch.randn(2, 5, 96, device='cuda', requires_grad=True) for _ in range(2))
    y, z = module(x, h)
    (y.sum() + (z * z).sum()).backward()
    assert all(p.grad is not None for p in module.parameters()) and x.grad is not None
    same, first = module(x)
    assert same is x and first.shape == x.shape
    plain = NormResidual(96).cuda()
    x.grad = h.grad = None
    y, z = plain(x, h)
    (z ** 3).sum().backward()
    assert ch.equal(x.grad, h.grad)


def test_gradient_against_differences():
    """Along one direction, with e = 2^-5: the third derivative is below 50 here (e^2 / 6 * 50 < 2^-6), and 400 values of size 1 with an
    error of 2^-22 each give 400 * 2^-22 / 2^-4 < 2^-9."""
    from ffcv_b200.training import norm_residual
    v, dy, dz = make((2, 5, 40), ch.float32, 'layer', 'rms', 'sample', True)
    leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
    gen = ch.Generator('cuda').manual_seed(4)

    def f(at):
        y, z = norm_residual(**at, norm='layer', post_norm='rms')
        return (y.double() * dy).sum() + (z.double() * dz).sum()

    grads = dict(zip(leaves, ch.autograd.grad(f(leaves), list(leaves.values()))))
    e = 2.0 ** -5
    for name in leaves:
        d = ch.randn(v[name].shape, generator=gen, device='cuda')
        d /= d.norm()
        up, down = (f({**v, name: v[name] + s * e * d}) for s in (1, -1))
        assert abs(float(up - down) / (2 * e) - float((grads[name] * d).sum())) < 2.0 ** -6 + 2.0 ** -9, name


def test_no_rows_the_same_bits_and_another_stream():
    from ffcv_b200.training import norm_residual_backward, norm_residual_forward
    v, dy, dz = make((16, 197, 96), ch.bfloat16, 'layer', 'rms', 'sample', True)
    how = {k: t for k, t in v.items() if k not in ('x', 'h')}
    how.update(norm='layer', post_norm='rms')

    def both():
        y, z, stats = norm_residual_forward(v['x'], v['h'], **how)
        return [y, z] + list(norm_residual_backward(dy, dz, v['x'], v['h'], stats, **how).values())

    first = both()
    side = ch.cuda.Stream()
    side.wait_stream(ch.cuda.current_stream())
    with ch.cuda.stream(side):
        second = both()
    side.synchronize()
    assert all(ch.equal(a, b) for a, b in zip(first, second))
    empty = {k: t[:0] if k in ('x', 'h', 'gate') else t for k, t in v.items()}
    how['gate'] = empty['gate']
    y, z, stats = norm_residual_forward(empty['x'], empty['h'], **how)
    grads = norm_residual_backward(dy[:0], dz[:0], empty['x'], empty['h'], stats, **how)
    assert y.shape == (0, 197, 96) and not grads['weight'].any() and not grads['scale'].any()


def test_refusals():
    from ffcv_b200.training import NormResidual, norm_residual_backward, norm_residual_forward
    x = ch.randn(2, 3, 16, device='cuda')
    w = ch.ones(16, device='cuda')
    for kw, kind in ((dict(norm='batch'), ValueError), (dict(norm=None), ValueError), (dict(gate=x), ValueError), (dict(scale=w), ValueError),
                     (dict(post_norm='rms'), ValueError), (dict(h=x[:1]), ValueError), (dict(h=x.half()), ValueError), (dict(weight=w[:8]), ValueError),
                     (dict(weight=w.cpu()), TypeError), (dict(weight=w, bias=w.half()), TypeError), (dict(h=x, post_weight=w), ValueError),
                     (dict(h=x, norm=None, weight=w), ValueError), (dict(h=x, gate=x[:1]), ValueError), (dict(h=x, gate=x.half()), ValueError)):
        with pytest.raises(kind):
            norm_residual_forward(x, **kw)
    with pytest.raises(TypeError):
        norm_residual_forward(x.cpu())
    with pytest.raises(TypeError):
        norm_residual_forward(x.double())
    with pytest.raises(ValueError):
        norm_residual_forward(ch.randn(1, 16385, device='cuda'))
    _, _, stats = norm_residual_forward(x, x)
    with pytest.raises(ValueError):
        norm_residual_backward(x[:1], x, x, x, stats)
    with pytest.raises(ValueError):
        NormResidual(16, norm='max')
