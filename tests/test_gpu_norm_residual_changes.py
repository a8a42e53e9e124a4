"""The seam between two blocks at the edges: nothing in it, gradients that are not there, streams and branches of two types."""
import pytest
import torch as ch

from test_gpu_norm_residual import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [ch.float32, ch.bfloat16], ids=str)
@pytest.mark.parametrize('shape', [(2, 0, 64), (0, 3, 64), (0, 64), (2, 0, 333)], ids=str)
@pytest.mark.parametrize('gate', [None, 'sample', 'row', 'token'])
def test_no_tokens(shape, gate, dtype):
    """Empty results and gradients; what is summed over no rows, a gate per sample among it, has a gradient of zeros."""
    from ffcv_b200.training import norm_residual, norm_residual_backward, norm_residual_forward
    width = shape[-1]
    v = dict(x=ch.randn(shape, device='cuda', dtype=dtype), h=ch.randn(shape, device='cuda', dtype=dtype), weight=ch.ones(width, device='cuda'),
             bias=ch.ones(width, device='cuda'), scale=ch.ones(width, device='cuda'))
    if gate == 'sample':
        v['gate'] = ch.randn(*shape[:-2], 1, width, device='cuda', dtype=dtype)
    elif gate == 'row':
        v['gate'] = ch.randn(width, device='cuda', dtype=dtype)
    elif gate == 'token':
        v['gate'] = ch.randn(shape, device='cuda', dtype=dtype)
    how = {k: t for k, t in v.items() if k not in ('x', 'h')}
    dirt = ch.full((1 << 16,), 7.0, device='cuda')  # (what is not written is not zero by chance)
    del dirt
    y, z, stats = norm_residual_forward(v['x'], v['h'], **how)
    assert y.shape == z.shape == shape
    grads = norm_residual_backward(ch.empty_like(y), ch.empty_like(z), v['x'], v['h'], stats, **how)
    assert set(grads) == set(v)
    assert all(g.shape == v[k].shape and g.dtype == v[k].dtype and not g.any() for k, g in grads.items())
    leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
    y, z = norm_residual(**leaves)
    (y.sum() + z.sum()).backward()
    assert all(t.grad is not None and not t.grad.any() for t in leaves.values())


@pytest.mark.parametrize('post, gate', [(None, None), ('rms', 'sample'), ('layer', 'token')])
@pytest.mark.parametrize('dtype, width', [(ch.float32, 96), (ch.bfloat16, 1024), (ch.float16, 333)], ids=str)
def test_without_the_norms_gradient(dtype, width, post, gate):
    """Where z had no use: as with a gradient of zeros, which nobody has to make."""
    from ffcv_b200.training import norm_residual, norm_residual_backward, norm_residual_forward
    v, dy, dz = make((3, 50, width), dtype, 'layer', post, gate, True)
    how = {k: t for k, t in v.items() if k not in ('x', 'h')}
    how.update(norm='layer', post_norm=post, eps=1e-6)
    y, z, stats = norm_residual_forward(v['x'], v['h'], **how)
    want = norm_residual_backward(dy, ch.zeros_like(dz), v['x'], v['h'], stats, **how)
    got = norm_residual_backward(dy, None, v['x'], v['h'], stats, **how)
    check(v, dy, ch.zeros_like(dz), 'layer', post, got=(y, z, got))
    assert set(got) == set(want) and not got['weight'].any() and not got['bias'].any()
    x, h = (t.clone().requires_grad_() for t in (v['x'], v['h']))
    y, z = norm_residual(x, h)
    ch.cuda.synchronize()
    ch.cuda.reset_peak_memory_stats()
    before = ch.cuda.memory_allocated()
    dx, dh = ch.autograd.grad(y, (x, h), dy)
    peak = ch.cuda.max_memory_allocated() - before
    assert ch.equal(dx, dy) and ch.equal(dh, dy) and peak <= x.numel() * x.element_size() + 2048


@pytest.mark.parametrize('stream, branch', [(ch.float32, ch.bfloat16), (ch.float32, ch.float16), (ch.bfloat16, ch.float32), (ch.bfloat16, ch.float16)], ids=str)
@pytest.mark.parametrize('gate', [None, 'sample'])
def test_stream_and_branch_of_two_types(stream, branch, gate):
    """As a sum takes them: in the wider type, with gradients in each one's own."""
    from ffcv_b200.training import norm_residual
    v, dy, dz = make((2, 9, 96), ch.float32, 'layer', 'rms', gate, True)
    v['x'], v['h'] = v['x'].to(stream), v['h'].to(branch)
    wide = ch.promote_types(stream, branch)
    leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
    same = {k: (t.to(wide) if k in ('x', 'h') else t).detach().requires_grad_() for k, t in v.items()}
    y, z = norm_residual(**leaves, post_norm='rms')
    want = norm_residual(**same, post_norm='rms')
    assert y.dtype == z.dtype == wide and ch.equal(y, want[0]) and ch.equal(z, want[1])
    got = ch.autograd.grad((y, z), list(leaves.values()), (dy.to(wide), dz.to(wide)))
    for k, g, w in zip(v, got, ch.autograd.grad(want, list(same.values()), (dy.to(wide), dz.to(wide)))):
        assert g.dtype == v[k].dtype and ch.equal(g, w.to(g.dtype))


def test_under_automatic_mixed_precision():
    """A stream in 32 bits whose blocks' products are made in 16."""
    from ffcv_b200.training import NormResidual
    join, linear = NormResidual(64, scale=0.1).cuda(), ch.nn.Linear(64, 64).cuda()
    x = ch.randn(2, 5, 64, device='cuda', requires_grad=True)
    with ch.autocast('cuda', dtype=ch.bfloat16):
        h = linear(x)
        assert h.dtype == ch.bfloat16
        y, z = join(x, h)
        out = linear(z)
    assert y.dtype == z.dtype == ch.float32 and out.dtype == ch.bfloat16
    (out.float().square().mean() + y.mean()).backward()
    assert all(p.grad is not None and bool(ch.isfinite(p.grad).all()) for p in (*join.parameters(), *linear.parameters(), x))


def test_other_types_are_refused_as_before():
    from ffcv_b200.training import norm_residual
    x = ch.randn(2, 3, 16, device='cuda')
    for a, b in ((x, x.double()), (x.double(), x), (x, x.int())):
        with pytest.raises(TypeError):
            norm_residual(a, b)
    with pytest.raises(ValueError):
        norm_residual(x, x.half()[:1])
    for bad in (dict(h=[1.0]), dict(h=1.0)):
        with pytest.raises(TypeError, match='not a tensor'):
            norm_residual(x, **bad)
    with pytest.raises(TypeError, match='not a tensor'):
        norm_residual([1.0], x)
