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
