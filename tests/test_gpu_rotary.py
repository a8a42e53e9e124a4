"""Rotary positions against complex multiplication in 64 bits.

Tolerance: an angle is right to 2^-25 of a turn, that is 2^-22 radians, sine and cosine to 2^-23 more, and two products and
their sum to 2^-23 of the larger; a result in 16 bits is off by half a unit in its last place more."""
import math

import pytest
import torch as ch

pytestmark = pytest.mark.gpu

TYPES = [ch.float32, ch.bfloat16, ch.float16]
UNIT = {t: ch.finfo(t).eps / 2 for t in TYPES}


def turned(a, positions, rotary, base, factor, scaling, length, back=False):
    r, axes = rotary.rotary_dim, rotary.axes
    dim = r // axes
    i = ch.arange(dim // 2, dtype=ch.float64, device=a.device)
    f = base ** (-2 * i / dim)
    amplitude = 1.0
    if scaling == 'linear':
        f = f / factor
    elif scaling == 'ntk':
        f = (base * factor ** (dim / (dim - 2))) ** (-2 * i / dim)
    elif scaling == 'ramp':
        keep = ((length * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        f, amplitude = f * ((1 - keep) / factor + keep), 0.1 * math.log(factor) + 1
    angle = positions.double()[..., None] * f
    angle = angle.flatten(-2) if axes == 2 else angle
    turn = ch.polar(ch.full_like(angle, amplitude), -angle if back else angle)[..., None, :]
    x = a.double()
    first, second = (x[..., :r // 2], x[..., r // 2:r]) if rotary.layout == 'half' else (x[..., 0:r:2], x[..., 1:r:2])
    z = ch.complex(first, second) * turn
    both = ch.cat([z.real, z.imag], -1) if rotary.layout == 'half' else ch.stack([z.real, z.imag], -1).flatten(-2)
    size = ch.complex(first, second).abs() * amplitude
    size = ch.cat([size, size], -1) if rotary.layout == 'half' else ch.stack([size, size], -1).flatten(-2)
    return ch.cat([both, x[..., r:]], -1), ch.cat([size, ch.zeros_like(x[..., r:])], -1)


def check(got, a, *how, back=False):
    want, size = turned(a, *how, back=back)
    bound = UNIT[got.dtype] * want.abs() + size * 2.0 ** -20 + (2.0 ** -25 if got.dtype == ch.float16 else 0)
    assert got.shape == a.shape and got.dtype == a.dtype
    assert bool(((got.double() - want).abs() <= bound).all())
    r = how[1].rotary_dim
    assert ch.equal(got[..., r:], a[..., r:])


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('batch, tokens, heads, kv_heads, head_dim, rotary_dim, axes', [
    (1, 1, 1, 1, 2, 2, 1), (2, 5, 3, 1, 64, 64, 1), (3, 17, 4, 2, 80, 40, 1), (1, 130, 12, 12, 64, 32, 2), (2, 33, 2, 2, 36, 20, 2),
    (1, 9, 5, 0, 128, 128, 2), (2, 70, 1, 1, 256, 256, 1), (1, 3, 2, 1, 66, 6, 1), (5, 196, 6, 3, 96, 96, 2), (1, 2, 1, 1, 4096, 4096, 1)])
def test_layouts(batch, tokens, heads, kv_heads, head_dim, rotary_dim, axes, layout, dtype):
    from ffcv_b200.training import RotaryPositions
    gen = ch.Generator('cuda').manual_seed(tokens)
    q = ch.randn((batch, tokens, heads, head_dim), generator=gen, device='cuda').to(dtype)
    k = ch.randn((batch, tokens, kv_heads, head_dim), generator=gen, device='cuda').to(dtype) if kv_heads else None
    shape = (batch, tokens) + ((2,) if axes == 2 else ())
    for positions in (ch.randint(0, 5000, shape, generator=gen, device='cuda'), ch.randint(0, 90, shape[1:], generator=gen, device='cuda'),
                      ch.rand(shape, generator=gen, device='cuda') * 77 - 20):
        rotary = RotaryPositions(head_dim, rotary_dim=rotary_dim, layout=layout, axes=axes)
        how = (positions, rotary, 10000.0, 1.0, 'none', 0)
        for transpose in (False, True):
            a, b = rotary.rotate(q, k, positions, transpose=transpose)
            check(a, q, *how, back=transpose)
            if k is not None:
                check(b, k, *how, back=transpose)
        mine, other = q.clone(), None if k is None else k.clone()
        c, d = rotary.rotate(mine, other, positions, inplace=True)
        assert c is mine and d is other and ch.equal(c, rotary.rotate(q, k, positions)[0])


@pytest.mark.parametrize('scaling', ['linear', 'ntk', 'ramp'])
@pytest.mark.parametrize('axes', [1, 2])
def test_scaling_and_far_positions(scaling, axes):
    from ffcv_b200.training import RotaryPositions
    rotary = RotaryPositions(64, base=500000.0, axes=axes, scaling=scaling, factor=8.0, original_length=4096)
    shape = (2, 50) + ((2,) if axes == 2 else ())
    for most in (4096, 1 << 20, 1 << 40):  # (the angle of 2^40 has 40 - 53 + 2 = -11 as last bit: 2^-12 of a radian's size)
        positions = ch.randint(0, most, shape, device='cuda')
        q = ch.randn(2, 50, 3, 64, device='cuda')
        got, none = rotary.rotate(q, None, positions)
        assert none is None
        want, size = turned(q, positions, rotary, 500000.0, 8.0, scaling, 4096)
        assert bool(((got.double() - want).abs() <= size * (2.0 ** -20 + most * 2.0 ** -51) + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
def test_strides(layout, dtype):
    """Views of a fused projection, heads before tokens, one key head for all, storage at an odd place."""
    from ffcv_b200.training import RotaryPositions
    rotary = RotaryPositions(64, rotary_dim=32, layout=layout)
    positions = ch.arange(100, 137, device='cuda')
    how = (positions, rotary, 10000.0, 1.0, 'none', 0)
    fused = ch.randn(3, 37, 5 + 2 * 2, 64, device='cuda').to(dtype)
    odd = ch.randn(3 * 37 * 5 * 64 + 1, device='cuda').to(dtype)[1:].view(3, 37, 5, 64)
    cases = [(fused[:, :, :5], fused[:, :, 5:7]), (fused[:, :, :5].transpose(1, 2).contiguous().transpose(1, 2), fused[:, :, 7:]),
             (odd, odd[:, :, 2:3]), (fused[:, :, :4], fused[:, :, 8:].expand(3, 37, 4, 64)),
             (fused[..., :5, :].transpose(2, 3).contiguous().transpose(2, 3), None)]
    for q, k in cases:
        a, b = rotary.rotate(q, k, positions)
        check(a, q, *how)
        if k is not None:
            check(b, k, *how)
    q, k = fused[:, :, :5], fused[:, :, 5:7]
    want, rest = rotary.rotate(q, k, positions), fused[:, :, 7:].clone()
    rotary.rotate(q, k, positions, inplace=True)
    assert ch.equal(q, want[0]) and ch.equal(k, want[1]) and ch.equal(fused[:, :, 7:], rest)


def test_autograd():
    """The gradient is the transpose, also of keys that all heads share, and turns against the formula."""
    from ffcv_b200.training import RotaryPositions, patch_positions
    rotary = RotaryPositions(32, axes=2, layout='interleaved', scaling='ramp', factor=2.0, original_length=64)
    positions = patch_positions(3, 5, 'cuda')
    assert positions.tolist() == [[r, c] for r in range(3) for c in range(5)]
    q, k = ch.randn(2, 15, 4, 32, device='cuda', requires_grad=True), ch.randn(2, 15, 1, 32, device='cuda', requires_grad=True)
    a, b = rotary(q, k, positions)
    da, db = ch.randn_like(a), ch.randn_like(b)
    dq, dk = ch.autograd.grad([a, b], [q, k], [da, db])
    how = (positions, rotary, 10000.0, 2.0, 'ramp', 64)
    check(dq, da, *how, back=True)
    check(dk, db, *how, back=True)
    shared = rotary(q, k.expand(2, 15, 4, 32), positions)[1]  # a broadcast input: its heads' gradients add up
    ds = ch.randn_like(shared)
    dk, = ch.autograd.grad(shared, k, ds)
    want, size = turned(ds, *how, back=True)
    assert bool(((dk.double() - want.sum(2, keepdim=True)).abs() <= size.sum(2, keepdim=True) * 2.0 ** -19).all())
    only, = ch.autograd.grad(rotary(q, None, positions), q, da)
    assert ch.equal(only, dq)
    e, d = 2.0 ** -4, ch.randn_like(q)  # linear: differences have no error but rounding's
    diff = ((rotary(q + e * d, None, positions) * da).sum() - (rotary(q - e * d, None, positions) * da).sum()) / (2 * e)
    assert abs(float(diff) - float((dq * d).sum())) < 2.0 ** -22 * q.numel() * 4 / e


def test_default_positions_empty_and_streams():
    from ffcv_b200.training import RotaryPositions
    rotary = RotaryPositions(16)
    q = ch.randn(2, 6, 2, 16, device='cuda')
    a, b = rotary.rotate(q, q)
    assert ch.equal(a, rotary.rotate(q, None, ch.arange(6, device='cuda'))[0]) and ch.equal(a, b)
    assert rotary.rotate(q[:, :0], q[:, :0])[0].shape == (2, 0, 2, 16)
    side = ch.cuda.Stream()
    side.wait_stream(ch.cuda.current_stream())
    with ch.cuda.stream(side):
        c = rotary.half().rotate(q)[0]  # (a module cast to 16 bits keeps its angles)
    side.synchronize()
    assert ch.equal(a, c)


def test_refusals():
    from ffcv_b200.training import RotaryPositions
    for bad in (dict(layout='both'), dict(axes=3), dict(rotary_dim=66), dict(rotary_dim=3), dict(rotary_dim=34, axes=2), dict(scaling='log'),
                dict(base=-1.0), dict(factor=0.0)):
        with pytest.raises(ValueError):
            RotaryPositions(64, **bad)
    rotary = RotaryPositions(64)
    q = ch.randn(2, 3, 4, 64, device='cuda')
    for args, kind in (((q[0],), ValueError), ((q[..., :32],), ValueError), ((q.cpu(),), TypeError), ((q.double(),), TypeError),
                       ((q, q.half()), ValueError), ((q, q[:1]), ValueError), ((q, None, ch.arange(4, device='cuda')), ValueError),
                       ((q, None, ch.arange(3)), ValueError), ((q, None, [0, 1, 2]), TypeError)):
        with pytest.raises(kind):
            rotary.rotate(*args)
    with pytest.raises(ValueError):
        RotaryPositions(64, axes=2).rotate(q)
    with pytest.raises(ValueError):
        rotary.rotate(q.transpose(2, 3).contiguous().transpose(2, 3), inplace=True)
    with pytest.raises(ValueError):
        rotary.rotate(q.clone().requires_grad_(), inplace=True)
