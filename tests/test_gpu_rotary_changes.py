"""Rotary positions among other operations: in place, with some gradients, and their digits in 32 bits."""
import math

import pytest
import torch as ch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('keys', [False, True])
@pytest.mark.parametrize('which', ['q', 'k'])
def test_in_place_is_seen_by_autograd(which, keys):
    """A backward pass that needs queries or keys as they were says so, also where the turning itself had no gradient to make."""
    from ffcv_b200.training import RotaryPositions
    if which == 'k' and not keys:
        return
    rotary = RotaryPositions(8)
    q, k = ch.randn(1, 3, 2, 8, device='cuda'), ch.randn(1, 3, 1, 8, device='cuda')
    w = ch.ones(8, device='cuda', requires_grad=True)
    out = ((q if which == 'q' else k) * w).sum()
    versions = q._version, k._version
    rotary.rotate(q, k if keys else None, inplace=True)
    assert q._version > versions[0] and (k._version > versions[1]) == keys
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.backward()
    leaf = ch.randn(1, 3, 2, 8, device='cuda', requires_grad=True)
    out = (leaf * leaf).sum()
    with ch.no_grad():
        rotary.rotate(leaf, inplace=True)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.backward()
    before = q.clone(), q._version
    rotary.rotate(q)
    assert q._version == before[1] and ch.equal(q, before[0])
    with ch.inference_mode():
        p = ch.randn(1, 3, 2, 8, device='cuda')
        want = rotary.rotate(p)[0]
        rotary.rotate(p, inplace=True)
        assert ch.equal(p, want)


def test_values_that_share_memory_are_not_turned_in_place():
    from ffcv_b200.training import RotaryPositions
    rotary = RotaryPositions(8)
    one, fused = ch.randn(2, 3, 1, 8, device='cuda'), ch.randn(2, 3, 5, 8, device='cuda')
    steps = ch.as_strided(fused, (2, 3, 4, 8), (120, 40, 4, 1))  # heads half over one another
    before = one.clone(), fused.clone()
    for args in ((one.expand(2, 3, 4, 8),), (fused, one.expand(2, 3, 4, 8)), (one.expand(2, 3, 1, 8)[:1].expand(2, 3, 1, 8),), (steps,), (fused, fused),
                 (fused[:, :, :2], fused)):
        with pytest.raises(ValueError, match='where another does'):
            rotary.rotate(*args, inplace=True)
    assert ch.equal(one, before[0]) and ch.equal(fused, before[1])
    assert rotary.rotate(one.expand(2, 3, 4, 8))[0].shape == (2, 3, 4, 8)
    want = rotary.rotate(fused[:, :, :4], fused[:, :, 4:])
    rotary.rotate(fused[:, :, :4], fused[:, :, 4:], inplace=True)  # parts of one projection
    assert ch.equal(fused[:, :, :4], want[0]) and ch.equal(fused[:, :, 4:], want[1])
    turned = fused.transpose(1, 2).contiguous().transpose(1, 2)
    want = rotary.rotate(turned)[0]
    rotary.rotate(turned, inplace=True)
    assert ch.equal(turned, want)
    rotary.rotate(fused[:, :0], fused[:, :0], inplace=True)


def plain(a, angle):
    """Turned with sines and cosines that are made in 64 bits and rounded once, in 32 bits: the usual table."""
    c, s = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    x, y = a[..., :a.shape[-1] // 2], a[..., a.shape[-1] // 2:]
    return ch.cat([x * c - y * s, y * c + x * s], -1)


@pytest.mark.parametrize('transpose', [False, True])
@pytest.mark.parametrize('kind', ['whole', 'float', 'patches'])
def test_digits_in_32_bits(kind, transpose):
    """The root of the mean square of the errors is that of the usual tables or less than a tenth more: whole and float positions of a
    long sequence, and an image's patches."""
    from ffcv_b200.training import RotaryPositions, patch_positions
    gen = ch.Generator('cuda').manual_seed(1)
    if kind == 'patches':
        rotary, positions, batch = RotaryPositions(64, axes=2), patch_positions(14, 14, 'cuda'), 64
    else:
        rotary, batch = RotaryPositions(64), 1
        positions = ch.arange(65536, device='cuda')
        positions = positions if kind == 'whole' else positions.float() + 0.25
    q = ch.randn((batch, positions.shape[0], 4, 64), generator=gen, device='cuda')
    dim = 64 // rotary.axes
    f = 10000.0 ** (-ch.arange(0, dim, 2, dtype=ch.float64, device='cuda') / dim)
    angle = positions.double()[..., None] * f
    angle = angle.flatten(-2) if kind == 'patches' else angle
    angle = -angle if transpose else angle
    turn = ch.polar(ch.ones_like(angle), angle)[:, None, :]
    z = ch.complex(q[..., :32].double(), q[..., 32:].double()) * turn
    want = ch.cat([z.real, z.imag], -1)
    error = lambda t: math.sqrt(float((t.double() - want).square().mean()))  # noqa: E731
    own, tables = error(rotary.rotate(q, None, positions, transpose=transpose)[0]), error(plain(q, angle))
    assert own <= 1.1 * tables, (own, tables)


def test_quarter_turns():
    """Positions about the places where the nearest quarter turn changes, on either side of zero."""
    from ffcv_b200.training import RotaryPositions
    rotary = RotaryPositions(2, base=1.0)  # one radian per unit of position
    near = ch.arange(-9, 10, device='cuda', dtype=ch.float64)[:, None] * (math.pi / 4) + ch.tensor([-1e-6, -1e-9, 0.0, 1e-9, 1e-6], device='cuda', dtype=ch.float64)
    positions = ch.cat([near.flatten().float(), ch.arange(-700, 700, device='cuda').float()])
    for where in (positions, ch.arange(-700, 700, device='cuda'), ch.tensor([-2 ** 40, 2 ** 40, -2 ** 53 + 1], device='cuda')):
        q = ch.tensor([1.0, 0.0], device='cuda').expand(1, where.numel(), 1, 2)
        got = rotary.rotate(q, None, where)[0][0, :, 0]
        # (the product of a position with turns of 2^-64: 2^-65 of a position; floats: 2^-53 of the angle)
        room = where.double().abs() * 2.0 ** -50 + 2.0 ** -23 + 2.0 ** -25
        want = ch.stack([where.double().cos(), where.double().sin()], 1)
        assert bool(((got.double() - want).abs() <= room[:, None]).all())


def test_only_wanted_gradients_are_made():
    """Of queries or keys alone, if only they need one: as many values are allocated as are asked for.  What was turned and then not used
    has a gradient of zeros."""
    from ffcv_b200.training import RotaryPositions
    rotary, where = RotaryPositions(64), ch.arange(256, device='cuda')
    q, k = ch.randn(2, 256, 4, 64, device='cuda'), ch.randn(2, 256, 2, 64, device='cuda')
    dq, dk = ch.randn_like(q), ch.randn_like(k)
    want = rotary.rotate(dq, dk, where, transpose=True)
    for needs in ((True, True), (True, False), (False, True)):
        a, b = q.clone().requires_grad_(needs[0]), k.clone().requires_grad_(needs[1])
        out, leaves = rotary(a, b, where), [t for t in (a, b) if t.requires_grad]
        ch.cuda.synchronize()
        ch.cuda.reset_peak_memory_stats()
        before = ch.cuda.memory_allocated()
        got = ch.autograd.grad(out, leaves, (dq, dk))
        peak = ch.cuda.max_memory_allocated() - before
        wanted = [w for w, need in zip(want, needs) if need]
        assert all(ch.equal(g, w) for g, w in zip(got, wanted)) and peak <= sum(w.numel() * 4 for w in wanted) + 2048
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    for use in (0, 1):
        got = ch.autograd.grad(rotary(a, b, where)[use], (a, b), (dq, dk)[use])
        assert ch.equal(got[use], want[use]) and not got[1 - use].any()
