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
