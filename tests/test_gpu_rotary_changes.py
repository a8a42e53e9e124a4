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
