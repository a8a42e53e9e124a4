"""Group norm with an activation without a GPU: what is refused, strides, and the workspace that a call asks for."""
import itertools
import math

import pytest
import torch as ch


def args(samples=2, positions=9, channels=8, groups=2, type_=0, param_type=0, act=0, eps=1e-5, x=256, weight=256, stats=256, y=256, dy=256, dx=256, dweight=256, dbias=256,
         strides=None):
    from ffcv_b200.training import _native as N
    return N.GROUP_NORM.pack(x, weight, 0, stats, y, dy, dx, dweight, dbias, samples, positions, channels, groups,
                             *(strides or (positions * channels, channels, positions * channels, channels)), 0, type_, param_type, act, eps, 0)


def test_structure_is_as_in_the_header():
    from ffcv_b200.training import _native as N
    assert N.GROUP_NORM.size == 9 * 8 + 8 * 8 + 6 * 4


def test_bad_arguments_come_back_as_codes():
    from ffcv_b200.training._native import lib
    for call in (lib.ffcvb_group_norm, lib.ffcvb_group_norm_backward):
        assert call(None, None, None) == -2 and b'no arguments' in lib.ffcvb_training_error()
        for bad in (dict(samples=-1), dict(samples=(1 << 24) + 1), dict(positions=-1), dict(positions=(1 << 30) + 1), dict(channels=0), dict(channels=7), dict(groups=0),
                    dict(groups=16), dict(channels=1 << 21, groups=1), dict(samples=1 << 24, channels=1 << 10, groups=1 << 10), dict(type_=3), dict(type_=-1),
                    dict(param_type=3), dict(act=4), dict(act=-1), dict(eps=-1.0), dict(eps=math.nan), dict(x=0), dict(stats=0), dict(strides=(-1, 8, 8, 8))):
            assert call(args(**bad), 256, None) == -2, bad
    assert lib.ffcvb_group_norm(args(y=0), 256, None) == -2
    for bad in (dict(dy=0), dict(dx=0, dweight=0, dbias=0)):
        assert lib.ffcvb_group_norm_backward(args(**bad), 256, None) == -2
    for workspace in (None, 8):
        assert lib.ffcvb_group_norm_backward(args(), workspace, None) == -2 and b'no workspace' in lib.ffcvb_training_error()


def test_workspace():
    """Of some percent of the values at most; none for a forward pass whose groups are held."""
    from ffcv_b200.training._native import lib
    assert lib.ffcvb_group_norm_workspace(None, 0) == 0
    assert lib.ffcvb_group_norm_workspace(args(), 0) == 0
    for samples, positions, channels, share, type_, backward in itertools.product([1, 3, 512], [1, 49, 1000, 1 << 20], [1, 30, 256, 4096], [1, 2], [0, 2], [0, 1]):
        if channels % share:
            continue
        size = lib.ffcvb_group_norm_workspace(args(samples, positions, channels, channels // share, type_), backward)
        assert 0 <= size <= 256 * 3 + samples * channels * 16 + samples * channels * (positions // 8 + 1) * 8


def test_strides_of_samples_and_positions():
    from ffcv_b200.training.group_norm import _strides
    x = ch.zeros(4, 10, 12, 6).movedim(-1, 1)  # channels last
    assert _strides(x) == (720, 6)
    assert _strides(x[:, :, 2:5]) == (720, 6) and _strides(x[:, :, :, 2:5]) is None and _strides(x[:, 2:4]) == (720, 6) and _strides(x[::2]) == (1440, 6)
    assert _strides(x.contiguous()) is None
    assert _strides(x[:, :, :1, 2:5]) == (720, 6) and _strides(x[:, :, :, 3:4]) == (720, 72) and _strides(x[:, :, 3:4, 3:4]) == (720, 6)
    assert _strides(ch.zeros(4, 6)) == (6, 6) and _strides(ch.zeros(4, 1, 5)) == (5, 1) and _strides(ch.zeros(1, 1, 5, 7)) == (35, 1)
    assert _strides(ch.zeros(4, 6, 1).expand(4, 6, 5)) is None
    assert _strides(ch.zeros(1, 3, 8).expand(4, 3, 8).movedim(2, 1)) == (0, 8)
    assert _strides(ch.zeros(0, 8, 3)) == _strides(ch.zeros(2, 8, 0)) == (0, 8)


def test_what_is_refused_before_a_gpu_is_looked_for():
    from ffcv_b200.training import GroupNormAct, group_norm_act, group_norm_act_forward
    x = ch.zeros(2, 8, 3, 3)
    for call in (lambda: group_norm_act(x, 2), lambda: group_norm_act_forward(x, 2), lambda: GroupNormAct(2, 8)(x)):
        with pytest.raises(TypeError, match='not on a GPU'):
            call()
    for bad in (dict(groups=3, channels=8), dict(groups=0, channels=8), dict(groups=2, channels=8, activation='tanh')):
        with pytest.raises(ValueError):
            GroupNormAct(**bad)
    assert repr(GroupNormAct(2, 8, 'silu')) == "GroupNormAct(2, 8, activation='silu', eps=1e-05, affine=True)"
    assert GroupNormAct(2, 8, affine=False).weight is None
