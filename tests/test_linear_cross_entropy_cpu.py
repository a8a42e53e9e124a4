"""Cross entropy of a linear layer without a GPU: what is refused, and the workspace that a call asks for."""
import itertools
import math

import pytest
import torch as ch


def args(rows=4, classes=5, width=8, kind=0, type_=2, smoothing=0.0, hidden=256, weight=256, target=256, row_loss=256, stats=256, ignore=0, from_stats=0,
         grads=(256, 256, 0), bias=0, hidden_stride=None, weight_stride=None, upstream=0, per_row=0):
    from ffcv_b200.training import _native as N
    return N.LINEAR_CROSS_ENTROPY.pack(hidden, weight, bias, target, upstream, *grads, 256, row_loss, stats, rows, classes, width,
                                       width if hidden_stride is None else hidden_stride, width if weight_stride is None else weight_stride, 1, -100,
                                       0, type_, kind, ignore, 1, per_row, from_stats, 0, smoothing, 1.0)


def test_structure_is_as_in_the_header():
    from ffcv_b200.training import _native as N
    assert N.LINEAR_CROSS_ENTROPY.size == 11 * 8 + 7 * 8 + 8 * 4 + 2 * 4


def test_bad_arguments_come_back_as_codes():
    from ffcv_b200.training._native import lib
    assert lib.ffcvb_linear_cross_entropy(None, None, None) == -2 and b'no arguments' in lib.ffcvb_training_error()
    assert lib.ffcvb_linear_cross_entropy_workspace(None) == 0
    for bad in (dict(type_=0), dict(type_=3), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(classes=0), dict(classes=(1 << 24) + 1), dict(width=0), dict(width=65537),
                dict(kind=2), dict(kind=-1), dict(kind=1, ignore=1), dict(smoothing=-0.1), dict(smoothing=math.nan), dict(hidden=0), dict(weight=0), dict(target=0),
                dict(row_loss=0), dict(stats=0), dict(from_stats=1, grads=(0, 0, 0)), dict(grads=(0, 0, 256)), dict(hidden_stride=7), dict(weight_stride=-8)):
        assert lib.ffcvb_linear_cross_entropy(args(**bad), 256, None) == -2, bad
        assert lib.ffcvb_linear_cross_entropy_workspace(args(**bad)) == 0, bad
    for workspace in (None, 128):
        assert lib.ffcvb_linear_cross_entropy(args(), workspace, None) == -2 and b'no workspace' in lib.ffcvb_training_error()


@pytest.mark.parametrize('rows,classes,width', itertools.product([1, 127, 1021, 65536, 1 << 24], [1, 1000, 21841, 1 << 20], [1, 8, 130, 1024]))
def test_workspace_is_bounded(rows, classes, width):
    """Whatever is wanted: it holds a part of the logits' gradient, and for each row some statistics."""
    from ffcv_b200.training._native import lib
    for ignore, grads, from_stats, bias, upstream in itertools.product([0, 1], itertools.product([0, 256], [0, 256], [0, 256]), [0, 1], [0, 256], [0, 256]):
        if (grads[2] and not bias) or (from_stats and not any(grads)):
            continue
        size = lib.ffcvb_linear_cross_entropy_workspace(args(rows, classes, width, ignore=ignore, grads=grads, from_stats=from_stats, bias=bias, upstream=upstream,
                                                             per_row=1))
        padded = -(-rows // 128) * 128
        wide = -(-width // 32) * 32
        held = max(256 << 20, padded * 512) + padded * 512  # a piece of the logits' gradient, of 256 classes at least
        most = 1 << 12
        if any(grads):
            most += held + held // 16 * (1 if grads[2] else 0) + held // 16
        if not from_stats:
            most += padded * (classes // 64 + 4) * 8
        most += padded * 8 + (padded + classes + 128) * (width + 8) * 2 * 2
        if any(grads):
            most += 148 * (padded + min(classes + 256, held // (2 * padded) + 256)) * wide * 4 if padded <= 148 * 128 else (padded + classes + 512) * wide * 4 * 2
        assert 0 <= size <= most


def test_what_is_refused_before_a_gpu_is_looked_for():
    from ffcv_b200.training import LinearCrossEntropy, linear_cross_entropy, linear_cross_entropy_with_grad
    x, w, labels = ch.randn(4, 6).bfloat16(), ch.randn(9, 6).bfloat16(), ch.zeros(4, dtype=ch.long)
    for call in (lambda: linear_cross_entropy(x, w, labels), lambda: linear_cross_entropy_with_grad(x, w, labels),
                 lambda: LinearCrossEntropy(6, 9, dtype=ch.bfloat16)(x, labels)):
        with pytest.raises(TypeError, match='not on a GPU'):
            call()


def test_module_is_named_as_a_linear_layer():
    from ffcv_b200.training import LinearCrossEntropy
    layer = LinearCrossEntropy(6, 9)
    assert {k: tuple(v.shape) for k, v in layer.state_dict().items()} == {'weight': (9, 6), 'bias': (9,)}
    layer.load_state_dict(ch.nn.Linear(6, 9).state_dict())
    assert layer.logits(ch.zeros(2, 6)).shape == (2, 9) and repr(layer) == 'LinearCrossEntropy(6, 9, bias=True)'
    assert LinearCrossEntropy(6, 9, bias=False).bias is None
