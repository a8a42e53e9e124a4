"""Distillation without a GPU: what is refused."""
import math

import pytest
import torch as ch


def test_structure_is_as_in_the_header():
    from ffcv_b200.training import _native as N
    assert N.DISTILLATION.size == 10 * 8 + 9 * 8 + 10 * 4 + 4 * 4


def test_bad_arguments_come_back_as_codes():
    from ffcv_b200.training import _native as N
    lib = N.lib

    def call(rows=4, classes=50, kept=5, type_=0, teacher_type=0, kind=0, ignore=0, mean=1, from_stats=0, tau=1.0, hard=0.0, smoothing=0.0, logits=16, teacher=16,
             where=16, target=16, row_loss=16, grad=0, stats=0, counted=16):
        return lib.ffcvb_distillation(N.DISTILLATION.pack(
            logits, teacher, where, target, 0, grad, 0, row_loss, stats, counted, rows, classes, kept, classes, kept, kept, 1, classes, -1,
            0, type_, teacher_type, 0, kind, ignore, mean, 0, from_stats, 0, tau, hard, smoothing, 1.0), None)

    assert lib.ffcvb_distillation(None, None) == -2 and b'no arguments' in lib.ffcvb_training_error()
    for bad in (dict(rows=-1), dict(rows=1 << 28), dict(classes=0), dict(classes=0x7fff0001), dict(kept=0), dict(kept=1025), dict(type_=3), dict(teacher_type=-1),
                dict(kind=2), dict(tau=0.0), dict(tau=-1.0), dict(tau=math.inf), dict(tau=math.nan), dict(hard=-0.1), dict(hard=1.5), dict(hard=math.nan),
                dict(smoothing=2.0), dict(logits=0), dict(teacher=0), dict(where=0), dict(target=0, hard=0.5), dict(row_loss=0), dict(from_stats=1),
                dict(from_stats=1, stats=16), dict(from_stats=1, grad=16), dict(ignore=1, target=0), dict(ignore=1, kind=1), dict(ignore=1, counted=0)):
        assert call(**bad) == -2, bad


def test_tensors_of_the_host_and_wrong_ones_are_refused():
    from ffcv_b200.training import Distillation, distillation, distillation_with_grad
    x, t, c = ch.randn(4, 6), ch.randn(4, 2), ch.zeros(4, 2, dtype=ch.int32)
    for call in (lambda: distillation(x, t, c), lambda: distillation_with_grad(x, t, c), lambda: Distillation(2.0)(x, t, c)):
        with pytest.raises(TypeError, match='not on a GPU'):
            call()
