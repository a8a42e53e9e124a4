"""Addresses between the boundaries that kernels read at are refused before any of them runs."""
from test_group_norm_cpu import args as group_norm


def test_group_norm():
    from ffcv_b200.training._native import lib
    for call in (lib.ffcvb_group_norm, lib.ffcvb_group_norm_backward):
        for at in (257, 258, 260, 263):
            assert call(group_norm(stats=at), 256, None) == -2 and b'stats begin on 8 bytes' in lib.ffcvb_training_error()


def test_distillation():
    from ffcv_b200.training import _native as N
    for at in (257, 260, 264, 271):
        args = N.DISTILLATION.pack(16, 16, 16, 16, 0, 16, 0, 16, at, 16, 4, 50, 5, 50, 5, 5, 1, 50, -1, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0, 1.0, 0.0, 0.0, 1.0)
        assert N.lib.ffcvb_distillation(args, None) == -2 and b'stats begin on 16 bytes' in N.lib.ffcvb_training_error()


def test_cross_entropy():
    from ffcv_b200.training import _native as N
    for at in (257, 260, 263):
        args = N.CROSS_ENTROPY.pack(16, 16, 0, 16, 0, 16, at, 0, 4, 5, 5, 1, 5, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0.0, 1.0)
        assert N.lib.ffcvb_cross_entropy(args, None) == -2 and b'stats begin on 8 bytes' in N.lib.ffcvb_training_error()


def test_norm_residual():
    from ffcv_b200.training import _native as N
    for at in (257, 260, 264, 271):
        args = N.NORM_RESIDUAL.pack(16, 16, 0, 0, 0, 0, 0, 0, at, 16, 16, *([0] * 5), *([0] * 5), 2, 8, 1, 8, 8, 8, 8, 8, 0, 0, 0, 1, 0, 0, 1e-6, 1.0)
        for call in (lambda: N.lib.ffcvb_norm_residual(args, None), lambda: N.lib.ffcvb_norm_residual_backward(args, 256, None)):
            assert call() == -2 and b'stats begin on 16 bytes' in N.lib.ffcvb_training_error()
