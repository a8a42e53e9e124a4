"""Addresses between the boundaries that kernels read at are refused before any of them runs."""
from test_group_norm_cpu import args as group_norm


def test_group_norm():
    from ffcv_b200.training._native import lib
    for call in (lib.ffcvb_group_norm, lib.ffcvb_group_norm_backward):
        for at in (257, 258, 260, 263):
            assert call(group_norm(stats=at), 256, None) == -2 and b'stats begin on 8 bytes' in lib.ffcvb_training_error()
