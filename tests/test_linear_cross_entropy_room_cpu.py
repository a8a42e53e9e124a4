"""The workspace of a linear layer's cross entropy, part by part: each buffer once, of the size that its kernels use."""
import itertools

import pytest
from test_linear_cross_entropy_cpu import args


def up(n, to):
    return -(-n // to) * to


@pytest.mark.parametrize('rows,classes,width', itertools.product([1, 127, 1021, 65536, 1 << 24], [1, 1000, 21841, 1 << 20], [1, 8, 130, 1024]))
@pytest.mark.parametrize('smoothing', [0.0, 0.1])
def test_workspace_has_each_part_once(rows, classes, width, smoothing):
    from ffcv_b200.training._native import lib
    padded, wide, even = up(rows, 256 if rows > 128 else 128), up(width, 32), up(width, 8)
    # classes at once: n of them in c pieces of the least c for which n / c of all rows, a multiple of 128, take 256 MB; in whole 256
    chunk = min(up(classes, 256), up((256 << 20) // (2 * up(rows, 128)) + 1, 256))
    for ignore, grads, from_stats, bias, upstream, odd in itertools.product([0, 1], itertools.product([0, 256], [0, 256], [0, 256]), [0, 1], [0, 256], [0, 256], [0, 2]):
        if (grads[2] and not bias) or (from_stats and not any(grads)):
            continue
        size = lib.ffcvb_linear_cross_entropy_workspace(args(rows, classes, width, ignore=ignore, grads=grads, from_stats=from_stats, bias=bias, upstream=upstream,
                                                             per_row=1, smoothing=smoothing, hidden=256 + odd, weight=256 + odd))
        most = 16 * 256  # (each part begins on 256 bytes)
        if ignore:
            most += 2 * 4 * padded + 4
        if upstream:
            most += 4
        if ignore or odd or width % 8:
            most += 2 * padded * even
        if odd or width % 8:
            most += 2 * up(classes, 128) * even
        if not from_stats:
            most += (12 if smoothing else 8) * padded * (up(classes, 256) // 64)
        if any(grads):
            most += 2 * padded * chunk
        if grads[0]:
            most += 4 * padded * wide
        if grads[1] and width % 8:
            most += 4 * chunk * wide
        if grads[0] or grads[1]:
            most += 2 * 148 * 128 * 256 * 4
        if grads[2]:
            most += 4 * padded // 32 * chunk
        assert 0 < size <= most
