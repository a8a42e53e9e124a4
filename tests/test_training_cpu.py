"""The training operators without a GPU: what is refused, how the optimizer lays its state out, frequencies, symbols."""
import ctypes
import math

import numpy as np
import pytest
import torch as ch


def test_tensors_of_the_host_are_refused():
    from ffcv_b200.training import AdamW, NormResidual, RotaryPositions, cross_entropy, cross_entropy_with_grad, norm_residual
    x = ch.randn(4, 6)
    for call in (lambda: cross_entropy(x, ch.zeros(4, dtype=ch.long)), lambda: cross_entropy_with_grad(x, ch.zeros(4, dtype=ch.long)),
                 lambda: norm_residual(x), lambda: NormResidual(6)(x), lambda: RotaryPositions(6)(x.view(1, 2, 2, 6)),
                 lambda: AdamW([ch.nn.Parameter(x)])):
        with pytest.raises(TypeError, match='not on a GPU'):
            call()


def test_layout_of_the_flat_state():
    from ffcv_b200.training._native import ADAMW_BLOCK, lib
    numel = np.array([1, 0, 256, 257, 8192, 100000], np.int64)
    start, sizes = np.zeros(6, np.int64), np.zeros(2, np.int64)
    total = lib.ffcvb_adamw_layout(6, numel.ctypes.data, start.ctypes.data, sizes.ctypes.data)
    assert ADAMW_BLOCK == 256
    assert start.tolist() == [0, 256, 256, 512, 1024, 9216] and total == 9216 + 100096
    chunk = 2048  # few values: a unit for each of a CTA's eight warps
    chunks = [-(-int(n) // chunk) for n in numel]
    assert sizes.tolist() == [6 * 24 + 8 * sum(chunks), 4 * sum(chunks)]
    table = np.zeros(int(sizes[0]), np.uint8)
    where = np.arange(6, dtype=np.uint64) * 4096
    assert lib.ffcvb_adamw_table(6, numel.ctypes.data, where.ctypes.data, table.ctypes.data) == 0
    tensors = table[:144].view(np.int64).reshape(6, 3)
    assert tensors[:, 0].tolist() == where.tolist() and tensors[:, 1].tolist() == numel.tolist() and tensors[:, 2].tolist() == start.tolist()
    of = table[144:].view(np.int32).reshape(-1, 2)
    assert of.tolist() == [[i, c] for i, n in enumerate(chunks) for c in range(n)]
    many = np.full(3, 40 << 20, np.int64)  # more than a chunk of four units for every place of a CTA
    lib.ffcvb_adamw_layout(3, many.ctypes.data, start.ctypes.data, sizes.ctypes.data)
    assert sizes[1] == 4 * 3 * (40 << 20) // 8192


def test_bad_arguments_come_back_as_codes():
    """No exception and no abort leaves a C entry, whatever the host's arguments are; nothing is launched."""
    from ffcv_b200.training import _native as N
    lib = N.lib
    for call in (lib.ffcvb_cross_entropy, lib.ffcvb_norm_residual, lib.ffcvb_rotary, lambda args, stream: lib.ffcvb_norm_residual_backward(args, None, stream)):
        assert call(None, None) == -2
        assert b'no arguments' in lib.ffcvb_training_error()
    assert lib.ffcvb_norm_residual_workspace(None) == 0
    assert lib.ffcvb_adamw_step(None, None, None, None, None, None, 0, None) == -2
    loss = lambda rows=4, classes=5, kind=0, type_=0, smoothing=0.0, logits=16, target=16, row_loss=16: N.CROSS_ENTROPY.pack(  # noqa: E731
        logits, target, 0, 0, 0, row_loss, 0, 0, rows, classes, classes, 1, classes, 0, 0, type_, kind, 0, 0, 1, 0, 0, smoothing, 1.0)
    for bad in (loss(rows=-1), loss(classes=0), loss(kind=3), loss(type_=3), loss(smoothing=1.5), loss(logits=0), loss(target=0), loss(row_loss=0),
                loss(smoothing=math.nan)):
        assert lib.ffcvb_cross_entropy(bad, None) == -2
    norm = lambda rows=2, width=8, norm=1, post=0, gate=0, x=16, h=16, gate_at=0, tokens=1, type_=0, y=16: N.NORM_RESIDUAL.pack(  # noqa: E731
        x, h, gate_at, 0, 0, 0, 0, 0, 16, y, 16, *([0] * 5), *([0] * 5), rows, width, tokens, width, width, width, width, width, 0, type_, 0, norm, post, gate,
        1e-6, 1.0)
    for bad in (norm(rows=-1), norm(width=0), norm(norm=3), norm(post=-1), norm(gate=3), norm(x=0), norm(gate=1, gate_at=0), norm(rows=3, gate=1, gate_at=16, tokens=2),
                norm(type_=7), norm(y=0), norm(h=0, norm=0)):
        assert lib.ffcvb_norm_residual(bad, None) == -2
    assert lib.ffcvb_norm_residual(norm(width=16385), None) == -6
    assert lib.ffcvb_norm_residual_backward(norm(), None, None) == -2  # no workspace
    for odd in (norm(width=1 << 40), norm(width=0), norm(rows=-3), norm(gate=1, tokens=0)):
        assert lib.ffcvb_norm_residual_workspace(odd) == 0
    assert lib.ffcvb_norm_residual_workspace(norm(rows=0)) >= 0
    assert lib.ffcvb_norm_residual(norm(rows=0), None) == 0
    rotary = lambda head_dim=8, rotary_dim=8, axes=1, heads=2, q=16, tokens=3: N.ROTARY.pack(  # noqa: E731
        q, 0, 16, 0, 16, 16, 16, 1, tokens, heads, 0, head_dim, rotary_dim, 0, *([0] * 12), 0, 0, 0, axes, 0, 0, 1.0, 0)
    for bad in (rotary(head_dim=0), rotary(rotary_dim=10), rotary(rotary_dim=7), rotary(axes=3), rotary(rotary_dim=6, axes=2), rotary(q=0), rotary(heads=-1),
                rotary(head_dim=8192, rotary_dim=8192)):
        assert lib.ffcvb_rotary(bad, None) == -2
    assert lib.ffcvb_rotary(rotary(tokens=0), None) == 0


def test_structures_are_as_in_the_header():
    """The packed formats have no padding: their sizes are those of the C structures (members of 8 bytes first)."""
    from ffcv_b200.training import _native as N
    for fmt, size in ((N.CROSS_ENTROPY, 8 * 8 + 6 * 8 + 8 * 4 + 2 * 4), (N.NORM_RESIDUAL, 21 * 8 + 8 * 8 + 6 * 4 + 2 * 4), (N.ROTARY, 7 * 8 + 19 * 8 + 8 * 4),
                      (N.ADAMW, 8 * 8 + 4 * 4 + 8), (N.ADAMW_GROUP, 40)):
        assert fmt.size == size and size % 8 == 0


@pytest.mark.parametrize('scaling', ['none', 'linear', 'ntk', 'ramp'])
@pytest.mark.parametrize('axes', [1, 2])
def test_rotary_frequencies(scaling, axes):
    from ffcv_b200.training import RotaryPositions
    r = RotaryPositions(64, rotary_dim=32, axes=axes, scaling=scaling, factor=4.0, original_length=1000)
    turns, steps = r._turns[ch.device('cpu')]
    assert turns.dtype == ch.float64 and turns.shape == (16,)
    f = (turns * 2 * math.pi)[:16 // axes]
    dim = 32 // axes
    plain = 10000.0 ** (-ch.arange(0, dim, 2, dtype=ch.float64) / dim)
    if scaling == 'none':
        assert ch.allclose(f, plain, rtol=1e-14)
    elif scaling == 'linear':
        assert ch.allclose(f, plain / 4, rtol=1e-14)
    elif scaling == 'ntk':  # the fastest pair as it was, the slowest slowed by the factor
        assert math.isclose(f[0], 1.0, rel_tol=1e-14) and math.isclose(f[-1], plain[-1] / 4, rel_tol=1e-12)
    else:
        turned = 1000 * plain / (2 * math.pi)
        assert ch.allclose(f[turned >= 32], plain[turned >= 32]) and ch.allclose(f[turned <= 1], plain[turned <= 1] / 4)
        assert math.isclose(r.amplitude, 0.1 * math.log(4) + 1)
    if axes == 2:
        assert ch.equal(turns[:8], turns[8:])
    whole = steps.numpy().view(np.uint64)
    assert all(abs(int(w) - t * 2 ** 64) <= 2 ** 12 for w, t in zip(whole, turns.tolist()))
    # a far position by whole numbers, as the kernel does it, against exact arithmetic
    position = 123456789
    for w, t in zip(whole.tolist(), turns.tolist()):
        left = (position * w) % 2 ** 64 / 2 ** 64
        exact = math.fmod(position * t, 1.0)
        assert min(abs(left - exact), 1 - abs(left - exact)) < 1e-7


def test_patch_positions():
    from ffcv_b200.training import patch_positions
    assert patch_positions(2, 3).tolist() == [[0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]


def test_symbols():
    from ffcv_b200 import libffcv
    for name in ('ffcvb_training_error', 'ffcvb_cross_entropy', 'ffcvb_norm_residual', 'ffcvb_norm_residual_backward', 'ffcvb_norm_residual_workspace',
                 'ffcvb_rotary', 'ffcvb_adamw_layout', 'ffcvb_adamw_table', 'ffcvb_adamw_step'):
        assert isinstance(getattr(libffcv.lib, name), ctypes._CFuncPtr)
