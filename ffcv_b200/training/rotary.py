"""Rotary positions of queries and keys: of tokens in a row, or of an image's patches by row and column."""
import math

import numpy as np
import torch as ch

from . import _native as N


def patch_positions(rows, cols, device=None):
    """``(rows * cols, 2)`` row and column of every patch of an image, row by row."""
    r = ch.arange(rows, device=device).repeat_interleave(cols)
    c = ch.arange(cols, device=device).repeat(rows)
    return ch.stack([r, c], 1)


def _overlaps(t):
    """Whether values of a tensor may share memory, as those of an expanded one do."""
    reach = 0  # of the dimensions within
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if n == 0:
            return False
        if stride <= reach:
            return True
        reach += (n - 1) * stride
    return False


class _Rotate(ch.autograd.Function):
    @staticmethod
    def forward(ctx, rotary, positions, q, k):
        ctx.rotary = rotary
        ctx.save_for_backward(positions)
        return rotary._run(q, k, *rotary._where(q, positions), False, False)

    @staticmethod
    @ch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        positions, = ctx.saved_tensors
        run, where = ctx.rotary._run, ctx.rotary._where(dq, positions)
        _, _, of_q, of_k = ctx.needs_input_grad
        if not of_q:
            return None, None, None, run(dk, None, *where, True, False)[0] if of_k else None
        dq, dk = run(dq, dk if of_k else None, *where, True, False)
        return None, None, dq, dk


class RotaryPositions(ch.nn.Module):
    """Turns pairs of values of every query and key by angles that grow with the token's position.

    Parameters
    ----------
    head_dim : int
        Values per head.
    rotary_dim : int
        The first values of a head, which are turned; the others stay as they are.  Default: all.
    base : float
        Pair i turns by ``base ** (-2 i / (rotary_dim / axes))`` radians per unit of position.
    layout : 'half' or 'interleaved'
        Pairs are ``rotary_dim / 2`` apart, or neighbours.
    axes : 1 or 2
        With 2 a token has two positions (row and column of a patch): the first half of the pairs turns by the
        first, the second half by the second.
    scaling : 'none', 'linear', 'ntk' or 'ramp'
        For positions ``factor`` times further out than a network was trained at (a larger image, a longer text).  'linear'
        divides all positions by it; 'ntk' raises the base, so that the slowest pair is slowed by it and the fastest not at
        all; 'ramp' divides for pairs with less than one turn over ``original_length`` positions, leaves those with more
        than 32, blends between, and multiplies queries and keys by ``0.1 ln(factor) + 1``.
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, layout='half', axes=1, scaling='none', factor=1.0,
                 original_length=2048):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if layout not in ('half', 'interleaved'):
            raise ValueError(f"layout must be 'half' or 'interleaved', not {layout!r}")
        if axes not in (1, 2):
            raise ValueError(f'axes must be 1 or 2, not {axes}')
        if not 0 < rotary_dim <= head_dim or rotary_dim % (2 * axes):
            raise ValueError(f'rotary_dim must be a multiple of {2 * axes}, at most head_dim, not {rotary_dim}')
        if scaling not in ('none', 'linear', 'ntk', 'ramp'):
            raise ValueError(f"scaling must be 'none', 'linear', 'ntk' or 'ramp', not {scaling!r}")
        if not base > 0 or not factor > 0 or not original_length > 0:
            raise ValueError('base, factor and original_length must be positive')
        self.head_dim, self.rotary_dim, self.layout, self.axes = head_dim, rotary_dim, layout, axes
        dim = rotary_dim // axes
        if scaling == 'ntk' and dim > 2:
            base = base * factor ** (dim / (dim - 2))
        f = base ** (-ch.arange(0, dim, 2, dtype=ch.float64) / dim)
        self.amplitude = 1.0
        if scaling == 'linear':
            f = f / factor
        elif scaling == 'ramp':
            keep = ((original_length * f / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
            f = f * ((1 - keep) / factor + keep)
            self.amplitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
        # turns per unit of position, in 64 bits whatever type the module is cast to: as floats, and in units of 2^-64 of a turn
        turns = (f / (2 * math.pi)).repeat(axes)
        steps = np.array([round(math.fmod(t, 1.0) * 2 ** 64) & (2 ** 64 - 1) for t in turns.tolist()], np.uint64)
        self._turns = {ch.device('cpu'): ch.stack([turns, ch.from_numpy(steps.view(np.float64))])}

    def extra_repr(self):
        return f'head_dim={self.head_dim}, rotary_dim={self.rotary_dim}, layout={self.layout!r}, axes={self.axes}'

    def _turns_on(self, device):
        turns = self._turns.get(device)
        if turns is None:
            turns = self._turns[device] = self._turns[ch.device('cpu')].to(device)
        return turns

    def _where(self, q, positions):
        """Positions as the kernel reads them, and the stride from one sequence to the next."""
        batch, tokens = q.shape[:2]
        if positions is None:
            if self.axes == 2:
                raise ValueError('positions are needed with two axes')
            positions = ch.arange(tokens, device=q.device)
        if not isinstance(positions, ch.Tensor):
            raise TypeError('positions is not a tensor')
        if positions.device != q.device:
            raise ValueError(f'positions are on {positions.device}, not on {q.device}')
        if positions.dtype not in (ch.int64, ch.float32):
            positions = positions.float() if positions.is_floating_point() else positions.long()
        own, shape = (tokens,) if self.axes == 1 else (tokens, 2), positions.shape
        if shape == own:
            return positions.contiguous(), 0
        if shape == (1,) + own:
            return positions[0].contiguous(), 0
        if shape == (batch,) + own:
            return positions.contiguous(), tokens * self.axes
        raise ValueError(f'positions must be of shape {own} or {(batch,) + own}, not {tuple(shape)}')

    def _check(self, q, k):
        N.require(q, 'q')
        if q.dim() != 4 or q.shape[3] != self.head_dim:
            raise ValueError(f'q must be (batch, tokens, heads, {self.head_dim}), not {tuple(q.shape)}')
        if k is not None:
            N.require(k, 'k', q)
            if k.dtype is not q.dtype or k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != self.head_dim:
                raise ValueError(f'k must be {q.dtype} {tuple(q.shape[:2])} + (heads, {self.head_dim}), not {k.dtype} {tuple(k.shape)}')

    def _run(self, q, k, where, stride, transpose, inplace):
        if inplace and ch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            raise ValueError('in place is for tensors without a gradient: autograd would not know of the change')
        if inplace and (q.stride(3) != 1 or (k is not None and k.stride(3) != 1)):
            raise ValueError('in place the values of a head must lie next to one another')
        if inplace and (_overlaps(q) or (k is not None and (_overlaps(k) or (k.data_ptr() == q.data_ptr() and q.numel() and k.numel())))):
            raise ValueError('in place no value may lie where another does: it would be turned more than once')
        if q.stride(3) != 1:
            q = q.contiguous()
        if k is not None and k.stride(3) != 1:
            k = k.contiguous()
        q_out = q if inplace else N.new_like(q)
        k_out = k if inplace or k is None else N.new_like(k)
        batch, tokens, heads, _ = q.shape
        qb, qt, qh, _ = q.stride()
        qob, qot, qoh, _ = q_out.stride()
        kv_heads, kb, kt, kh, kob, kot, koh = 0, 0, 0, 0, 0, 0, 0
        if k is not None:
            kv_heads = k.shape[2]
            kb, kt, kh, _ = k.stride()
            kob, kot, koh, _ = k_out.stride()
        index, turns = q.get_device(), self._turns_on(q.device).data_ptr()
        args = N.ROTARY.pack(
            q.data_ptr(), N.ptr(k), q_out.data_ptr(), N.ptr(k_out), where.data_ptr(), turns, turns + 4 * self.rotary_dim,
            batch, tokens, heads, kv_heads, self.head_dim, self.rotary_dim, stride, qb, qt, qh, kb, kt, kh, qob, qot, qoh, kob, kot, koh,
            index, N.TYPES[q.dtype], where.dtype == ch.float32, self.axes, self.layout == 'interleaved', transpose, self.amplitude, 0)
        if inplace:  # (a backward pass that needs what they were says so)
            ch.autograd.graph.increment_version(q if k is None else (q, k))
        N.check(N.lib.ffcvb_rotary(args, N.raw_stream(index)))
        return q_out, k_out

    def rotate(self, q, k=None, positions=None, transpose=False, inplace=False):
        """``(q, k)`` turned, without autograd.  ``transpose`` turns the other way, which is the gradient's way: given the
        gradients of what ``rotate`` returned, it returns those of what it was given.  ``inplace`` writes over q and k, no value of which may
        share memory with another."""
        self._check(q, k)
        return self._run(q, k, *self._where(q, positions), transpose, inplace)

    def forward(self, q, k=None, positions=None):
        """Queries and keys, (batch, tokens, heads, head_dim) with any strides, at integer or float positions of
        shape (tokens,) or (batch, tokens), with a last dimension of 2 for two axes; default 0, 1, ...  Keys may have
        fewer heads.  Returns ``(q, k)``, or the queries alone without keys."""
        self._check(q, k)
        where = self._where(q, positions)[0]
        if k is None:
            return _Rotate.apply(self, where, q, None)[0]
        return _Rotate.apply(self, where, q, k)
