"""The seam between two blocks of a residual network: the norm behind a block, its gate and residual scale, the sum with
the residual stream, and the norm before the next block, in one kernel each way."""
import torch as ch

from . import _native as N

_NORMS = {None: 0, 'layer': 1, 'rms': 2}
_NO_GATE, _SAMPLE, _TOKEN = range(3)
_PARAMS = ('weight', 'bias', 'post_weight', 'post_bias', 'scale')


def _gate_kind(x, gate):
    """Whether a gate has a row per row of x or per sample, and a sample's rows; None for other shapes."""
    if gate is None:
        return _NO_GATE, 1
    if gate.shape == x.shape:
        return _TOKEN, 1
    if x.dim() >= 2 and gate.shape[-1:] == x.shape[-1:]:
        if gate.shape in (x.shape[:-2] + (1, x.shape[-1]), x.shape[:-2] + x.shape[-1:]):
            return _SAMPLE, x.shape[-2]
        if gate.numel() == x.shape[-1]:
            return _SAMPLE, x.numel() // x.shape[-1]
    return None, 1


def _rows(t, width):
    """(rows, width) with neighbouring values together: a view where the strides allow it."""
    t = t.reshape(-1, width)
    return t if t.stride(1) == 1 or width == 1 else t.contiguous()


class _Call:
    """A checked call: what the forward and the backward pass have in common."""

    def __init__(self, x, h, norm, weight, bias, post_norm, post_weight, post_bias, gate, scale, eps):
        self.type = N.require(x, 'x')
        if x.dim() < 1 or not 1 <= x.shape[-1] <= N.NORM_MAX_WIDTH:
            raise ValueError(f'x must have 1 to {N.NORM_MAX_WIDTH} values in its last dimension, not {tuple(x.shape)}')
        if norm not in _NORMS or post_norm not in _NORMS:
            raise ValueError("norms are 'layer', 'rms' or None")
        if h is None:
            if norm is None:
                raise ValueError('nothing to do: neither a branch nor a norm')
            if post_norm is not None or gate is not None or scale is not None:
                raise ValueError('post_norm, gate and scale go with a branch h')
        elif N.require(h, 'h', x) != self.type or h.shape != x.shape:
            raise ValueError(f'h must be {x.dtype} {tuple(x.shape)}, not {h.dtype} {tuple(h.shape)}')
        if norm is None and (weight is not None or bias is not None):
            raise ValueError('weight and bias go with a norm')
        if post_norm is None and (post_weight is not None or post_bias is not None):
            raise ValueError('post_weight and post_bias go with a post_norm')
        self.number, self.scale = 1.0, scale
        if scale is not None and not isinstance(scale, ch.Tensor):
            self.number, self.scale = float(scale), None
        self.width = width = x.shape[-1]
        self.weight, self.bias, self.post_weight, self.post_bias = weight, bias, post_weight, post_bias
        self.param_dtype, self.param_type = ch.float32, 0
        first = True
        for name in _PARAMS:
            p = getattr(self, name)
            if p is None:
                continue
            kind = N.require(p, name, x)
            if p.shape != (width,):
                raise ValueError(f'{name} must be of shape ({width},), not {tuple(p.shape)}')
            if not first and p.dtype != self.param_dtype:
                raise TypeError('weights, biases and scale must be of one type')
            self.param_dtype, self.param_type, first = p.dtype, kind, False
            if width > 1 and p.stride(0) != 1:
                setattr(self, name, p.contiguous())
        self.gate_kind, self.tokens = _gate_kind(x, gate)
        if gate is not None and (N.require(gate, 'gate', x) != self.type or self.gate_kind is None):
            raise ValueError(f'gate must be {x.dtype}, with a row per row or per sample of {tuple(x.shape)}, not {gate.dtype} {tuple(gate.shape)}')
        self.shape, self.device = x.shape, x.device
        self.x, self.h = _rows(x, width), None if h is None else _rows(h, width)
        self.gate_shape = None if gate is None else gate.shape
        self.gate = None if gate is None else _rows(gate, width)
        self.norm, self.post_norm, self.eps = _NORMS[norm], _NORMS[post_norm], float(eps)

    def plain(self):
        """Whether the branch is added as it is, so that its gradient is the stream's."""
        return self.post_norm == 0 and self.gate is None and self.scale is None and self.number == 1.0

    def pack(self, stats, y=None, z=None, dy=None, dz=None, dx=None, dh=None, dgate=None, params=(0,) * 5, workspace=0):
        x, h, gate = self.x, self.h, self.gate
        p = N.ptr
        return N.NORM_RESIDUAL.pack(
            x.data_ptr(), p(h), p(gate), p(self.weight), p(self.bias), p(self.post_weight), p(self.post_bias), p(self.scale),
            p(stats), p(y), p(z), p(dy), p(dz), p(dx), p(dh), p(dgate), *params, workspace,
            x.shape[0], self.width, self.tokens, x.stride(0), 0 if h is None else h.stride(0), 0 if gate is None else gate.stride(0),
            0 if dy is None else dy.stride(0), 0 if dz is None else dz.stride(0),
            self.device.index, self.type, self.param_type, self.norm, self.post_norm, self.gate_kind, self.eps, self.number)

    def forward(self):
        new = lambda: ch.empty(self.shape, dtype=self.x.dtype, device=self.device)  # noqa: E731
        y, z = None if self.h is None else new(), new() if self.norm else None
        stats = ch.empty((self.x.shape[0], 4), device=self.device)
        N.check(N.lib.ffcvb_norm_residual(self.pack(stats, y, z), N.stream_of(self.x)))
        return y, z, stats

    def backward(self, stats, dy, dz, wanted):
        """The gradients named in `wanted`, which holds only what the call was given."""
        dtype, device = self.x.dtype, self.device
        for name, g in (('dy', dy), ('dz', dz)):
            if g is not None and (N.require(g, name, self.x) != self.type or g.shape != self.shape):
                raise ValueError(f'{name} must be {dtype} {tuple(self.shape)}, not {g.dtype} {tuple(g.shape)}')
        if dz is not None and self.norm == 0:
            raise ValueError('dz goes with a norm')
        dy, dz = (None if g is None else _rows(g, self.width) for g in (dy, dz))
        if dz is None and self.norm:  # the kernel reads one where there is a norm
            dz = ch.zeros_like(self.x)
        new = lambda: ch.empty(self.shape, dtype=dtype, device=device)  # noqa: E731
        plain = self.plain()
        out = {}
        if 'x' in wanted or (plain and 'h' in wanted):
            out['x'] = new()
        if 'h' in wanted:
            out['h'] = out['x'] if plain else new()
        for name in _PARAMS:
            if name in wanted:
                out[name] = ch.empty(self.width, dtype=self.param_dtype, device=device)
        if 'gate' in wanted:
            out['gate'] = ch.empty(self.gate_shape, dtype=dtype, device=device)
        how = dict(dy=dy, dz=dz, dx=out.get('x'), dh=None if plain else out.get('h'), dgate=out.get('gate'),
                   params=tuple(N.ptr(out.get(name)) for name in _PARAMS))
        room = N.lib.ffcvb_norm_residual_workspace(self.pack(stats, **how))
        workspace = ch.empty(room, dtype=ch.uint8, device=device)
        N.check(N.lib.ffcvb_norm_residual_backward(self.pack(stats, workspace=workspace.data_ptr(), **how), N.stream_of(self.x)))
        return out


def norm_residual_forward(x, h=None, *, norm='layer', weight=None, bias=None, post_norm=None, post_weight=None, post_bias=None,
                          gate=None, scale=None, eps=1e-6):
    """``(y, z, stats)`` of :func:`norm_residual` without autograd; ``stats`` is what
    :func:`norm_residual_backward` needs besides the arguments.  ``y`` is None without h, ``z`` without a norm."""
    return _Call(x, h, norm, weight, bias, post_norm, post_weight, post_bias, gate, scale, eps).forward()


def norm_residual_backward(dy, dz, x, h, stats, *, norm='layer', weight=None, bias=None, post_norm=None, post_weight=None,
                           post_bias=None, gate=None, scale=None, eps=1e-6):
    """Gradients of all tensors that :func:`norm_residual_forward` was given, by their names, from those of y and z (None: 0).
    Where the branch is added as it is, the entries 'x' and 'h' are one tensor."""
    call = _Call(x, h, norm, weight, bias, post_norm, post_weight, post_bias, gate, scale, eps)
    given = dict(x=x, h=h, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate, scale=call.scale)
    return call.backward(stats, dy, dz, {name for name, t in given.items() if t is not None})


class _NormResidual(ch.autograd.Function):
    NAMES = ('x', 'h', 'weight', 'bias', 'post_weight', 'post_bias', 'gate', 'scale')

    @staticmethod
    def forward(ctx, how, x, h, weight, bias, post_weight, post_bias, gate, scale):
        norm, post_norm, number, eps = how
        call = _Call(x, h, norm, weight, bias, post_norm, post_weight, post_bias, gate, scale if scale is not None else number, eps)
        y, z, stats = call.forward()
        ctx.how = how
        ctx.save_for_backward(x, h, weight, bias, post_weight, post_bias, gate, scale, stats)
        ctx.set_materialize_grads(False)
        return y, z

    @staticmethod
    @ch.autograd.function.once_differentiable
    def backward(ctx, dy, dz):
        norm, post_norm, number, eps = ctx.how
        x, h, weight, bias, post_weight, post_bias, gate, scale, stats = ctx.saved_tensors
        if dy is None and dz is None:
            return (None,) * 9
        call = _Call(x, h, norm, weight, bias, post_norm, post_weight, post_bias, gate, scale if scale is not None else number, eps)
        wanted = {name for name, needed in zip(_NormResidual.NAMES, ctx.needs_input_grad[1:]) if needed}
        grads = call.backward(stats, dy, dz, wanted)
        return (None,) + tuple(grads[name] if name in wanted else None for name in _NormResidual.NAMES)


def norm_residual(x, h=None, *, norm='layer', weight=None, bias=None, post_norm=None, post_weight=None, post_bias=None,
                  gate=None, scale=None, eps=1e-6):
    """``u = post_norm(h); y = x + scale * gate * u; z = norm(y)``; returns ``(y, z)``.

    Parameters
    ----------
    x : float32, float16 or bfloat16 CUDA tensor (..., tokens, width)
        The residual stream.
    h : the same, or None
        The block's output.  Without it y is x.
    norm, post_norm : 'layer', 'rms' or None
        Norms over the last dimension, with ``weight`` and ``bias``, ``post_weight`` and ``post_bias`` (width,), each of
        which may be None.  Without ``norm`` z is None.
    gate : of x's type
        A factor per value (the shape of x), or per sample and channel: (..., 1, width), (..., width), (width,); other
        shapes that broadcast are expanded first.
    scale : float, or tensor (width,)
        The residual scale.

    Everything is computed in 32 bits; y is rounded when it is stored, and z is made from what it was before.
    """
    if gate is not None:
        gate = gate.to(x.dtype)
        if _gate_kind(x, gate)[0] is None:
            gate = gate.expand(x.shape).contiguous()
    number = None
    if scale is not None and not isinstance(scale, ch.Tensor):
        number, scale = float(scale), None
    y, z = _NormResidual.apply((norm, post_norm, number, eps), x, h, weight, bias, post_weight, post_bias, gate, scale)
    return (x if h is None else y), z


class NormResidual(ch.nn.Module):
    """:func:`norm_residual` with its weights.

    Parameters
    ----------
    width : int
    norm, post_norm : 'layer', 'rms' or None
    scale : float or None
        Start value of a residual scale per channel; None: no scale.
    """

    def __init__(self, width, norm='layer', post_norm=None, scale=None, eps=1e-6, device=None, dtype=None):
        super().__init__()
        for kind in (norm, post_norm):
            if kind not in _NORMS:
                raise ValueError(f"norms are 'layer', 'rms' or None, not {kind!r}")
        self.width, self.norm, self.post_norm, self.eps = width, norm, post_norm, eps
        new = lambda on, value: ch.nn.Parameter(ch.full((width,), value, device=device, dtype=dtype)) if on else None  # noqa: E731
        self.weight, self.bias = new(norm is not None, 1.0), new(norm == 'layer', 0.0)
        self.post_weight, self.post_bias = new(post_norm is not None, 1.0), new(post_norm == 'layer', 0.0)
        self.scale = new(scale is not None, 0.0 if scale is None else float(scale))

    def extra_repr(self):
        return f'{self.width}, norm={self.norm!r}, post_norm={self.post_norm!r}, scale={self.scale is not None}, eps={self.eps}'

    def forward(self, x, h=None, gate=None):
        """``(y, z)``: the stream with the block's output h added, and its norm.  Without h: x, and its norm."""
        if h is None:
            return norm_residual(x, norm=self.norm, weight=self.weight, bias=self.bias, eps=self.eps)
        return norm_residual(x, h, norm=self.norm, weight=self.weight, bias=self.bias, post_norm=self.post_norm,
                             post_weight=self.post_weight, post_bias=self.post_bias, gate=gate, scale=self.scale, eps=self.eps)
