"""The seam between two blocks of a residual network: the norm behind a block, its gate and residual scale, the sum with
the residual stream, and the norm before the next block, in one kernel each way."""
import torch as ch

from . import _native as N

_NORMS = {None: 0, 'layer': 1, 'rms': 2}
_NO_GATE, _SAMPLE, _TOKEN = range(3)
_PARAMS = ('weight', 'bias', 'post_weight', 'post_bias', 'scale')
_NAMES = ('x', 'h', 'weight', 'bias', 'post_weight', 'post_bias', 'gate', 'scale')


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


class _Call:
    """A checked call: what the forward and the backward pass have in common."""
    __slots__ = ('x', 'h', 'gate', 'scale', 'width', 'rows', 'type', 'param_dtype', 'param_type', 'index', 'norm', 'post_norm', 'gate_kind',
                 'tokens', 'eps', 'number', 'given', 'strides', 'kept')

    def __init__(self, x, h, norm, weight, bias, post_norm, post_weight, post_bias, gate, scale, eps):
        self.type = N.require(x, 'x')
        shape = x.shape
        if len(shape) < 1 or not 1 <= shape[-1] <= N.NORM_MAX_WIDTH:
            raise ValueError(f'x must have 1 to {N.NORM_MAX_WIDTH} values in its last dimension, not {tuple(shape)}')
        if norm not in _NORMS or post_norm not in _NORMS:
            raise ValueError("norms are 'layer', 'rms' or None")
        if h is None:
            if norm is None:
                raise ValueError('nothing to do: neither a branch nor a norm')
            if post_norm is not None or gate is not None or scale is not None:
                raise ValueError('post_norm, gate and scale go with a branch h')
        elif N.require(h, 'h', x) != self.type or h.shape != shape:
            raise ValueError(f'h must be {x.dtype} {tuple(shape)}, not {h.dtype} {tuple(h.shape)}')
        if norm is None and (weight is not None or bias is not None):
            raise ValueError('weight and bias go with a norm')
        if post_norm is None and (post_weight is not None or post_bias is not None):
            raise ValueError('post_weight and post_bias go with a post_norm')
        self.number = 1.0
        if scale is not None and not isinstance(scale, ch.Tensor):
            self.number, scale = float(scale), None
        self.x, self.h, self.gate, self.scale = x, h, gate, scale
        self.width = width = shape[-1]
        self.rows = x.numel() // width
        self.index = x.get_device()
        self.param_dtype, self.param_type, self.kept = None, 0, []
        at = [0] * 8  # addresses of x, h, gate, and the parameters
        for k, p in enumerate((weight, bias, post_weight, post_bias, scale)):
            if p is None:
                continue
            kind = N.require(p, _PARAMS[k], x)
            if p.shape != (width,):
                raise ValueError(f'{_PARAMS[k]} must be of shape ({width},), not {tuple(p.shape)}')
            if self.param_dtype is None:
                self.param_dtype, self.param_type = p.dtype, kind
            elif p.dtype is not self.param_dtype:
                raise TypeError('weights, biases and scale must be of one type')
            if not p.is_contiguous():
                p = p.contiguous()
                self.kept.append(p)
            at[3 + k] = p.data_ptr()
        self.gate_kind, self.tokens = _gate_kind(x, gate)
        self.tokens = max(1, self.tokens)  # (samples without tokens have no rows)
        if gate is not None and (N.require(gate, 'gate', x) != self.type or self.gate_kind is None):
            raise ValueError(f'gate must be {x.dtype}, with a row per row or per sample of {tuple(shape)}, not {gate.dtype} {tuple(gate.shape)}')
        at[0], x_stride = self.rows_of(x)
        at[1], h_stride = self.rows_of(h)
        at[2], gate_stride = self.rows_of(gate)
        self.given, self.strides = at, (x_stride, h_stride, gate_stride)
        self.norm, self.post_norm, self.eps = _NORMS[norm], _NORMS[post_norm], float(eps)

    def rows_of(self, t):
        """Address of rows whose values lie together, and the stride from one to the next: a view where the strides allow it."""
        if t is None:
            return 0, 0
        if t.is_contiguous():
            return t.data_ptr(), self.width
        t = t.reshape(-1, self.width)
        if self.width > 1 and t.stride(1) != 1:
            t = t.contiguous()
        self.kept.append(t)
        return t.data_ptr(), t.stride(0)

    def plain(self):
        """Whether the branch is added as it is, so that its gradient is the stream's."""
        return self.post_norm == 0 and self.gate is None and self.scale is None and self.number == 1.0

    def pack(self, stats, *places):
        """places: y, z; dy, dz; dx, dh, dgate; the parameters' gradients; dy's and dz's strides."""
        return N.NORM_RESIDUAL.pack(
            *self.given, stats.data_ptr(), *places[:12], self.rows, self.width, self.tokens, *self.strides, *places[12:], self.index,
            self.type, self.param_type, self.norm, self.post_norm, self.gate_kind, self.eps, self.number)

    def forward(self):
        x = self.x
        y, z = None if self.h is None else N.new_like(x), N.new_like(x) if self.norm else None
        stats = ch.empty(4 * self.rows, dtype=ch.float32, device=x.device)
        N.check(N.lib.ffcvb_norm_residual(self.pack(stats, N.ptr(y), N.ptr(z), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), N.raw_stream(self.index)))
        return y, z, stats

    def backward(self, stats, dy, dz, wanted):
        """The gradients of x, h, weight, bias, post_weight, post_bias, gate and scale, of which `wanted` says which ones (only such as
        the call was given), else None."""
        x = self.x
        for name, g in (('dy', dy), ('dz', dz)):
            if g is not None and (N.require(g, name, x) != self.type or g.shape != x.shape):
                raise ValueError(f'{name} must be {x.dtype} {tuple(x.shape)}, not {g.dtype} {tuple(g.shape)}')
        if dz is not None and self.norm == 0:
            raise ValueError('dz goes with a norm')
        dy_at, dy_stride = self.rows_of(dy)
        dz_at, dz_stride = self.rows_of(dz)
        of_x, of_h, of_weight, of_bias, of_post_weight, of_post_bias, of_gate, of_scale = wanted
        plain = self.plain()
        dx = N.new_like(x) if of_x or (plain and of_h) else None
        dh = None if not of_h else dx if plain else N.new_like(x)
        dgate = N.new_like(self.gate) if of_gate else None
        if of_gate and self.rows == 0:  # samples' gates may be there all the same
            dgate.zero_()
        new, device = ch.empty, x.device
        params = [new(self.width, dtype=self.param_dtype, device=device) if of else None
                  for of in (of_weight, of_bias, of_post_weight, of_post_bias, of_scale)]
        ptr = N.ptr
        args = self.pack(stats, 0, 0, dy_at, dz_at, ptr(dx), 0 if plain else ptr(dh), ptr(dgate), *map(ptr, params), dy_stride, dz_stride)
        workspace = new(N.lib.ffcvb_norm_residual_workspace(args), dtype=ch.uint8, device=device)
        N.check(N.lib.ffcvb_norm_residual_backward(args, workspace.data_ptr(), N.raw_stream(self.index)))
        return dx if of_x else None, dh, *params[:4], dgate, params[4]


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
    if not isinstance(stats, ch.Tensor) or stats.shape != (4 * call.rows,) or stats.dtype != ch.float32 or not stats.is_contiguous() or stats.device != x.device:
        raise ValueError('stats must be what the forward pass of the same call gave')
    if stats.data_ptr() % 16:  # (kept in the middle of another tensor)
        stats = stats.clone()
    grads = call.backward(stats, dy, dz, [t is not None for t in (x, h, weight, bias, post_weight, post_bias, gate, call.scale)])
    return {name: g for name, g in zip(_NAMES, grads) if g is not None}


class _NormResidual(ch.autograd.Function):
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
        return (None,) + tuple(call.backward(stats, dy, dz, ctx.needs_input_grad[1:]))


def norm_residual(x, h=None, *, norm='layer', weight=None, bias=None, post_norm=None, post_weight=None, post_bias=None,
                  gate=None, scale=None, eps=1e-6):
    """``u = post_norm(h); y = x + scale * gate * u; z = norm(y)``; returns ``(y, z)``.

    Parameters
    ----------
    x : float32, float16 or bfloat16 CUDA tensor (..., tokens, width)
        The residual stream.
    h : the same, or None
        The block's output.  Without it y is x.  A branch of another type than the stream's (of 16 bits beside 32, as automatic mixed
        precision makes it): both are taken in the wider of the two.
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
    if isinstance(h, ch.Tensor) and isinstance(x, ch.Tensor) and h.dtype is not x.dtype and h.dtype in N.TYPES and x.dtype in N.TYPES:
        wide = ch.promote_types(x.dtype, h.dtype)
        x, h = x.to(wide), h.to(wide)
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
