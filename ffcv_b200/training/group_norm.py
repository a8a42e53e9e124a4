"""Group norm with an activation behind it, of images that lie channels last, in one pass each way."""
import torch as ch

from . import _native as N

_ACTIVATIONS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3}
_NAMES = ('x', 'weight', 'bias')


def _strides(t):
    """Strides of samples and positions of (samples, channels, ...) whose channels lie together and whose positions are evenly apart, or
    None.  Dimensions of one value may have any stride."""
    shape = t.shape
    if len(shape) == 4 and t.is_contiguous(memory_format=ch.channels_last):  # (as most are: 1 us and not 3)
        channels = shape[1]
        return shape[2] * shape[3] * channels, channels
    samples, channels, *sides = shape
    if t.numel() == 0:
        return 0, channels
    stride = t.stride()
    if channels > 1 and stride[1] != 1:
        return None
    position, along = None, 1  # the innermost dimension's stride, positions within it
    for size, step in zip(reversed(sides), reversed(stride[2:])):
        if size == 1:
            continue
        if position is None:
            position = step
        elif step != position * along:
            return None
        along *= size
    position = channels if position is None else position
    if along > 1 and position < channels:  # (positions that share memory)
        return None
    return stride[0] if samples > 1 else along * position, position


def _last(t):
    """Channels last, in new memory."""
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


def _new(t):
    """Room for a dense result of a tensor's shape, channels last."""
    if t.dim() == 4 and t.is_contiguous(memory_format=ch.channels_last):
        return ch.empty_like(t)
    samples, channels, *sides = t.shape
    return ch.empty((samples, *sides, channels), dtype=t.dtype, device=t.device).movedim(-1, 1)


class _Call:
    """A checked call: what the forward and the backward pass have in common."""
    __slots__ = ('x', 'weight', 'bias', 'strides', 'sizes', 'type', 'param_dtype', 'param_type', 'activation', 'eps', 'index')

    def __init__(self, x, groups, weight, bias, activation, eps):
        self.type = N.require(x, 'x')
        if x.dim() < 2 or x.shape[1] == 0:
            raise ValueError(f'x must be (samples, channels, ...), not {tuple(x.shape)}')
        samples, channels = x.shape[:2]
        if isinstance(groups, bool) or not isinstance(groups, int) or groups < 1 or channels % groups != 0:
            raise ValueError(f'groups must divide the {channels} channels, {groups!r} does not')
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activations are 'relu', 'silu', 'gelu' or None, not {activation!r}")
        if not eps >= 0.0:
            raise ValueError(f'eps must not be below 0, as {eps} is')
        self.param_dtype, self.param_type = None, 0
        for name, p in (('weight', weight), ('bias', bias)):
            if p is None:
                continue
            kind = N.require(p, name, x)
            if p.shape != (channels,):
                raise ValueError(f'{name} must be of shape ({channels},), not {tuple(p.shape)}')
            if self.param_dtype is None:
                self.param_dtype, self.param_type = p.dtype, kind
            elif p.dtype is not self.param_dtype:
                raise TypeError('weight and bias must be of one type')
        self.weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
        self.bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        self.x, self.strides = self.laid(x)
        positions = 1
        for side in x.shape[2:]:
            positions *= side
        self.sizes, self.activation, self.eps, self.index = (samples, positions, channels, groups), _ACTIVATIONS[activation], float(eps), x.get_device()

    @staticmethod
    def laid(t):
        strides = _strides(t)
        if strides is None:
            t = _last(t)
            strides = _strides(t)
        return t, strides

    def pack(self, stats, y, dy, dx, dweight, dbias, dy_strides):
        return N.GROUP_NORM.pack(self.x.data_ptr(), N.ptr(self.weight), N.ptr(self.bias), stats.data_ptr(), *map(N.ptr, (y, dy, dx, dweight, dbias)),
                                 *self.sizes, *self.strides, *dy_strides, self.index, self.type, self.param_type, self.activation, self.eps, 0)

    def room(self, args, backward):
        size = N.lib.ffcvb_group_norm_workspace(args, backward)
        return ch.empty(size, dtype=ch.uint8, device=self.x.device) if size else None

    def forward(self):
        y = _new(self.x)
        stats = ch.empty((self.sizes[0], self.sizes[3], 2), dtype=ch.float32, device=self.x.device)
        args = self.pack(stats, y, None, None, None, None, (0, 0))
        workspace = self.room(args, 0)
        N.check(N.lib.ffcvb_group_norm(args, N.ptr(workspace), N.raw_stream(self.index)))
        return y, stats

    def backward(self, dy, stats, wanted):
        """The gradients of x, weight and bias, of which `wanted` says which ones (only such as the call was given), else None."""
        x = self.x
        if N.require(dy, 'dy', x) != self.type or dy.shape != x.shape:
            raise ValueError(f'dy must be {x.dtype} {tuple(x.shape)}, not {dy.dtype} {tuple(dy.shape)}')
        if stats.shape != (self.sizes[0], self.sizes[3], 2) or stats.dtype != ch.float32 or not stats.is_contiguous() or stats.device != x.device:
            raise ValueError('stats must be what the forward pass of the same call gave')
        if stats.data_ptr() % 8:  # (kept in the middle of another tensor)
            stats = stats.clone()
        dy, dy_strides = self.laid(dy)
        dx = _new(x) if wanted[0] else None
        dweight, dbias = (ch.empty_like(p) if w else None for p, w in zip((self.weight, self.bias), wanted[1:]))
        if dx is not None or dweight is not None or dbias is not None:
            args = self.pack(stats, None, dy, dx, dweight, dbias, dy_strides)
            workspace = self.room(args, 1)
            N.check(N.lib.ffcvb_group_norm_backward(args, N.ptr(workspace), N.raw_stream(self.index)))
        return dx, dweight, dbias


def group_norm_act_forward(x, groups, *, weight=None, bias=None, activation=None, eps=1e-5):
    """``(y, stats)`` of :func:`group_norm_act` without autograd; ``stats`` (samples, groups, 2) are each group's mean and
    1 / deviation, which :func:`group_norm_act_backward` needs besides the arguments."""
    return _Call(x, groups, weight, bias, activation, eps).forward()


def group_norm_act_backward(dy, x, stats, groups, *, weight=None, bias=None, activation=None, eps=1e-5):
    """Gradients of x, and of weight and bias where there are, by their names, from that of y."""
    grads = _Call(x, groups, weight, bias, activation, eps).backward(dy, stats, (True, weight is not None, bias is not None))
    return {name: g for name, g in zip(_NAMES, grads) if g is not None}


class _GroupNormAct(ch.autograd.Function):
    @staticmethod
    def forward(ctx, how, x, weight, bias):
        groups, activation, eps = how
        y, stats = _Call(x, groups, weight, bias, activation, eps).forward()
        ctx.how = how
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @ch.autograd.function.once_differentiable
    def backward(ctx, dy):
        groups, activation, eps = ctx.how
        x, weight, bias, stats = ctx.saved_tensors
        return (None, *_Call(x, groups, weight, bias, activation, eps).backward(dy, stats, ctx.needs_input_grad[1:]))


def group_norm_act(x, groups, weight=None, bias=None, *, activation=None, eps=1e-5):
    """``activation(group_norm(x))``, channels last.

    Parameters
    ----------
    x : float32, float16 or bfloat16 CUDA tensor (samples, channels, ...)
        Images, or anything else with positions behind the channels, or none.  Channels should lie next to one another in memory, as in
        what ``ToTorchImage`` hands over; other tensors are copied first.  The result lies that way, whatever x does.
    groups : int
        Groups of neighbouring channels, each of which is normed over its channels and all positions of a sample.
    weight, bias : (channels,), of one type, each or both None
    activation : 'relu', 'silu', 'gelu' or None
    eps : float

    Everything is computed in 32 bits and rounded once.  The backward pass keeps x, not y.
    """
    return _GroupNormAct.apply((groups, activation, eps), x, weight, bias)


class GroupNormAct(ch.nn.Module):
    """:func:`group_norm_act` with its weights, which are named as those of a ``torch.nn.GroupNorm``."""

    def __init__(self, groups, channels, activation=None, eps=1e-5, affine=True, device=None, dtype=None):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activations are 'relu', 'silu', 'gelu' or None, not {activation!r}")
        if groups < 1 or channels % groups != 0:
            raise ValueError(f'groups must divide the {channels} channels, {groups!r} does not')
        self.groups, self.channels, self.activation, self.eps = groups, channels, activation, eps
        new = lambda value: ch.nn.Parameter(ch.full((channels,), value, device=device, dtype=dtype)) if affine else None  # noqa: E731
        self.weight, self.bias = new(1.0), new(0.0)

    def extra_repr(self):
        return f'{self.groups}, {self.channels}, activation={self.activation!r}, eps={self.eps}, affine={self.weight is not None}'

    def forward(self, x):
        return group_norm_act(x, self.groups, self.weight, self.bias, activation=self.activation, eps=self.eps)
