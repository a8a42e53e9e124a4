"""Cross entropy of a classifier's last layer whose logits are never kept, with the gradients of what goes into it."""
import torch as ch

from . import _native as N

_LABELS, _MIXED = range(2)
_REDUCTIONS = ('mean', 'sum', 'none')
_MOST_ROWS, _MOST_CLASSES, _MOST_WIDTH = 1 << 24, 1 << 24, 1 << 16


def _rows(t):
    """Rows that do not overlap and whose values lie together."""
    return t if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


class _Call:
    """A checked call: what the forward and the backward pass have in common."""
    __slots__ = ('hidden', 'weight', 'bias', 'target', 'kind', 'type', 'ignore', 'mean', 'smoothing', 'sizes')

    def __init__(self, hidden, weight, labels, mixed, bias, smoothing, ignore_index, reduction):
        self.type = N.require(hidden, 'hidden')
        if hidden.dtype == ch.float32:
            raise TypeError('hidden must be float16 or bfloat16; logits of 32-bit values go to cross_entropy')
        if hidden.dim() != 2 or not 1 <= hidden.shape[1] <= _MOST_WIDTH or hidden.shape[0] > _MOST_ROWS:
            raise ValueError(f'hidden must be (samples, width), at most {_MOST_ROWS} by {_MOST_WIDTH}, not {tuple(hidden.shape)}')
        n, width = hidden.shape
        if N.require(weight, 'weight', hidden) != self.type:
            raise TypeError(f'weight must be {hidden.dtype} as hidden is, not {weight.dtype}')
        if weight.dim() != 2 or weight.shape[1] != width or not 1 <= weight.shape[0] <= _MOST_CLASSES:
            raise ValueError(f'weight must be (classes, {width}), at most {_MOST_CLASSES} classes, not {tuple(weight.shape)}')
        classes = weight.shape[0]
        if bias is not None:
            if N.require(bias, 'bias', hidden) != self.type:
                raise TypeError(f'bias must be {hidden.dtype} as hidden is, not {bias.dtype}')
            if bias.shape != (classes,):
                raise ValueError(f'bias must be of shape ({classes},), not {tuple(bias.shape)}')
            bias = bias.contiguous()
        if (labels is None) == (mixed is None):
            raise ValueError('give exactly one of labels and mixed')
        if not 0.0 <= smoothing <= 1.0:
            raise ValueError(f'label_smoothing must be in [0, 1], not {smoothing}')
        if reduction not in _REDUCTIONS:
            raise ValueError(f'reduction must be one of {_REDUCTIONS}, not {reduction!r}')
        if labels is not None:
            self.kind, shape = _LABELS, (n,)
            if not isinstance(labels, ch.Tensor) or labels.dtype not in (ch.int64, ch.int32):
                raise TypeError('labels must be an int64 or int32 tensor')
            target = labels if labels.dtype == ch.int64 else labels.long()
        else:
            self.kind, shape = _MIXED, (n, 3)
            N.require(mixed, 'mixed', hidden)
            target = mixed if mixed.dtype == ch.float32 else mixed.float()
        if target.shape != shape:
            raise ValueError(f'targets must be of shape {shape}, not {tuple(target.shape)}')
        if self.kind == _MIXED and target.stride(1) != 1:
            target = target.contiguous()
        if target.device != hidden.device:
            raise ValueError(f'targets are on {target.device}, not on {hidden.device}')
        if ignore_index is not None and labels is None:
            raise ValueError('ignore_index goes with labels')
        self.hidden, self.weight, self.bias, self.target = _rows(hidden), _rows(weight), bias, target
        self.ignore, self.mean, self.smoothing, self.sizes = ignore_index, reduction == 'mean', float(smoothing), (n, classes, width)

    def run(self, grads, rows_at, loss_at, stats=None, upstream=None, per_row=False, from_stats=False, scale=1.0):
        """grads: of hidden, weight and bias, or None; rows_at, loss_at: addresses for a loss per sample, and for their mean or sum, or 0; without
        `stats` they are in the workspace."""
        x, w, t, ignore = self.hidden, self.weight, self.target, self.ignore
        index = x.get_device()

        def pack(stats_at):
            return N.LINEAR_CROSS_ENTROPY.pack(
                x.data_ptr(), w.data_ptr(), N.ptr(self.bias), t.data_ptr(), N.ptr(upstream), *map(N.ptr, grads), loss_at, rows_at, stats_at,
                *self.sizes, x.stride(0), w.stride(0), t.stride(0), -1 if ignore is None else ignore,
                index, self.type, self.kind, ignore is not None, self.mean, per_row, from_stats, 0, self.smoothing, scale)

        args = pack(16 if stats is None else stats.data_ptr())
        size = N.lib.ffcvb_linear_cross_entropy_workspace(args)
        workspace = ch.empty(size if stats is not None else size + 16 * self.sizes[0], dtype=ch.uint8, device=x.device)
        at = workspace.data_ptr()
        if stats is None:
            args = pack(at + size)
        N.check(N.lib.ffcvb_linear_cross_entropy(args, at, N.raw_stream(index)))

    def room_for(self, wanted):
        """Room for the gradients of hidden, weight and bias that are wanted."""
        n, classes, width = self.sizes
        new = lambda *shape: ch.empty(shape, dtype=self.hidden.dtype, device=self.hidden.device)  # noqa: E731
        return (new(n, width) if wanted[0] else None, new(classes, width) if wanted[1] else None,
                new(classes) if wanted[2] and self.bias is not None else None)


def linear_cross_entropy_with_grad(hidden, weight, labels=None, *, mixed=None, bias=None, label_smoothing=0.0, ignore_index=None,
                                   reduction='mean', grad_scale=1.0):
    """The loss of ``hidden @ weight.T + bias`` and the gradients of the three: ``(loss, grad_hidden, grad_weight, grad_bias)``.

    The logits are never in memory as a whole: they are made on the tensor cores in 32 bits, once for the loss and once more,
    some classes at a time, for the gradients.

    Parameters
    ----------
    hidden : float16 or bfloat16 CUDA tensor (samples, width)
    weight : of hidden's type (classes, width)
    labels : int64 or int32 (samples,)
        One class per sample.
    mixed : float (samples, 3)
        What ``LabelMixup`` makes: a class, the class mixed in, and the share of the first.  Where the two are the same their shares add up.
    bias : of hidden's type (classes,), or None
        ``grad_bias`` is None without it.
    label_smoothing : float
        Share of the target that is spread over all classes.
    ignore_index : int
        Samples with this label count for nothing: their hidden values are not even read, and take no time.  (Other labels
        outside the classes make a sample's loss NaN, its gradient, and with it the weights'.)
    reduction : 'mean', 'sum' or 'none'
        With 'none' the loss is a value per sample, and the gradients those of their sum.
    grad_scale : float
        Factor of the gradients, applied before they are rounded to 16 bits: with float16 the loss scale.

    The loss is float32.  The gradient of the logits is rounded to 16 bits before it is multiplied with weights and hidden values; the
    bias' is the sum of it as it was before.  With a gradient
    per sample from behind (``reduction='none'`` and autograd) it is held relative to the largest of these among the samples that count: in
    float16 in steps of 2^-38 of that, so a sample with a billionth of the largest keeps few digits.  One that is infinite or NaN
    makes its own sample's hidden gradient NaN, and those of the weights and the bias, which are sums over the samples.

    A kernel whose own copies or products do not come to an end gives up after two seconds; the call has returned by then, and what is missing is
    NaN, in the loss too.
    """
    call = _Call(hidden, weight, labels, mixed, bias, label_smoothing, ignore_index, reduction)
    n = hidden.shape[0]
    grads = call.room_for((True, True, True))
    loss = ch.empty(n + 1, dtype=ch.float32, device=hidden.device)
    at = loss.data_ptr()
    call.run(grads, at, 0 if reduction == 'none' else at + 4 * n, scale=grad_scale)
    return (loss[:n] if reduction == 'none' else loss[n], *grads)


class _LinearCrossEntropy(ch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, call, reduction):
        n = hidden.shape[0]
        ctx.per_row = reduction == 'none'
        loss = ch.empty(n if ctx.per_row else (), dtype=ch.float32, device=hidden.device)
        stats = ch.empty(4 * n if ctx.per_row else 5 * n, dtype=ch.float32, device=hidden.device)
        if ctx.per_row:
            call.run((None, None, None), loss.data_ptr(), 0, stats)
        else:
            call.run((None, None, None), stats.data_ptr() + 16 * n, loss.data_ptr(), stats)
        ctx.save_for_backward(call.hidden, call.weight, call.bias, call.target, stats)
        call.hidden = call.weight = call.bias = call.target = None  # (autograd keeps them, and sees to it that nobody changes them)
        ctx.call = call
        return loss

    @staticmethod
    @ch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        call = ctx.call
        call.hidden, call.weight, call.bias, call.target, stats = ctx.saved_tensors
        grads = call.room_for(ctx.needs_input_grad[:3])
        if any(g is not None for g in grads):
            call.run(grads, 0, 0, stats, upstream.float().contiguous(), ctx.per_row, True)
        call.hidden = call.weight = call.bias = call.target = None
        return (*grads, None, None)


def linear_cross_entropy(hidden, weight, labels=None, *, mixed=None, bias=None, label_smoothing=0.0, ignore_index=None, reduction='mean'):
    """The loss as a function of hidden values, weights and bias that autograd knows; see :func:`linear_cross_entropy_with_grad`
    for the arguments.  The gradients are made in the backward pass, where a loss scale is known.  Under autocast hidden values, weights and
    bias are taken in its type, as a linear layer takes them."""
    if ch.is_autocast_enabled('cuda'):
        dtype = ch.get_autocast_dtype('cuda')
        hidden, weight, bias = (t.to(dtype) if isinstance(t, ch.Tensor) and t.is_cuda and t.dtype in N.TYPES else t for t in (hidden, weight, bias))
    call = _Call(hidden, weight, labels, mixed, bias, label_smoothing, ignore_index, reduction)
    return _LinearCrossEntropy.apply(call.hidden, call.weight, call.bias, call, reduction)


class LinearCrossEntropy(ch.nn.Module):
    """The last layer of a classifier together with its loss against class labels or the ``[label, label of the sample mixed in,
    lambda]`` rows of ``LabelMixup``.  Weights are named as those of a ``torch.nn.Linear``."""

    def __init__(self, width, classes, bias=True, label_smoothing=0.0, ignore_index=None, reduction='mean', device=None, dtype=None):
        super().__init__()
        self.label_smoothing, self.ignore_index, self.reduction = label_smoothing, ignore_index, reduction
        layer = ch.nn.Linear(width, classes, bias=bias, device=device, dtype=dtype)  # (its start values)
        self.weight, self.bias = layer.weight, layer.bias

    def extra_repr(self):
        return f'{self.weight.shape[1]}, {self.weight.shape[0]}, bias={self.bias is not None}'

    def logits(self, hidden):
        """What the loss is of: for predictions."""
        return ch.nn.functional.linear(hidden, self.weight, self.bias)

    def forward(self, hidden, target):
        if target.is_floating_point():
            return linear_cross_entropy(hidden, self.weight, mixed=target, bias=self.bias, label_smoothing=self.label_smoothing,
                                        reduction=self.reduction)
        return linear_cross_entropy(hidden, self.weight, target, bias=self.bias, label_smoothing=self.label_smoothing,
                                    ignore_index=self.ignore_index, reduction=self.reduction)
