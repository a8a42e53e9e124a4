"""Cross entropy against class labels, the rows of ``LabelMixup``, or probabilities, and its gradient."""
import torch as ch

from . import _native as N

_LABELS, _MIXED, _SOFT = range(3)
_REDUCTIONS = ('mean', 'sum', 'none')


class _Call:
    """A checked call: what the forward and the backward pass have in common."""
    __slots__ = ('logits', 'target', 'kind', 'type', 'target_type', 'ignore', 'mean', 'smoothing')

    def __init__(self, logits, labels, mixed, soft, smoothing, ignore_index, reduction):
        self.type = N.require(logits, 'logits')
        if logits.dim() != 2 or logits.shape[1] == 0:
            raise ValueError(f'logits must be (samples, classes), not {tuple(logits.shape)}')
        if (labels is None) + (mixed is None) + (soft is None) != 2:
            raise ValueError('give exactly one of labels, mixed and soft')
        if not 0.0 <= smoothing <= 1.0:
            raise ValueError(f'label_smoothing must be in [0, 1], not {smoothing}')
        if reduction not in _REDUCTIONS:
            raise ValueError(f'reduction must be one of {_REDUCTIONS}, not {reduction!r}')
        n, classes = logits.shape
        self.target_type = 0
        if labels is not None:
            self.kind, target, shape = _LABELS, labels, (n,)
            if not isinstance(labels, ch.Tensor) or labels.dtype not in (ch.int64, ch.int32):
                raise TypeError('labels must be an int64 or int32 tensor')
            target = labels if labels.dtype == ch.int64 else labels.long()
        elif mixed is not None:
            self.kind, target, shape = _MIXED, mixed, (n, 3)
            N.require(mixed, 'mixed', logits)
            target = mixed if mixed.dtype == ch.float32 else mixed.float()
            if target.stride(1) != 1:
                target = target.contiguous()
        else:
            self.kind, target, shape = _SOFT, soft, (n, classes)
            self.target_type = N.require(soft, 'soft', logits)
            if soft.requires_grad:
                raise ValueError('soft: there is no gradient with respect to the probabilities')
            if target.stride(1) != 1:
                target = target.contiguous()
        if target.shape != shape:
            raise ValueError(f'targets must be of shape {shape}, not {tuple(target.shape)}')
        if target.device != logits.device:
            raise ValueError(f'targets are on {target.device}, not on {logits.device}')
        if ignore_index is not None and labels is None:
            raise ValueError('ignore_index goes with labels')
        self.logits = logits if logits.stride(1) == 1 else logits.contiguous()
        self.target, self.ignore, self.mean, self.smoothing = target, ignore_index, reduction == 'mean', float(smoothing)

    def run(self, grad, rows_at, loss_at, stats=None, upstream=None, per_row=False, from_stats=False, scale=1.0):
        """rows_at, loss_at: addresses for a loss per sample, and for their mean or sum, or 0."""
        x, t, ignore = self.logits, self.target, self.ignore
        rows, classes = x.shape
        counted = ch.empty(1, dtype=ch.float32, device=x.device) if ignore is not None and self.mean else None
        index = x.get_device()
        args = N.CROSS_ENTROPY.pack(
            x.data_ptr(), t.data_ptr(), N.ptr(upstream), N.ptr(grad), loss_at, rows_at, N.ptr(stats), N.ptr(counted),
            rows, classes, x.stride(0), t.stride(0), classes, -1 if ignore is None else ignore,
            index, self.type, self.kind, self.target_type, ignore is not None, self.mean, per_row, from_stats, self.smoothing, scale)
        N.check(N.lib.ffcvb_cross_entropy(args, N.raw_stream(index)))


def cross_entropy_with_grad(logits, labels=None, *, mixed=None, soft=None, label_smoothing=0.0, ignore_index=None,
                            reduction='mean', grad_scale=1.0):
    """The loss and its gradient with respect to the logits in one pass: ``(loss, grad)``.

    Parameters
    ----------
    logits : float32, float16 or bfloat16 CUDA tensor (samples, classes)
    labels : int64 or int32 (samples,)
        One class per sample.
    mixed : float (samples, 3)
        What ``LabelMixup`` makes: a class, the class mixed in, and the share of the first.  Where the two are the
        same their shares add up (``MixupToOneHot`` keeps the second one only, as the reference does).
    soft : float (samples, classes)
        Probabilities.
    label_smoothing : float
        Share of the target that is spread over all classes.
    ignore_index : int
        Samples with this label count for nothing.  (Other labels outside the classes make a sample's loss and
        gradient NaN.)
    reduction : 'mean', 'sum' or 'none'
        With 'none' the loss is a value per sample, and the gradient that of their sum.
    grad_scale : float
        Factor of the gradient, applied before it is rounded to the logits' type: with float16 logits the loss scale.

    The loss is float32.  A sample whose logits are all -inf has loss and gradient 0.
    """
    call = _Call(logits, labels, mixed, soft, label_smoothing, ignore_index, reduction)
    n = logits.shape[0]
    loss, grad = ch.empty(n + 1, dtype=ch.float32, device=logits.device), N.new_like(call.logits)
    at = loss.data_ptr()
    call.run(grad, at, 0 if reduction == 'none' else at + 4 * n, scale=grad_scale)
    return loss[:n] if reduction == 'none' else loss[n], grad


class _CrossEntropy(ch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call, reduction):
        n = logits.shape[0]
        ctx.per_row = reduction == 'none'
        # the result is a tensor of its own (a part of another one could not be changed in place); losses of rows that are not are behind the statistics
        loss = ch.empty(n if ctx.per_row else (), dtype=ch.float32, device=logits.device)
        stats = ch.empty(2 * n if ctx.per_row else 3 * n, dtype=ch.float32, device=logits.device)
        if ctx.per_row:
            call.run(None, loss.data_ptr(), 0, stats)
        else:
            call.run(None, stats.data_ptr() + 8 * n, loss.data_ptr(), stats)
        ctx.save_for_backward(call.logits, call.target, stats)
        call.logits = call.target = None  # (autograd keeps them, and sees to it that nobody changes them)
        ctx.call = call
        return loss

    @staticmethod
    @ch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        call = ctx.call
        call.logits, call.target, stats = ctx.saved_tensors
        grad = N.new_like(call.logits)
        upstream = upstream.float().contiguous()
        call.run(grad, 0, 0, stats, upstream, ctx.per_row, True)
        call.logits = call.target = None
        return grad, None, None


def cross_entropy(logits, labels=None, *, mixed=None, soft=None, label_smoothing=0.0, ignore_index=None, reduction='mean'):
    """The loss as a function of the logits that autograd knows; see :func:`cross_entropy_with_grad` for the arguments.
    The gradient is made in the backward pass, where a loss scale is known."""
    call = _Call(logits, labels, mixed, soft, label_smoothing, ignore_index, reduction)
    return _CrossEntropy.apply(call.logits, call, reduction)


class MixupCrossEntropy(ch.nn.Module):
    """Cross entropy of logits against the ``[label, label of the sample mixed in, lambda]`` rows of ``LabelMixup``
    (to go behind ``ToTensor`` and ``ToDevice`` in the label pipeline), or against plain int labels."""

    def __init__(self, label_smoothing=0.0, ignore_index=None, reduction='mean'):
        super().__init__()
        self.label_smoothing, self.ignore_index, self.reduction = label_smoothing, ignore_index, reduction

    def forward(self, logits, target):
        if target.is_floating_point():
            return cross_entropy(logits, mixed=target, label_smoothing=self.label_smoothing, reduction=self.reduction)
        return cross_entropy(logits, target, label_smoothing=self.label_smoothing, ignore_index=self.ignore_index,
                             reduction=self.reduction)
