"""Loss of logits against a teacher's largest logits, with the loss against labels beside it, and its gradient."""
import math

import torch as ch

from . import _native as N

_LABELS, _MIXED = range(2)
_REDUCTIONS = ('mean', 'sum', 'none')


def _rows(t):
    return t if t.stride(1) == 1 else t.contiguous()


class _Call:
    """A checked call: what the forward and the backward pass have in common."""
    __slots__ = ('logits', 'teacher', 'classes', 'target', 'kind', 'type', 'teacher_type', 'ignore', 'mean', 'smoothing', 'temperature', 'hard')

    def __init__(self, logits, teacher_logits, teacher_classes, labels, mixed, temperature, hard_weight, smoothing, ignore_index, reduction):
        self.type = N.require(logits, 'logits')
        if logits.dim() != 2 or logits.shape[1] == 0:
            raise ValueError(f'logits must be (samples, classes), not {tuple(logits.shape)}')
        n = logits.shape[0]
        self.teacher_type = N.require(teacher_logits, 'teacher_logits', logits)
        if teacher_logits.dim() != 2 or teacher_logits.shape[0] != n or not 1 <= teacher_logits.shape[1] <= N.DISTILLATION_MOST:
            raise ValueError(f'teacher_logits must be ({n}, 1 to {N.DISTILLATION_MOST}), not {tuple(teacher_logits.shape)}')
        if teacher_logits.requires_grad:
            raise ValueError('teacher_logits: there is no gradient with respect to the teacher')
        if not isinstance(teacher_classes, ch.Tensor) or teacher_classes.dtype not in (ch.int64, ch.int32):
            raise TypeError('teacher_classes must be an int64 or int32 tensor')
        if teacher_classes.shape != teacher_logits.shape:
            raise ValueError(f'teacher_classes must be of shape {tuple(teacher_logits.shape)}, not {tuple(teacher_classes.shape)}')
        if not (math.isfinite(temperature) and 1e-30 <= temperature <= 1e30):
            raise ValueError(f'temperature must be above 0, not {temperature}')
        if not 0.0 <= hard_weight <= 1.0:
            raise ValueError(f'hard_weight must be in [0, 1], not {hard_weight}')
        if not 0.0 <= smoothing <= 1.0:
            raise ValueError(f'label_smoothing must be in [0, 1], not {smoothing}')
        if reduction not in _REDUCTIONS:
            raise ValueError(f'reduction must be one of {_REDUCTIONS}, not {reduction!r}')
        if labels is not None and mixed is not None:
            raise ValueError('give at most one of labels and mixed')
        if labels is None and mixed is None and hard_weight != 0.0:
            raise ValueError('hard_weight goes with labels or mixed')
        if ignore_index is not None and labels is None:
            raise ValueError('ignore_index goes with labels')
        self.kind, target = _LABELS, None
        if labels is not None:
            if not isinstance(labels, ch.Tensor) or labels.dtype not in (ch.int64, ch.int32):
                raise TypeError('labels must be an int64 or int32 tensor')
            target, shape = labels if labels.dtype == ch.int64 else labels.long(), (n,)
        elif mixed is not None:
            N.require(mixed, 'mixed', logits)
            self.kind, target, shape = _MIXED, mixed if mixed.dtype == ch.float32 else mixed.float(), (n, 3)
        if target is not None:
            if target.shape != shape:
                raise ValueError(f'targets must be of shape {shape}, not {tuple(target.shape)}')
            if self.kind == _MIXED:
                target = _rows(target)
        for name, t in (('teacher_classes', teacher_classes), ('targets', target)):
            if t is not None and t.device != logits.device:
                raise ValueError(f'{name} are on {t.device}, not on {logits.device}')
        self.logits, self.teacher, self.classes, self.target = _rows(logits), _rows(teacher_logits), _rows(teacher_classes), target
        self.ignore, self.mean, self.smoothing = ignore_index, reduction == 'mean', float(smoothing)
        self.temperature, self.hard = float(temperature), float(hard_weight)

    def run(self, grad, rows_at, loss_at, stats=None, upstream=None, per_row=False, from_stats=False, scale=1.0):
        """rows_at, loss_at: addresses for a loss per sample, and for their mean or sum, or 0."""
        x, t, c, target, ignore = self.logits, self.teacher, self.classes, self.target, self.ignore
        rows, classes = x.shape
        counted = ch.empty(1, dtype=ch.float32, device=x.device) if ignore is not None and self.mean else None
        index = x.get_device()
        args = N.DISTILLATION.pack(
            x.data_ptr(), t.data_ptr(), c.data_ptr(), N.ptr(target), N.ptr(upstream), N.ptr(grad), loss_at, rows_at, N.ptr(stats), N.ptr(counted),
            rows, classes, t.shape[1], x.stride(0), t.stride(0), c.stride(0), 0 if target is None else target.stride(0), classes,
            -1 if ignore is None else ignore, index, self.type, self.teacher_type, c.dtype == ch.int64, self.kind, ignore is not None, self.mean, per_row,
            from_stats, 0, self.temperature, self.hard, self.smoothing, scale)
        N.check(N.lib.ffcvb_distillation(args, N.raw_stream(index)))


def distillation_with_grad(logits, teacher_logits, teacher_classes, labels=None, *, mixed=None, temperature=1.0, hard_weight=0.0,
                           label_smoothing=0.0, ignore_index=None, reduction='mean', grad_scale=1.0):
    """The loss of logits against a teacher's largest ones and its gradient with respect to the logits in one pass: ``(loss, grad)``.

    With q the softmax of a sample's teacher logits over the temperature and p that of its logits over all classes, the loss is
    ``(1 - hard_weight) * temperature ** 2 * sum(q * log(q / p)) + hard_weight * cross_entropy``.

    Parameters
    ----------
    logits : float32, float16 or bfloat16 CUDA tensor (samples, classes)
    teacher_logits : float32, float16 or bfloat16 (samples, kept)
        The teacher's largest logits of each sample, 1 to 1024 of them, as a data set keeps them (``NDArrayField``).
    teacher_classes : int64 or int32 (samples, kept)
        Their classes.  Entries with a class below 0, or a logit of -inf, are none: samples may have fewer than others.  The shares of a class
        that comes more than once add up.  A sample without entries has no loss against the teacher; one with a class above the last one a
        loss and gradient of NaN.
    labels, mixed, label_smoothing
        For the cross entropy, with a ``hard_weight`` above 0; see :func:`cross_entropy_with_grad`.
    temperature : float
        Of both softmaxes, not of the cross entropy.
    hard_weight : float
        Share of the cross entropy.
    ignore_index : int
        Samples with this label count for nothing, whatever the ``hard_weight``.
    reduction : 'mean', 'sum' or 'none'
        With 'none' the loss is a value per sample, and the gradient that of their sum.
    grad_scale : float
        Factor of the gradient, applied before it is rounded to the logits' type: with float16 logits the loss scale.

    The loss is float32.  A sample whose logits are all -inf has loss and gradient 0.
    """
    call = _Call(logits, teacher_logits, teacher_classes, labels, mixed, temperature, hard_weight, label_smoothing, ignore_index, reduction)
    n = logits.shape[0]
    loss, grad = ch.empty(n + 1, dtype=ch.float32, device=logits.device), N.new_like(call.logits)
    at = loss.data_ptr()
    call.run(grad, at, 0 if reduction == 'none' else at + 4 * n, scale=grad_scale)
    return loss[:n] if reduction == 'none' else loss[n], grad


class _Distillation(ch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call, reduction):
        n = logits.shape[0]
        ctx.per_row = reduction == 'none'
        loss = ch.empty(n if ctx.per_row else (), dtype=ch.float32, device=logits.device)
        stats = ch.empty(4 * n if ctx.per_row else 5 * n, dtype=ch.float32, device=logits.device)
        if ctx.per_row:
            call.run(None, loss.data_ptr(), 0, stats)
        else:
            call.run(None, stats.data_ptr() + 16 * n, loss.data_ptr(), stats)
        ctx.save_for_backward(call.logits, call.teacher, call.classes, call.target, stats)
        call.logits = call.teacher = call.classes = call.target = None  # (autograd keeps them, and sees to it that nobody changes them)
        ctx.call = call
        return loss

    @staticmethod
    @ch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        call = ctx.call
        call.logits, call.teacher, call.classes, call.target, stats = ctx.saved_tensors
        grad = N.new_like(call.logits)
        call.run(grad, 0, 0, stats, upstream.float().contiguous(), ctx.per_row, True)
        call.logits = call.teacher = call.classes = call.target = None
        return grad, None, None


def distillation(logits, teacher_logits, teacher_classes, labels=None, *, mixed=None, temperature=1.0, hard_weight=0.0, label_smoothing=0.0,
                 ignore_index=None, reduction='mean'):
    """The loss as a function of the logits that autograd knows; see :func:`distillation_with_grad` for the arguments.
    The gradient is made in the backward pass, where a loss scale is known."""
    call = _Call(logits, teacher_logits, teacher_classes, labels, mixed, temperature, hard_weight, label_smoothing, ignore_index, reduction)
    return _Distillation.apply(call.logits, call, reduction)


class Distillation(ch.nn.Module):
    """:func:`distillation` of logits from a teacher's largest ones, with class labels, the ``[label, label of the sample mixed in,
    lambda]`` rows of ``LabelMixup``, or without (``hard_weight=0``)."""

    def __init__(self, temperature=1.0, hard_weight=0.0, label_smoothing=0.0, ignore_index=None, reduction='mean'):
        super().__init__()
        self.temperature, self.hard_weight, self.label_smoothing = temperature, hard_weight, label_smoothing
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, logits, teacher_logits, teacher_classes, target=None):
        how = dict(temperature=self.temperature, hard_weight=self.hard_weight, label_smoothing=self.label_smoothing, reduction=self.reduction)
        if target is None or target.is_floating_point():
            return distillation(logits, teacher_logits, teacher_classes, mixed=target, **how)
        return distillation(logits, teacher_logits, teacher_classes, target, ignore_index=self.ignore_index, **how)
