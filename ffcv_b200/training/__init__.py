"""Operators of the training step that the loader's batches go into: losses for mixed labels, for a linear layer's
outputs that are not kept and for a teacher's logits, the norms and residual joins of a network's blocks, the group
norm of convolutions with its activation, positions of image patches, and the optimizer.  No counterpart in the
reference, whose work ends with the batch.

Every operator is a hand-written kernel behind a call of ``libffcv_b200.so`` and runs on the current stream of its
tensors' device; there is no CPU form.
"""
from .adamw import AdamW
from .cross_entropy import MixupCrossEntropy, cross_entropy, cross_entropy_with_grad
from .distillation import Distillation, distillation, distillation_with_grad
from .group_norm import GroupNormAct, group_norm_act, group_norm_act_backward, group_norm_act_forward
from .linear_cross_entropy import LinearCrossEntropy, linear_cross_entropy, linear_cross_entropy_with_grad
from .norm_residual import NormResidual, norm_residual, norm_residual_backward, norm_residual_forward
from .rotary import RotaryPositions, patch_positions

__all__ = ['AdamW', 'MixupCrossEntropy', 'cross_entropy', 'cross_entropy_with_grad', 'Distillation', 'distillation',
           'distillation_with_grad', 'GroupNormAct', 'group_norm_act', 'group_norm_act_forward', 'group_norm_act_backward',
           'LinearCrossEntropy', 'linear_cross_entropy', 'linear_cross_entropy_with_grad', 'NormResidual', 'norm_residual',
           'norm_residual_forward', 'norm_residual_backward', 'RotaryPositions', 'patch_positions']
