"""Distillation of class logits from a teacher's top logits, one HIP kernel a direction.

The hard labels of a head's sampled RoIs come from ``rbbox_target`` (mmdet/core/rbbox/rbbox_target.py:8-93); this is the
soft side: for every RoI the teacher's k best class logits and their indices, however many classes there are.  Reduction
and ``avg_factor`` as in the reference's losses (mmdet/models/losses/utils.py).  Compute: ``obb_topk_distill_*``
(include/obbops.h) behind the autograd node of aidet_amd/csrc/obbops_torch_train.cpp; fp32 whatever the type of the logits; the same bits on every run.
"""
from torch import nn

from . import torch_ext


def topk_distill_loss(logits, teacher_values, teacher_indices, temperature=1.0, weight=None, reduction='mean',
                      avg_factor=None):
    """``weight * T^2 * KL(softmax(teacher / T) || softmax(logits / T))`` per row, the teacher's distribution being over
    its k entries (renormalised), the student's over all classes.

    Args:
        logits (Tensor): (..., C) student logits, float32 / bfloat16 / float16; rows may have any pitch
        teacher_values (Tensor): (..., k) teacher logits, a constant (no gradient); k <= 1024
        teacher_indices (Tensor): (..., k) int64 / int32 classes; an index outside [0, C) marks an absent entry, an index
            that comes twice counts twice
        temperature (float): T, from 1e-6 to 1e6
        weight (Tensor, optional): (...) weight per row, a constant
        reduction (str): 'none' | 'mean' | 'sum'
        avg_factor (float, optional): with 'mean', the sum is divided by it instead of by the number of rows ('none' is not
            touched by it, 'sum' refuses it)

    Returns:
        fp32: the rows' losses (...) or a scalar (0 where there are no rows).  A row without an entry and a row of weight
        0 have loss and gradient 0, whatever their logits hold.

    TypeError: a type that is not served; ValueError: shapes or numbers that do not fit, a weight that wants a gradient;
    NotImplementedError: a tensor that is not on a HIP device, dual logits or weights (there is no forward-mode derivative).
    """
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError('temperature must lie in [1e-6, 1e6], but got {}'.format(temperature))
    if reduction not in ('none', 'mean', 'sum'):
        raise ValueError("reduction must be 'none', 'mean' or 'sum', but got {!r}".format(reduction))
    scale = -1. if reduction == 'none' else 1.
    if avg_factor is not None:
        if reduction == 'sum':
            raise ValueError("avg_factor goes with reduction='mean'")
        if not float(avg_factor) > 0:
            raise ValueError('avg_factor must be positive, but got {}'.format(avg_factor))
        if reduction == 'mean':
            scale = 1. / float(avg_factor)
    elif reduction == 'mean' and hasattr(logits, 'shape'):
        scale = 1. / max(logits.shape[:-1].numel(), 1)
    return torch_ext.ext().topk_distill(logits, teacher_values, teacher_indices, temperature, weight, scale)


class TopkDistillLoss(nn.Module):
    """``loss_weight * topk_distill_loss`` with the construction and call conventions of the reference's losses
    (mmdet/models/losses/cross_entropy_loss.py)."""

    def __init__(self, temperature=1.0, reduction='mean', loss_weight=1.0):
        super(TopkDistillLoss, self).__init__()
        self.temperature = temperature
        self.reduction = reduction
        self.loss_weight = loss_weight

    def forward(self, logits, teacher_values, teacher_indices, weight=None, avg_factor=None, reduction_override=None):
        assert reduction_override in (None, 'none', 'mean', 'sum')
        reduction = reduction_override if reduction_override else self.reduction
        return self.loss_weight * topk_distill_loss(logits, teacher_values, teacher_indices, self.temperature, weight,
                                                    reduction, avg_factor)
