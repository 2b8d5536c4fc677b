"""Distillation of class logits from a teacher's top logits, one HIP kernel a direction.

The hard labels of a head's sampled RoIs come from ``rbbox_target`` (mmdet/core/rbbox/rbbox_target.py:8-93); this is the
soft side: for every RoI the teacher's k best class logits and their indices, however many classes there are.  Reduction
and ``avg_factor`` as in the reference's losses (mmdet/models/losses/utils.py).  Compute: ``obb_topk_distill_*``
(include/obbops.h); fp32 whatever the type of the logits; the same bits on every run.
"""
import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib


def _rows(t, cols):
    t = t.detach().reshape(t.shape[:-1].numel(), cols)
    if (cols > 1 and t.stride(1) != 1) or (t.size(0) > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, max(t.stride(0), cols)


def _ptr(t):
    return None if t is None else t.data_ptr()


class TopkDistillFunction(Function):

    @staticmethod
    def forward(ctx, logits, values, indices, weight, temperature, scale):
        """`scale`: None = the rows' losses, else scale * their sum."""
        classes, k = logits.size(-1), values.size(-1)
        dev = logits.device
        rows_shape = logits.shape[:-1]
        with _lib.on_device(dev):
            s, ld = _rows(logits, classes)
            v, i = values.detach().contiguous(), indices.contiguous()
            w = None if weight is None else weight.detach().to(torch.float32).contiguous()
            rows = rows_shape.numel()
            row_loss = torch.empty(rows_shape, dtype=torch.float32, device=dev)
            stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if logits.requires_grad else None
            total = None if scale is None else torch.empty((), dtype=torch.float32, device=dev)
            if rows > 0 or total is not None:
                nbytes = _lib.lib().obb_topk_distill_workspace_bytes(rows, classes)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
                _lib.check(_lib.lib().obb_topk_distill_forward(
                    s.data_ptr(), ld, rows, classes, _lib.DTYPES[s.dtype], v.data_ptr(), i.data_ptr(), k, _lib.DTYPES[v.dtype],
                    i.element_size(), temperature, _ptr(w), row_loss.data_ptr(), _ptr(stats), 1. if scale is None else scale,
                    _ptr(total), _ptr(ws), nbytes, _lib.stream_ptr(dev)))
        ctx.args = (temperature, scale)
        ctx.save_for_backward(logits, v, i, w, stats)
        return row_loss if scale is None else total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        logits, v, i, w, stats = ctx.saved_tensors
        temperature, scale = ctx.args
        classes, dev = logits.size(-1), logits.device
        with _lib.on_device(dev):
            d = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
            if d.numel() > 0:
                s, ld = _rows(logits, classes)
                g = grad.to(torch.float32).contiguous()
                _lib.check(_lib.lib().obb_topk_distill_backward(
                    s.data_ptr(), ld, s.size(0), classes, _lib.DTYPES[s.dtype], v.data_ptr(), i.data_ptr(), v.size(-1),
                    _lib.DTYPES[v.dtype], i.element_size(), temperature, _ptr(w), stats.data_ptr(), g.data_ptr(),
                    1 if scale is None else 0, 1. if scale is None else scale, d.data_ptr(), classes, _lib.stream_ptr(dev)))
        return d, None, None, None, None, None


def topk_distill_loss(logits, teacher_values, teacher_indices, temperature=1.0, weight=None, reduction='mean',
                      avg_factor=None):
    """``weight * T^2 * KL(softmax(teacher / T) || softmax(logits / T))`` per row, the teacher's distribution being over
    its k entries (renormalised), the student's over all classes.

    Args:
        logits (Tensor): (..., C) student logits, float32 / bfloat16 / float16; rows may have any pitch
        teacher_values (Tensor): (..., k) teacher logits, a constant (no gradient); k <= 1024
        teacher_indices (Tensor): (..., k) int64 / int32 classes; an index outside [0, C) marks an absent entry, an index
            that comes twice counts twice
        temperature (float): T > 0
        weight (Tensor, optional): (...) weight per row, a constant
        reduction (str): 'none' | 'mean' | 'sum'
        avg_factor (float, optional): with 'mean', the sum is divided by it instead of by the number of rows

    Returns:
        fp32: the rows' losses (...) or a scalar (0 where there are no rows).  A row without an entry and a row of weight
        0 have loss and gradient 0, whatever their logits hold.
    """
    for name, t in (('logits', logits), ('teacher_values', teacher_values), ('teacher_indices', teacher_indices),
                    ('weight', weight)):
        if not isinstance(t, torch.Tensor):
            if t is None and name == 'weight':
                continue
            raise TypeError('{} must be a Tensor, but got {}'.format(name, type(t)))
        if not t.is_cuda:
            raise NotImplementedError('topk_distill_loss runs on a HIP device only ({} is on {})'.format(name, t.device))
        if t.device != logits.device:
            raise ValueError('logits are on {}, {} on {}'.format(logits.device, name, t.device))
    if logits.dtype not in _lib.DTYPES or teacher_values.dtype not in _lib.DTYPES:
        raise TypeError('logits and teacher_values must be float32, bfloat16 or float16: got {} and {}'.format(
            logits.dtype, teacher_values.dtype))
    if teacher_indices.dtype not in (torch.int64, torch.int32):
        raise TypeError('teacher_indices must be int64 or int32, but got {}'.format(teacher_indices.dtype))
    if logits.dim() < 1 or teacher_values.dim() != logits.dim() or teacher_values.shape[:-1] != logits.shape[:-1] \
            or teacher_indices.shape != teacher_values.shape:
        raise ValueError('logits must be (..., C), teacher_values and teacher_indices (..., k): got {}, {} and {}'.format(
            tuple(logits.shape), tuple(teacher_values.shape), tuple(teacher_indices.shape)))
    if teacher_values.size(-1) > _lib.DISTILL_MAX_K:
        raise ValueError('at most {} teacher entries a row, but got {}'.format(_lib.DISTILL_MAX_K, teacher_values.size(-1)))
    if weight is not None:
        if weight.shape != logits.shape[:-1] or not weight.is_floating_point():
            raise ValueError('weight must be floating and {}, but got {} of {}'.format(
                tuple(logits.shape[:-1]), weight.dtype, tuple(weight.shape)))
        if weight.requires_grad:
            raise ValueError('weight is a constant: no gradient reaches it')
    temperature = float(temperature)
    if not 0. < temperature < 3e38:
        raise ValueError('temperature must be positive and finite, but got {}'.format(temperature))
    if reduction not in ('none', 'mean', 'sum'):
        raise ValueError("reduction must be 'none', 'mean' or 'sum', but got {!r}".format(reduction))
    scale = None if reduction == 'none' else 1.
    if avg_factor is not None:
        if reduction != 'mean':
            raise ValueError("avg_factor goes with reduction='mean'")
        if not float(avg_factor) > 0:
            raise ValueError('avg_factor must be positive, but got {}'.format(avg_factor))
        scale = 1. / float(avg_factor)
    elif reduction == 'mean':
        scale = 1. / max(logits.shape[:-1].numel(), 1)
    return TopkDistillFunction.apply(logits, teacher_values, teacher_indices, weight, temperature, scale)


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
