"""Fused linear layer: ``act(x @ weight.T + bias + residual)`` as one HIP kernel, with its gradients.

What the heads' FC trunks are made of (``nn.Linear`` + ``ReLU``, mmdet/models/bbox_heads/convfc_bbox_head.py:175-188,
rbbox_head.py:157-195) and, on channels-last maps, the 1 x 1 convolutions of a bottleneck with its shortcut and ReLU
(mmdet/models/backbones/resnet.py:101-125).  Compute: ``obb_linear_*`` (include/obbops.h) behind the autograd node of
aidet_amd/csrc/obbops_torch_train.cpp.  fp32, bf16 and fp16 tensors; products and sums in fp32, one rounding to the type at
the end; the same bits on every run.
"""
from torch import nn

from . import _lib, torch_ext


def _act_code(act):
    code = _lib.ACTS.get(act) if isinstance(act, str) else None
    if code is None:
        raise ValueError('act must be one of {}, but got {!r}'.format(sorted(_lib.ACTS), act))
    return code


def fused_linear(x, weight, bias=None, residual=None, act='none'):
    """``act(x @ weight.T + bias + residual)``.

    Args:
        x (Tensor): (..., K); rows may have any pitch
        weight (Tensor): (N, K)
        bias (Tensor, optional): (N,)
        residual (Tensor, optional): (..., N), added BEFORE the activation (the shortcut of a bottleneck); an expanded
            row is read in place
        act (str): 'none' | 'relu' | 'gelu' (exact) | 'silu'

    All tensors are of one type (float32, bfloat16 or float16) and on one HIP device; under ``torch.autocast`` they are cast
    to its type first, as those of ``torch.nn.functional.linear`` are.  Differentiable once with respect to
    every tensor.  TypeError: a type that is not served, or several; ValueError: shapes that do not fit, an unknown act;
    NotImplementedError: a tensor that is not on a HIP device, or a dual tensor (there is no forward-mode derivative).
    """
    return torch_ext.ext().fused_linear(x, weight, bias, residual, _act_code(act))


class FusedLinear(nn.Linear):
    """``nn.Linear`` (its construction, parameters and ``state_dict``) followed by `act`, one kernel; ``forward`` takes an
    optional residual that is added before the activation."""

    def __init__(self, in_features, out_features, bias=True, act='none'):
        super(FusedLinear, self).__init__(in_features, out_features, bias=bias)
        _act_code(act)
        self.act = act

    def forward(self, x, residual=None):
        return fused_linear(x, self.weight, self.bias, residual, self.act)

    def extra_repr(self):
        return super(FusedLinear, self).extra_repr() + ', act={}'.format(self.act)
