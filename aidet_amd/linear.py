"""Fused linear layer: ``act(x @ weight.T + bias + residual)`` as one HIP kernel, with its gradients.

What the heads' FC trunks are made of (``nn.Linear`` + ``ReLU``, mmdet/models/bbox_heads/convfc_bbox_head.py:175-188,
rbbox_head.py:157-195) and, on channels-last maps, the 1 x 1 convolutions of a bottleneck with its shortcut and ReLU
(mmdet/models/backbones/resnet.py:101-125).  Compute: ``obb_linear_*`` (include/obbops.h).  fp32, bf16 and fp16 tensors;
products and sums in fp32, one rounding to the type at the end; the same bits on every run.
"""
import torch
from torch import nn
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib


def _rows(t, cols):
    """`t` (..., cols) as rows the kernels read in place: (tensor, row pitch); copied only where its last dimension is
    not contiguous or its rows overlap."""
    t = t.detach().reshape(t.shape[:-1].numel(), cols)
    if (cols > 1 and t.stride(1) != 1) or (t.size(0) > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t, max(t.stride(0), cols)


def _workspace(m, n, k, dtype, op, device):
    nbytes = _lib.lib().obb_linear_workspace_bytes(m, n, k, _lib.DTYPES[dtype], op)
    return (torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None), nbytes


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, residual, act, want_z):
    n, k = weight.shape
    y = torch.empty(x.shape[:-1] + (n, ), dtype=x.dtype, device=x.device)
    z = torch.empty(y.shape, dtype=torch.float32, device=x.device) if want_z else None
    if y.numel() == 0:
        return y, z
    with _lib.on_device(x.device):
        x2, ldx = _rows(x, k)
        w2, ldw = _rows(weight, k)
        res = bias1 = None
        ldr = 0
        if bias is not None:
            bias1 = bias.detach().contiguous()
        if residual is not None:
            res = residual.detach().reshape(y.shape[:-1].numel(), n)
            if res.size(0) > 1 and res.stride(0) == 0 and (n == 1 or res.stride(1) == 1):
                ldr = 0                                     # (one row for all)
            else:
                res, ldr = _rows(res, n)
        m = x2.size(0)
        ws, nbytes = _workspace(m, n, k, x.dtype, _lib.LINEAR_FORWARD, x.device)
        _lib.check(_lib.lib().obb_linear_forward(
            x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(bias1), _ptr(res), ldr, m, n, k, _lib.DTYPES[x.dtype],
            _lib.ACTS[act], y.data_ptr(), _ptr(z), _ptr(ws), nbytes, _lib.stream_ptr(x.device)))
    return y, z


class FusedLinearFunction(Function):

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        # gelu and silu keep the pre-activation, in 32 bits: their slope is taken where the forward was; relu needs y only
        smooth = act in ('gelu', 'silu')
        y, z = _forward(x, weight, bias, residual, act, smooth)
        ctx.act = act
        ctx.save_for_backward(x, weight, z if smooth else (y if act == 'relu' else None))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        x, weight, kept = ctx.saved_tensors
        act = ctx.act
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        n, k = weight.shape
        m = x.shape[:-1].numel()
        dx = dw = db = dz = None
        L, code = _lib.lib(), _lib.DTYPES[x.dtype]
        with _lib.on_device(x.device):
            stream = _lib.stream_ptr(x.device)
            dy = grad_output.contiguous()
            dz = dy
            want_dz = act != 'none' and (need_x or need_w or need_r)
            if want_dz:
                dz = torch.empty_like(dy)
            if need_b:
                db = torch.empty(n, dtype=x.dtype, device=x.device)
            if want_dz or need_b:
                ws, nbytes = _workspace(m, n, k, x.dtype, _lib.LINEAR_ACT_BACKWARD, x.device) if need_b else (None, 0)
                _lib.check(L.obb_linear_act_backward(
                    dy.data_ptr(), _ptr(kept) if act == 'relu' else None, _ptr(kept) if act in ('gelu', 'silu') else None,
                    m, n, code, _lib.ACTS[act], dz.data_ptr() if want_dz else None, _ptr(db), _ptr(ws), nbytes, stream))
            if need_x:
                dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
                w2, ldw = _rows(weight, k)
                ws, nbytes = _workspace(m, n, k, x.dtype, _lib.LINEAR_BACKWARD_INPUT, x.device)
                _lib.check(L.obb_linear_backward_input(dz.data_ptr(), w2.data_ptr(), ldw, m, n, k, code, dx.data_ptr(), _ptr(ws),
                                                       nbytes, stream))
            if need_w:
                dw = torch.empty(n, k, dtype=x.dtype, device=x.device)
                x2, ldx = _rows(x, k)
                ws, nbytes = _workspace(m, n, k, x.dtype, _lib.LINEAR_BACKWARD_WEIGHT, x.device)
                _lib.check(L.obb_linear_backward_weight(dz.data_ptr(), x2.data_ptr(), ldx, m, n, k, code, dw.data_ptr(), _ptr(ws),
                                                        nbytes, stream))
        return dx, dw, db, (dz if need_r else None), None


def _check(x, weight, bias, residual, act):
    for name, t in (('x', x), ('weight', weight), ('bias', bias), ('residual', residual)):
        if not isinstance(t, torch.Tensor):
            if t is None and name in ('bias', 'residual'):
                continue
            raise TypeError('{} must be a Tensor, but got {}'.format(name, type(t)))
        if not t.is_cuda:
            raise NotImplementedError('fused_linear runs on a HIP device only ({} is on {})'.format(name, t.device))
        if t.dtype not in _lib.DTYPES or t.dtype != x.dtype:
            raise TypeError('fused_linear takes tensors of one type, float32, bfloat16 or float16: x is {}, {} is {}'.format(
                x.dtype, name, t.dtype))
        if t.device != x.device:
            raise ValueError('x is on {}, {} on {}'.format(x.device, name, t.device))
    if act not in _lib.ACTS:
        raise ValueError('act must be one of {}, but got {!r}'.format(sorted(_lib.ACTS), act))
    if weight.dim() != 2 or x.dim() < 1 or x.size(-1) != weight.size(1):
        raise ValueError('x must be (..., K) and weight (N, K): got {} and {}'.format(tuple(x.shape), tuple(weight.shape)))
    if bias is not None and tuple(bias.shape) != (weight.size(0), ):
        raise ValueError('bias must be ({},), but got {}'.format(weight.size(0), tuple(bias.shape)))
    if residual is not None and residual.shape != x.shape[:-1] + (weight.size(0), ):
        raise ValueError('residual must have the shape of the output, {}, but got {}'.format(
            tuple(x.shape[:-1]) + (weight.size(0), ), tuple(residual.shape)))


def fused_linear(x, weight, bias=None, residual=None, act='none'):
    """``act(x @ weight.T + bias + residual)``.

    Args:
        x (Tensor): (..., K); rows may have any pitch
        weight (Tensor): (N, K)
        bias (Tensor, optional): (N,)
        residual (Tensor, optional): (..., N), added BEFORE the activation (the shortcut of a bottleneck); an expanded
            row is read in place
        act (str): 'none' | 'relu' | 'gelu' (exact) | 'silu'

    All tensors are of one type: float32, bfloat16 or float16.  Differentiable once with respect to every tensor.
    """
    _check(x, weight, bias, residual, act)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return FusedLinearFunction.apply(x, weight, bias, residual, act)
    return _forward(x, weight, bias, residual, act, False)[0]


class FusedLinear(nn.Linear):
    """``nn.Linear`` (its construction, parameters and ``state_dict``) followed by `act`, one kernel; ``forward`` takes an
    optional residual that is added before the activation."""

    def __init__(self, in_features, out_features, bias=True, act='none'):
        super(FusedLinear, self).__init__(in_features, out_features, bias=bias)
        if act not in _lib.ACTS:
            raise ValueError('act must be one of {}, but got {!r}'.format(sorted(_lib.ACTS), act))
        self.act = act

    def forward(self, x, residual=None):
        return fused_linear(x, self.weight, self.bias, residual, self.act)

    def extra_repr(self):
        return super(FusedLinear, self).extra_repr() + ', act={}'.format(self.act)
