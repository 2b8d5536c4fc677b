"""Distillation from a teacher's top logits (aidet_amd.distill, obb_topk_distill_*): refusals on the CPU, values and
gradients on the GPU against a plain implementation in 64 bits.

Tolerances, u = 2^-24.  exp2 of an argument a is good to (|a| + 4) u relative: a is a product of fp32 numbers (three roundings) and
the function itself.  Terms that carry a sum have |a| <= A = 1.4427 max|s - max| / T <= 60 here.  A sum of n positive terms
in fp32: each rounding at most u of the total, the partial sums of a lane, a wave and a workgroup: n / 256 + 16 of them.
So q and p are good to (A + n / 256 + 24) u relative, log p and log q to that absolutely plus 4 u of their size, a row's
loss to T^2 times their sum over p (which sums to 1); the gradient is rounded to the logits' type: eps / 2 of it.
"""
import ctypes

import pytest
import torch

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = 'cuda:0'


def reference(logits, values, indices, temp, weight):
    """row losses, gradient of their sum, allowed errors of both; in 64 bits"""
    s, t = logits.double(), values.double()
    classes = s.size(1)
    here = (indices >= 0) & (indices < classes)
    idx = indices.long().masked_fill(~here, 0)
    t = t.masked_fill(~here, -float('inf')) / temp
    some = (t > -float('inf')).any(1)
    w = torch.ones(s.size(0), dtype=torch.float64, device=s.device) if weight is None else weight.double()
    live = some & (w != 0)
    s = s.masked_fill(~live[:, None], 0.) / temp
    t = t.masked_fill(~live[:, None], 0.)
    log_p = t - torch.logsumexp(t, 1, keepdim=True)
    log_q = s - torch.logsumexp(s, 1, keepdim=True)
    p, q = log_p.exp(), log_q.exp()
    picked = log_q.gather(1, idx)
    term = torch.where(p > 0, p * (log_p - picked), torch.zeros_like(p))
    loss = temp ** 2 * w * term.sum(1)
    full = torch.zeros_like(s).scatter_add_(1, idx, p.masked_fill(~here, 0.))
    grad = temp * w[:, None] * (q - full)
    for v in (loss, grad):
        v[~live] = 0.
    finite = torch.where(s.isfinite(), s, torch.zeros_like(s))
    arg = 1.4427 * (finite.amax(1) - finite.amin(1)).clamp(max=90.)
    rel = (arg + classes / 256 + values.size(1) / 256 + 24) * U
    size = torch.where(p > 0, p * (log_p.abs() + picked.abs()), torch.zeros_like(p)).sum(1)
    tol_loss = temp ** 2 * w * (2 * rel + 8 * U + (rel + 8 * U) * size)
    tol_grad = temp * w[:, None] * (rel[:, None] + 8 * U) * (q + full) + torch.finfo(logits.dtype).eps / 2 * grad.abs()
    floor = 2.0 ** -24 if logits.dtype == torch.float16 else 2.0 ** -126
    return loss, grad, tol_loss, tol_grad + floor


def make(rows, classes, k, dtype, seed=0, noise=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = (torch.randn(rows, classes, generator=g, device=DEV) * 3).to(dtype)
    teacher = (logits.float() + noise * torch.randn(rows, classes, generator=g, device=DEV)).to(dtype)
    values, indices = teacher.topk(k, 1)
    return logits, values, indices


def check(logits, values, indices, temp=1.0, weight=None):
    from aidet_amd import topk_distill_loss
    want, grad, tol, tol_grad = reference(logits, values, indices, temp, weight)
    x = logits.detach().requires_grad_(True)
    got = topk_distill_loss(x, values, indices, temp, weight, 'none')
    assert got.dtype == torch.float32 and got.shape == (logits.size(0), )
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), (float(off.max()), int(off.argmax()))
    up = torch.linspace(0.5, 2., max(logits.size(0), 1), device=DEV)[:logits.size(0)]
    have, = torch.autograd.grad(got, x, up)
    f = up.double()[:, None]
    off = (have.double() - grad * f).abs() - (tol_grad * f + 4 * U * (grad * f).abs())
    assert have.dtype == logits.dtype and bool((off <= 0).all()), (float(off.max()), int(off.argmax()))
    # the scalar reductions: the same rows' losses, summed in a fixed order; their gradient: g scale of the rows'
    for reduction, factor, scale in (('sum', None, 1.), ('mean', None, 1. / max(logits.size(0), 1)), ('mean', 7.5, 1 / 7.5)):
        total = topk_distill_loss(x, values, indices, temp, weight, reduction, factor)
        assert total.shape == () and abs(float(total) - float(got.double().sum()) * scale) <= 4 * U * abs(float(total)) + 1e-30
        have, = torch.autograd.grad(2 * total, x)
        off = (have.double() - 2 * scale * grad).abs() - (2 * scale * (tol_grad + 4 * U * grad.abs())) - (2.0 ** -24 if logits.dtype == torch.float16 else 0)
        assert bool((off <= 0).all()), (reduction, float(off.max()))
    return got


# ---- refusals: no GPU ----------------------------------------------------------------------------------------------------
class _Cuda(torch.Tensor):
    """a CPU tensor that says it is on the GPU: what the wrapper checks before any device work"""
    is_cuda = True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def _idx(*shape, dtype=torch.int64):
    return _fake(*shape, dtype=dtype)


@pytest.mark.parametrize('args, kwargs, error', [
    (([1.], _fake(3, 2), _idx(3, 2)), {}, TypeError),
    ((torch.zeros(3, 4), _fake(3, 2), _idx(3, 2)), {}, NotImplementedError),
    ((_fake(3, 4, dtype=torch.float64), _fake(3, 2), _idx(3, 2)), {}, TypeError),
    ((_fake(3, 4), _idx(3, 2), _idx(3, 2)), {}, TypeError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2, dtype=torch.int16)), {}, TypeError),
    ((_fake(3, 4), _fake(2, 2), _idx(2, 2)), {}, ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 3)), {}, ValueError),
    ((_fake(3, 4), _fake(3, 1025), _idx(3, 1025)), {}, ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(temperature=0.), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(temperature=float('nan')), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(temperature=1e-7), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(temperature=float('inf')), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(weight=_fake(2)), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(weight=_idx(3)), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(weight=_fake(3).requires_grad_(True)), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(reduction='max'), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(reduction='sum', avg_factor=3.), ValueError),
    ((_fake(3, 4), _fake(3, 2), _idx(3, 2)), dict(avg_factor=0.), ValueError),
])
def test_wrapper_refusals(args, kwargs, error):
    from aidet_amd import topk_distill_loss
    with pytest.raises(error):
        topk_distill_loss(*args, **kwargs)


@pytest.mark.parametrize('device', ['cpu', pytest.param(DEV, marks=pytest.mark.gpu)])
def test_refuses_dual_tensors(device):
    """logits or weights that are dual tensors; the teacher's values are a constant in forward mode too"""
    import torch.autograd.forward_ad as fwad
    from aidet_amd import topk_distill_loss
    logits, values, weight = (torch.ones(*s, device=device) for s in ((3, 4), (3, 2), (3, )))
    indices = torch.arange(2, device=device).expand(3, 2)
    for grad in (True, False):
        with fwad.dual_level(), torch.set_grad_enabled(grad):
            def dual(t):
                return fwad.make_dual(t, torch.ones_like(t))
            for args in ((dual(logits), values, indices, 1., weight), (logits, values, indices, 1., dual(weight))):
                with pytest.raises(NotImplementedError, match='forward-mode'):
                    topk_distill_loss(*args)
            if device != 'cpu':
                assert torch.equal(topk_distill_loss(logits, dual(values), indices, 1., weight), topk_distill_loss(logits, values, indices, 1., weight))


def test_c_abi_refusals_without_gpu():
    from aidet_amd import _lib
    L = _lib.lib()
    one, null = ctypes.c_void_p(256), None     # (never dereferenced: validation fails first)

    def fwd(rows=3, classes=4, ld=4, dtype=0, k=2, vtype=0, ib=8, temp=1., s=one, row_loss=one):
        return L.obb_topk_distill_forward(s, ld, rows, classes, dtype, one, one, k, vtype, ib, temp, null, row_loss, null, 1., null, null, 0, null)
    for bad in (dict(rows=-1), dict(classes=-1), dict(k=1025), dict(dtype=3), dict(vtype=-1), dict(ib=2), dict(temp=0.),
                dict(temp=float('nan')), dict(temp=float('inf')), dict(ld=3), dict(s=null), dict(row_loss=null), dict(rows=1 << 31)):
        assert fwd(**bad) == _lib.OBB_EINVAL, bad
    assert fwd(rows=0) == _lib.OBB_OK
    b = L.obb_topk_distill_backward
    assert b(one, 4, 3, 4, 0, one, one, 2, 0, 8, 1., null, null, one, 0, 1., one, 4, null) == _lib.OBB_EINVAL      # no stats
    assert b(one, 4, 3, 4, 0, one, one, 2, 0, 8, 1., null, one, one, 2, 1., one, 4, null) == _lib.OBB_EINVAL       # grad_stride
    assert b(one, 4, 3, 4, 0, one, one, 2, 0, 8, 1., null, one, one, 0, 1., one, 3, null) == _lib.OBB_EINVAL       # pitch of dlogits
    assert b(null, 4, 0, 4, 0, null, null, 2, 0, 8, 1., null, null, null, 0, 1., null, 4, null) == _lib.OBB_OK


# ---- values and gradients --------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, classes, k', [(1, 1, 1), (3, 2, 1), (200, 16, 4), (7, 16, 16), (65, 33, 5), (130, 81, 20), (50, 1000, 64), (9, 1025, 256),
                                              (20, 4096, 7), (6, 8191, 100), (5, 20001, 32), (2, 131072, 1024), (1, 300007, 50)])
def test_sizes(rows, classes, k, dtype):
    check(*make(rows, classes, min(k, classes), dtype, seed=rows + classes))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('temp', [0.5, 1.0, 3.0, 8.0])
@pytest.mark.parametrize('rows, classes, k', [(100, 16, 3), (40, 1203, 50), (3, 70000, 40)])
def test_temperature_and_weights(rows, classes, k, temp, dtype):
    logits, values, indices = make(rows, classes, k, dtype, seed=1)
    g = torch.Generator(device=DEV).manual_seed(2)
    weight = torch.rand(rows, generator=g, device=DEV) * (torch.rand(rows, generator=g, device=DEV) < 0.7)
    check(logits, values, indices, temp, weight)


@pytest.mark.gpu
@pytest.mark.parametrize('rows, classes, k', [(40, 16, 4), (24, 500, 30), (3, 40000, 60)])
def test_absent_entries_empty_rows_and_zero_weights(rows, classes, k):
    """rows with fewer entries or none, indices outside the classes (with NaN and infinities in their values), rows of
    weight 0 and empty rows full of NaN"""
    for dtype in TYPES:
        logits, values, indices = make(rows, classes, k, dtype, seed=3)
        values = values.clone()
        have = torch.arange(rows, device=DEV) % (k + 1)
        absent = torch.arange(k, device=DEV) >= have[:, None]
        indices = torch.where(absent, torch.full_like(indices, -1), indices)
        indices[absent & (torch.arange(k, device=DEV) % 3 == 1)] = classes
        indices[absent & (torch.arange(k, device=DEV) % 3 == 2)] = 1 << 40
        values[absent] = float('nan')
        values[absent & (torch.arange(k, device=DEV) % 2 == 1)] = float('inf')
        weight = torch.ones(rows, device=DEV)
        weight[1] = 0.
        logits = logits.clone()
        logits[0] = float('nan')          # no entry at all
        logits[1] = float('nan')          # weight 0
        got = check(logits, values, indices, 2.0, weight)
        assert float(got[0]) == 0. and float(got[1]) == 0.
        # every entry -inf: a row without a distribution
        values[2:] = -float('inf')
        assert not check(logits, values, indices, 2.0, weight).any()


@pytest.mark.gpu
@pytest.mark.parametrize('rows, classes, k', [(12, 16, 5), (6, 600, 40), (2, 50000, 70)])
def test_masked_logits_and_masked_teacher(rows, classes, k):
    """-inf and the type's lowest value in either side's masked places; -inf under an entry is an infinite loss"""
    from aidet_amd import topk_distill_loss
    for dtype in TYPES:
        for low in (-float('inf'), torch.finfo(dtype).min):
            logits, values, indices = make(rows, classes, k, dtype, seed=4)
            keep = torch.zeros(rows, classes, dtype=torch.bool, device=DEV).scatter_(1, indices, True)
            mask = (torch.arange(classes, device=DEV) % 3 == 0)[None] & ~keep
            logits = logits.masked_fill(mask, low)
            values = values.clone()
            values[:, k // 2] = low                       # p = 0
            check(logits, values, indices)
            logits[0, indices[0, k // 2]] = -float('inf')  # q = 0 where p = 0: nothing
            check(logits, values, indices)
        logits[0, indices[0, 0]] = -float('inf')           # q = 0 where p > 0
        x = logits.detach().requires_grad_(True)
        loss = topk_distill_loss(x, values, indices, reduction='none')
        assert float(loss[0]) == float('inf') and bool(loss[1:].isfinite().all())
        grad, = torch.autograd.grad(loss, x, torch.ones_like(loss))
        assert bool(grad.isfinite().all())
        logits[0] = -float('inf')                          # no class left: NaN, as log_softmax, in this row alone
        loss = topk_distill_loss(logits, values, indices, reduction='none')
        assert bool(loss[0].isnan()) and bool(loss[1:].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize('rows, classes, k', [(7, 13, 5), (5, 200, 9), (4, 1021, 9), (4, 3001, 9), (2, 66001, 20)])
def test_nan_stays_in_its_row(rows, classes, k):
    """a NaN logit -- also where every other one is -inf -- makes its row NaN and no other"""
    from aidet_amd import topk_distill_loss
    for dtype in TYPES:
        logits, values, indices = make(rows, classes, k, dtype, seed=12)
        want = topk_distill_loss(logits, values, indices, reduction='none')
        for fill in (None, -float('inf')):
            for at in (0, classes // 2, classes - 1):
                x = logits.clone()
                if fill is not None:
                    x[1] = fill
                x[1, at] = float('nan')
                x.requires_grad_(True)
                got = topk_distill_loss(x, values, indices, reduction='none')
                assert bool(got[1].isnan()) and torch.equal(got[[0] + list(range(2, rows))], want[[0] + list(range(2, rows))])
                grad, = torch.autograd.grad(got, x, torch.ones_like(got))
                assert bool(grad[1].isnan().all()) and bool(grad[0].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize('rows, classes, k', [(10, 16, 6), (5, 3000, 50), (2, 66000, 64)])
def test_same_index_twice(rows, classes, k):
    for dtype in TYPES:
        logits, values, indices = make(rows, classes, k, dtype, seed=5)
        indices = indices.clone()
        indices[:, 1::2] = indices[:, 0::2][:, :indices[:, 1::2].size(1)]
        check(logits, values, indices)
        check(logits, values, torch.zeros_like(indices))
        check(logits, values.float(), indices.int())


@pytest.mark.gpu
def test_layouts():
    from aidet_amd import topk_distill_loss
    for rows, classes, k in ((20, 17, 4), (6, 2049, 9), (2, 40001, 33)):
        for dtype in TYPES:
            logits, values, indices = make(rows, classes, k, dtype, seed=6)
            want = check(logits, values, indices)
            for pad, start in ((8, 0), (8, 8), (3, 1)):
                wide = torch.full((rows, classes + pad + start), float('nan'), dtype=dtype, device=DEV)
                wide[:, start:start + classes] = logits
                check(wide[:, start:start + classes], values, indices)
            assert torch.equal(topk_distill_loss(logits.t().contiguous().t(), values, indices, reduction='none'), want)
            got = topk_distill_loss(logits.view(1, rows, classes), values.t().contiguous().t().view(1, rows, k), indices.view(1, rows, k), reduction='none')
            assert torch.equal(got, want[None])
            one = topk_distill_loss(logits[0], values[0], indices[0])
            assert one.shape == () and abs(float(one) - float(want[0])) <= 4 * U * abs(float(want[0]))


@pytest.mark.gpu
def test_empty_sizes():
    from aidet_amd import topk_distill_loss
    x = torch.zeros(0, 5, device=DEV, requires_grad=True)
    v, i = torch.zeros(0, 2, device=DEV), torch.zeros(0, 2, dtype=torch.int64, device=DEV)
    loss = topk_distill_loss(x, v, i)
    assert float(loss) == 0. and torch.autograd.grad(loss, x)[0].shape == (0, 5)
    assert topk_distill_loss(x, v, i, reduction='none').shape == (0, )
    x = torch.randn(3, 5, device=DEV, requires_grad=True)
    loss = topk_distill_loss(x, torch.zeros(3, 0, device=DEV), torch.zeros(3, 0, dtype=torch.int64, device=DEV))
    assert float(loss) == 0. and not torch.autograd.grad(loss, x)[0].any()


@pytest.mark.gpu
def test_rows_past_32_bits():
    """logits whose last rows begin past 2^32 bytes (and 2^31 elements): those rows alone give the same bits"""
    from aidet_amd import topk_distill_loss
    rows, classes = 9, 1 << 28
    logits = torch.zeros(rows, classes, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(7)
    logits[-1] = torch.randn(classes, generator=g, device=DEV).to(torch.bfloat16)
    values = torch.randn(rows, 6, generator=g, device=DEV)
    indices = torch.randint(0, classes, (rows, 6), generator=g, device=DEV)
    x = logits.requires_grad_(True)
    loss = topk_distill_loss(x, values, indices, reduction='none')
    y = logits.detach()[-1:].clone().requires_grad_(True)
    alone = topk_distill_loss(y, values[-1:], indices[-1:], reduction='none')
    assert abs(float(loss[-1]) - float(alone)) <= 64 * U * abs(float(alone))
    up = torch.zeros(rows, device=DEV)
    up[-1] = 1e6
    grad, = torch.autograd.grad(loss, x, up)
    want, = torch.autograd.grad(alone, y, up[-1:])
    assert not grad[:-1].any()
    assert float((grad[-1:].float() - want.float()).abs().max()) <= 2.0 ** -8 * float(want.float().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize('rows, classes, k', [((1 << 28) + 17, 2, 1), ((1 << 24) + 17, 65, 257)])
def test_more_rows_than_a_launch_holds(rows, classes, k):
    """a launch has fewer than 2^32 threads, 16 or 256 of them a row here: every row is served, with the bits of a small call"""
    from aidet_amd import topk_distill_loss
    g = torch.Generator(device=DEV).manual_seed(47)
    logits = torch.empty(rows, classes, device=DEV, dtype=torch.float16)
    few = torch.randn(1 << 16, classes, generator=g, device=DEV).half()
    for r in range(0, rows, 1 << 16):                       # (rows repeat: 2^16 different ones, and a shift)
        logits[r:r + (1 << 16)] = few[:rows - r]
    values = torch.randn(1, k, generator=g, device=DEV).half().expand(rows, k)
    indices = (torch.arange(k, device=DEV, dtype=torch.int32) % classes).expand(rows, k).contiguous()
    logits.requires_grad_(True)
    loss = topk_distill_loss(logits, values, indices, reduction='none')
    grad, = torch.autograd.grad(loss, logits, torch.ones_like(loss))
    want = topk_distill_loss(few, values[:1 << 16], indices[:1 << 16], reduction='none')
    want_grad, = torch.autograd.grad(topk_distill_loss(few.requires_grad_(True), values[:1 << 16], indices[:1 << 16], reduction='sum'), few)
    for r in range(0, rows, 1 << 16):
        n = min(1 << 16, rows - r)
        assert torch.equal(loss[r:r + n], want[:n]) and torch.equal(grad[r:r + n], want_grad[:n]), r


@pytest.mark.gpu
def test_long_rows_behind_the_last_full_launch():
    """a call of more rows than one launch takes whose last launch has few of them, long enough to be cut into parts if they were a
    call of their own: 137 GB of logits, losses only"""
    from aidet_amd import topk_distill_loss
    rows, classes = (1 << 23) + 17, 8192
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip('needs 160 GB of free memory')
    g = torch.Generator(device=DEV).manual_seed(53)
    few = torch.randn(256, classes, generator=g, device=DEV).half()
    logits = torch.empty(rows, classes, device=DEV, dtype=torch.float16)
    logits[:1 << 23].view(-1, 256, classes).copy_(few)
    logits[1 << 23:] = few[:17]
    values, indices = few.float().topk(2, 1)
    values, indices = values.repeat(1 << 15, 1), indices.int().repeat(1 << 15, 1)
    values, indices = torch.cat([values, values[:17]]), torch.cat([indices, indices[:17]])
    loss = topk_distill_loss(logits, values, indices, reduction='none')
    del logits
    torch.cuda.empty_cache()
    want, _, tol, _ = reference(few, values[:256], indices[:256], 1., None)
    for part in (loss[:1 << 23].view(-1, 256), loss[1 << 23:][None]):
        n = part.size(1)
        assert bool(((part.double() - want[:n]).abs() <= tol[:n]).all())


@pytest.mark.gpu
def test_against_differences():
    """fp32 against central differences of the plain form in 64 bits (h = 1e-5: good to ~1e-9)"""
    for rows, classes, k in ((6, 16, 4), (4, 1500, 40)):
        logits, values, indices = make(rows, classes, k, torch.float32, seed=8)
        from aidet_amd import topk_distill_loss
        x = logits.detach().requires_grad_(True)
        grad, = torch.autograd.grad(topk_distill_loss(x, values, indices, 2.0, reduction='sum'), x)
        g = torch.Generator(device=DEV).manual_seed(9)
        for _ in range(4):
            d = torch.randn(rows, classes, generator=g, device=DEV).double()
            f = [reference(logits.double() + h * d, values, indices, 2.0, None)[0].sum() for h in (1e-5, -1e-5)]
            want, have = (f[0] - f[1]) / 2e-5, (grad.double() * d).sum()
            size = ((grad.double() * d) ** 2).sum().sqrt()
            assert abs(float(have - want)) <= 2e-5 * float(size) + 1e-6 * abs(float(want))


@pytest.mark.gpu
def test_same_bits_other_streams_and_replays():
    from aidet_amd import topk_distill_loss
    for rows, classes, k in ((300, 16, 4), (30, 1203, 100), (2, 200000, 64)):
        logits, values, indices = make(rows, classes, k, torch.bfloat16, seed=10)
        x = logits.clone().requires_grad_(True)

        def step():
            loss = topk_distill_loss(x, values, indices, 2.0)
            return loss.detach(), torch.autograd.grad(loss, x)[0]
        want = step()
        torch.cuda.synchronize()
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(step(), want))
        streams = [torch.cuda.Stream() for _ in range(3)]
        outs = []
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for o in outs for p, q in zip(o, want))
        with torch.cuda.stream(streams[0]):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for i in range(4):
            with torch.no_grad():
                x.copy_(logits.roll(i + 1, 1))
            want = step()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want)), i


@pytest.mark.gpu
def test_module_follows_the_losses_conventions():
    from aidet_amd import TopkDistillLoss, topk_distill_loss
    logits, values, indices = make(12, 16, 4, torch.float32, seed=11)
    m = TopkDistillLoss(temperature=2.0, loss_weight=0.25)
    w = torch.ones(12, device=DEV)
    assert torch.equal(m(logits, values, indices, w, avg_factor=5.), 0.25 * topk_distill_loss(logits, values, indices, 2.0, w, avg_factor=5.))
    assert m(logits, values, indices, reduction_override='none').shape == (12, )


@pytest.mark.parametrize('device', ['cpu', pytest.param(DEV, marks=pytest.mark.gpu)])
def test_avg_factor_of_unreduced_losses(device, monkeypatch):
    """heads pass avg_factor whatever the reduction: 'none' leaves the rows' losses as they are, as the reference's losses do"""
    from aidet_amd import TopkDistillLoss, topk_distill_loss, torch_ext
    args = [torch.randn(5, 7, device=device), torch.randn(5, 2, device=device), torch.arange(2, device=device).expand(5, 2).contiguous()]
    if device == 'cpu':
        class Ext:
            @staticmethod
            def topk_distill(logits, values, indices, temperature, weight, scale):
                return scale
        monkeypatch.setattr(torch_ext, 'ext', Ext)
        assert topk_distill_loss(*args, reduction='none', avg_factor=3.) == -1
        assert topk_distill_loss(*args, reduction='mean', avg_factor=4.) == 0.25
        return
    want = topk_distill_loss(*args, reduction='none')
    assert want.shape == (5, ) and torch.equal(topk_distill_loss(*args, reduction='none', avg_factor=3.), want)
    assert torch.equal(TopkDistillLoss(loss_weight=0.5)(*args, avg_factor=3., reduction_override='none'), 0.5 * want)
    with pytest.raises(ValueError):
        topk_distill_loss(*args, reduction='sum', avg_factor=3.)


@pytest.mark.gpu
@pytest.mark.parametrize('rows, classes, k', [(1, 1, 1), (1, 9, 1), (4, 1, 1), (5, 9, 2)])
def test_tensors_with_the_negative_bit(rows, classes, k):
    """float tensors that are the imaginary part of a conjugate, at sizes at which they pass for contiguous ones and at others"""
    from aidet_amd import topk_distill_loss

    def pair(*shape):
        t = torch.view_as_complex(torch.randn(*shape, 2, device=DEV)).conj().imag
        assert t.is_neg()
        return t, t.clone().resolve_neg()
    torch.manual_seed(4)
    inputs = [pair(rows, classes), pair(rows, k), pair(rows), pair(rows)]
    indices = torch.arange(k, device=DEV).expand(rows, k).contiguous()
    results = []
    for logits, values, weight, up in zip(*inputs):
        logits = logits.detach().requires_grad_(True)
        loss = topk_distill_loss(logits, values, indices, 1., weight, 'none')
        results.append((loss.detach(), torch.autograd.grad(loss, logits, up)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_a_head_learns_from_a_teachers_top_logits():
    """FC trunk, class logits, loss and gradients together: against the same chain in 64 bits.  Whole steps of fp32: the
    trunk's and the loss's errors (at most 1e-5 relative each at these sizes, by the tolerances of their own tests) pass
    through sums of independent signs: 1e-4 of a gradient's largest value is allowed"""
    from aidet_amd import FusedLinear, topk_distill_loss
    torch.manual_seed(0)
    trunk = torch.nn.ModuleList([FusedLinear(12 * 49, 96, act='gelu'), FusedLinear(96, 96, act='gelu')]).to(DEV)
    cls = FusedLinear(96, 16).to(DEV)
    feats = torch.randn(70, 12, 7, 7, device=DEV)
    teacher = torch.randn(70, 16, device=DEV) * 2
    values, indices = teacher.topk(4, 1)
    h = feats.flatten(1)
    for fc in trunk:
        h = fc(h)
    params = list(trunk.parameters()) + list(cls.parameters())
    loss = topk_distill_loss(cls(h), values, indices, 2.0)
    grads = torch.autograd.grad(loss, params)
    p64 = [p.detach().double().requires_grad_(True) for p in params]
    h = feats.flatten(1).double()
    for i in (0, 2):
        h = torch.nn.functional.gelu(h @ p64[i].t() + p64[i + 1])
    log_q = torch.log_softmax((h @ p64[4].t() + p64[5]) / 2, 1).gather(1, indices)
    log_p = torch.log_softmax(values.double() / 2, 1)
    want = 4 * (log_p.exp() * (log_p - log_q)).sum(1).mean()
    assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
    for g, v in zip(grads, torch.autograd.grad(want, p64)):
        assert float((g.double() - v).abs().max()) <= 1e-4 * float(v.abs().max())
