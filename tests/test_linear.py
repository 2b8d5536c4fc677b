"""Fused linear layer (aidet_amd.linear, obb_linear_*): refusals on the CPU, values and gradients on the GPU against a
plain implementation in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32; half a step of the output's type is eps / 2 relative.
* A sum of K products kept in fp32 makes at most K roundings of at most u times a partial sum; partial sums of terms with
  independent signs have the size s = sqrt(sum of the squared terms), and the roundings are independent too: their sum has
  a deviation below sqrt(K) u s.  8 of those are allowed, plus 8 u of every operand of the epilogue.
* |act'| <= 1.13 for every activation; the functions themselves are good to a few u.
* dz is rounded to the type once before the gradients' products: another eps / 2 of every term, independent: 4 times
  eps / 2 sqrt(sum of the squared terms).  act'' <= 0.8 brings the error of z into dz.
"""
import ctypes

import pytest
import torch

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEV = 'cuda:0'


def act64(z, act):
    if act == 'relu':
        return z.clamp(min=0)
    if act == 'gelu':
        return 0.5 * z * torch.erfc(-z / 2 ** 0.5)
    if act == 'silu':
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    if act == 'relu':
        return (z > 0).double()
    if act == 'gelu':
        return 0.5 * torch.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    if act == 'silu':
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def half_step(t):
    return torch.finfo(t).eps / 2


def product64(a, b):
    """a (M, K) @ b (K, N) in 64 bits, and the deviation's unit: sqrt of the sum of the squared terms."""
    a, b = a.double(), b.double()
    return a @ b, ((a * a) @ (b * b)).sqrt()


def summed(s, terms, more):
    """allowed error of fp32 sums of `terms` products, `more` = epilogue operands' size"""
    return 8 * (terms + 8) ** 0.5 * U * s + 8 * U * more


def tiny(t):
    return 2 * torch.finfo(t).tiny if t != torch.float16 else 2.0 ** -24     # (fp16: values below its normal range step by 2^-24)


def make(m, k, n, dtype, bias, residual, seed=0, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(m, k + pad, generator=g, device=DEV).to(dtype)[:, :k]
    w = (torch.randn(n, k, generator=g, device=DEV) * max(k, 1) ** -0.5).to(dtype)
    b = torch.randn(n, generator=g, device=DEV).to(dtype) if bias else None
    r = torch.randn(m, n, generator=g, device=DEV).to(dtype) if residual else None
    return x, w, b, r


def reference(x, w, b, r, act):
    """(y64, z64, allowed error of z, of y)"""
    z, s = product64(x, w.t())
    more = z.abs()
    for t in (b, r):
        if t is not None:
            z = z + t.double()
            more = more + t.double().abs()
    ez = summed(s, x.size(1), more)
    y = act64(z, act)
    return y, z, ez, 1.13 * ez + 4 * U * (y.abs() + z.abs()) + half_step(x.dtype) * y.abs() + tiny(x.dtype)


def check(x, w, b, r, act):
    from aidet_amd import fused_linear
    got = fused_linear(x, w, b, r, act)
    want, _, _, tol = reference(x.reshape(-1, x.size(-1)), w, b, None if r is None else r.reshape(-1, w.size(0)), act)
    assert got.dtype == x.dtype and got.shape == x.shape[:-1] + (w.size(0), )
    off = (got.reshape(want.shape).double() - want).abs() - tol
    assert bool((off <= 0).all()), (float(off.max()), int(off.argmax()))
    return got


# ---- refusals and host logic: no GPU ------------------------------------------------------------------------------------
def test_refuses_what_it_cannot_serve():
    from aidet_amd import FusedLinear, fused_linear
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    with pytest.raises(TypeError):
        fused_linear([[1.]], w)
    with pytest.raises(NotImplementedError):
        fused_linear(x, w)
    with pytest.raises(ValueError):
        FusedLinear(4, 5, act='tanh')
    m = FusedLinear(4, 5, act='silu')
    assert set(m.state_dict()) == {'weight', 'bias'} and 'act=silu' in repr(m)
    m.load_state_dict(torch.nn.Linear(4, 5).state_dict())


class _Cuda(torch.Tensor):
    """a CPU tensor that says it is on the GPU: what the wrapper checks before any device work"""
    is_cuda = True


def _fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


@pytest.mark.parametrize('args, error', [
    ((_fake(3, 4), _fake(5, 4, dtype=torch.float16)), TypeError),
    ((_fake(3, 4, dtype=torch.float64), _fake(5, 4, dtype=torch.float64)), TypeError),
    ((_fake(3, 4), _fake(5, 3)), ValueError),
    ((_fake(3, 4), _fake(5, 4, 1)), ValueError),
    ((_fake(3, 4), _fake(5, 4), _fake(4)), ValueError),
    ((_fake(3, 4), _fake(5, 4), _fake(5, 1)), ValueError),
    ((_fake(3, 4), _fake(5, 4), None, _fake(1, 5)), ValueError),
    ((_fake(3, 4), _fake(5, 4), None, None, 'tanh'), ValueError),
    ((_fake(3, 4), _fake(5, 4), torch.zeros(5)), NotImplementedError),
])
def test_wrapper_refusals(args, error):
    from aidet_amd import fused_linear
    with pytest.raises(error):
        fused_linear(*args)


def _dual_is_refused(device, match):
    """every argument a dual tensor in turn, with and without grad mode"""
    import torch.autograd.forward_ad as fwad
    from aidet_amd import fused_linear
    base = [torch.ones(*s, device=device) for s in ((3, 4), (5, 4), (5, ), (3, 5))]
    for i in range(4):
        for grad in (True, False):
            with fwad.dual_level(), torch.set_grad_enabled(grad):
                args = list(base)
                args[i] = fwad.make_dual(base[i], torch.ones_like(base[i]))
                with pytest.raises(NotImplementedError, match=match):
                    fused_linear(*args)


def test_refuses_dual_tensors():
    _dual_is_refused('cpu', 'forward-mode')


@pytest.mark.gpu
def test_refuses_dual_tensors_on_the_device():
    from aidet_amd import fused_linear
    _dual_is_refused(DEV, 'forward-mode')
    _dual_is_refused(DEV, 'fused_linear')
    x, w, b, _ = make(3, 4, 5, torch.float32, True, False)
    check(x, w, b, None, 'silu')                # (and afterwards it serves)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        _dual_is_refused(DEV, 'forward-mode')
        assert fused_linear(x, w).dtype == torch.bfloat16


def test_c_abi_refusals_without_gpu():
    from aidet_amd import _lib
    L = _lib.lib()
    one, null = ctypes.c_void_p(256), None     # (never dereferenced: validation fails first)
    f = L.obb_linear_forward
    assert f(one, 4, one, 4, null, null, 0, -1, 5, 4, 0, 0, one, null, null, 0, null) == _lib.OBB_EINVAL
    assert f(one, 4, one, 4, null, null, 0, 3, 5, 4, 9, 0, one, null, null, 0, null) == _lib.OBB_EINVAL
    assert f(one, 4, one, 4, null, null, 0, 3, 5, 4, 0, 7, one, null, null, 0, null) == _lib.OBB_EINVAL
    assert b'activation' in L.obb_last_error()
    assert f(one, 3, one, 4, null, null, 0, 3, 5, 4, 0, 0, one, null, null, 0, null) == _lib.OBB_EINVAL
    assert f(one, 4, one, 4, null, one, 3, 3, 5, 4, 0, 0, one, null, null, 0, null) == _lib.OBB_EINVAL
    assert b'pitch' in L.obb_last_error()
    assert f(null, 4, one, 4, null, null, 0, 3, 5, 4, 0, 0, one, null, null, 0, null) == _lib.OBB_EINVAL
    assert f(null, 4, null, 4, null, null, 0, 0, 5, 4, 0, 0, null, null, null, 0, null) == _lib.OBB_OK
    assert L.obb_linear_act_backward(one, null, null, 3, 5, 0, 1, one, null, null, 0, null) == _lib.OBB_EINVAL    # relu: no y
    assert L.obb_linear_act_backward(one, one, null, 3, 5, 0, 2, one, null, null, 0, null) == _lib.OBB_EINVAL     # gelu: no z
    assert L.obb_linear_act_backward(one, one, one, 3, 5, 0, 1, null, null, null, 0, null) == _lib.OBB_EINVAL
    assert L.obb_linear_act_backward(one, one, one, 3, 5, 0, 1, one, one, null, 0, null) == _lib.OBB_EWORKSPACE
    assert L.obb_linear_backward_input(one, one, 3, 3, 5, 4, 0, one, null, 0, null) == _lib.OBB_EINVAL
    assert L.obb_linear_backward_weight(one, null, 4, 3, 5, 4, 0, one, null, 0, null) == _lib.OBB_EINVAL
    assert L.obb_linear_backward_weight(one, one, 4, 3, 5, 4, 3, one, null, 0, null) == _lib.OBB_EINVAL
    assert L.obb_linear_workspace_bytes(-1, 5, 4, 0, 0) == 0


def test_c_abi_refuses_launches_past_the_limit():
    """a dimension of a launch has fewer than 2^32 threads: a call that would need more says so"""
    from aidet_amd import _lib
    L = _lib.lib()
    one, null, big = ctypes.c_void_p(256), None, 1 << 46     # (never dereferenced: refused before any launch)
    wide = (1 << 31) - 1
    for dtype in range(3):
        for rc in (L.obb_linear_forward(one, 8, one, 8, null, null, 0, 1 << 33, 64, 8, dtype, 0, one, null, one, big, null),
                   L.obb_linear_forward(one, 9, one, 9, null, null, 0, 40, wide, 9, dtype, 0, one, null, one, big, null),
                   L.obb_linear_backward_input(one, one, 64, 1 << 33, 8, 64, dtype, one, one, big, null),
                   L.obb_linear_backward_weight(one, one, 40, 8, wide, 40, dtype, one, one, big, null),
                   L.obb_linear_act_backward(one, one, null, 3, wide, dtype, 1, one, one, one, big, null)):
            assert rc == _lib.OBB_EINVAL and b'threads' in L.obb_last_error(), (dtype, rc, L.obb_last_error())


@pytest.mark.parametrize('op', range(4))
@pytest.mark.parametrize('dtype', range(3))
def test_workspaces_of_empty_sizes(op, dtype):
    """each size zero in turn and together: a number of bytes that an empty output or an empty sum needs"""
    from aidet_amd import _lib
    size = _lib.lib().obb_linear_workspace_bytes
    for m, n, k in ((0, 5, 8), (4, 0, 8), (4, 5, 0), (0, 0, 8), (0, 5, 0), (4, 0, 0), (0, 0, 0)):
        have = size(m, n, k, dtype, op)
        assert have == (256 if op == _lib.LINEAR_ACT_BACKWARD and n else 0), (m, n, k, have)


# ---- values --------------------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 64, 64), (2, 7, 3), (17, 33, 65), (64, 64, 64), (1, 4096, 1000), (5, 1024, 16), (63, 129, 257), (128, 256, 128),
         (200, 1000, 80), (257, 512, 255), (1000, 72, 40), (300, 2056, 520), (4097, 24, 8), (33, 12544, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m, k, n', SIZES)
def test_forward_sizes(m, k, n, dtype):
    x, w, b, r = make(m, k, n, dtype, True, True, seed=m + k + n)
    check(x, w, b, r, 'relu')
    check(x, w, None, None, 'none')


@pytest.fixture
def cut():
    """``cut(tile, splits)`` forces how products are cut (where that is possible); restored afterwards"""
    from aidet_amd import _lib

    def force(tile, splits):
        _lib.set_tuning(_lib.TUNE_LINEAR_TILE, tile)
        _lib.set_tuning(_lib.TUNE_LINEAR_SPLITS, splits)
    yield force
    force(-1, -1)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('tile', [256, 192, 128, 64])
@pytest.mark.parametrize('splits', [1, 2, 8])
def test_every_cut(tile, splits, dtype, cut):
    """each tile and number of splits on sizes that end inside tiles, slabs and splits, forward and gradients, aligned and not"""
    for m, k, n in ((300, 1096, 264), (300, 1001, 263), (40, 72, 24)):
        x, w, b, r = make(m, k, n, dtype, True, True, seed=tile + splits)
        dy = torch.randn(m, n, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).to(dtype)
        cut(tile, splits)
        check(x, w, b, r, 'relu')
        check_gradients(x, w, b, r, 'gelu', dy)


@pytest.mark.gpu
@pytest.mark.parametrize('forced', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m', [1, 2, 16, 17, 32, 33])
def test_few_rows(m, dtype, forced, cut):
    """rows up to 32 by one launch: K of one element, that ends inside a chunk, a block and a wave's share; odd N and pitches"""
    from aidet_amd import fused_linear
    if forced:
        cut(16, 1)
    for k, n, pad in ((1024, 1024, 0), (1, 17, 0), (3, 5, 0), (7, 40, 1), (8, 16, 0), (255, 31, 1), (256, 33, 0), (257, 100, 3), (1001, 1023, 3),
                      (2047, 65, 1), (2048, 64, 0), (4100, 20, 4)):
        x, w, b, r = make(m, k, n, dtype, True, True, seed=m + k, pad=pad)
        check(x, w, b, r, 'gelu')
        check(x, w, None, None, 'relu')
    x, w, b, _ = make(m, 0, 50, dtype, True, False)
    assert torch.equal(fused_linear(x, w, b, None, 'silu'), fused_linear(x.new_zeros(m, 1), w.new_zeros(50, 1), b, None, 'silu'))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_few_rows_keep_infinities_and_nans_to_their_rows(dtype):
    """a NaN or an infinity in a row of x or of w reaches that row or column alone, at the end of K too, and nothing outside K is read into a sum"""
    from aidet_amd import fused_linear
    k, n = 1000, 500
    x, w, _, _ = make(5, k + 24, n, dtype, False, False, seed=3)
    w = torch.cat([w[:, :k], torch.full((n, 24), float('nan'), device=DEV, dtype=dtype)], 1)[:, :k]     # (NaN behind every row)
    x = torch.cat([x[:, :k], torch.full((5, 24), float('inf'), device=DEV, dtype=dtype)], 1)[:, :k]
    want = check(x, w, None, None, 'none')
    x2, w2 = x.clone(), w.clone()
    x2[1, k - 1], x2[3, 0], w2[7, k - 1] = float('nan'), float('inf'), float('nan')
    y = fused_linear(x2, w2)
    assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[:, 7]).all())
    assert not bool(torch.isfinite(y[3]).any())
    keep = [0, 2, 4]
    cols = [c for c in range(n) if c != 7]
    assert torch.equal(y[keep][:, cols], want[keep][:, cols])


@pytest.mark.gpu
@pytest.mark.parametrize('m, k, n', [(4096, 128, 4352), (4000, 200, 4360), (2300, 192, 8200), (4104, 72, 4360)])
def test_more_tiles_than_the_device_holds(m, k, n, cut):
    """a workgroup takes several tiles one after the other, whole ones and ones that end inside, with few slabs each"""
    cut(256, 1)
    for dtype in TYPES[1:]:
        x, w, b, r = make(m, k, n, dtype, True, True, seed=19)
        check(x, w, b, r, 'silu')
        check(x, w, None, None, 'none')
        x, w, b, _ = make(n, k, m, dtype, True, False, seed=20)
        dy = torch.randn(n, m, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).to(dtype)
        check_gradients(x, w, b, None, 'gelu', dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['none', 'relu', 'gelu', 'silu'])
@pytest.mark.parametrize('bias, residual', [(False, False), (True, False), (False, True), (True, True)])
def test_forward_epilogue(act, bias, residual, dtype):
    x, w, b, r = make(150, 200, 136, dtype, bias, residual, seed=3)
    check(x, w, b, r, act)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m, n', [(3, 512), (300, 256)])
def test_forward_layouts(m, n, dtype):
    """rows of a wider buffer, unaligned starts, transposed storage, leading dimensions, an expanded residual"""
    k = 320
    x, w, b, r = make(m, k, n, dtype, True, True, seed=5)
    want = check(x, w, b, r, 'silu')
    from aidet_amd import fused_linear
    for pad, start in ((8, 0), (8, 8), (1, 0), (5, 3), (3, 1)):
        wide = torch.full((m, k + start + pad), float('nan'), dtype=dtype, device=DEV)
        wide[:, start:start + k] = x
        wide_w = torch.full((n, k + start + pad), float('nan'), dtype=dtype, device=DEV)
        wide_w[:, start:start + k] = w
        wide_r = torch.full((m, n + start + pad), float('nan'), dtype=dtype, device=DEV)
        wide_r[:, start:start + n] = r
        got = check(wide[:, start:start + k], wide_w[:, start:start + k], b, wide_r[:, start:start + n], 'silu')
        assert got.is_contiguous()
    assert torch.equal(fused_linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r, 'silu'), want)
    assert torch.equal(fused_linear(x.view(1, m, k), w, b, r.view(1, m, n), 'silu'), want[None])
    row = r[:1].expand(m, n)
    assert torch.equal(fused_linear(x, w, b, row, 'silu'), fused_linear(x, w, b, row.contiguous(), 'silu'))
    one = fused_linear(x[0], w, b, r[0], 'silu')
    assert one.shape == (n, ) and torch.equal(one, fused_linear(x[:1], w, b, r[:1], 'silu')[0])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_empty_sizes(dtype):
    from aidet_amd import fused_linear
    x, w, b, r = make(0, 8, 5, dtype, True, True)
    assert fused_linear(x, w, b, r, 'relu').shape == (0, 5)
    x, w, b, r = make(4, 0, 5, dtype, True, True)
    assert torch.equal(fused_linear(x, w, b, r, 'none'), (b.float() + r.float()).to(dtype))
    x, w, b, r = make(4, 8, 0, dtype, True, True)
    assert fused_linear(x, w, b, r, 'relu').shape == (4, 0)
    # gradients of an empty batch: zeros for what is there
    x, w, b, _ = make(0, 8, 5, dtype, True, False)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(fused_linear(*leaves, act='gelu').float().sum(), leaves)
    assert dx.shape == (0, 8) and not dw.any() and not db.any() and dw.shape == w.shape


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['none', 'relu', 'gelu', 'silu'])
@pytest.mark.parametrize('m, k, n', [(4, 8, 0), (4, 0, 5), (0, 8, 5), (0, 0, 5), (4, 0, 0), (0, 8, 0), (0, 0, 0)])
def test_gradients_of_empty_sizes(m, k, n, act, dtype):
    """every gradient has its tensor's shape: zeros where nothing is summed, with no terms in the product dz alone remains"""
    x, w, b, r = make(m, k, n, dtype, True, True, seed=2)
    dy = torch.ones(m, n, device=DEV, dtype=dtype)
    dx, dw, db, dr = gradients(x, w, b, r, act, dy)
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape and dr.shape == r.shape
    assert not dx.any() if n == 0 else True
    assert not dw.any()
    if m and n:
        check_gradients(x, w, b, r, act, dy)
    else:
        assert not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m', [2, 150])
def test_infinities_and_nans_stay_in_their_rows(m, dtype):
    """IEEE: an infinite or NaN input reaches its row's (weight: its column's) outputs and no other"""
    from aidet_amd import fused_linear
    k, n = 264, 200
    x, w, b, _ = make(m, k, n, dtype, True, False, seed=8)
    clean = fused_linear(x, w, b)
    x2, w2 = x.clone(), w.clone()
    x2[1, 5] = float('inf')
    w2[7] = 0
    got = fused_linear(x2, w2, b)
    want = x2.double() @ w2.double().t() + b.double()     # (+-inf by the weight's sign; NaN at the zero weights)
    assert torch.equal(got[1].isnan(), want[1].isnan()) and torch.equal(got[1].isinf(), want[1].isinf())
    assert torch.equal(got[1][got[1].isinf()].double(), want[1][want[1].isinf()])
    others = [c for c in range(n) if c != 7]
    assert torch.equal(got[0][others], clean[0][others]) and bool((got[0, 7] == b[7]))
    x2[1, 5] = float('nan')
    got = fused_linear(x2, w, b)
    assert bool(got[1].isnan().all()) and torch.equal(got[0], clean[0])
    w2 = w.clone()
    w2[3, 2] = -float('inf')
    got = fused_linear(x, w2, b)
    assert bool(got[:, 3].isinf().all()) and torch.equal(got[:, 4:], clean[:, 4:])
    assert torch.equal(got[:, 3] > 0, x[:, 2] < 0)


@pytest.mark.gpu
@pytest.mark.parametrize('m', [1, 130])
@pytest.mark.parametrize('size', [2.0 ** 60, 2.0 ** -60])
def test_fp32_keeps_its_range(m, size):
    """products of very large and very small factors: relative accuracy as at 1"""
    x, w, b, _ = make(m, 500, 140, torch.float32, False, False, seed=9)
    check(x * size, w / size, None, None, 'none')
    check(x * size, w * min(size, 1.), None, None, 'none')


@pytest.mark.gpu
@pytest.mark.parametrize('m', [3, 20])
def test_few_fp32_rows_at_the_ends_of_the_range(m, cut):
    """the product of few rows: one term a sum, a power of two the other factor: exact, the largest numbers and denormal ones too"""
    from aidet_amd import fused_linear
    cut(16, 1)
    g = torch.Generator(device=DEV).manual_seed(31)
    x, w = torch.zeros(m, 200, device=DEV), torch.zeros(40, 200, device=DEV)
    w[:, 199] = 1.
    w[::2, 199] = 0.5
    x[:, 199] = torch.finfo(torch.float32).max
    assert torch.equal(fused_linear(x, w), (x[:, 199:].double() * w[:, 199].double()).float())
    x[:, 199] = (torch.randint(1, 1 << 20, (m, ), generator=g, device=DEV).double() * 2.0 ** -148).float()
    assert torch.equal(fused_linear(x, w), (x[:, 199:].double() * w[:, 199].double()).float())


@pytest.mark.gpu
@pytest.mark.parametrize('m, n', [(3, 40), (140, 200)])
def test_fp32_numbers_at_the_ends_of_the_range(m, n):
    """one factor a power of two, one term a sum: the products are exact, also of the largest and of denormal numbers"""
    from aidet_amd import fused_linear
    g = torch.Generator(device=DEV).manual_seed(18)
    x = torch.zeros(m, 64, device=DEV)
    top = torch.finfo(torch.float32).max
    x[:, 0] = top * (1 - torch.rand(m, generator=g, device=DEV) * 2.0 ** -9)
    x[0, 0], x[1, 0] = top, -top
    w = torch.zeros(n, 64, device=DEV)
    w[:, 0] = 1.
    w[::2, 0] = 0.5
    assert torch.equal(fused_linear(x, w), (x[:, :1].double() * w[:, 0].double()).float())
    assert torch.equal(fused_linear(x[:, :1], w[:, :1]), fused_linear(x, w))
    x[:, 0] = (torch.randint(1, 1 << 20, (m, ), generator=g, device=DEV).double() * 2.0 ** -149).float()
    want = x[:, :1].double() * w[:, 0].double()
    assert float((fused_linear(x, w).double() - want).abs().max()) <= 2.0 ** -133       # (parts below bf16's last bit vanish)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_activations_at_infinity(dtype):
    """gelu and silu of +-inf are inf and 0, their slopes 1 and 0; NaN stays NaN"""
    from aidet_amd import fused_linear
    inf = float('inf')
    x = torch.tensor([[inf], [-inf], [float('nan')], [200.], [-200.], [0.]], device=DEV, dtype=dtype).expand(6, 1).contiguous()
    w = torch.ones(9, 1, device=DEV, dtype=dtype)
    for act in ('gelu', 'silu', 'relu'):
        r = torch.zeros(6, 9, device=DEV, dtype=dtype, requires_grad=True)
        y = fused_linear(x, w, None, r, act)
        assert torch.equal(y[[0, 1, 3, 4, 5]].abs(), torch.tensor([inf, 0., 200., 0., 0.], device=DEV, dtype=dtype)[:, None].expand(5, 9))
        assert bool(y[2].isnan().all())
        dr, = torch.autograd.grad(y, r, torch.ones_like(y))
        assert torch.equal(dr[[0, 1, 3, 4]], torch.tensor([1., 0., 1., 0.], device=DEV, dtype=dtype)[:, None].expand(4, 9))


@pytest.mark.gpu
@pytest.mark.parametrize('m', [33, 140])
def test_fp32_products_next_to_the_largest_number(m):
    """factors that 8 bits round up to the next power of two: the rounded ones' product overflows where the product does not.
    One term a sum, the other factor a power of two: exact; then terms that add up to less than the largest number, in any order."""
    from aidet_amd import fused_linear
    g = torch.Generator(device=DEV).manual_seed(37)
    x, w = torch.zeros(m, 200, device=DEV), torch.zeros(140, 200, device=DEV)
    x[:, 7] = ((2 - 2.0 ** -9 * torch.rand(m, generator=g, device=DEV).double()) * 2.0 ** 63).float()
    x[0, 7], x[1::2, 7] = 1.998 * 2.0 ** 63, -x[1::2, 7]
    w[:, 7] = 2.0 ** 64 * (1 - 2 * (torch.arange(140, device=DEV) % 3 == 0).float())
    want = (x[:, 7:8].double() * w[:, 7].double()).float()
    assert bool(want.isfinite().all()) and torch.equal(fused_linear(x, w), want)
    leaf = w.clone().requires_grad_(True)                   # (the gradients' products too: dy @ w, dy^T @ x)
    dw, = torch.autograd.grad(fused_linear(x, leaf), leaf, torch.ones(m, 140, device=DEV) * 2.0 ** -20)
    assert bool(dw.isfinite().all())
    xl = torch.ones(m, 200, device=DEV, requires_grad=True)
    dy = torch.zeros(m, 140, device=DEV)
    dy[:, 3] = x[:, 7]
    dx, = torch.autograd.grad(fused_linear(xl, w), xl, dy)
    assert torch.equal(dx[:, 7], (x[:, 7].double() * w[3, 7].double()).float())
    x[:, 8:12], w[:, 8:12] = x[:, 7:8] / 16, w[:, 7:8] * -1
    check(x, w, None, None, 'none')
    x[0, 20], w[1, 20] = float('inf'), 0.                  # (an infinite operand in the same tile, beside them)
    y = fused_linear(x, w)
    assert bool(y[0].isnan().all()) and bool(y[1:].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize('m, n', [(20, 140), (33, 140), (140, 200), (300, 70)])
@pytest.mark.parametrize('small, large', [(2.0 ** -112, 2.0 ** 60), (2.0 ** -120, 2.0 ** 60), (2.0 ** -127, 2.0 ** 100), (2.0 ** -141, 2.0 ** 110),
                                          (2.0 ** -60, 2.0 ** -40), (2.0 ** -126, 1.)])
def test_fp32_products_of_small_numbers(small, large, m, n):
    """operands down to denormal numbers times large ones, sums among them: the accuracy of fp32 products whichever kernel the
    number of rows selects, and whichever operand is the small one; the gradients' products as well.  Outputs that are denormal themselves
    (the last size) are off by half of their step more: 2^-150, within the allowance of the smallest normal number."""
    g = torch.Generator(device=DEV).manual_seed(41)
    k = 500
    x = (torch.randn(m, k, generator=g, device=DEV).double() * small).float()
    w = torch.randn(n, k, generator=g, device=DEV) * large
    check(x, w, None, None, 'none')
    check(w[:, :k], x, None, None, 'none')
    check(x[:, 3:8], w[:, 3:8], None, None, 'none')
    one = torch.ones(m, k, device=DEV)
    check_gradients(one, w, None, None, 'none', (torch.randn(m, n, generator=g, device=DEV).double() * small).float())
    check_gradients(x, torch.zeros_like(w), None, None, 'none', torch.randn(m, n, generator=g, device=DEV) * large)


@pytest.mark.gpu
@pytest.mark.parametrize('split', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['gelu', 'silu'])
def test_activations_everywhere(act, dtype, split, cut):
    """z from -13 to 8 (silu from -87), in every number of the type or densely: the activation to its own accuracy, relative to the
    value, the tail too; z is exact here (a factor of 1, one term).  fp32: q is a polynomial of 1 u, five roundings of its sum that count,
    reciprocal, exp2 and two products of at most 2 u each: 14 u; z - z q next to -1 is 1 - 0.34 / 0.16 of that.  The exponential of silu
    alike, its root squared.  16 u.  16 bits: (16 + 3 z^2) u -- silu (16 + 3 |z|) u -- and half a step of the type.  And in fp32 the error of normal
    inputs is no larger than that of the elementary form, 0.5 z (1 + erf(z / sqrt 2)) and z / (1 + exp(-z)), but a tenth."""
    from aidet_amd import fused_linear
    low = -13 if act == 'gelu' else -87
    if dtype == torch.float32:
        z = torch.cat([torch.linspace(low, 8, 40001, device=DEV), torch.linspace(-0.05, 0.05, 4000, device=DEV)])
    else:
        z = torch.arange(-32768, 32768, device=DEV).to(torch.int16).view(dtype)
        z = z[(z.float() >= low) & (z.float() <= 8)]
    k = 256 if split else 1
    cut(64, 2) if split else None
    x, w = torch.zeros(z.numel(), k, device=DEV, dtype=dtype), torch.zeros(8, k, device=DEV, dtype=dtype)
    x[:, 0], w[:, 0] = z, 1.
    y = fused_linear(x, w, None, None, act)
    assert bool((y == y[:, :1]).all())
    got, d = y[:, 0].double(), z.double()
    want = act64(d, act)
    own = 16 * U if dtype == torch.float32 else (16 + 3 * (d * d if act == 'gelu' else d.abs())) * U + half_step(dtype)
    step = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126      # (half a step of fp16; the exponentials end at the smallest normal number)
    off = (got - want).abs() - own * want.abs() - step
    assert bool((off <= 0).all()), (float(z[off.argmax()]), float(off.max()))
    if dtype == torch.float32:
        z = torch.randn(1 << 18, 1, generator=torch.Generator(device=DEV).manual_seed(43), device=DEV)
        plain = 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5)) if act == 'gelu' else z / (1 + torch.exp(-z))
        want = act64(z.double(), act)
        x = torch.zeros(1 << 18, k, device=DEV)
        x[:, :1] = z
        got = fused_linear(x, w, None, None, act)[:, :1]
        off, off_plain = ((((t.double() - want) / want) ** 2).mean().sqrt() for t in (got, plain))
        assert float(off) <= 1.1 * float(off_plain), (float(off), float(off_plain))


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['gelu', 'silu'])
def test_slopes_everywhere(act):
    """the slope over the same range, fp32: 8 u absolute, and 8 u (1 + z^2) of z's size times the density in the tail"""
    z = torch.linspace(-13, 8, 40001, device=DEV)[:, None]
    r = z.clone().requires_grad_(True)
    from aidet_amd import fused_linear
    y = fused_linear(torch.zeros(z.numel(), 1, device=DEV), torch.zeros(1, 1, device=DEV), None, r, act)
    got, = torch.autograd.grad(y, r, torch.ones_like(y))
    d = z.double()
    off = (got.double() - slope64(d, act)).abs()
    assert float(off.max()) <= 8 * U
    tail = d < -5
    size = d.abs() * torch.exp(-d * d / 2) if act == 'gelu' else d.abs() * torch.exp(d)
    assert bool((off[tail] <= (8 * U * (1 + d * d) * size)[tail]).all())


@pytest.mark.gpu
def test_pitches_past_32_bits():
    """rows 2^31 and more elements apart"""
    from aidet_amd import fused_linear
    pitch, k = (1 << 30) + 8, 40
    buf = torch.empty(4 * pitch, dtype=torch.bfloat16, device=DEV)
    x, w, b, _ = make(4, k, 130, torch.bfloat16, True, False, seed=10)
    far = buf.as_strided((4, k), (pitch, 1))
    far.copy_(x)
    assert torch.equal(fused_linear(far, w, b, act='relu'), fused_linear(x, w, b, act='relu'))
    x, w, b, _ = make(130, k, 4, torch.bfloat16, True, False, seed=11)
    far.copy_(w)
    assert torch.equal(fused_linear(x, far, b, act='relu'), fused_linear(x, w, b, act='relu'))


# ---- gradients -----------------------------------------------------------------------------------------------------------
def gradients(x, w, b, r, act, dy):
    from aidet_amd import fused_linear
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in (x, w, b, r)]
    return torch.autograd.grad(fused_linear(*args, act=act), leaves, dy)


def check_gradients(x, w, b, r, act, dy):
    dtype = x.dtype
    h = half_step(dtype)
    got = list(gradients(x, w, b, r, act, dy))
    _, z, ez, _ = reference(x, w, b, r, act)
    dz = dy.double() * slope64(z, act)
    edz = dy.double().abs() * (0.8 * ez + 8 * U) + h * dz.abs() + tiny(dtype)      # per element, independent of each other

    def product(a, ea, c):            # (a +- ea) @ c
        p, s = product64(a, c)
        spread = 4 * ((ea * ea) @ (c.double() ** 2)).sqrt()
        return p, summed(s, a.size(1), p.abs()) + spread + h * p.abs() + tiny(dtype)
    want = [product(dz, edz, w), product(dz.t(), edz.t(), x)]
    if b is not None:
        want.append((dz.sum(0), summed((dz * dz).sum(0).sqrt(), x.size(0), dz.sum(0).abs()) + 4 * ((edz - h * dz.abs()) ** 2).sum(0).sqrt()
                     + h * dz.sum(0).abs() + tiny(dtype)))
    if r is not None:
        want.append((dz, edz))
    for g, (v, tol), name in zip(got, want, ['x', 'w'] + ['b'] * (b is not None) + ['r'] * (r is not None)):
        off = (g.double() - v).abs() - tol
        assert g.dtype == dtype and bool((off <= 0).all()), (name, float(off.max()), int(off.argmax()))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m, k, n', [(1, 1, 1), (1, 200, 96), (3, 70, 33), (64, 64, 64), (65, 257, 129), (256, 512, 384), (700, 40, 24), (130, 1031, 17),
                                     (2050, 136, 72)])
def test_gradients_sizes(m, k, n, dtype):
    x, w, b, r = make(m, k, n, dtype, True, True, seed=m + n)
    dy = torch.randn(m, n, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(dtype)
    check_gradients(x, w, b, r, 'silu', dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('act', ['none', 'gelu', 'silu'])
@pytest.mark.parametrize('bias, residual', [(False, False), (True, True)])
def test_gradients_epilogue(act, bias, residual, dtype):
    x, w, b, r = make(140, 96, 200, dtype, bias, residual, seed=4, pad=8)
    dy = torch.randn(140, 200, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(dtype)
    check_gradients(x, w, b, r, act, dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m, k, n', [(90, 60, 130), (200, 128, 64)])
def test_gradients_relu(m, k, n, dtype):
    """whole numbers and a bias of a half: z is exact and never 0, so every gradient has one value -- and an exact one
    while its sum stays below 2^24 (fp32) and within the type"""
    g = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randint(-2, 3, (m, k), generator=g, device=DEV).to(dtype)
    w = torch.randint(-2, 3, (n, k), generator=g, device=DEV).to(dtype)
    b = torch.full((n, ), 0.5, device=DEV, dtype=dtype)
    dy = torch.randint(-2, 3, (m, n), generator=g, device=DEV).to(dtype)
    dx, dw, db = gradients(x, w, b, None, 'relu', dy)
    dz = dy.double() * ((x.double() @ w.double().t() + 0.5) > 0)
    for got, want in ((dx, dz @ w.double()), (dw, dz.t() @ x.double()), (db, dz.sum(0))):
        assert torch.equal(got, want.to(dtype))


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32 against central differences of the plain form in 64 bits, gelu: (f(t + h d) - f(t - h d)) / 2h for random
    directions d.  The difference quotient is good to ~1e-9 relative (h = 1e-5); the kernel's sums to the tolerance below:
    a scalar product of ~1e4 terms, each within 2e-6 of its size, independent."""
    m, k, n = 37, 50, 41
    x, w, b, r = make(m, k, n, torch.float32, True, True, seed=12)
    g = torch.Generator(device=DEV).manual_seed(13)
    dy = torch.randn(m, n, generator=g, device=DEV)
    grads = gradients(x, w, b, r, 'gelu', dy)
    base = [t.double() for t in (x, w, b, r)]
    for i, got in enumerate(grads):
        d = torch.randn(base[i].shape, generator=g, device=DEV).double()

        def f(h):
            t = list(base)
            t[i] = t[i] + h * d
            return (dy.double() * act64(t[0] @ t[1].t() + t[2] + t[3], 'gelu')).sum()
        want = (f(1e-5) - f(-1e-5)) / 2e-5
        have = (got.double() * d).sum()
        size = ((got.double() * d) ** 2).sum().sqrt()
        assert abs(float(have - want)) <= 2e-5 * float(size) + 1e-6 * abs(float(want)), (i, float(have), float(want))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_gradients_only_where_wanted_and_broadcast(dtype):
    from aidet_amd import fused_linear
    x, w, b, _ = make(50, 64, 40, dtype, True, False, seed=14)
    row = torch.randn(40, device=DEV).to(dtype).requires_grad_(True)
    w.requires_grad_(True)
    y = fused_linear(x, w, b, row.expand(50, 40), 'none')
    dw, dr = torch.autograd.grad(y.float().sum(), (w, row))       # (an expanded gradient of y)
    assert torch.equal(dr, torch.full_like(dr, 50.))
    v, s = product64(torch.ones(40, 50, device=DEV), x)
    assert bool(((dw.double() - v).abs() <= summed(s, 50, v.abs()) + half_step(dtype) * v.abs()).all())
    # each gradient alone, with and without a bias before the residual
    for with_bias in (True, False):
        xs = x.detach().requires_grad_(True)
        bs = b.detach().requires_grad_(True) if with_bias else None
        rs = torch.randn(50, 40, device=DEV).to(dtype).requires_grad_(True)
        y = fused_linear(xs, w, bs, rs, 'silu')
        up = torch.randn(50, 40, device=DEV).to(dtype)
        leaves = [xs, w] + ([bs] if with_bias else []) + [rs]
        every = torch.autograd.grad(y, leaves, up, retain_graph=True)
        for leaf, want in zip(leaves, every):
            alone, = torch.autograd.grad(y, leaf, up, retain_graph=True)
            assert torch.equal(alone, want)
    # the same weight twice in one graph: the gradients add
    x.requires_grad_(True)
    sq = (torch.randn(64, 64, device=DEV) / 8).to(dtype).requires_grad_(True)
    h = fused_linear(x, sq, act='silu')
    both, = torch.autograd.grad(fused_linear(h, sq).float().sum(), sq, retain_graph=True)
    assert both.shape == sq.shape and bool(both.isfinite().all())
    with pytest.raises(RuntimeError):                             # differentiable once
        gx, = torch.autograd.grad(h.float().sum(), x, create_graph=True)
        gx.float().sum().backward()


@pytest.mark.gpu
def test_same_bits_every_run():
    for dtype in TYPES:
        x, w, b, r = make(700, 3000, 260, dtype, True, True, seed=15)
        dy = torch.randn(700, 260, device=DEV).to(dtype)
        first = gradients(x, w, b, r, 'gelu', dy)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, gradients(x, w, b, r, 'gelu', dy)))


@pytest.mark.gpu
def test_other_stream_and_two_at_once():
    from aidet_amd import fused_linear
    x, w, b, r = make(600, 2000, 300, torch.bfloat16, True, True, seed=16)
    want = fused_linear(x, w, b, r, 'gelu')
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([fused_linear(x, w, b, r, 'gelu') for _ in range(4)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for per in outs for o in per)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_captured_step_replays(dtype):
    """forward + backward captured, replayed on changed inputs with eager work between: every replay the eager bits"""
    from aidet_amd import fused_linear
    x, w, b, r = make(90, 1100, 130, dtype, True, True, seed=17)
    dy = torch.randn(90, 130, device=DEV).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x.contiguous(), w, b, r)]

    def step():
        y = fused_linear(*leaves, act='gelu')
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(90, 1100, device=DEV))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), i


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_infinite_gradients_of_units_that_are_off(dtype):
    """relu: where y is 0 the gradient of y reaches nothing, whatever it holds"""
    from aidet_amd import fused_linear
    x, w, b, r = make(70, 200, 67, dtype, True, True, seed=23)
    leaves = [t.requires_grad_(True) for t in (x.contiguous(), w, b, r)]
    y = fused_linear(*leaves, act='relu')
    dy = torch.randn(70, 67, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV).to(dtype)
    dy = torch.where(y > 0, dy, torch.zeros_like(dy))
    odd = dy.clone()
    for i, bad in enumerate((float('inf'), float('-inf'), float('nan'))):
        odd[i::3] = torch.where(y[i::3] > 0, dy[i::3], torch.full_like(dy[i::3], bad))
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, odd)
    assert all(bool(torch.isfinite(t).all()) and torch.equal(t, u) for t, u in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES[1:])
def test_autocast_casts_as_a_linear_layer_does(dtype):
    from aidet_amd import FusedLinear, fused_linear
    x, w, b, r = make(33, 120, 50, torch.float32, True, True, seed=29)
    layer = FusedLinear(120, 50, act='silu').to(DEV)
    with torch.autocast('cuda', dtype=dtype):
        y = fused_linear(x, w, b.to(torch.float16), r, 'silu')
        z = layer(x.to(dtype), r)
    assert y.dtype == dtype and z.dtype == dtype
    assert torch.equal(y, fused_linear(x.to(dtype), w.to(dtype), b.to(torch.float16).to(dtype), r.to(dtype), 'silu'))
    z.sum().backward()
    assert layer.weight.grad.dtype == torch.float32 and bool(layer.weight.grad.abs().sum() > 0)
    dy = torch.ones_like(z)
    a, c = layer.weight.detach().to(dtype).requires_grad_(True), layer.bias.detach().to(dtype)
    want, = torch.autograd.grad(fused_linear(x.to(dtype), a, c, r.to(dtype), 'silu'), a, dy)
    assert torch.equal(layer.weight.grad, want.float())


@pytest.mark.gpu
def test_capture_beside_an_eager_graph_of_the_default_stream():
    """a captured backward pass whose leaves' accumulators belong to the default stream is refused; afterwards it is served"""
    from aidet_amd import fused_linear, topk_distill_loss
    w = torch.randn(24, 40, device=DEV, requires_grad=True)
    x = torch.randn(9, 40, device=DEV)
    logits = torch.randn(9, 24, device=DEV, requires_grad=True)
    values, indices = torch.randn(9, 4, device=DEV), torch.arange(36, device=DEV).reshape(9, 4) % 24

    def linear():
        return fused_linear(x, w, act='silu').square().sum()

    def distill():
        return topk_distill_loss(logits, values, indices)
    for loss, leaf in ((linear, w), (distill, logits)):
        kept = loss()
        kept.backward()
        want, leaf.grad = leaf.grad, None
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match='graph of the same leaves'):
            with torch.cuda.graph(graph):
                loss().backward()
        torch.cuda.synchronize()
        del kept
        leaf.grad = None
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            kept = loss()                    # (alive during the capture, but not of the default stream)
            kept.backward()
        torch.cuda.current_stream().wait_stream(s)
        leaf.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss().backward()
        for _ in range(3):
            leaf.grad.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(leaf.grad, want)
        del kept
        leaf.grad = None


@pytest.mark.gpu
@pytest.mark.parametrize('way', ['autocast', 'view'])
def test_capture_beside_an_eager_graph_whose_leaves_are_behind_other_nodes(way):
    """the same where the leaf reaches the layer through a cast of autocast, or a product and a view"""
    from aidet_amd import fused_linear
    w = torch.randn(24, 40, device=DEV, requires_grad=True)
    x = torch.randn(9, 40, device=DEV)

    def loss():
        if way == 'view':
            return fused_linear(x, (w * 2).view(24, 40), act='silu').square().sum()
        with torch.autocast('cuda', dtype=torch.bfloat16, cache_enabled=False):
            return fused_linear(x, w, act='silu').float().square().sum()
    kept = loss()
    kept.backward()
    want, w.grad = w.grad, None
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match='graph of the same leaves'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            loss().backward()
    torch.cuda.synchronize()
    del kept
    w.grad = None
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss().backward()
    torch.cuda.current_stream().wait_stream(s)
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss().backward()
    for _ in range(3):
        w.grad.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w.grad, want)
    w.grad = None


def lazily_negative(*shape):
    """(a float tensor whose negative bit is set, the same numbers in memory): the imaginary part of a conjugate"""
    t = torch.view_as_complex(torch.randn(*shape, 2, device=DEV)).conj().imag
    assert t.is_neg()
    return t, t.clone().resolve_neg()


@pytest.mark.gpu
@pytest.mark.parametrize('m, k, n', [(5, 1, 3), (5, 4, 1), (1, 1, 1), (6, 7, 8)])
def test_tensors_with_the_negative_bit(m, k, n):
    """sizes at which such a tensor passes for a contiguous one, and others; as gradients of the output too"""
    from aidet_amd import fused_linear
    torch.manual_seed(3)
    pairs = [lazily_negative(*s) for s in ((m, k), (n, k), (n, ), (m, n))]
    dy, plain_dy = lazily_negative(m, n)
    results = []
    for which, up in ((0, dy), (1, plain_dy)):
        leaves = [p[which].detach().requires_grad_(True) for p in pairs]
        y = fused_linear(*leaves, act='silu')
        results.append([y.detach()] + list(torch.autograd.grad(y, leaves, up)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
