"""The cases by which the fused linear layer and the top-logit distillation loss are measured.

Two operators, in two directions each:

* ``linear``:  ``z = x @ w.T + bias + residual``, ``y = act(z)``; a training pass also returns the gradients of ``x``,
  ``w``, ``bias`` and ``residual`` for a given gradient of ``y``.
* ``distill``: ``p = softmax(values / T)`` over a row's k teacher entries, ``q = softmax(logits / T)`` over all classes,
  ``loss_r = T^2 sum_j p_j (log p_j - log q_j)``; rows may carry weights and may miss entries (index -1); a training pass
  returns the mean loss and the gradient of the logits, an evaluating one the losses of the rows.
"""
import math

import torch

own = False

_TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def _linear(name, m, k, n, dtype, act, bias=True, residual=False, train=False, pad=0):
    return dict(name=name, op='linear', m=m, k=k, n=n, dtype=dtype, act=act, bias=bias, residual=residual, train=train,
                pad=pad)


def _distill(name, rows, classes, k, dtype, temperature, weighted=False, missing=False, train=True, index='int64'):
    return dict(name=name, op='distill', rows=rows, classes=classes, k=k, dtype=dtype, temperature=temperature,
                weighted=weighted, missing=missing, train=train, index=index)


def listed():
    return [
        # one RoI through the second FC layer of a head: a call's latency
        _linear('single_row_bf16', 1, 1024, 1024, 'bf16', 'relu'),
        # the first FC layer of a head on a tile's 2000 proposals (256 channels x 7 x 7), as the detector runs it
        _linear('trunk_fc1_fp32', 2000, 12544, 1024, 'fp32', 'relu'),
        # the same in half the bytes
        _linear('trunk_fc1_bf16', 2000, 12544, 1024, 'bf16', 'relu'),
        # a handful of RoIs scored again: bound by the weights
        _linear('few_rows_fp16', 24, 12544, 1024, 'fp16', 'silu'),
        # the last 1x1 convolution of a bottleneck on a 256 x 256 channels-last map: folded norm, shortcut, ReLU
        _linear('pointwise_residual_fp32', 65536, 64, 256, 'fp32', 'relu', residual=True),
        # a wide layer over a long batch: the largest product
        _linear('wide_gelu_bf16', 8192, 4096, 16384, 'bf16', 'gelu'),
        # a training step of the first FC layer on 2 x 512 sampled RoIs
        _linear('train_fc1_bf16', 1024, 12544, 1024, 'bf16', 'relu', train=True),
        # odd sizes, rows that are not aligned, every gradient
        _linear('train_odd_fp32', 777, 1111, 515, 'fp32', 'gelu', residual=True, train=True, pad=3),
        # a head's 16 classes on a tile's 2000 proposals, the 4 best of the teacher, weights of the sampled RoIs
        _distill('head_classes_fp32', 2000, 16, 4, 'fp32', 2.0, weighted=True),
        # a large vocabulary of odd size
        _distill('vocabulary_bf16', 4096, 50001, 32, 'bf16', 1.0, missing=True),
        # few rows, long ones
        _distill('few_long_rows_fp32', 8, 262144, 128, 'fp32', 1.0),
        # scoring a checkpoint: losses only
        _distill('evaluate_fp16', 1000, 1203, 100, 'fp16', 4.0, train=False, index='int32'),
    ]


def _log_size(rng, low, high):
    """A size whose logarithm is spread evenly; half of them are odd, some a multiple of 64."""
    size = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    how = rng.random()
    if how < 0.4:
        size |= 1
    elif how < 0.8 and size >= 64:
        size -= size % 64
    return max(low, min(high, size))


def draw(rng):
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    train = rng.random() < 0.5
    if rng.random() < 0.6:
        while True:
            m, k, n = _log_size(rng, 1, 65536), _log_size(rng, 8, 16384), _log_size(rng, 8, 16384)
            flops = 2 * m * k * n * (3 if train else 1)
            if flops <= 1.0e12 and m * (k + 2 * n) <= 3e8:
                break
        # the gradient of a ReLU jumps where z is within a rounding of 0: in 32 bits a training pass takes a smooth one
        act = rng.choice(['none', 'gelu', 'silu'] if train and dtype == 'fp32' else ['none', 'relu', 'gelu', 'silu'])
        case = _linear('', m, k, n, dtype, act, bias=rng.random() < 0.8, residual=rng.random() < 0.4, train=train,
                       pad=rng.choice([0, 0, 0, 1, 8]))
    else:
        while True:
            rows, classes = _log_size(rng, 1, 65536), _log_size(rng, 4, 262144)
            if rows * classes <= 2.0e8:
                break
        k = min(classes, _log_size(rng, 1, 256))
        case = _distill('', rows, classes, k, dtype, rng.choice([1.0, 2.0, 4.0]), weighted=rng.random() < 0.5,
                        missing=rng.random() < 0.3, train=train, index=rng.choice(['int64', 'int32']))
    del case['name']
    return case


def prepare(case, seed):
    dtype = _TYPES[case['dtype']]
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device='cuda')

    if case['op'] == 'linear':
        m, k, n = case['m'], case['k'], case['n']
        state = dict(op='linear', act=case['act'], train=case['train'])
        # (rows of a wider buffer where `pad` is set)
        state['x'] = normal(m, k + case['pad']).to(dtype)[:, :k]
        state['w'] = (normal(n, k) * k ** -0.5).to(dtype)
        state['bias'] = (normal(n) * 0.1).to(dtype) if case['bias'] else None
        state['residual'] = normal(m, n).to(dtype) if case['residual'] else None
        if case['train']:
            state['grad'] = normal(m, n).to(dtype)
            for name in ('x', 'w', 'bias', 'residual'):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    rows, classes, k = case['rows'], case['classes'], case['k']
    logits = (normal(rows, classes) * 3).to(dtype)
    # the teacher: the student's logits with noise of their own, its k best
    teacher = logits.float()
    teacher = (teacher + normal(rows, classes)).to(dtype)
    values, indices = teacher.topk(k, dim=1)
    if case['missing']:   # rows with fewer entries, some with none
        have = torch.randint(0, k + 1, (rows, 1), generator=gen, device='cuda')
        indices = torch.where(torch.arange(k, device='cuda') < have, indices, torch.full_like(indices, -1))
    weight = None
    if case['weighted']:  # sampled RoIs: weight 1, others 0
        weight = (torch.rand(rows, generator=gen, device='cuda') < 0.75).float()
    return dict(op='distill', logits=logits.requires_grad_(case['train']), values=values.contiguous(),
                indices=indices.to(torch.int32 if case['index'] == 'int32' else torch.int64).contiguous(), weight=weight,
                temperature=case['temperature'], train=case['train'])


def _act(z, act):
    if act == 'relu':
        return z.clamp(min=0)
    if act == 'gelu':
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == 'silu':
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == 'relu':
        return (z > 0).to(z.dtype)
    if act == 'gelu':
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == 'silu':
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    return torch.ones_like(z)


def _plain_linear(s):
    dtype = s['x'].dtype
    x, w = s['x'].float(), s['w'].float()
    z = x @ w.t()
    if s['bias'] is not None:
        z = z + s['bias'].float()
    if s['residual'] is not None:
        z = z + s['residual'].float()
    y = _act(z, s['act']).to(dtype)
    if not s['train']:
        return y
    dz = s['grad'].float() * _act_slope(z, s['act'])
    out = [y, (dz @ w).to(dtype), (dz.t() @ x).to(dtype)]
    if s['bias'] is not None:
        out.append(dz.sum(0).to(dtype))
    if s['residual'] is not None:
        out.append(dz.to(dtype))
    return out


def _plain_distill(s):
    temp, logits = s['temperature'], s['logits']
    x = logits.float() / temp
    x = x - x.amax(1, keepdim=True)
    lse = x.exp().sum(1, keepdim=True).log()
    there = s['indices'] >= 0
    some = there.any(1, keepdim=True)
    t = (s['values'].float() / temp).masked_fill(~there, -math.inf)
    t = t - t.amax(1, keepdim=True).masked_fill(~some, 0.)
    t_lse = t.exp().sum(1, keepdim=True).log().masked_fill(~some, 0.)
    p = (t - t_lse).exp()
    index = s['indices'].long().clamp(min=0)
    log_ratio = (t - t_lse).masked_fill(~there, 0.) - (x.gather(1, index) - lse)
    loss = temp * temp * (p * log_ratio).sum(1)
    if s['weight'] is not None:
        loss = loss * s['weight']
    if not s['train']:
        return loss
    grad = (x - lse).exp() * some.float()
    grad.scatter_add_(1, index, -p)
    scale = temp / loss.numel()
    grad = grad * (scale if s['weight'] is None else scale * s['weight'][:, None])
    return loss.mean(), grad.to(logits.dtype)


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return _plain_linear(s) if s['op'] == 'linear' else _plain_distill(s)
    import aidet_amd
    if s['op'] == 'linear':
        y = aidet_amd.fused_linear(s['x'], s['w'], s['bias'], s['residual'], act=s['act'])
        if not s['train']:
            return y
        leaves = [s[name] for name in ('x', 'w', 'bias', 'residual') if s[name] is not None]
        return [y.detach()] + list(torch.autograd.grad(y, leaves, s['grad']))
    loss = aidet_amd.topk_distill_loss(s['logits'], s['values'], s['indices'], temperature=s['temperature'],
                                       weight=s['weight'], reduction='mean' if s['train'] else 'none')
    if not s['train']:
        return loss
    return loss.detach(), torch.autograd.grad(loss, s['logits'])[0]


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'linear':
        m, k, n = case['m'], case['k'], case['n']
        once = m * k + n * k + (n if case['bias'] else 0) + (m * n if case['residual'] else 0)
        if not case['train']:
            return {'bytes': size * (once + m * n), 'flops': 2 * m * n * k}
        # read: the inputs and the gradient of y; written: y and a gradient for each input
        return {'bytes': size * (2 * once + 2 * m * n), 'flops': 6 * m * n * k}
    rows, classes, k = case['rows'], case['classes'], case['k']
    lists = rows * k * (size + (4 if case['index'] == 'int32' else 8)) + (4 * rows if case['weighted'] else 0)
    if not case['train']:
        return {'bytes': size * rows * classes + lists + 4 * rows, 'flops': 4 * rows * classes}
    return {'bytes': 2 * size * rows * classes + lists + 4, 'flops': 8 * rows * classes}


def exact(case, seed):
    s = prepare(case, seed)
    wide = {name: v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v for name, v in s.items()}
    if case['op'] == 'linear':
        leaves = [wide[name].requires_grad_(case['train']) for name in ('x', 'w', 'bias', 'residual')
                  if wide[name] is not None]
        z = torch.nn.functional.linear(wide['x'], wide['w'], wide['bias'])
        z = z if wide['residual'] is None else z + wide['residual']
        f = torch.nn.functional
        y = {'none': lambda v: v, 'relu': f.relu, 'gelu': f.gelu, 'silu': f.silu}[case['act']](z)
        if not case['train']:
            return y
        return [y.detach()] + list(torch.autograd.grad(y, leaves, wide['grad']))
    temp = case['temperature']
    logits = wide['logits'].requires_grad_(case['train'])
    log_q = torch.log_softmax(logits / temp, 1)
    # rows without an entry have no loss; the others' missing places have no probability
    have = s['indices'] >= 0
    log_p = torch.where(have, wide['values'] / temp, torch.full_like(wide['values'], -1e300))
    log_p = torch.log_softmax(log_p, 1)
    p = torch.where(have, log_p.exp(), torch.zeros_like(log_p))
    picked = log_q.gather(1, torch.where(have, s['indices'], torch.zeros_like(s['indices'])).long())
    losses = torch.where(have, p * (log_p - picked), torch.zeros_like(p)).sum(1) * temp ** 2
    if s['weight'] is not None:
        losses = losses * wide['weight']
    if not case['train']:
        return losses
    loss = losses.sum() / case['rows']
    return loss.detach(), torch.autograd.grad(loss, logits)[0]
