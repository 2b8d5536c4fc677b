"""The fused linear layer and the distillation loss inside the detector: heads, bottlenecks, pyramid, a head's training step.

Tolerances.  The fused and the plain layer are the same sums of fp32 products in another order: a layer of K terms is off by
less than 8 sqrt(K + 8) 2^-24 of sqrt(sum of the squared terms) on either side (the bound of test_linear.py), which for
outputs of about that size is 16 sqrt(K + 8) 2^-24 of a layer's largest value: 1.1e-4 at K = 12544, 2e-5 at K = 512.  Layers
in a row add theirs (weights are random: no layer amplifies), so L layers of at most K terms are allowed L times that.
"""
import numpy as np
import pytest
import torch

DEV = 'cuda:0'


def _near(got, want, layers, k):
    tol = layers * 16 * (k + 8) ** 0.5 * 2.0 ** -24 * float(want.abs().max())
    assert got.shape == want.shape and float((got - want).abs().max()) <= tol, (float((got - want).abs().max()), tol)


def test_folding_is_dropped_with_the_weights_it_came_from():
    from aidet_amd.models.theta_obb_rcnn import Bottleneck, ThetaOBBRCNN
    import torch.nn as nn
    torch.manual_seed(0)
    b = Bottleneck(16, 4).eval()
    names = set(b.state_dict())
    b.fold()
    assert b.folded and set(b.state_dict()) == names and b.w3.shape == (16, 4)
    x = torch.randn(1, 16, 5, 6)
    with torch.no_grad():
        want = nn.functional.conv2d(x, b.conv1.weight)
        want = b.bn1(want)
        got = nn.functional.conv2d(x, b.w1[:, :, None, None], b.b1)
    assert float((got - want).abs().max()) < 1e-5
    b.load_state_dict(b.state_dict())
    assert not b.folded and b.w1 is None
    b.fold()
    b.train()
    assert not b.folded
    m = ThetaOBBRCNN()
    assert not m.bbox_head.fused_linear and not m.neck.fused_linear      # (as before unless asked for)
    keys = set(m.state_dict())
    assert set(m.fold_pointwise().state_dict()) == keys and m.neck.fused_linear
    assert set(ThetaOBBRCNN(fused_linear=True).state_dict()) == keys


@pytest.fixture
def calls(monkeypatch):
    """every map counts as channels-last on a device and `pointwise` is a plain convolution here: the list of its calls"""
    import aidet_amd.models.theta_obb_rcnn as mod
    made = []

    def plain(x, weight, bias=None, residual=None, act='none'):
        made.append(tuple(weight.shape))
        y = torch.nn.functional.conv2d(x, weight[:, :, None, None], bias)
        y = y if residual is None else y + residual
        return y.relu() if act == 'relu' else y
    monkeypatch.setattr(mod, '_channels_last', lambda x: True)
    monkeypatch.setattr(mod, 'pointwise', plain)
    return made


def test_a_folded_bottleneck_in_training_mode_normalises_by_the_batch(calls):
    """fold() after train(), and a norm alone in training mode: the batch's statistics, running ones updated; fold() of a
    module in training mode serves once it is in eval mode, unless a pass has moved the statistics it was made of"""
    import copy
    from aidet_amd.models.theta_obb_rcnn import Bottleneck
    torch.manual_seed(3)
    for norms in (('bn1', 'bn2', 'bn3'), ('bn1', ), ('bn3', )):
        plain = Bottleneck(16, 4).eval()
        for name in norms:
            getattr(plain, name).train()
        if len(norms) == 3:
            plain.train()
        folded = copy.deepcopy(plain)
        folded.fold()
        assert folded.folded
        x = torch.randn(2, 16, 5, 6)
        with torch.no_grad():
            want, got = plain(x), folded(x)
            assert torch.equal(want, got) and not calls
            assert all(torch.equal(u, v) for u, v in zip(plain.state_dict().values(), folded.state_dict().values()))
            assert torch.equal(plain.eval()(x), folded.eval()(x)) and not calls    # (what was folded is not what it is now)
            folded.train()
            folded.fold()
            folded.eval()
            near = folded(x)
        assert calls == [(4, 16), (16, 4)] and float((near - plain(x)).abs().max()) < 1e-5
        calls.clear()


def test_training_mode_and_loading_end_the_folding_of_the_whole_detector(calls):
    """train() and loading weights end it in the pyramid as in the bottlenecks; eval() does not"""
    from aidet_amd.models.theta_obb_rcnn import Bottleneck, ThetaOBBRCNN

    def on():
        return {m.neck.fused_linear} | {b.folded for b in m.modules() if isinstance(b, Bottleneck)}
    m = ThetaOBBRCNN().eval().fold_pointwise()
    feats = [torch.randn(1, c, 16 >> i, 16 >> i) for i, c in enumerate((256, 512, 1024, 2048))]
    with torch.no_grad():
        m.neck(feats)
    assert on() == {True} and len(calls) == 4
    m.eval()
    assert on() == {True}
    m.train()
    assert on() == {False}
    m.eval().fold_pointwise()
    m.load_state_dict(m.state_dict())
    assert on() == {False}
    with torch.no_grad():
        m.neck(feats)
    assert len(calls) == 4
    m.neck.train()                      # (of a part of the detector: it is the detector's own train() that ends it)
    m.fold_pointwise()
    assert on() == {True}


def test_layers_with_hooks_of_their_own_are_called(calls, monkeypatch):
    """a hook of any kind on a layer, or a layer of another class in its place: that layer is called as a module, the others stay
    fused; without hooks none is called"""
    import aidet_amd.models.theta_obb_rcnn as mod
    nn = torch.nn
    rows = []

    def plain(x, weight, bias=None, residual=None, act='none'):
        rows.append(tuple(weight.shape))
        y = nn.functional.linear(x, weight, bias)
        return y.relu() if act == 'relu' else y
    monkeypatch.setattr(mod, 'fused_linear', plain)
    torch.manual_seed(5)

    def hooked(layer, kind):
        seen = []
        register = getattr(layer, 'register_' + kind)
        return seen, register(lambda m, *a: seen.append(m) and None)
    # heads
    head = mod.SharedFCHead(5, in_channels=2, fc_out_channels=8, fused_linear=True)
    x = torch.randn(3, 2, 7, 7)
    want = head(x)
    assert len(rows) == 4
    for kind in ('forward_hook', 'forward_pre_hook', 'full_backward_hook', 'full_backward_pre_hook'):
        for layer in (head.shared_fcs[0], head.shared_fcs[1], head.fc_cls, head.fc_reg):
            rows.clear()
            seen, handle = hooked(layer, kind)
            got = head(x)
            sum(g.sum() for g in got).backward()
            handle.remove()
            assert seen == [layer] and len(rows) == 3
            assert all(torch.allclose(g, w, atol=1e-6) for g, w in zip(got, want))

    class Doubled(nn.Linear):
        def forward(self, x):
            return 2 * super(Doubled, self).forward(x)
    rows.clear()
    first = head.shared_fcs[0]
    head.shared_fcs[0] = Doubled(98, 8)
    head.shared_fcs[0].load_state_dict({k: v / 2 for k, v in first.state_dict().items()})
    assert all(torch.allclose(g, w, atol=1e-6) for g, w in zip(head(x), want)) and len(rows) == 3
    # bottlenecks
    block = mod.Bottleneck(16, 4).eval()
    block.fold()
    x = torch.randn(1, 16, 5, 6)
    with torch.no_grad():
        want = block(x)
        assert len(calls) == 2
        for kind in ('forward_hook', 'forward_pre_hook'):
            for layer in (block.conv1, block.bn1, block.conv3, block.bn3):
                calls.clear()
                seen, handle = hooked(layer, kind)
                got = block(x)
                handle.remove()
                assert seen == [layer] and not calls and torch.allclose(got, want, atol=1e-5)
        assert block.folded and torch.equal(block(x), want)
    # pyramid
    neck = mod.FPN((3, 4, 5), 6, 4)
    neck.fused_linear = True
    feats = [torch.randn(1, c, 16 >> i, 16 >> i) for i, c in enumerate((3, 4, 5))]
    calls.clear()
    want = neck(feats)
    assert len(calls) == 3
    for layer in neck.lateral_convs:
        calls.clear()
        seen, handle = hooked(layer, 'forward_hook')
        got = neck(feats)
        handle.remove()
        assert seen == [layer] and len(calls) == 2 and all(torch.allclose(g, w, atol=1e-5) for g, w in zip(got, want))


@pytest.mark.gpu
def test_heads_on_fused_layers():
    from aidet_amd.models.theta_obb_rcnn import SharedFCHead
    torch.manual_seed(1)
    for n in (0, 1, 37, 500):
        plain = SharedFCHead(5).to(DEV)
        fused = SharedFCHead(5, fused_linear=True).to(DEV)
        fused.load_state_dict(plain.state_dict())
        x = torch.randn(n, 256, 7, 7, device=DEV)
        with torch.no_grad():
            want, got = plain(x), fused(x)
        for w, g in zip(want, got):
            assert g.shape == w.shape
            if n:
                _near(g, w, 3, 12544)


@pytest.mark.gpu
def test_pyramid_on_fused_layers():
    from aidet_amd.models import build_detector, demo_inputs
    model = build_detector(torch.device(DEV)).to(memory_format=torch.channels_last)
    for m in model.backbone.modules():            # (norms that do something)
        if isinstance(m, torch.nn.BatchNorm2d):
            torch.nn.init.uniform_(m.running_var, 0.5, 2.0)
            torch.nn.init.normal_(m.running_mean, std=0.1)
            torch.nn.init.uniform_(m.weight, 0.5, 1.0)
            torch.nn.init.normal_(m.bias, std=0.1)
    img, _ = demo_inputs(DEV, 256)
    img = img.contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        want = model.extract_feat(img)
        model.fold_pointwise()
        got = model.extract_feat(img)
        assert all(g.is_contiguous(memory_format=torch.channels_last) for g in got[:4])
        for g, w in zip(got, want):
            _near(g, w, 16 * 3 + 2, 512)            # (16 bottlenecks of up to 3 convolutions, lateral, output)
        model.fold_pointwise(False)
        for g, w in zip(model.extract_feat(img), want):
            _near(g, w, 16 * 3 + 2, 512)


@pytest.mark.gpu
def test_the_fused_paths_run(monkeypatch):
    """channels-last tile: two fused layers a bottleneck and one a level, all by the kernel, where the detector is folded and none
    where it is not; every head layer where the heads are fused; what they give is the unfused detector's within the layers' bound"""
    import aidet_amd.models.theta_obb_rcnn as mod
    made = []
    kernel = mod.fused_linear

    def counted(x, weight, *args, **kwargs):
        made.append(tuple(weight.shape))
        return kernel(x, weight, *args, **kwargs)
    monkeypatch.setattr(mod, 'fused_linear', counted)
    dev = torch.device(DEV)
    models = [mod.build_detector(dev, fused_linear=f).to(memory_format=torch.channels_last) for f in (False, True)]
    img, _ = mod.demo_inputs(dev, 256)
    img = img.contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        want = models[0].extract_feat(img)
        pooled = torch.randn(50, 256, 7, 7, device=dev)
        heads = [h(pooled) for h in (models[0].bbox_head, models[0].rbbox_head)]
        assert not made
        got = models[1].fold_pointwise().extract_feat(img)
        assert len(made) == 2 * 16 + 4
        for g, w in zip(got, want):
            _near(g, w, 16 * 3 + 2, 512)
        made.clear()
        for head, outs in zip((models[1].bbox_head, models[1].rbbox_head), heads):
            for g, w in zip(head(pooled), outs):
                _near(g, w, 3, 12544)
        assert len(made) == 8
        made.clear()
        models[1].fold_pointwise(False).extract_feat(img)
        assert not made
        # (the convolutions of a model that is not channels-last give maps that are not, and are served by themselves)
        mod.build_detector(dev).fold_pointwise().extract_feat(img.contiguous())
        assert not made


@pytest.mark.gpu
def test_detector_tile_on_fused_layers():
    from aidet_amd.models import build_detector, demo_inputs
    dev = torch.device(DEV)
    model = build_detector(dev, rotated_nms=True, fused_linear=True).to(memory_format=torch.channels_last).fold_pointwise()
    img, meta = demo_inputs(dev, 512)
    img = img.contiguous(memory_format=torch.channels_last)
    bb, rb = model.simple_test(img, meta)
    assert len(bb) == len(rb) == 15 and all(b.shape[1] == 5 for b in bb) and all(r.shape[1] == 6 for r in rb)
    assert all(np.isfinite(b).all() for b in bb + rb)


@pytest.mark.gpu
def test_a_heads_distillation_step():
    """x -> FC trunk -> class logits -> loss -> gradients of every layer and of the pooled features, fused against plain
    layers and the loss in 64 bits.  The logits are within the layers' bound; the loss and its gradient are smooth in them, the
    gradients' products one layer deeper each: 8 layers' bound of the largest value."""
    from aidet_amd.models.theta_obb_rcnn import SharedFCHead
    torch.manual_seed(2)
    plain = SharedFCHead(5, fc_out_channels=128).to(DEV).double()
    for fc in plain.shared_fcs:
        torch.nn.init.zeros_(fc.bias)
    torch.nn.init.normal_(plain.fc_cls.weight, std=0.1)
    fused = SharedFCHead(5, fc_out_channels=128, fused_linear=True).to(DEV)
    fused.load_state_dict({k: v.float() for k, v in plain.state_dict().items()})
    plain.load_state_dict({k: v.double() for k, v in fused.state_dict().items()})
    x = torch.randn(96, 256, 7, 7, device=DEV)
    teacher = 2 * torch.randn(96, 16, device=DEV)
    values, indices = teacher.topk(4, 1)
    weights = (torch.arange(96, device=DEV) % 4 != 0).float()
    x1, x2 = x.clone().requires_grad_(True), x.double().requires_grad_(True)
    loss = fused.distill_loss(x1, values, indices, 2.0, weights, 72.)
    params = [p for p in fused.parameters()]
    grads = torch.autograd.grad(loss, [x1] + params, allow_unused=True)
    # (a pre-activation within a rounding of 0 would have two gradients: there is none among these)
    h = x2.flatten(1)
    for fc in plain.shared_fcs:
        z = fc(h)
        assert float(z.abs().min()) > 1e-7
        h = z.relu()
    log_q = torch.log_softmax(plain.fc_cls(h) / 2, 1).gather(1, indices)
    log_p = torch.log_softmax(values.double() / 2, 1)
    want = (weights * 4 * (log_p.exp() * (log_p - log_q)).sum(1)).sum() / 72
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    refs = torch.autograd.grad(want, [x2] + [p for p in plain.parameters()], allow_unused=True)
    for g, r in zip(grads, refs):
        assert (g is None) == (r is None)
        if g is not None:
            tol = 8 * 16 * (12544 + 8) ** 0.5 * 2.0 ** -24 * float(r.abs().max())
            assert float((g.double() - r).abs().max()) <= tol
    assert grads[1:].count(None) == 2             # (fc_reg has no part in it)
