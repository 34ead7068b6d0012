"""The 8-bit options of the convolution stacks (backbone.py: pointwise='int8', checkpoints='int8') and the autograd
bindings under them (quant.linear_int8, conv_kept, norm_act_kept)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import yolo_tf_amd as y
from yolo_tf_amd import backbone as bb, quant
from tests import quant_cases as qc
from tests.test_backbone import _fill, _load_conv_golden

pytestmark = pytest.mark.gpu


def _layer(cin, cout, kernel, stride, act, pointwise, checkpoints, dev):
    layer = bb.ConvBN(cin, cout, kernel, stride, activation=act)
    layer.pointwise, layer.checkpoints = pointwise, checkpoints
    with torch.no_grad():
        layer.conv.bias.normal_()
        layer.bn.weight.normal_(1, 0.2)
        layer.bn.bias.normal_(0, 0.2)
    return layer.to(dev).to(memory_format=torch.channels_last).train()


def test_the_forward_pass_with_checkpoints_is_the_plain_one(gpu):
    """Against the NumPy restatement of the blocks, as the float32 stack is tested."""
    gold = _load_conv_golden()
    t = lambda a: torch.from_numpy(gold[a]).float().to(gpu).contiguous(memory_format=torch.channels_last)
    close = lambda got, name: np.testing.assert_allclose(got.detach().cpu().numpy(), gold[name], rtol=1e-4, atol=1e-4, err_msg=name)

    def kept(m):
        for layer in m.modules():
            if isinstance(layer, bb.ConvBN):
                layer.checkpoints = 'int8'
        return m.to(gpu)

    for name, cout, k, stride, act in (('c3', 7, 3, 1, True), ('c3s2', 6, 3, 2, True), ('c1', 4, 1, 1, False)):
        layer = kept(_fill(bb.ConvBN(5, cout, k, stride, activation=act), gold, 'layer.%s.' % name))
        close(layer(t('layer.x')), 'layer.%s.y' % name)
        with torch.no_grad():
            close(layer(t('layer.x')), 'layer.%s.y' % name)
    close(kept(_fill(bb.DarknetBlock(4, 8, 2), gold, 'block.'))(t('block.x')), 'block.y')
    header = kept(_fill(bb.Yolo3Header(6, 8, 11, pyramid_channels=5), gold, 'header.'))
    pred, conv5 = header(t('header.bottom'), t('header.pyramid'))
    close(conv5, 'header.conv5')
    close(pred, 'header.pred')


def test_running_statistics_are_batch_norms(gpu):
    torch.manual_seed(1)
    plain = _layer(16, 24, 3, 1, True, 'float32', 'float32', gpu)
    kept = _layer(16, 24, 3, 1, True, 'float32', 'int8', gpu)
    kept.load_state_dict(plain.state_dict())
    x = torch.randn(3, 16, 10, 9, device=gpu).contiguous(memory_format=torch.channels_last)
    for _ in range(2):
        plain(x)
        kept(x)
    for name in ('running_mean', 'running_var'):
        assert torch.allclose(getattr(plain.bn, name), getattr(kept.bn, name), rtol=1e-5, atol=1e-6)
    assert int(kept.bn.num_batches_tracked) == int(plain.bn.num_batches_tracked) == 2
    # a stack put into evaluation mode normalises with them
    assert torch.allclose(plain.eval()(x), kept.eval()(x), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize('kernel,stride,act,shortcut', [(1, 1, True, False), (1, 1, False, False), (3, 1, True, True), (3, 2, True, False)])
def test_gradients_of_a_layer_with_checkpoints(gpu, kernel, stride, act, shortcut):
    """Against autograd in 64 bits without any code.  The checkpoint's xhat is off by at most half a step of its row, the
    convolution's input by at most half a step of its own: dz moves by off_z (as derived for the normalisation), the
    weights' gradient by off_z * |x| + |dz| * half a step of x, the input's by off_z * |w|."""
    torch.manual_seed(10 * kernel + stride)
    cin, cout = 20, 24
    layer = _layer(cin, cout, kernel, stride, act, 'float32', 'int8', gpu)
    x = torch.randn(2, cin, 9, 11)
    slope = bb.LEAKY_SLOPE if act else 1.0
    d = lambda t: t.detach().cpu().double()
    x64 = d(x).requires_grad_()
    p = {k: d(v).requires_grad_() for k, v in layer.named_parameters()}
    padded = bb._pad_same(x64, kernel, stride)
    z = F.conv2d(padded, p['conv.weight'], p['conv.bias'], stride)
    z.retain_grad()
    xhat = (z - z.mean((0, 2, 3), keepdim=True)) / torch.sqrt(z.var((0, 2, 3), unbiased=False, keepdim=True) + bb.BN_EPSILON)
    u = xhat * p['bn.weight'].view(1, -1, 1, 1) + p['bn.bias'].view(1, -1, 1, 1)
    res = torch.randn_like(u)
    da = torch.randn_like(u) * (u.detach().abs() > 1e-3)          # elements next to zero could land on either side in float32
    a = torch.where(u > 0, u, slope * u) + (res if shortcut else 0)
    (a * da).sum().backward()

    cl = lambda t: t.detach().float().to(gpu).contiguous(memory_format=torch.channels_last)
    xg, rg = cl(x).requires_grad_(), cl(res).requires_grad_()
    out = layer(xg, residual=rg if shortcut else None)
    assert torch.allclose(out.detach().cpu().double(), a.detach(), rtol=1e-4, atol=1e-4)
    (out * cl(da)).sum().backward()
    if shortcut:
        assert torch.equal(rg.grad.cpu(), da.float())

    m = z.numel() // cout
    half_n = xhat.detach().abs().amax(1, keepdim=True) / 63 / 2 * (1 + 1e-3)
    du = torch.where(u.detach() > 0, da, slope * da)
    off_gamma = (du.abs() * half_n).sum((0, 2, 3))
    g = (p['bn.weight'].detach().abs() / torch.sqrt(z.detach().var((0, 2, 3), unbiased=False) + bb.BN_EPSILON)).view(1, -1, 1, 1)
    v = lambda t: t.view(1, -1, 1, 1)
    off_z = g * ((xhat.detach().abs() + half_n) * v(off_gamma) + half_n * v((du * xhat.detach()).sum((0, 2, 3)).abs())) / m
    size_z = g * (du.abs() + v(du.abs().mean((0, 2, 3))) + xhat.detach().abs() * v((du * xhat.detach()).abs().mean((0, 2, 3))))
    half_x = padded.detach().abs().amax(1, keepdim=True) / 127 / 2 * (1 + 1e-3)
    from torch.nn.grad import conv2d_input, conv2d_weight
    wshape, pshape = p['conv.weight'].shape, padded.shape
    ax = padded.detach().abs()
    dz = z.grad.abs()
    wg = lambda xx, zz: conv2d_weight(xx, wshape, zz, stride)
    rel = (1 + 4 * np.sqrt(3 * m)) * qc.U * 4                    # float32 sums over the rows, and dz's own float32 steps
    bound_w = wg(ax, off_z) + wg(half_x.expand_as(ax), dz + off_z) + rel * wg(ax, size_z)
    assert ((d(layer.conv.weight.grad) - p['conv.weight'].grad).abs() <= bound_w).all()
    bound_x = conv2d_input(pshape, p['conv.weight'].detach().abs(), off_z + rel * size_z, stride)
    top, left = bb.same_padding(9, kernel, stride)[0], bb.same_padding(11, kernel, stride)[0]
    bound_x = bound_x[:, :, top:top + 9, left:left + 11]
    assert ((d(xg.grad) - x64.grad).abs() <= bound_x).all()
    assert ((d(layer.bn.weight.grad) - p['bn.weight'].grad).abs() <= off_gamma + rel * (du * xhat.detach()).abs().sum((0, 2, 3))).all()
    assert ((d(layer.bn.bias.grad) - p['bn.bias'].grad).abs() <= rel * du.abs().sum((0, 2, 3))).all()


def test_pointwise_layer_in_integers(gpu):
    """linear_int8 and its gradients through a layer: the codes' own arithmetic in 64 bits."""
    torch.manual_seed(3)
    layer = _layer(48, 40, 1, 1, False, 'int8', 'float32', gpu)
    x = torch.randn(2, 48, 7, 5, device=gpu).contiguous(memory_format=torch.channels_last).requires_grad_()
    rows = x.permute(0, 2, 3, 1)
    z = quant.linear_int8(rows, layer.conv.weight.reshape(40, 48), layer.conv.bias)
    assert torch.equal(layer(x), layer.bn(z.permute(0, 3, 1, 2)))
    q, s = qc.rows_of(rows.detach().cpu().reshape(-1, 48).numpy())
    wq, ws = qc.rows_of(layer.conv.weight.detach().cpu().reshape(40, 48).numpy())
    xv, wv = q * s[:, None].astype(np.float64), wq * ws[:, None].astype(np.float64)
    want = xv @ wv.T + qc.f64(layer.conv.bias)
    zf = qc.f64(z).reshape(-1, 40)
    assert (np.abs(zf - want) <= 3 * qc.U * np.abs(xv @ wv.T) + 2.1 * qc.U * np.abs(want)).all()
    dz = torch.randn_like(z)
    z.backward(dz)
    d = qc.f64(dz).reshape(-1, 40)
    assert (np.abs(qc.f64(layer.conv.weight.grad).reshape(40, 48) - d.T @ xv) <= qc.sum_bound(np.abs(d).T @ np.abs(xv), 3 * 70)).all()
    assert (np.abs(qc.f64(layer.conv.bias.grad) - d.sum(0)) <= qc.sum_bound(np.abs(d).sum(0), 70)).all()
    gx = qc.f64(x.grad.permute(0, 2, 3, 1)).reshape(-1, 48)
    assert (np.abs(gx - d @ wv) <= qc.sum_bound(np.abs(d) @ np.abs(wv), 120)).all()
    with torch.no_grad():
        assert torch.equal(quant.linear_int8(rows, layer.conv.weight.reshape(40, 48), layer.conv.bias), z)


def test_inputs_of_few_channels_are_kept_as_they_are(gpu):
    torch.manual_seed(4)
    x = torch.randn(1, 3, 12, 12, device=gpu).contiguous(memory_format=torch.channels_last)
    w = torch.randn(8, 3, 3, 3, device=gpu, requires_grad=True)
    got, = torch.autograd.grad(quant.conv_kept(x, w, None, 1).square().sum(), w)
    want, = torch.autograd.grad(F.conv2d(x, w).square().sum(), w)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize('pointwise,checkpoints', [('float32', 'int8'), ('int8', 'float32'), ('int8', 'int8')])
def test_both_stacks_train_and_detect_with_the_options(gpu, pointwise, checkpoints):
    """Runs the class API with the options in its configuration: a training step moves every parameter that the plain
    stack's step moves, with finite values, and detection runs."""
    rng = np.random.default_rng(2)
    B, size, C = 2, 96, 3
    images = torch.from_numpy(rng.uniform(0, 255, size=(B, size, size, 3)).astype(np.float32)).cuda()
    gt = torch.from_numpy(y.synth.make_ground_truth(3, B, 2, 4, size, C)).cuda()

    def batches():
        while True:
            yield images, gt
    base = dict(mode='train', data_shape=[size, size, 3], num_classes=C, weight_decay=1e-4, keep_prob=0.5,
                data_format='channels_last', batch_size=B, coord_scale=1, noobj_scale=1, obj_scale=5., class_scale=1.,
                nms_score_threshold=0.5, nms_max_boxes=10, nms_iou_threshold=0.5, rescore_confidence=False,
                pointwise=pointwise, checkpoints=checkpoints)
    for cls, extra in ((y.YOLOv2, dict(priors=[[1., 1.], [2., 1.5]])), (y.YOLOv3, dict(num_priors=3, priors=y.synth.V3_PRIORS))):
        torch.manual_seed(6)
        prov = dict(num_train=2 * B, num_val=0, train_generator=(None, batches()), val_generator=None)
        net = cls(dict(base, **extra), prov)
        assert np.isfinite(float(net.train_one_epoch(1e-4)))
        stack = net.head_provider
        assert (stack.pointwise, stack.checkpoints) == (pointwise, checkpoints)
        params = dict(stack.named_parameters())
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in params.values())
        assert all(float(p.grad.abs().max()) > 0 for n, p in params.items() if n.endswith(('conv.weight', 'bn.weight', 'bn.bias')))
        scores, bbox, class_id = net.test_one_image(images[:1])
        assert np.isfinite(scores).all() and bbox.shape == (len(scores), 4)


def test_a_step_with_checkpoints_holds_less_memory(gpu):
    torch.manual_seed(7)
    held = {}
    images = torch.rand(8, 160, 160, 3, device=gpu) * 255
    for mode in ('float32', 'int8'):
        net = bb.Darknet53Heads(4, 3, checkpoints=mode).to(gpu)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        heads = net(images)
        torch.cuda.synchronize()
        held[mode] = torch.cuda.memory_allocated() - before
        sum(h.square().mean() for h in heads).backward()
        del net, heads
    # two bytes and two scales of four bytes a pixel, of at least 32 channels, against twelve bytes (shortcut sums and
    # resized maps included): well under a half
    assert held['int8'] < held['float32'] / 2


def test_a_step_under_autocast(gpu):
    """The convolutions in bfloat16, the checkpoints beside them: gradients of the parameters' own type, near the plain
    stack's under the same autocast."""
    torch.manual_seed(9)
    grads = {}
    x = torch.randn(2, 32, 12, 12, device=gpu).contiguous(memory_format=torch.channels_last)
    da = torch.randn(2, 48, 12, 12, device=gpu)
    for mode in ('float32', 'int8'):
        for kernel in (1, 3):
            torch.manual_seed(9)
            layer = _layer(32, 48, kernel, 1, True, 'float32', mode, gpu)
            with torch.autocast('cuda', dtype=torch.bfloat16):
                out = layer(x)
            (out.float() * da).sum().backward()
            grads[mode, kernel] = layer.conv.weight.grad
            assert layer.conv.weight.grad.dtype == torch.float32 and torch.isfinite(layer.conv.weight.grad).all()
    for kernel in (1, 3):
        a, b = grads['int8', kernel], grads['float32', kernel]
        # bfloat16 convolutions (2^-8 a term) and codes (2^-8 of a row's largest) on both sides of sums over 288 pixels
        assert float((a - b).norm() / b.norm()) < 0.05


def _pointwise_layer(gpu):
    torch.manual_seed(21)
    layer = _layer(64, 48, 1, 1, True, 'int8', 'int8', gpu)
    x = torch.randn(2, 64, 13, 13, device=gpu).contiguous(memory_format=torch.channels_last).requires_grad_()
    res = torch.randn(2, 48, 13, 13, device=gpu).contiguous(memory_format=torch.channels_last)
    da = torch.randn(2, 48, 13, 13, device=gpu).contiguous(memory_format=torch.channels_last)
    return layer, x, res, da


def test_a_graph_kept_for_a_second_backward_gives_the_same_again(gpu):
    layer, x, res, da = _pointwise_layer(gpu)
    leaves = [x] + list(layer.parameters())
    out = layer(x, residual=res)
    first = torch.autograd.grad(out, leaves, da, retain_graph=True)
    second = torch.autograd.grad(out, leaves, da)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, da)


def test_a_layer_captured_with_its_backward_replays_beside_eager_steps(gpu):
    layer, x, res, da = _pointwise_layer(gpu)
    leaves = [x] + list(layer.parameters())

    def step():
        out = layer(x, residual=res)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, da))

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream(gpu).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(4):
        torch.manual_seed(100 + seed)
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            da.copy_(torch.randn_like(da))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [g.clone() for g in got]
        assert all(torch.equal(a, b) for a, b in zip(replayed, step()))


def test_options_are_checked():
    with pytest.raises(ValueError, match='pointwise'):
        bb.Darknet19Head(2, 1, pointwise='int4')
    with pytest.raises(ValueError, match='checkpoints'):
        bb.Darknet53Heads(2, 3, checkpoints='bf16')


OPTIONS = [('float32', 'int8'), ('int8', 'float32'), ('int8', 'int8')]


@pytest.mark.parametrize('pointwise,checkpoints', OPTIONS)
def test_a_layer_whose_weights_a_hook_makes(gpu, pointwise, checkpoints):
    """torch.nn.utils.prune sets conv.weight in a hook before each call."""
    from torch.nn.utils import prune
    torch.manual_seed(34)
    layers = [_layer(32, 24, 1, 1, True, *mode, gpu) for mode in (('float32', 'float32'), (pointwise, checkpoints))]
    layers[1].load_state_dict(layers[0].state_dict())
    x = torch.randn(2, 32, 9, 7, device=gpu)
    fresh, mask = torch.randn(24, 32, 1, 1, device=gpu), torch.rand(24, 32, 1, 1, device=gpu) > 0.5
    for layer in layers:
        prune.custom_from_mask(layer.conv, 'weight', mask)
        with torch.no_grad():
            layer.conv.weight_orig.copy_(fresh)
    want, got = (layer(x) for layer in layers)
    # as the stack's golden values are compared: the same convolution, the normalisation in float32
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize('pointwise,checkpoints', OPTIONS)
def test_hooks_of_the_modules_inside_run(gpu, pointwise, checkpoints):
    torch.manual_seed(35)
    block = bb.DarknetBlock(16, 32, 1)
    for m in block.modules():
        if isinstance(m, bb.ConvBN):
            m.pointwise, m.checkpoints = pointwise, checkpoints
    block.to(gpu).train()
    x, seen = torch.randn(2, 16, 8, 8, device=gpu), []
    want = block(x)
    unit = block.units[0]
    for name, m in (('unit', unit), ('second', unit[1]), ('conv', unit[0].conv), ('bn', unit[0].bn)):
        m.register_forward_hook(lambda m, a, out, name=name: seen.append((name, out)))
    got = block(x)
    seen = dict(seen)
    assert set(seen) == {'unit', 'second', 'conv', 'bn'}
    down = block.down(x)
    assert torch.equal(seen['unit'], seen['second']) and torch.allclose(down + seen['unit'], got, rtol=1e-5, atol=1e-5)
    if pointwise == 'float32':
        assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)


class _HalvedConv(torch.nn.Conv2d):
    def forward(self, x):
        return super().forward(x) * torch.linspace(0, 1, x.shape[-1], device=x.device)


class _ShiftedNorm(torch.nn.BatchNorm2d):
    def forward(self, x):
        return super().forward(x) + 1


@pytest.mark.parametrize('pointwise,checkpoints', OPTIONS)
@pytest.mark.parametrize('swap', ['conv', 'dilation', 'bn'])
def test_modules_put_in_the_place_of_a_layers_own_are_called(gpu, swap, pointwise, checkpoints):
    torch.manual_seed(36)
    layers = [_layer(32, 24, 1 if swap != 'dilation' else 3, 1, True, *mode, gpu) for mode in (('float32', 'float32'), (pointwise, checkpoints))]
    x = torch.randn(2, 32, 9, 7, device=gpu)
    new = {'conv': lambda: _HalvedConv(32, 24, 1), 'dilation': lambda: torch.nn.Conv2d(32, 24, 3, dilation=2),
           'bn': lambda: _ShiftedNorm(24)}[swap]
    for layer in layers:
        setattr(layer, 'conv' if swap in ('conv', 'dilation') else 'bn', new().to(gpu))
    layers[1].load_state_dict(layers[0].state_dict())
    want, got = (layer(x) for layer in layers)
    if swap in ('conv', 'dilation') or pointwise == 'float32':
        assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)
    else:                        # the codes of both operands: 0.7 % each of a deviation, five times that at the most of 24 x 126
        assert float((got - want).abs().max()) < 0.1


def test_cumulative_statistics(gpu):
    """momentum None: running statistics are the batches' mean, as torch.optim.swa_utils.update_bn sets it."""
    from torch.optim.swa_utils import update_bn
    torch.manual_seed(37)
    plain = _layer(16, 24, 3, 1, True, 'float32', 'float32', gpu)
    kept = _layer(16, 24, 3, 1, True, 'float32', 'int8', gpu)
    kept.load_state_dict(plain.state_dict())
    batches = [torch.randn(3, 16, 10, 9, device=gpu) * (i + 1) for i in range(3)]
    for layer in (plain, kept):
        update_bn(batches, layer)
    assert int(kept.bn.num_batches_tracked) == 3
    for name in ('running_mean', 'running_var'):
        assert torch.allclose(getattr(plain.bn, name), getattr(kept.bn, name), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize('change', [dict(affine=False), dict(track_running_stats=False), dict(momentum=None)])
def test_normalisations_of_other_settings(gpu, change):
    torch.manual_seed(38)
    layers = [_layer(16, 24, 3, 1, True, 'float32', mode, gpu) for mode in ('float32', 'int8')]
    for layer in layers:
        layer.bn = torch.nn.BatchNorm2d(24, **change).to(gpu)
    layers[1].load_state_dict(layers[0].state_dict())
    for _ in range(2):
        x = torch.randn(2, 16, 9, 7, device=gpu)
        want, got = (layer(x) for layer in layers)
        assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)
    for (name, a), (_, b) in zip(layers[0].named_buffers(), layers[1].named_buffers()):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6), name


@pytest.mark.parametrize('autocast', [False, True])
@pytest.mark.parametrize('kind', ['type', 'broadcast'])
def test_a_shortcut_of_another_type_or_shape_is_added_as_by_the_plain_layer(gpu, kind, autocast):
    """The plain layer's sum promotes and broadcasts.  The product in integers, so that two calls give the same bits."""
    torch.manual_seed(31)
    layer = _layer(16, 24, 1, 1, True, 'int8', 'int8', gpu)
    x = torch.randn(2, 16, 9, 7, device=gpu)
    shape = (2, 24, 9, 7) if kind == 'type' else (1, 24, 1, 1)
    res = torch.randn(shape, device=gpu, dtype=torch.float32 if autocast else torch.float64 if kind == 'type' else torch.float32).requires_grad_()
    with torch.autocast('cuda', dtype=torch.bfloat16, enabled=autocast):
        out, alone = layer(x, residual=res), layer(x)
    assert out.dtype == (torch.result_type(res, alone)) and torch.equal(out, res + alone)
    da = torch.randn_like(out)
    out.backward(da)
    assert torch.equal(res.grad, da.sum_to_size(shape))
    assert all(torch.isfinite(p.grad).all() for p in layer.parameters())


@pytest.mark.parametrize('checkpoints', ['float32', 'int8'])
def test_a_pointwise_layer_under_autocast_takes_the_types_of_the_plain_one(gpu, checkpoints):
    torch.manual_seed(32)
    layer = _layer(32, 48, 1, 1, True, 'int8', checkpoints, gpu)
    plain = _layer(32, 48, 1, 1, True, 'float32', 'float32', gpu)
    plain.load_state_dict(layer.state_dict())
    x = torch.randn(2, 32, 12, 12, device=gpu).requires_grad_()
    with torch.autocast('cuda', dtype=torch.bfloat16):
        out, want = layer(x), plain(x)
        half = layer(x.detach().bfloat16())
        assert layer(x.detach().half()).dtype == plain(x.detach().half()).dtype == torch.bfloat16
    assert out.dtype == want.dtype == torch.bfloat16
    assert torch.equal(out, half)
    out.sum().backward()
    assert x.grad.dtype == torch.float32 and all(p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all() for p in layer.parameters())


@pytest.mark.parametrize('pointwise,checkpoints', OPTIONS)
def test_a_residual_block_under_autocast(gpu, pointwise, checkpoints):
    """Forward and backward of a block with shortcuts: types, and the distance to the plain block under the same autocast.
    A rounding of relative size e (codes: a row's largest is about three deviations, so 3 / 127 / sqrt(12) = 0.7 % for each
    operand of a product; bfloat16 0.2 %) moves that share of the activations' inputs across zero, e * 0.8 of them, and each
    takes 0.9 of its gradient along: sqrt(0.008 * 0.8) * 0.9 = 7 % in the gradient for each of five layers on either path,
    16 % if they are independent; three times that for their correlation."""
    grads = {}
    x = torch.randn(2, 16, 16, 16, device=gpu)
    da = torch.randn(2, 32, 8, 8, device=gpu)
    for mode in (('float32', 'float32'), (pointwise, checkpoints)):
        torch.manual_seed(33)
        block = bb.DarknetBlock(16, 32, 2)
        for m in block.modules():
            if isinstance(m, bb.ConvBN):
                m.pointwise, m.checkpoints = mode
        block.to(gpu).to(memory_format=torch.channels_last).train()
        with torch.autocast('cuda', dtype=torch.bfloat16):
            out = block(x)
        assert out.dtype == torch.bfloat16
        (out.float() * da).sum().backward()
        grads[mode] = {n: p.grad for n, p in block.named_parameters()}
    for name, want in grads['float32', 'float32'].items():
        got = grads[pointwise, checkpoints][name]
        assert got.dtype == torch.float32 and torch.isfinite(got).all()
        if not name.endswith('conv.bias'):                       # zero but for roundings: the normalisation takes the mean off
            assert float((got - want).norm() / want.norm()) < 0.5, name


@pytest.mark.parametrize('stride', [2, (2, 2), [2, 2], (1, 2), (1,)])
def test_conv_kept_takes_the_strides_of_a_convolution(gpu, stride):
    """The output is the plain convolution's; the gradients are those of the values that the codes stand for."""
    torch.manual_seed(39)
    x = torch.randn(2, 16, 11, 9, device=gpu).contiguous(memory_format=torch.channels_last).requires_grad_()
    w, b = torch.randn(12, 16, 3, 3, device=gpu, requires_grad=True), torch.randn(12, device=gpu, requires_grad=True)
    out = quant.conv_kept(x, w, b, stride)
    held = quant.dequantize_rows(*quant.quantize_rows(x.permute(0, 2, 3, 1))).permute(0, 3, 1, 2).detach().requires_grad_()
    # sums of 144 terms of about 0.64 in float32, in any order: (1 + 4 sqrt(144)) 2^-24 * 92
    assert torch.allclose(out, F.conv2d(x, w, b, stride), rtol=0, atol=3e-4)
    dy = torch.randn_like(out)
    got = torch.autograd.grad(out, (x, w, b), dy)
    want = torch.autograd.grad(F.conv2d(held, w, b, stride), (held, w, b), dy)
    for g, v in zip(got, want):                              # the library's convolutions in float32 on both sides
        assert torch.allclose(g, v, rtol=1e-4, atol=1e-3)
    with torch.no_grad():
        assert torch.allclose(quant.conv_kept(x, w, b, stride), out, rtol=0, atol=3e-4)
