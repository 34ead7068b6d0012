"""The 8-bit row operators without a GPU: refusals of the Python layer and of the C ABI, workspace sizes, and
the plain statements that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

from yolo_tf_amd import _abi, quant
from tests import quant_cases as qc

OK = (0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000)        # addresses that the host never dereferences
F32, BF16, F16, I8 = 0, 1, 2, 3


def _refused(rc, code, text):
    assert rc == code, _abi.load().yh_last_error()
    assert text in _abi.load().yh_last_error().decode()


def test_no_cpu_path():
    x, q, s = torch.zeros(3, 8), torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)
    g = torch.ones(8)
    for call in (lambda: quant.quantize_rows(x), lambda: quant.dequantize_rows(q, s), lambda: quant.matmul_int8(x, q, s),
                 lambda: quant.weight_grad(x, q, s), lambda: quant.input_grad(x, q, s), lambda: quant.norm_act(x, g, g, 1e-3, 0.1),
                 lambda: quant.norm_act_backward(x, quant.NormKept(q, (3, 8), 3, 16, g, 0.1))):
        with pytest.raises(RuntimeError, match='no CPU path'):
            call()
    with pytest.raises(TypeError, match='torch tensor'):
        quant.quantize_rows(np.zeros((3, 8), np.float32))


def test_the_stack_options_have_no_cpu_path():
    from yolo_tf_amd import backbone as bb
    for option in (dict(pointwise='int8'), dict(checkpoints='int8')):
        net = bb.Darknet19Head(2, 1, **option)
        with pytest.raises(RuntimeError, match='no CPU path'):
            net(torch.zeros(1, 32, 32, 3))


def test_calls_without_a_device_say_so():
    if torch.cuda.is_available():
        pytest.skip('a HIP device is present')
    lib = _abi.load()
    _refused(lib.yh_quantize_rows(OK[0], F32, 8, 4, 8, OK[1], 16, OK[2], None), _abi.YH_ERR_NO_DEVICE, 'no HIP device')
    _refused(lib.yh_input_grad(OK[0], F32, 8, OK[1], 16, OK[2], 4, 8, 16, OK[3], 16, None), _abi.YH_ERR_NO_DEVICE, 'no HIP device')


def test_refusals_of_the_code_calls():
    lib = _abi.load()
    inv, lim, ali = _abi.YH_ERR_INVALID_ARG, _abi.YH_ERR_LIMIT, _abi.YH_ERR_ALIGN
    q = lambda x=OK[0], t=F32, ldx=8, rows=4, k=8, c=OK[1], ldc=16, s=OK[2]: lib.yh_quantize_rows(x, t, ldx, rows, k, c, ldc, s, None)
    _refused(q(t=I8), inv, 'dtype')
    _refused(q(t=9), inv, 'dtype')
    _refused(q(rows=-1), inv, 'negative')
    _refused(q(k=0), inv, 'channels')
    _refused(q(rows=_abi.YH_MAX_ROWS), lim, 'rows')
    _refused(q(k=_abi.YH_MAX_ROW_CHANNELS + 1), lim, 'channels')
    _refused(q(x=None), inv, 'x is null')
    _refused(q(x=0x1002), ali, 'x is not aligned')
    _refused(q(x=0x1001, t=BF16), ali, 'x is not aligned')
    _refused(q(c=None), inv, 'codes is null')
    _refused(q(s=None), inv, 'scale is null')
    _refused(q(s=0x2002), ali, 'scale')
    _refused(q(ldc=7), inv, 'codes: 7 elements')
    _refused(q(ldx=-8), inv, 'x: -8 elements')
    _refused(q(ldx=1 << 36), lim, 'not below 2^36')
    assert q(x=None, c=None, s=None, rows=0) == _abi.YH_OK            # nothing to do
    d = lambda c=OK[0], ldc=16, s=OK[1], rows=4, k=8, x=OK[2], t=F16, ldx=8: lib.yh_dequantize_rows(c, ldc, s, rows, k, x, t, ldx, None)
    _refused(d(t=I8), inv, 'dtype')
    _refused(d(ldx=7), inv, 'x: 7 elements')
    _refused(d(x=0x2001), ali, 'x is not aligned')
    _refused(d(s=None), inv, 'scale is null')
    assert d(rows=0) == _abi.YH_OK


def test_refusals_of_the_products():
    lib = _abi.load()
    inv, lim, ali, wsp = _abi.YH_ERR_INVALID_ARG, _abi.YH_ERR_LIMIT, _abi.YH_ERR_ALIGN, _abi.YH_ERR_WORKSPACE

    def m(x=OK[0], xt=F32, ldx=8, xs=None, rows=4, k=8, w=OK[1], ldw=8, ws=OK[2], n=5, b=None, y=OK[3], yt=F32, ldy=5, c=None, ldc=0,
          s=None, work=OK[4], size=1 << 20):
        return lib.yh_matmul_int8(x, xt, ldx, xs, rows, k, w, ldw, ws, n, b, y, yt, ldy, c, ldc, s, work, size, None)

    _refused(m(xt=4), inv, 'x_dtype')
    _refused(m(yt=I8), inv, 'y_dtype')
    _refused(m(xs=OK[5]), inv, 'x_scale belongs')
    _refused(m(xt=I8), inv, 'x_scale is null')
    _refused(m(xt=I8, xs=OK[5], c=OK[5], ldc=8, s=OK[6]), inv, 'given as codes')
    _refused(m(c=OK[5], ldc=8), inv, 'scale is null')
    _refused(m(s=OK[5], ldc=8), inv, 'codes is null')
    _refused(m(c=OK[5], ldc=7, s=OK[6]), inv, 'codes: 7')
    _refused(m(w=None), inv, 'w is null')
    _refused(m(ws=None), inv, 'w_scale is null')
    _refused(m(b=0x7002), ali, 'bias')
    _refused(m(ldy=4), inv, 'y: 4')
    wide = dict(rows=5000, k=5000, ldx=5000, ldw=5000)               # a size whose codes pass through a workspace
    _refused(m(work=None, **wide), wsp, 'workspace')
    _refused(m(size=5000 * 5000 - 1, **wide), wsp, 'workspace')
    _refused(m(work=0x5008, size=1 << 30, **wide), ali, 'workspace')
    _refused(m(k=1 << 16, n=1 << 16), lim, 'weights')
    _refused(m(rows=(1 << 26) - 65, k=1 << 15), lim, '2^36')
    _refused(m(rows=1 << 20, n=1 << 16), lim, '2^36')
    assert m(rows=0) == _abi.YH_OK

    def wg(dy=OK[0], t=F32, ld=5, c=OK[1], ldc=8, s=OK[2], rows=100000, n=5, k=8, dw=OK[3], db=OK[4], work=OK[5], size=1 << 30):
        return lib.yh_weight_grad(dy, t, ld, c, ldc, s, rows, n, k, dw, db, work, size, None)

    _refused(wg(t=I8), inv, 'dtype')
    _refused(wg(dy=None), inv, 'dy is null')
    _refused(wg(c=None), inv, 'codes is null')
    _refused(wg(s=None), inv, 'scale is null')
    _refused(wg(dw=None), inv, 'dw is null')
    _refused(wg(db=0x4002), ali, 'db')
    _refused(wg(work=None), wsp, 'workspace')
    _refused(wg(size=16), wsp, 'workspace')
    ig = lambda dy=OK[0], t=F32, ld=5, w=OK[1], ldw=8, ws=OK[2], rows=4, n=5, k=8, dx=OK[3], ldx=8: lib.yh_input_grad(
        dy, t, ld, w, ldw, ws, rows, n, k, dx, ldx, None)
    _refused(ig(t=I8), inv, 'dtype')
    _refused(ig(ldx=7), inv, 'dx: 7')
    _refused(ig(ws=None), inv, 'w_scale is null')
    _refused(ig(dx=0x4001, t=F16), ali, 'dx')
    assert ig(rows=0) == _abi.YH_OK


def test_refusals_of_the_norm():
    lib = _abi.load()
    inv, ali, wsp = _abi.YH_ERR_INVALID_ARG, _abi.YH_ERR_ALIGN, _abi.YH_ERR_WORKSPACE

    def f(z=OK[0], ldz=8, r=None, ldr=0, t=F32, rows=4, c=8, g=OK[1], b=OK[1], eps=1e-3, a=OK[2], lda=8, kept=OK[3], ldk=16, s=OK[4],
          mean=OK[5], inv_=OK[5], rm=None, rv=None, work=OK[6], size=1 << 20):
        return lib.yh_norm_act_forward(z, ldz, r, ldr, t, rows, c, g, b, eps, 0.1, a, lda, kept, ldk, s, mean, inv_, rm, rv, 0.01,
                                       work, size, None)

    _refused(f(rows=0), inv, 'no rows')
    _refused(f(t=I8), inv, 'dtype')
    _refused(f(eps=-1e-9), inv, 'eps')
    _refused(f(eps=float('nan')), inv, 'eps')
    _refused(f(g=None), inv, 'gamma')
    _refused(f(mean=None), inv, 'mean')
    _refused(f(kept=None), inv, 'kept and scale')
    _refused(f(s=None), inv, 'kept and scale')
    _refused(f(rm=OK[0]), inv, 'running_mean and running_var')
    _refused(f(r=0x1002), ali, 'residual')
    _refused(f(lda=7), inv, 'a: 7')
    _refused(f(ldk=7), inv, 'kept: 7')
    _refused(f(rows=100000, size=8), wsp, 'workspace')

    def b(da=OK[0], ld=8, t=F32, rows=4, c=8, kept=OK[1], ldk=8, s=OK[2], g=OK[3], i=OK[3], dz=OK[4], ldz=8, dg=OK[5], db=OK[5],
          work=OK[6], size=1 << 20):
        return lib.yh_norm_act_backward(da, ld, t, rows, c, kept, ldk, s, g, i, 0.1, dz, ldz, dg, db, work, size, None)

    _refused(b(rows=0), inv, 'no rows')
    _refused(b(kept=None), inv, 'kept is null')
    _refused(b(s=None), inv, 'scale')
    _refused(b(dg=None), inv, 'dgamma')
    _refused(b(dz=0x5002), ali, 'dz')
    _refused(b(rows=100000, work=None), wsp, 'workspace')


def test_workspace_sizes():
    lib = _abi.load()
    n = ctypes.c_size_t(7)
    ask = lambda fn, *a: (_abi.check(fn(*a, ctypes.byref(n))), n.value)[1]
    # zero, or the codes and their scales
    for rows, k, n_out in ((1, 1, 1), (100, 33, 5), (5000, 5000, 500), (173056, 256, 128), (43264, 1536, 425), (60000, 1000, 1000)):
        assert ask(lib.yh_matmul_int8_workspace_bytes, rows, k, n_out, F32, 0) in (0, rows * ((k + 15) // 16 * 16 + 4))
        assert ask(lib.yh_matmul_int8_workspace_bytes, rows, k, n_out, F32, 1) == 0
        assert ask(lib.yh_matmul_int8_workspace_bytes, rows, k, n_out, I8, 0) == 0
    assert ask(lib.yh_matmul_int8_workspace_bytes, 5000, 5000, 500, F32, 0) > 0
    assert ask(lib.yh_weight_grad_workspace_bytes, 0, 64, 64) == 0
    # the pieces of the rows never take more than their number times the result, and that number is bounded
    for rows, a, b in ((1, 1, 1), (700000, 64, 128), (10816, 512, 1024), (50000, 1536, 1536)):
        assert ask(lib.yh_weight_grad_workspace_bytes, rows, a, b) <= 1024 * (a * b + a) * 4
    assert ask(lib.yh_norm_act_workspace_bytes, 1, 1, F32) == 0                # few rows are summed by one workgroup a channel
    assert 0 < ask(lib.yh_norm_act_workspace_bytes, 700000, 64, BF16) <= 64 * 1100 * 16
    assert lib.yh_norm_act_workspace_bytes(0, 8, F32, ctypes.byref(n)) == _abi.YH_ERR_INVALID_ARG
    for fn, a in ((lib.yh_matmul_int8_workspace_bytes, (1, 1, 1, 0, 0)), (lib.yh_weight_grad_workspace_bytes, (1, 1, 1)),
                  (lib.yh_norm_act_workspace_bytes, (1, 1, 0))):
        _refused(fn(*a, None), _abi.YH_ERR_INVALID_ARG, 'bytes is null')


def test_the_plain_statement_of_the_codes():
    x = np.array([[0, 0, 0], [127, 1.5, -2.5], [1, 0.25, -1], [2.0 ** -111, 0, 0], [np.inf, 1, 2], [np.nan, 0, 0]], np.float32)
    q, s = qc.rows_of(x)
    assert q.tolist() == [[0, 0, 0], [127, 2, -2], [127, 32, -127], [0, 0, 0], [0, 0, 0], [0, 0, 0]]
    assert s[:2].tolist() == [0, 1] and s[3] == 0 and np.isnan(s[4:]).all()


def test_channel_counts_that_do_not_fit_a_call_are_refused(monkeypatch):
    """2^32 + 5 channels would reach the library as 5."""
    monkeypatch.setattr(quant, '_device_of', lambda x, what: x.device)            # tensors without memory
    most = _abi.YH_MAX_ROW_CHANNELS
    meta = lambda *shape, dtype=torch.float32: torch.empty(shape, device='meta', dtype=dtype)
    codes = lambda *shape: meta(*shape, dtype=torch.int8)
    for n in (most + 1, 2 ** 31, 2 ** 32 + 5):
        g = meta(n)
        for call in (lambda: quant.quantize_rows(meta(1, n)), lambda: quant.dequantize_rows(codes(1, n), meta(1)),
                     lambda: quant.matmul_int8(meta(2, n), codes(3, n), meta(3)), lambda: quant.matmul_int8(meta(2, 4), codes(n, 4), g),
                     lambda: quant.weight_grad(meta(2, n), codes(2, 4), meta(2)), lambda: quant.weight_grad(meta(2, 4), codes(2, n), meta(2)),
                     lambda: quant.input_grad(meta(2, n), codes(n, 4), g), lambda: quant.input_grad(meta(2, 4), codes(4, n), meta(4)),
                     lambda: quant.norm_act(meta(2, n), g, g, 1e-3, 0.1)):
            with pytest.raises(_abi.YhError, match='channels exceed') as refusal:
                call()
            assert refusal.value.code == _abi.YH_ERR_LIMIT
    assert quant._rows(meta(3, most), 'x')[1:] == (3, most, most)


def test_a_convolution_with_hooks_or_of_another_kind_is_called():
    """... by a layer that would otherwise run its product in integers, which the CPU refuses."""
    from yolo_tf_amd import backbone as bb

    class Doubled(torch.nn.Conv2d):
        def forward(self, x):
            return 2 * super().forward(x)
    x, seen = torch.randn(2, 8, 5, 5, requires_grad=True), []
    for change in (lambda m: m.conv.register_forward_hook(lambda *a: seen.append('after')),
                   lambda m: m.conv.register_forward_pre_hook(lambda *a: seen.append('before')),
                   lambda m: m.conv.register_full_backward_hook(lambda *a: seen.append('backward')),
                   lambda m: setattr(m, 'conv', Doubled(8, 4, 1)), lambda m: setattr(m, 'conv', torch.nn.Conv2d(8, 4, 1, groups=4)),
                   lambda m: setattr(m.conv, 'forward', lambda x: x[:, :4])):
        layer = bb.ConvBN(8, 4, 1)
        layer.pointwise = 'int8'
        with pytest.raises(RuntimeError, match='no CPU path'):
            layer(x)
        change(layer)
        layer(x).sum().backward()
    assert sorted(seen) == ['after', 'backward', 'before']
