"""Row operators in 8 bits for the convolution stacks: activation checkpoints, the
pointwise (1x1) convolution in 8-bit integers with its gradients, and batch
normalisation with leaky ReLU on an 8-bit checkpoint (kernels: csrc/yh_rows.hip,
csrc/yh_product.hip; declarations and definitions: include/yolohead.h).

A "row" is one pixel: tensors are [..., channels] in float32, bfloat16 or float16
on a HIP device, NHWC for an activation; leading dimensions that have one stride
between them (a channel slice of a wider tensor, say) are read in place, others are
copied first.  Calls go to the current stream of the tensors' device; outputs and
scratch come from torch's allocator, so a call can be captured into a graph.  There
is no CPU path: without a HIP device these functions raise.

The functions of the first half compute; the second half binds them to autograd, for
backbone.ConvBN (`pointwise='int8'`, `checkpoints='int8'`).  Their gradients take
the roundings for the identity (straight through) and cannot be differentiated
again.  As with every autograd function, a backward pass is captured into a graph
only while no eager graph of the same parameters is alive."""
import ctypes

import torch
import torch.nn.functional as F
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _abi

_TYPES = {torch.float32: _abi.YH_FLOAT32, torch.bfloat16: _abi.YH_BFLOAT16, torch.float16: _abi.YH_FLOAT16}


# ------------------------------------------------------------------ helpers
# The smallest calls take a few microseconds on the device, so the host's share counts: no call makes a tensor, a view
# or a library query that it can do without.
_sizes = {}                  # workspace sizes by (query, its arguments): they depend on nothing else


def _device_of(x, what):
    if not isinstance(x, torch.Tensor):
        raise TypeError('%s must be a torch tensor on a HIP device' % what)
    dev = x.device
    if dev.type != 'cuda':
        raise RuntimeError('%s must live on a HIP device (got %s); there is no CPU path' % (what, dev))
    return dev


def _float_type(dtype, what):
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError('%s must be float32, bfloat16 or float16, got %s' % (what, dtype))
    return code


def _check_channels(n, what):
    """Refuses what the library would, before a count beyond 32 bits is cut to what fits its argument."""
    if n > _abi.YH_MAX_ROW_CHANNELS:
        raise _abi.YhError(_abi.YH_ERR_LIMIT, '%s: %d channels exceed %d' % (what, n, _abi.YH_MAX_ROW_CHANNELS))


def _rows(x, what):
    """x as [rows, channels] with adjacent channels: (tensor that owns the memory, rows, channels, elements between rows)."""
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError('%s must be [..., channels] with at least one channel, got %s' % (what, tuple(shape)))
    cols = shape[-1]
    _check_channels(cols, what)
    if x.is_contiguous():
        return x, x.numel() // cols, cols, cols
    x = x.detach()
    if x.dim() != 2:
        x = x.reshape(-1, cols)
    if cols > 1 and x.stride(1) != 1:
        x = x.contiguous()
    rows = x.shape[0]
    return x, rows, cols, x.stride(0) if rows > 1 else cols


def _vector(v, n, dev, what):
    """A float32 vector of n adjacent values on `dev`."""
    if not isinstance(v, torch.Tensor) or v.dtype != torch.float32 or v.device != dev or v.numel() != n:
        raise ValueError('%s must be %d float32 values on %s' % (what, n, dev))
    return v if v.is_contiguous() else v.detach().contiguous()


def _codes(q, dev, what):
    if not isinstance(q, torch.Tensor) or q.dtype != torch.int8 or q.device != dev:
        raise ValueError('%s must be int8 codes on %s' % (what, dev))
    return _rows(q, what)


def _new_codes(x, shape):
    """int8 codes of x's `shape` whose rows start at multiples of 16 bytes: a view of a wider buffer where needed."""
    cols = shape[-1]
    if cols % 16 == 0:
        return x.new_empty(shape, dtype=torch.int8), cols
    wide = (cols + 15) // 16 * 16
    return x.new_empty(shape[:-1] + (wide,), dtype=torch.int8)[..., :cols], wide


def _call(dev, fn, *args):
    """One library call on `dev`'s current stream."""
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        _abi.check(rc)


def _scratch(fn_name, owner, *sizes):
    """(pointer, bytes, tensor that keeps it) of a workspace for one call, on the device of the tensor `owner`."""
    n = _sizes.get((fn_name, sizes))
    if n is None:
        out = ctypes.c_size_t(0)
        _abi.check(getattr(_abi.load(), fn_name)(*sizes, ctypes.byref(out)))
        if len(_sizes) > 4096:
            _sizes.clear()
        n = _sizes[(fn_name, sizes)] = out.value
    if n == 0:
        return None, 0, None
    ws = owner.new_empty(n, dtype=torch.uint8)
    return ws.data_ptr(), n, ws


# ------------------------------------------------------------------ row codes
def quantize_rows(x):
    """(codes int8 shaped like x, scale float32 [...]) of the rows of x: scale = max|x| / 127, code =
    x / scale rounded.  A row of zeros has the scale 0; one with an infinity or a NaN the scale NaN."""
    dev = _device_of(x, 'x')
    kind = _float_type(x.dtype, 'x')
    xr, rows, cols, ld = _rows(x, 'x')
    shape = tuple(x.shape)
    codes, ldc = _new_codes(x, shape)
    scale = x.new_empty(shape[:-1], dtype=torch.float32)
    _call(dev, _abi.load().yh_quantize_rows, xr.data_ptr(), kind, ld, rows, cols, codes.data_ptr(), ldc, scale.data_ptr())
    return codes, scale


def dequantize_rows(codes, scale, dtype=torch.float32):
    """The values that row codes stand for: codes * scale, in `dtype`."""
    dev = _device_of(codes, 'codes')
    kind = _float_type(dtype, 'dtype')
    qr, rows, cols, ld = _codes(codes, dev, 'codes')
    scale = _vector(scale, rows, dev, 'scale')
    x = codes.new_empty(codes.shape, dtype=dtype)
    _call(dev, _abi.load().yh_dequantize_rows, qr.data_ptr(), ld, scale.data_ptr(), rows, cols, x.data_ptr(), kind, cols)
    return x


# ------------------------------------------------------------------ products
def matmul_int8(x, w_codes, w_scale, bias=None, x_scale=None, out_dtype=None, want_codes=False):
    """A pointwise convolution in 8-bit integers: x [..., K] times the rows of w_codes [N, K], scaled by each
    row's and each output channel's scale, plus bias [N]: [..., N] in out_dtype (default: x's type).
    x: float rows, whose codes are taken within the call; or int8 codes with x_scale [...] (out_dtype then
    defaults to float32).  w_codes, w_scale: quantize_rows of the weights.  want_codes: returns
    (y, codes, scale), the checkpoint that weight_grad reads."""
    dev = _device_of(x, 'x')
    lib = _abi.load()
    xr, rows, k, ldx = _rows(x, 'x')
    wr, n, wk, ldw = _codes(w_codes, dev, 'w_codes')
    if w_codes.dim() != 2 or wk != k:
        raise ValueError('w_codes must be [N, %d], got %s' % (k, tuple(w_codes.shape)))
    _check_channels(n, 'w_codes')
    w_scale = _vector(w_scale, n, dev, 'w_scale')
    if bias is not None:
        bias = _vector(bias, n, dev, 'bias')
    whole = x.dtype == torch.int8
    if whole:
        if x_scale is None or want_codes:
            raise ValueError('int8 codes need x_scale, and are the codes already')
        kind, x_scale = _abi.YH_INT8, _vector(x_scale, rows, dev, 'x_scale')
        out_dtype = torch.float32 if out_dtype is None else out_dtype
    else:
        if x_scale is not None:
            raise ValueError('x_scale belongs to int8 codes')
        kind = _float_type(x.dtype, 'x')
        out_dtype = x.dtype if out_dtype is None else out_dtype
    out_kind = _float_type(out_dtype, 'out_dtype')
    shape = tuple(x.shape)
    y = x.new_empty(shape[:-1] + (n,), dtype=out_dtype)
    codes = scale = None
    ldc = 0
    if want_codes:
        codes, ldc = _new_codes(x, shape)
        scale = x.new_empty(shape[:-1], dtype=torch.float32)
    ws, nbytes, keep = _scratch('yh_matmul_int8_workspace_bytes', x, rows, k, n, kind, 1 if want_codes else 0)
    _call(dev, lib.yh_matmul_int8, xr.data_ptr(), kind, ldx, x_scale.data_ptr() if whole else None, rows, k,
          wr.data_ptr(), ldw, w_scale.data_ptr(), n, None if bias is None else bias.data_ptr(), y.data_ptr(), out_kind, n,
          codes.data_ptr() if want_codes else None, ldc, scale.data_ptr() if want_codes else None, ws, nbytes)
    return (y, codes, scale) if want_codes else y


def weight_grad(dy, codes, scale, want_bias=False):
    """dw [N, K] float32 = dy^T times the values of the row codes, from dy [..., N] and codes [..., K] with
    scale [...]; with want_bias (dw, db [N]), db the sum of dy's rows."""
    dev = _device_of(dy, 'dy')
    kind = _float_type(dy.dtype, 'dy')
    dr, rows, n, ldd = _rows(dy, 'dy')
    qr, qrows, k, ldq = _codes(codes, dev, 'codes')
    if qrows != rows:
        raise ValueError('dy has %d rows, codes %d' % (rows, qrows))
    scale = _vector(scale, rows, dev, 'scale')
    dw = dy.new_empty((n, k), dtype=torch.float32)
    db = dy.new_empty((n,), dtype=torch.float32) if want_bias else None
    ws, nbytes, keep = _scratch('yh_weight_grad_workspace_bytes', dy, rows, n, k)
    _call(dev, _abi.load().yh_weight_grad, dr.data_ptr(), kind, ldd, qr.data_ptr(), ldq, scale.data_ptr(), rows, n, k,
          dw.data_ptr(), db.data_ptr() if want_bias else None, ws, nbytes)
    return (dw, db) if want_bias else dw


def input_grad(dy, w_codes, w_scale):
    """dx [..., K] in dy's type = dy [..., N] times the values of the weight codes [N, K]."""
    dev = _device_of(dy, 'dy')
    kind = _float_type(dy.dtype, 'dy')
    dr, rows, n, ldd = _rows(dy, 'dy')
    wr, wn, k, ldw = _codes(w_codes, dev, 'w_codes')
    if w_codes.dim() != 2 or wn != n:
        raise ValueError('w_codes must be [%d, K], got %s' % (n, tuple(w_codes.shape)))
    w_scale = _vector(w_scale, n, dev, 'w_scale')
    dx = dy.new_empty(tuple(dy.shape[:-1]) + (k,))
    _call(dev, _abi.load().yh_input_grad, dr.data_ptr(), kind, ldd, wr.data_ptr(), ldw, w_scale.data_ptr(), rows, n, k,
          dx.data_ptr(), k)
    return dx


# ------------------------------------------------------------------ normalisation
class NormKept:
    """What norm_act leaves for norm_act_backward: one byte a value (`kept`: the activation's side and xhat in seven
    bits) with a scale for each row, mean and invstd [C] float32, and the call's gamma and slope.  Everything but gamma
    lies in one buffer, `store`: rows * pitch bytes, the scales, mean, invstd; the rest are views of it."""

    __slots__ = ('store', 'shape', 'rows', 'pitch', 'gamma', 'slope')

    def __init__(self, store, shape, rows, pitch, gamma, slope):
        self.store, self.shape, self.rows, self.pitch, self.gamma, self.slope = store, shape, rows, pitch, gamma, slope

    def _floats(self, at, n):
        begin = self.rows * (self.pitch + (4 if self.pitch else 0)) if at else self.rows * self.pitch
        begin += 4 * self.shape[-1] if at == 2 else 0
        return self.store[begin:begin + 4 * n].view(torch.float32)

    @property
    def kept(self):
        """int8, shaped like z; None if nothing was kept."""
        if not self.pitch:
            return None
        return self.store[:self.rows * self.pitch].view(torch.int8).view(self.shape[:-1] + (self.pitch,))[..., :self.shape[-1]]

    @property
    def scale(self):
        return self._floats(0, self.rows).view(self.shape[:-1]) if self.pitch else None

    @property
    def mean(self):
        return self._floats(1, self.shape[-1])

    @property
    def invstd(self):
        return self._floats(2, self.shape[-1])


def norm_act(z, gamma, beta, eps, slope, residual=None, running=None, momentum=0.01, want_kept=True):
    """Batch normalisation of z [..., C] on its own statistics, leaky ReLU of `slope` (1: none) and a shortcut:
    (a shaped like z, NormKept), NormKept without its checkpoint if want_kept is False.
    running: (mean, var) buffers [C], updated in place with `momentum` as torch.nn.BatchNorm2d does (one row
    counts its variance as it is)."""
    dev = _device_of(z, 'z')
    kind = _float_type(z.dtype, 'z')
    zr, rows, c, ldz = _rows(z, 'z')
    gr, beta = _vector(gamma, c, dev, 'gamma'), _vector(beta, c, dev, 'beta')
    rr, ldr = None, 0
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != z.shape or residual.dtype != z.dtype or residual.device != dev:
            raise ValueError('residual must be %s in %s on %s' % (tuple(z.shape), z.dtype, dev))
        rr, _, _, ldr = _rows(residual, 'residual')
    rm = rv = None
    if running is not None:
        rm, rv = running
        for t in (rm, rv):
            if _vector(t, c, dev, 'running').data_ptr() != t.data_ptr():
                raise ValueError('the running statistics must be contiguous: they are updated in place')
    shape, slope = tuple(z.shape), float(slope)
    a = z.new_empty(shape)
    pitch = (c + 15) // 16 * 16 if want_kept else 0
    head = rows * (pitch + 4) if want_kept else 0
    store = z.new_empty(head + 8 * c, dtype=torch.uint8)
    at = store.data_ptr()
    ws, nbytes, keep = _scratch('yh_norm_act_workspace_bytes', z, rows, c, kind)
    _call(dev, _abi.load().yh_norm_act_forward, zr.data_ptr(), ldz, None if rr is None else rr.data_ptr(), ldr, kind, rows, c,
          gr.data_ptr(), beta.data_ptr(), float(eps), slope, a.data_ptr(), c,
          at if want_kept else None, pitch, at + rows * pitch if want_kept else None, at + head, at + head + 4 * c,
          None if rm is None else rm.data_ptr(), None if rv is None else rv.data_ptr(), float(momentum), ws, nbytes)
    return a, NormKept(store, shape, rows, pitch, gamma, slope)


def norm_act_backward(da, kept):
    """(dz, dgamma [C], dbeta [C]) of norm_act from a's gradient and the NormKept (which reads gamma as it is now); the
    residual's gradient is da."""
    dev = _device_of(da, 'da')
    kind = _float_type(da.dtype, 'da')
    if not kept.pitch:
        raise ValueError('the forward call kept nothing (want_kept=False)')
    if tuple(da.shape) != kept.shape or kept.store.device != dev:
        raise ValueError('da must be shaped like the forward call\'s z, %s, on %s; got %s' % (kept.shape, kept.store.device, tuple(da.shape)))
    dr, rows, c, ldd = _rows(da, 'da')
    gamma = _vector(kept.gamma, c, dev, 'gamma')
    dz = da.new_empty(kept.shape)
    dgamma, dbeta = da.new_empty(c, dtype=torch.float32), da.new_empty(c, dtype=torch.float32)
    at = kept.store.data_ptr()
    scale = at + rows * kept.pitch
    ws, nbytes, keep = _scratch('yh_norm_act_workspace_bytes', da, rows, c, kind)
    _call(dev, _abi.load().yh_norm_act_backward, dr.data_ptr(), ldd, kind, rows, c, at, kept.pitch, scale,
          gamma.data_ptr(), scale + 4 * rows + 4 * c, kept.slope, dz.data_ptr(), c, dgamma.data_ptr(), dbeta.data_ptr(), ws, nbytes)
    return dz, dgamma, dbeta


# ------------------------------------------------------------------ autograd
class _LinearInt8(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, keep):
        w_codes, w_scale = quantize_rows(weight)
        ctx.types = weight.dtype, None if bias is None else bias.dtype
        bias = None if bias is None else bias.float()
        if not keep:
            return matmul_int8(x, w_codes, w_scale, bias)
        y, codes, scale = matmul_int8(x, w_codes, w_scale, bias, want_codes=True)
        ctx.save_for_backward(codes, scale, w_codes, w_scale)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scale, w_codes, w_scale = ctx.saved_tensors
        dx = input_grad(dy, w_codes, w_scale) if ctx.needs_input_grad[0] else None
        dw = db = None
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw, db = weight_grad(dy, codes, scale, want_bias=True)
            dw = dw.to(ctx.types[0])
            db = None if ctx.types[1] is None else db.to(ctx.types[1])
        return dx, dw, db, None


def linear_int8(x, weight, bias=None):
    """x [..., K] times weight [N, K] (float, quantised by its rows in the call) plus bias, in 8-bit integers, with
    gradients: the codes of x are the checkpoint that the weights' gradient is computed from.  The result has x's type,
    under autocast too."""
    return _LinearInt8.apply(x, weight, bias, torch.is_grad_enabled())


KEEP_CODES_FROM = 8          # channels; shorter rows take no less memory as codes (rows of 16 bytes and a scale)


class _ConvKept(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, stride):
        y = F.conv2d(x, weight, bias, stride)
        codes, scale = quantize_rows(x.permute(0, 2, 3, 1))
        ctx.save_for_backward(codes, scale, weight)
        ctx.stride, ctx.has_bias, ctx.dtype = stride, bias is not None, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scale, weight = ctx.saved_tensors
        n, k = weight.shape[:2]
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        own = weight.to(dy.dtype)                           # under autocast the convolution ran in dy's type
        dx = dw = db = None
        if weight.shape[2:] == (1, 1) and ctx.stride == (1, 1):
            rows = dy.permute(0, 2, 3, 1)
            if need_x:
                dx = (rows.reshape(-1, n) @ own.reshape(n, k)).view(codes.shape).permute(0, 3, 1, 2)
            if need_w or need_b:
                dw, db = weight_grad(rows, codes, scale, want_bias=True)
                dw = dw.view(weight.shape)
        else:
            x = dequantize_rows(codes, scale, dy.dtype).permute(0, 3, 1, 2)
            dx, dw, db = torch.ops.aten.convolution_backward(dy.contiguous(memory_format=torch.channels_last), x, own, [n] if ctx.has_bias else None,
                                                             ctx.stride, [0, 0], [1, 1], False, [0, 0], 1, [need_x, need_w, need_b and ctx.has_bias])
        return (dx.to(ctx.dtype) if need_x else None, dw.to(weight.dtype) if need_w else None,
                db.to(weight.dtype) if need_b and ctx.has_bias else None, None)


def conv_kept(x, weight, bias, stride):
    """F.conv2d(x, weight, bias, stride) of an NCHW tensor that keeps x for the backward pass as row codes (a byte a
    value and a scale a pixel) in the place of x itself.  The output is the plain convolution's; the weights'
    gradient is that of the values the codes stand for.  stride: one number or two."""
    stride = (int(stride),) * 2 if not isinstance(stride, (tuple, list)) else (int(stride[0]), int(stride[-1]))
    if not torch.is_grad_enabled() or x.shape[1] < KEEP_CODES_FROM:
        return F.conv2d(x, weight, bias, stride)
    return _ConvKept.apply(x, weight, bias, stride)


class _NormAct(Function):
    @staticmethod
    def forward(ctx, z, gamma, beta, eps, slope, residual, running, momentum, keep):
        a, kept = norm_act(z, gamma, beta, eps, slope, residual, running, momentum, want_kept=keep)
        if keep:
            ctx.save_for_backward(kept.store, gamma)
            ctx.layout = kept.shape, kept.rows, kept.pitch, kept.slope
        return a

    @staticmethod
    @once_differentiable
    def backward(ctx, da):
        store, gamma = ctx.saved_tensors
        shape, rows, pitch, slope = ctx.layout
        dz, dgamma, dbeta = norm_act_backward(da, NormKept(store, shape, rows, pitch, gamma, slope))
        return dz, dgamma, dbeta, None, None, da if ctx.needs_input_grad[5] else None, None, None, None


def norm_act_kept(z, gamma, beta, eps, slope, residual=None, running=None, momentum=0.01):
    """norm_act with gradients for z, gamma, beta and the residual, from its 8-bit checkpoint."""
    return _NormAct.apply(z, gamma, beta, eps, slope, residual, running, momentum, torch.is_grad_enabled())
