"""The 8-bit row operators (yolo_tf_amd.quant) against plain statements in 64 bits."""
import numpy as np
import pytest
import torch

from yolo_tf_amd import quant
from tests import quant_cases as qc

pytestmark = pytest.mark.gpu

# rows and channels: one, odd, wavefront and tile edges, several row plans, a row longer than a wavefront's registers
SHAPES = [(1, 1), (1, 1024), (3, 5), (7, 64), (65, 33), (127, 255), (33, 771), (130, 1536), (9, 6150), (4099, 32), (41, 2048), (21, 3001), (5, 4097)]


def _randn(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32))


def _hard_rows(rng, m, k):
    """Rows of many sizes, some zero, one constant, one with a single value far above the others."""
    x = _randn(rng, m, k) * torch.exp(3 * _randn(rng, m, 1))
    if m > 2:
        x[1] = 0
        x[2] = 0.25
    if m > 5:
        x[3] *= 2.0 ** -120                       # under the smallest row that counts
        x[4] *= 1e30
        x[5, k // 2] = 1e6
    return x


# ------------------------------------------------------------------ codes
@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,k', SHAPES)
def test_row_codes_are_the_definitions(gpu, m, k, dtype):
    rng = np.random.default_rng(m * 7 + k)
    x = _hard_rows(rng, m, k)
    if dtype == torch.float16:
        x = x.clamp(-60000, 60000)
    x = x.to(dtype)
    codes, scale = quant.quantize_rows(x.to(gpu))
    q, s = qc.rows_of(x.float().numpy())
    assert codes.shape == x.shape and scale.shape == (m,)
    assert np.array_equal(scale.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), q)
    for out in qc.TYPES:
        back = quant.dequantize_rows(codes, scale, out).cpu()
        want = (torch.from_numpy(q).float() * torch.from_numpy(s)[:, None]).to(out)
        assert back.dtype == out and torch.equal(back, want)


def test_codes_are_within_half_a_step_and_ties_go_to_even(gpu):
    # with a largest value of 127 the scale is 1 and r is 1: halves are ties
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5, 3.49, -3.51]])
    codes, scale = quant.quantize_rows(x.to(gpu))
    assert scale.item() == 1.0
    assert codes.cpu().tolist() == [[127, 0, 2, 2, 0, -2, 126, -126, 3, -4]]
    rng = np.random.default_rng(3)
    x = _randn(rng, 64, 300)
    codes, scale = quant.quantize_rows(x.to(gpu))
    back = qc.f64(codes) * qc.f64(scale)[:, None]
    # half a step, and the rounding of r and of the scale, each half a float32 step of at most 127 steps
    assert (np.abs(back - qc.f64(x)) <= qc.f64(scale)[:, None] * (0.5 + 2 * 127 * qc.U)).all()


def test_rows_with_infinities_and_nans_become_nan_and_no_other_row(gpu):
    rng = np.random.default_rng(4)
    x = _randn(rng, 40, 96)
    x[3, 95] = float('inf')
    x[4, 0] = float('nan')
    x[5, 7] = -float('inf')
    codes, scale = quant.quantize_rows(x.to(gpu))
    q, s = qc.rows_of(x.numpy())
    assert np.array_equal(scale.cpu().numpy(), s, equal_nan=True) and np.isnan(s[3:6]).all()
    assert np.array_equal(codes.cpu().numpy(), q)
    w, ws = quant.quantize_rows(_randn(rng, 17, 96).to(gpu))
    y = quant.matmul_int8(x.to(gpu), w, ws)
    assert torch.isnan(y[3:6]).all() and torch.isfinite(y[:3]).all() and torch.isfinite(y[6:]).all()


@pytest.mark.parametrize('dtype', qc.TYPES)
def test_strides_of_every_kind_are_read_in_place_or_copied(gpu, dtype):
    rng = np.random.default_rng(5)
    wide = _randn(rng, 6, 5, 4, 83).to(dtype).to(gpu)
    views = [wide[..., 3:70], wide[:, ::2, :, 1:], wide.permute(0, 3, 1, 2), wide[0, 0].t(), wide[:, :, :, :1],
             wide[0, 0, :1].expand(7, 83), wide[..., 0:64:2], wide[1:2, 2:3, 1:2]]
    for v in views:
        codes, scale = quant.quantize_rows(v)
        want_codes, want_scale = quant.quantize_rows(v.contiguous().clone())
        assert codes.shape == v.shape and torch.equal(codes, want_codes) and torch.equal(scale, want_scale)


@pytest.mark.parametrize('m,k,n,pitch', [(37, 45, 21, 61), (9001, 45, 21, 61), (9001, 450, 300, 461)])
def test_nothing_behind_a_row_or_the_last_row_is_written(gpu, m, k, n, pitch):
    import ctypes
    from yolo_tf_amd import _abi
    lib = _abi.load()
    rng = np.random.default_rng(6)
    x = _randn(rng, m, k).to(gpu)
    codes = torch.full((m + 2, pitch), 55, dtype=torch.int8, device=gpu)
    scale = torch.full((m + 2,), -7.0, device=gpu)
    st = ctypes.c_void_p(torch.cuda.current_stream(gpu).cuda_stream)
    _abi.check(lib.yh_quantize_rows(x.data_ptr(), 0, k, m, k, codes.data_ptr(), pitch, scale.data_ptr(), st))
    assert (codes[:m, k:] == 55).all() and (codes[m:] == 55).all() and (scale[m:] == -7).all()
    for kind, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        out = torch.full((m + 2, pitch), 9.0, dtype=dtype, device=gpu)
        _abi.check(lib.yh_dequantize_rows(codes.data_ptr(), pitch, scale.data_ptr(), m, k, out.data_ptr(), kind, pitch, st))
        assert (out[:m, k:] == 9).all() and (out[m:] == 9).all() and (out[:m, :k] != 9).any()
        w, ws = quant.quantize_rows(_randn(rng, n, k).to(gpu))
        y = torch.full((m + 2, pitch), 9.0, dtype=dtype, device=gpu)
        _abi.check(lib.yh_matmul_int8(codes.data_ptr(), 3, pitch, scale.data_ptr(), m, k, w.data_ptr(), w.stride(0), ws.data_ptr(), n,
                                      None, y.data_ptr(), kind, pitch, None, 0, None, None, 0, st))
        assert (y[:m, n:] == 9).all() and (y[m:] == 9).all()
        dy = _randn(rng, m, n).to(dtype).to(gpu)
        dx = torch.full((m + 2, pitch), 9.0, dtype=dtype, device=gpu)
        _abi.check(lib.yh_input_grad(dy.data_ptr(), kind, n, w.data_ptr(), w.stride(0), ws.data_ptr(), m, n, k, dx.data_ptr(), pitch, st))
        assert (dx[:m, k:] == 9).all() and (dx[m:] == 9).all()


# ------------------------------------------------------------------ products
PRODUCTS = [(1, 1, 1), (1, 1024, 255), (2, 77, 3), (5, 16, 64), (16, 65, 17), (40, 64, 32), (129, 255, 130), (300, 129, 257),
            (169, 1024, 512), (2000, 48, 27), (6000, 256, 640), (8, 6000, 20),
            # weights kept in LDS: one to sixteen lanes a row, whole and ragged rows; large tiles with a ragged end
            (9000, 20, 16), (5000, 100, 130), (4500, 129, 200), (4500, 256, 70), (8200, 300, 64), (12000, 300, 520), (17000, 512, 256),
            (16500, 100, 130), (20001, 255, 100), (16390, 256, 70), (16385, 300, 64),
            # matrices and last tiles of fewer than four columns
            (700, 1, 90), (701, 2, 90), (702, 3, 40), (500, 130, 66), (400, 258, 70)]


def _layer(rng, k, n, dev):
    w = _randn(rng, n, k) * float(np.sqrt(2.6 / k)) * torch.exp(_randn(rng, n, 1))
    return quant.quantize_rows(w.to(dev))


def _product_bound(p, y, out):
    # the sum as a float32, two products, one addition, each half a step; one rounding to the output's type
    return 3 * qc.U * np.abs(p) + (qc.U + qc.HALF_STEP[out]) * 1.01 * np.abs(y) + qc.TINY[out]


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,k,n', PRODUCTS)
def test_integer_product(gpu, m, k, n, dtype):
    rng = np.random.default_rng(m + 3 * k + 5 * n)
    x = (_randn(rng, m, k) * torch.exp(_randn(rng, m, 1))).to(dtype)
    w, ws = _layer(rng, k, n, gpu)
    bias = _randn(rng, n)
    y, codes, scale = quant.matmul_int8(x.to(gpu), w, ws, bias.to(gpu), want_codes=True)
    q, s = qc.rows_of(x.float().numpy())
    assert np.array_equal(codes.cpu().numpy(), q) and np.array_equal(scale.cpu().numpy(), s)
    p = (q @ qc.f64(w).T) * s.astype(np.float64)[:, None] * qc.f64(ws)[None, :]
    want = p + qc.f64(bias)[None, :]
    assert y.dtype == dtype and y.shape == (m, n)
    assert (np.abs(qc.f64(y) - want) <= _product_bound(p, want, dtype)).all()
    # the other forms of the call: without the codes, from the codes, without a bias
    assert torch.equal(quant.matmul_int8(x.to(gpu), w, ws, bias.to(gpu)), y)
    assert torch.equal(quant.matmul_int8(codes, w, ws, bias.to(gpu), x_scale=scale, out_dtype=dtype), y)
    bare = quant.matmul_int8(codes, w, ws, x_scale=scale, out_dtype=dtype)
    assert (np.abs(qc.f64(bare) - p) <= _product_bound(p, p, dtype)).all()


def test_integer_product_at_the_ends_of_the_codes(gpu):
    """Every code +-127: the largest sums; with 65536 terms they reach 2^30 and have to stay whole."""
    m, k, n = 3, 65536, 5
    x = torch.full((m, k), 127, dtype=torch.int8, device=gpu)
    x[1] = -127
    w = torch.full((n, k), 127, dtype=torch.int8, device=gpu)
    w[2, 1::2] = -127
    one = torch.ones(8, device=gpu)
    y = quant.matmul_int8(x, w, one[:n], x_scale=one[:m])
    want = qc.f64(x) @ qc.f64(w).T
    assert np.array_equal(qc.f64(y), want.astype(np.float32).astype(np.float64))


def _grads(rng, m, n, dtype):
    return (_randn(rng, m, n) * torch.exp(_randn(rng, m, 1)) * 1e-3).to(dtype)


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,k,n', PRODUCTS + [(0, 40, 30), (70000, 32, 64), (33001, 250, 512), (16640, 512, 512)])
def test_weight_gradient(gpu, m, k, n, dtype):
    rng = np.random.default_rng(m + 7 * k + n)
    dy = _grads(rng, m, n, dtype)
    x = _randn(rng, m, k) * torch.exp(_randn(rng, m, 1))
    codes, scale = quant.quantize_rows(x.to(gpu))
    dw, db = quant.weight_grad(dy.to(gpu), codes, scale, want_bias=True)
    d, xv = qc.f64(dy), qc.f64(codes) * qc.f64(scale)[:, None]
    assert dw.shape == (n, k) and db.shape == (n,) and dw.dtype == db.dtype == torch.float32
    # three products to a term
    assert (np.abs(qc.f64(dw) - d.T @ xv) <= qc.sum_bound(np.abs(d).T @ np.abs(xv), 3 * m) + 1e-36).all()
    assert (np.abs(qc.f64(db) - d.sum(0)) <= qc.sum_bound(np.abs(d).sum(0), m)).all()
    assert torch.equal(quant.weight_grad(dy.to(gpu), codes, scale), dw)


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,k,n', PRODUCTS)
def test_input_gradient(gpu, m, k, n, dtype):
    rng = np.random.default_rng(m + 11 * k + n)
    dy = _grads(rng, m, n, dtype)
    w, ws = _layer(rng, k, n, gpu)
    dx = quant.input_grad(dy.to(gpu), w, ws)
    d, wv = qc.f64(dy), qc.f64(w) * qc.f64(ws)[:, None]
    want = d @ wv
    assert dx.shape == (m, k) and dx.dtype == dtype
    bound = qc.sum_bound(np.abs(d) @ np.abs(wv), 3 * n) + qc.HALF_STEP[dtype] * 1.01 * np.abs(want) + qc.TINY[dtype] + 1e-36
    assert (np.abs(qc.f64(dx) - want) <= bound).all()


def test_gradients_against_differences(gpu):
    """The product is linear in the values of both operands: central differences of sum(dy * y) in 64 bits are its
    gradient up to the rounding of the differences themselves."""
    rng = np.random.default_rng(12)
    m, k, n = 6, 20, 9
    x, dy = _randn(rng, m, k), _randn(rng, m, n)
    w, ws = _layer(rng, k, n, gpu)
    codes, scale = quant.quantize_rows(x.to(gpu))
    dw, db = quant.weight_grad(dy.to(gpu), codes, scale, want_bias=True)
    dx = quant.input_grad(dy.to(gpu), w, ws)
    xv, wv, d = qc.f64(codes) * qc.f64(scale)[:, None], qc.f64(w) * qc.f64(ws)[:, None], qc.f64(dy)
    b = np.zeros(n)

    def loss(xv, wv, b):
        return float((d * (xv @ wv.T + b)).sum())

    h = 2.0 ** -10
    for grad, arg in ((dx, 0), (dw, 1), (db, 2)):
        at = [xv, wv, b]
        flat = qc.f64(grad).reshape(-1)
        for i in range(0, flat.size, 7):
            up, down = [a.copy() for a in at], [a.copy() for a in at]
            up[arg].reshape(-1)[i] += h
            down[arg].reshape(-1)[i] -= h
            diff = (loss(*up) - loss(*down)) / (2 * h)
            # at most 20 terms a gradient, of magnitudes below 8 here; the differences lose 2^-52 * |loss| / h
            assert abs(diff - flat[i]) <= (1 + 4 * np.sqrt(60)) * qc.U * 20 * 8 + 1e-9


def test_non_finite_gradients_reach_what_they_touch(gpu):
    rng = np.random.default_rng(13)
    m, k, n = 200, 48, 40
    dy = _randn(rng, m, n)
    dy[17, 5] = float('inf')
    dy[18, 6] = float('nan')
    w, ws = _layer(rng, k, n, gpu)
    dx = quant.input_grad(dy.to(gpu), w, ws).cpu()
    bad = torch.zeros(m, dtype=torch.bool)
    bad[17:19] = True
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    codes, scale = quant.quantize_rows(_randn(rng, m, k).to(gpu))
    dw, db = quant.weight_grad(dy.to(gpu), codes, scale, want_bias=True)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[5:7] = True
    assert torch.isnan(dw.cpu()[bad]).all() and torch.isfinite(dw.cpu()[~bad]).all()
    assert not torch.isfinite(db.cpu()[bad]).any() and torch.isfinite(db.cpu()[~bad]).all()


# ------------------------------------------------------------------ normalisation
NORMS = [(1, 1), (1, 40), (2, 3), (8, 1), (7, 64), (169, 1024), (333, 255), (50, 771), (64, 1536), (5, 6150), (4100, 32), (20000, 7), (700, 2049), (333, 4096), (31, 4100), (3001, 1300), (9, 3001)]


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,c', NORMS)
def test_norm_forward(gpu, m, c, dtype):
    rng = np.random.default_rng(m + c)
    z = (_randn(rng, m, c) * torch.exp(0.5 * _randn(rng, c)) + 3 * _randn(rng, c)).to(dtype)
    res = _randn(rng, m, c).to(dtype)
    gamma, beta = 1 + 0.3 * _randn(rng, c), 0.3 * _randn(rng, c)
    running = [_randn(rng, c).to(gpu), _randn(rng, c).abs().to(gpu)]
    before = [qc.f64(t) for t in running]
    eps, slope = 1e-3, 0.1
    a, kept = quant.norm_act(z.to(gpu), gamma.to(gpu), beta.to(gpu), eps, slope, residual=res.to(gpu), running=running, momentum=0.01)
    z64 = qc.f64(z)
    mean, var = z64.mean(0), z64.var(0)
    # the statistics are computed in 64 bits and rounded once
    one = 1.001 * qc.U
    assert (np.abs(qc.f64(kept.mean) - mean) <= one * np.abs(mean) + 1e-12).all()
    assert (np.abs(qc.f64(kept.invstd) - 1 / np.sqrt(var + eps)) <= one / np.sqrt(var + eps)).all()
    unbiased = var * (m / (m - 1)) if m > 1 else var
    for got, old, new in zip(running, before, (mean, unbiased)):
        want = 0.99 * old + 0.01 * new
        assert (np.abs(qc.f64(got) - want) <= one * np.abs(want) + 1e-12).all()
    # from the statistics on, every step is a float32 operation of its own: the same bits
    zf, rf = z.float().numpy(), res.float().numpy()
    want, xhat, side = qc.normed(zf, gamma.numpy(), beta.numpy(), kept.mean.cpu().numpy(), kept.invstd.cpu().numpy(), slope, rf)
    assert a.dtype == dtype and torch.equal(a.cpu(), torch.from_numpy(want).to(dtype))
    q, s = qc.rows_of(xhat, 63)
    assert np.array_equal(kept.scale.cpu().numpy(), s)
    assert np.array_equal(kept.kept.cpu().numpy(), (2 * q + side).astype(np.int8))
    # and without the options
    bare, none = quant.norm_act(z.to(gpu), gamma.to(gpu), beta.to(gpu), eps, slope, want_kept=False)
    want, _, _ = qc.normed(zf, gamma.numpy(), beta.numpy(), kept.mean.cpu().numpy(), kept.invstd.cpu().numpy(), slope)
    assert torch.equal(bare.cpu(), torch.from_numpy(want).to(dtype)) and none.kept is None
    with pytest.raises(ValueError, match='kept nothing'):
        quant.norm_act_backward(bare, none)


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,c', NORMS)
def test_norm_backward(gpu, m, c, dtype):
    rng = np.random.default_rng(2 * m + c)
    z = (_randn(rng, m, c) + _randn(rng, c)).to(dtype)
    gamma, beta = 1 + 0.3 * _randn(rng, c), 0.3 * _randn(rng, c)
    da = _grads(rng, m, c, dtype)
    slope = np.float32(0.1)
    _, kept = quant.norm_act(z.to(gpu), gamma.to(gpu), beta.to(gpu), 1e-3, float(slope))
    dz, dgamma, dbeta = quant.norm_act_backward(da.to(gpu), kept)
    byte = kept.kept.cpu().numpy()
    side = (byte & 1).astype(bool)
    xq = ((byte >> 1).astype(np.float32) * kept.scale.cpu().numpy()[:, None]).astype(np.float64)
    d32 = da.float().numpy()
    du = np.where(side, d32, (slope * d32).astype(np.float32)).astype(np.float64)
    one = 1.001 * qc.U
    for got, terms in ((dbeta, du), (dgamma, du * xq)):
        assert (np.abs(qc.f64(got) - terms.sum(0)) <= one * np.abs(terms.sum(0)) + 2.0 ** -45 * np.abs(terms).sum(0)).all()
    g = qc.f64(gamma) * qc.f64(kept.invstd)
    cb, cg = du.sum(0) / m, (du * xq).sum(0) / m
    want = g * (du - cb - xq * cg)
    # on any of the three terms: the sum rounded, times 1 / M (two more), two subtractions, g (a product) and the product
    # with it, seven half steps in all; the third term has one more, from the product with xq
    bound = np.abs(g) * 8.01 * qc.U * (np.abs(du) + np.abs(cb) + np.abs(xq * cg)) + qc.HALF_STEP[dtype] * 1.01 * np.abs(want) + qc.TINY[dtype] + 1e-40
    assert dz.dtype == dtype and (np.abs(qc.f64(dz) - want) <= bound).all()


def test_norm_gradient_against_differences_of_the_exact_function(gpu):
    """Against the function without any rounding.  The checkpoint's xhat is off by half a step of its row (and a float32
    rounding), which moves dgamma by at most sum |du| * half steps and dz by the two products it enters."""
    rng = np.random.default_rng(21)
    m, c, eps, slope = 24, 6, 1e-3, 0.1
    z, da = _randn(rng, m, c), _randn(rng, m, c)
    gamma, beta = 1 + 0.3 * _randn(rng, c), 0.3 * _randn(rng, c)
    _, kept = quant.norm_act(z.to(gpu), gamma.to(gpu), beta.to(gpu), eps, slope)
    dz, dgamma, dbeta = (qc.f64(t) for t in quant.norm_act_backward(da.to(gpu), kept))
    z, da, gamma, beta = qc.f64(z), qc.f64(da), qc.f64(gamma), qc.f64(beta)

    def loss(z, gamma, beta):
        xhat = (z - z.mean(0)) / np.sqrt(z.var(0) + eps)
        u = xhat * gamma + beta
        return (da * np.where(u > 0, u, slope * u)).sum(), u, xhat

    _, u, xhat = loss(z, gamma, beta)
    h = 1e-6
    assert np.abs(u).min() > 50 * h                       # no element crosses zero in a difference
    inv = 1 / np.sqrt(z.var(0) + eps)
    du = np.where(u > 0, da, slope * da)
    half = 0.5 * qc.f64(kept.scale)[:, None] * (1 + 1e-4)
    off_gamma = (np.abs(du) * half).sum(0)
    off_z = np.abs(gamma * inv) * ((np.abs(xhat) + half) * off_gamma + half * np.abs((du * xhat).sum(0))) / m
    fd = 1e-8                                             # of the differences: h^2 and 2^-52 / h
    for i in range(m):
        for j in range(c):
            d = np.zeros((m, c))
            d[i, j] = h
            diff = (loss(z + d, gamma, beta)[0] - loss(z - d, gamma, beta)[0]) / (2 * h)
            assert abs(diff - dz[i, j]) <= off_z[i, j] + 1e-5 * abs(diff) + 1e-6 + fd
    for j in range(c):
        d = np.zeros(c)
        d[j] = h
        diff = (loss(z, gamma + d, beta)[0] - loss(z, gamma - d, beta)[0]) / (2 * h)
        assert abs(diff - dgamma[j]) <= off_gamma[j] + 1e-5 * abs(diff) + fd
        diff = (loss(z, gamma, beta + d)[0] - loss(z, gamma, beta - d)[0]) / (2 * h)
        assert abs(diff - dbeta[j]) <= 1e-5 * abs(diff) + 1e-6 + fd


def test_norm_statistics_survive_a_large_mean_and_a_constant_channel(gpu):
    rng = np.random.default_rng(22)
    m, c = 5000, 12
    z = _randn(rng, m, c)
    z[:, 3] = 7.5
    z[:, 4] += 1e5
    z[:, 5] = 1e6 + torch.round(z[:, 5] * 4) / 4
    ones, zeros = torch.ones(c), torch.zeros(c)
    a, kept = quant.norm_act(z.to(gpu), ones.to(gpu), zeros.to(gpu), 1e-3, 1.0)
    z64 = qc.f64(z)
    assert (np.abs(qc.f64(kept.mean) - z64.mean(0)) <= 1.001 * qc.U * np.abs(z64.mean(0)) + 1e-12).all()
    inv = 1 / np.sqrt(z64.var(0) + 1e-3)
    assert (np.abs(qc.f64(kept.invstd) - inv) <= 1.001 * qc.U * inv).all()
    assert (a[:, 3] == 0).all()


def test_norm_with_a_nan_channel_leaves_the_other_channels_activation(gpu):
    rng = np.random.default_rng(23)
    z = _randn(rng, 100, 16)
    z[5, 2] = float('nan')
    z[6, 9] = float('inf')
    a, kept = quant.norm_act(z.to(gpu), torch.ones(16, device=gpu), torch.zeros(16, device=gpu), 1e-3, 0.1)
    good = [c for c in range(16) if c not in (2, 9)]
    assert torch.isnan(a[:, [2, 9]]).all() and torch.isfinite(a[:, good]).all()
    dz, dgamma, dbeta = quant.norm_act_backward(torch.ones(100, 16, device=gpu), kept)
    assert torch.isnan(dz).all() and torch.isnan(dgamma).all() and torch.isfinite(dbeta[good]).all()


# ------------------------------------------------------------------ streams, graphs, offsets
def test_calls_follow_the_current_stream(gpu):
    rng = np.random.default_rng(31)
    x = _randn(rng, 5000, 256).to(gpu)
    w, ws = _layer(rng, 256, 96, gpu)
    want = quant.matmul_int8(x, w, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(gpu)
    for _ in range(3):
        with torch.cuda.stream(side):
            y = torch.empty(1 << 24, device=gpu).normal_()          # work in front of the call on its stream
            late = (y[:1] * 0).expand(5000, 256) + x
            got = quant.matmul_int8(late, w, ws)
        side.synchronize()
        assert torch.equal(got, want)


def test_a_training_step_captured_into_two_graphs_replays_beside_eager_calls(gpu):
    """Product, both gradients and a norm step in a graph; another graph and eager calls run between the replays."""
    rng = np.random.default_rng(32)

    def make(m, k, n):
        s = dict(x=_randn(rng, m, k).to(gpu), da=_randn(rng, m, n).to(gpu), gamma=(1 + 0.1 * _randn(rng, n)).to(gpu),
                 beta=(0.1 * _randn(rng, n)).to(gpu))
        s['w'], s['ws'] = _layer(rng, k, n, gpu)
        return s

    def step(s):
        z, codes, scale = quant.matmul_int8(s['x'], s['w'], s['ws'], want_codes=True)
        a, kept = quant.norm_act(z, s['gamma'], s['beta'], 1e-3, 0.1)
        dz, dg, db = quant.norm_act_backward(s['da'], kept)
        return [a, dz, dg, db, quant.weight_grad(dz, codes, scale), quant.input_grad(dz, s['w'], s['ws'])]

    states = [make(3000, 64, 128), make(169, 255, 40)]
    graphs, outs = [], []
    for s in states:
        side = torch.cuda.Stream(gpu)
        with torch.cuda.stream(side):
            step(s)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s)
        graphs.append(g)
        outs.append(out)
    for turn in range(4):
        for s in states:
            s['x'].copy_(_randn(rng, *s['x'].shape))
            s['da'].copy_(_randn(rng, *s['da'].shape))
        want = [step(s) for s in states]
        torch.cuda.synchronize()
        for g in (graphs if turn % 2 else graphs[::-1]):
            g.replay()
        again = step(states[0])
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert all(torch.equal(p, q) for p, q in zip(w, o))
        assert all(torch.equal(p, q) for p, q in zip(want[0], again))


def test_offsets_beyond_32_bits(gpu):
    """A buffer whose last rows lie past 2^32 elements (codes) and 2^31 (float32)."""
    rows, k, ld = 70001, 48, 65536
    codes = torch.empty((rows, ld), dtype=torch.int8, device=gpu)[:, :k]
    rng = np.random.default_rng(33)
    x = _randn(rng, rows, k).to(gpu)
    q, s = quant.quantize_rows(x)
    codes.copy_(q)
    assert codes.stride(0) * (rows - 1) > 2 ** 32
    w, ws = _layer(rng, k, 20, gpu)
    assert torch.equal(quant.matmul_int8(codes, w, ws, x_scale=s), quant.matmul_int8(q, w, ws, x_scale=s))
    dy = _randn(rng, rows, 20).to(gpu)
    assert torch.equal(quant.weight_grad(dy, codes, s), quant.weight_grad(dy, q, s))
    assert torch.equal(quant.dequantize_rows(codes, s), quant.dequantize_rows(q, s))
    del codes, q
    wide = torch.empty((rows, 32768), dtype=torch.float32, device=gpu)[:, :k]
    wide.copy_(x)
    assert wide.stride(0) * (rows - 1) > 2 ** 31
    for a, b in zip(quant.quantize_rows(wide), quant.quantize_rows(x)):
        assert torch.equal(a, b)
    ones = torch.ones(k, device=gpu)
    (a, ka), (b, kb) = quant.norm_act(wide, ones, ones, 1e-3, 0.1), quant.norm_act(x, ones, ones, 1e-3, 0.1)
    assert torch.equal(a, b) and torch.equal(ka.kept, kb.kept)
    for p, r in zip(quant.norm_act_backward(wide, ka), quant.norm_act_backward(x, kb)):
        assert torch.equal(p, r)
    assert torch.equal(quant.input_grad(wide, *_layer(np.random.default_rng(1), 9, k, gpu)), quant.input_grad(x, *_layer(np.random.default_rng(1), 9, k, gpu)))


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,k,n,gap', [(5, 7, 3, 1), (300, 37, 21, 9), (4500, 129, 130, 3), (40000, 30, 5, 2), (3000, 515, 70, 6), (60, 2051, 9, 5)])
def test_what_lies_between_the_rows_has_no_effect(gpu, m, k, n, gap, dtype):
    """Vectors may run over a row's end: the same bits whether NaN and whole codes lie there or the next row."""
    rng = np.random.default_rng(38)

    def apart(v):
        wide = torch.full((v.shape[0], v.shape[1] + gap), 127 if v.dtype == torch.int8 else float('nan'), dtype=v.dtype, device=gpu)
        wide[:, :v.shape[1]] = v
        return wide[:, :v.shape[1]]

    x, dy = _randn(rng, m, k).to(dtype).to(gpu), _randn(rng, m, n).to(dtype).to(gpu)
    w, ws = _layer(rng, k, n, gpu)
    q, s = (v.contiguous() for v in quant.quantize_rows(x))
    w = w.contiguous()
    for got, want in ((quant.quantize_rows(apart(x)), (q, s)),
                      ((quant.dequantize_rows(apart(q), s),), (quant.dequantize_rows(q, s),)),
                      (quant.matmul_int8(apart(x), apart(w), ws, want_codes=True), (quant.matmul_int8(x, w, ws), q, s)),
                      ((quant.matmul_int8(apart(q), apart(w), ws, x_scale=s),), (quant.matmul_int8(q, w, ws, x_scale=s),)),
                      (quant.weight_grad(apart(dy), apart(q), s, want_bias=True), quant.weight_grad(dy, q, s, want_bias=True)),
                      ((quant.input_grad(apart(dy), apart(w), ws),), (quant.input_grad(dy, w, ws),))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    gamma, beta = (1 + 0.1 * _randn(rng, k)).to(gpu), (0.1 * _randn(rng, k)).to(gpu)
    res = x.flip(0).contiguous()
    a, kept = quant.norm_act(apart(x), gamma, beta, 1e-3, 0.1, residual=apart(res))
    b, same = quant.norm_act(x, gamma, beta, 1e-3, 0.1, residual=res)
    assert torch.equal(a, b) and torch.equal(kept.kept, same.kept) and torch.equal(kept.scale, same.scale)
    da = _randn(rng, m, k).to(dtype).to(gpu)
    assert all(torch.equal(g, h) for g, h in zip(quant.norm_act_backward(apart(da), kept), quant.norm_act_backward(da, same)))


@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,n,k', [(1, 161, 1), (70, 1122, 13), (169, 512, 200), (130, 300, 3), (64, 193, 64)])
def test_input_grad_of_few_tiles(gpu, m, n, k, dtype):
    """Long sums taken by several teams: against 64 bits, the terms within the float32 sum's bound."""
    rng = np.random.default_rng(39)
    w, ws = _layer(rng, k, n, gpu)
    dy = _randn(rng, m, n).to(dtype)
    got = quant.input_grad(dy.to(gpu), w, ws).double().cpu()
    values = w.double().cpu() * ws.double().cpu()[:, None]
    want, size = dy.double() @ values, dy.double().abs() @ values.abs()
    # a term: one rounding of dy * w_scale; the sum: n + 3 additions of three pieces a term; the result's own rounding
    bound = size * (3 * n + 8) * 2.0 ** -24 + want.abs() * (torch.finfo(dtype).eps / 2)
    assert bool(((got - want).abs() <= bound + 1e-30).all())


def test_pitches_beyond_the_short_offsets(gpu):
    """Rows 2^22 elements apart and more take the loads with 64-bit offsets."""
    rng = np.random.default_rng(34)
    m, k, n, ld = 70, 40, 24, (1 << 22) + 16
    x, dy = _randn(rng, m, k).to(gpu), _randn(rng, m, n).to(gpu)
    q, s = quant.quantize_rows(x)
    far_q = torch.empty((m, ld), dtype=torch.int8, device=gpu)[:, :k]
    far_q.copy_(q)
    far_dy = torch.empty((m, ld), dtype=torch.float32, device=gpu)[:, :n]
    far_dy.copy_(dy)
    w, ws = _layer(rng, k, n, gpu)
    far_w = torch.empty((n, ld), dtype=torch.int8, device=gpu)[:, :k]
    far_w.copy_(w)
    assert torch.equal(quant.weight_grad(far_dy, far_q, s), quant.weight_grad(dy, q, s))
    assert torch.equal(quant.input_grad(far_dy, far_w, ws), quant.input_grad(dy, w, ws))
    # the tile form of the product: more channels than the other forms take
    big = torch.randint(-127, 128, (m, 5000), dtype=torch.int8, device=gpu)
    far_big = torch.empty((m, ld), dtype=torch.int8, device=gpu)[:, :5000]
    far_big.copy_(big)
    wb, wbs = _layer(rng, 5000, n, gpu)
    assert torch.equal(quant.matmul_int8(far_big, wb, wbs, x_scale=s), quant.matmul_int8(big, wb, wbs, x_scale=s))


@pytest.mark.parametrize('m,c', [(50, 40), (3000, 130), (9, 6150)])
def test_norm_in_place(gpu, m, c):
    """The activation may overwrite the shortcut, and dz its gradient da."""
    import ctypes
    from yolo_tf_amd import _abi
    lib = _abi.load()
    rng = np.random.default_rng(35)
    z, res, da = (_randn(rng, m, c).to(gpu) for _ in range(3))
    gamma, beta = (1 + 0.1 * _randn(rng, c)).to(gpu), (0.1 * _randn(rng, c)).to(gpu)
    a, kept = quant.norm_act(z, gamma, beta, 1e-3, 0.1, residual=res)
    dz, dgamma, dbeta = quant.norm_act_backward(da, kept)
    st = ctypes.c_void_p(torch.cuda.current_stream(gpu).cuda_stream)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device=gpu)
    out, stats = res.clone(), torch.empty(2, c, device=gpu)
    _abi.check(lib.yh_norm_act_forward(z.data_ptr(), c, out.data_ptr(), c, 0, m, c, gamma.data_ptr(), beta.data_ptr(), 1e-3, 0.1,
                                       out.data_ptr(), c, None, 0, None, stats[0].data_ptr(), stats[1].data_ptr(), None, None, 0.0,
                                       ws.data_ptr(), ws.numel(), st))
    assert torch.equal(out, a)
    grad, sums = da.clone(), torch.empty(2, c, device=gpu)
    codes, scale = kept.kept, kept.scale
    _abi.check(lib.yh_norm_act_backward(grad.data_ptr(), c, 0, m, c, codes.data_ptr(), kept.pitch, scale.data_ptr(), gamma.data_ptr(),
                                        kept.invstd.data_ptr(), 0.1, grad.data_ptr(), c, sums[0].data_ptr(), sums[1].data_ptr(),
                                        ws.data_ptr(), ws.numel(), st))
    assert torch.equal(grad, dz) and torch.equal(sums[0], dgamma) and torch.equal(sums[1], dbeta)


def test_rows_of_one_number_repeated(gpu):
    """Inputs expanded along the rows or the channels (pitch 0, adjacent equal values) are read like any other."""
    rng = np.random.default_rng(36)
    w, ws = _layer(rng, 64, 30, gpu)
    row, one = _randn(rng, 1, 64).to(gpu), _randn(rng, 200, 1).to(gpu)
    for v in (row.expand(200, 64), one.expand(200, 64)):
        assert torch.equal(quant.matmul_int8(v, w, ws), quant.matmul_int8(v.contiguous(), w, ws))
        codes, scale = quant.quantize_rows(v.contiguous())
        dy = _randn(rng, 1, 30).to(gpu).expand(200, 30)
        assert torch.equal(quant.weight_grad(dy, codes, scale), quant.weight_grad(dy.contiguous(), codes, scale))
        assert torch.equal(quant.input_grad(dy, w, ws), quant.input_grad(dy.contiguous(), w, ws))


def test_two_threads_at_once(gpu):
    import threading
    rng = np.random.default_rng(37)
    cases = [(torch.randn(5000, 256, device=gpu), *_layer(rng, 256, 96, gpu)), (torch.randn(300, 512, device=gpu), *_layer(rng, 512, 70, gpu))]
    want = [quant.matmul_int8(*c) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(gpu)):
            for _ in range(50):
                if not torch.equal(quant.matmul_int8(*cases[i % 2]), want[i % 2]):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []


def test_empty_batches(gpu):
    x = torch.empty((0, 7, 32), device=gpu)
    codes, scale = quant.quantize_rows(x)
    assert codes.shape == (0, 7, 32) and scale.shape == (0, 7)
    assert quant.dequantize_rows(codes, scale).shape == (0, 7, 32)
    w, ws = quant.quantize_rows(torch.randn(5, 32, device=gpu))
    assert quant.matmul_int8(x, w, ws).shape == (0, 7, 5)
    assert quant.input_grad(torch.empty((0, 7, 5), device=gpu), w, ws).shape == (0, 7, 32)
    dw, db = quant.weight_grad(torch.empty((0, 7, 5), device=gpu), codes, scale, want_bias=True)
    assert (dw == 0).all() and (db == 0).all() and dw.shape == (5, 32)
    with pytest.raises(Exception, match='no rows'):
        quant.norm_act(x, torch.ones(32, device=gpu), torch.ones(32, device=gpu), 1e-3, 0.1)


@pytest.mark.parametrize('positive', [True, False])
@pytest.mark.parametrize('dtype', qc.TYPES)
@pytest.mark.parametrize('m,k,n', [(1, 1, 1), (500, 40, 66), (33001, 40, 3), (70001, 64, 64), (9000, 300, 130), (20011, 2100, 2000)])
def test_bias_gradient_is_a_sum_in_64_bits(gpu, m, k, n, dtype, positive):
    """One rounding to float32 of a sum in 64 bits, whatever the pieces of the rows (the last size is one piece of 626 steps);
    values of one sign, whose errors would add up, and of both, whose sum is far below its terms."""
    g = torch.Generator(device=gpu).manual_seed(m + k)
    dy = torch.rand(m, n, generator=g, device=gpu) + 0.5 if positive else torch.randn(m, n, generator=g, device=gpu)
    dy = dy.to(dtype)
    codes = torch.randint(-127, 128, (m, k), generator=g, device=gpu, dtype=torch.int8)
    scale = torch.rand(m, generator=g, device=gpu)
    _, db = quant.weight_grad(dy, codes, scale, want_bias=True)
    want, size = dy.double().sum(0), dy.double().abs().sum(0)
    # half a step of float32, and m additions in 64 bits on either side
    assert ((db.double() - want).abs() <= qc.U * want.abs() + 2 * m * 2.0 ** -53 * size).all()


def test_the_backward_pass_reads_gamma_as_it_is_now(gpu):
    """Twice the gamma, twice the input gradient, bit for bit; also where gamma's values are not adjacent."""
    torch.manual_seed(41)
    z, da, beta = torch.randn(300, 40, device=gpu), torch.randn(300, 40, device=gpu), torch.randn(40, device=gpu)
    for gamma in (torch.randn(40, device=gpu), torch.randn(40, 2, device=gpu)[:, 1]):
        _, kept = quant.norm_act(z, gamma, beta, 1e-3, 0.1)
        first = quant.norm_act_backward(da, kept)
        gamma.mul_(2)
        second = quant.norm_act_backward(da, kept)
        assert torch.equal(second[0], 2 * first[0])
        assert torch.equal(second[1], first[1]) and torch.equal(second[2], first[2])


def test_four_threads_all_finish_with_the_right_values(gpu):
    """Each of four threads on a stream of its own makes its 50 calls; an error in one of them is an error here."""
    from concurrent.futures import ThreadPoolExecutor
    rng = np.random.default_rng(38)
    layer = lambda k, n: quant.quantize_rows(torch.from_numpy(rng.standard_normal((n, k)).astype(np.float32)).to(gpu))
    x = [torch.randn(5000, 256, device=gpu), torch.randn(300, 512, device=gpu)]
    dy = [torch.randn(5000, 96, device=gpu), torch.randn(300, 70, device=gpu)]
    w = [layer(256, 96), layer(512, 70)]
    g, b = torch.rand(256, device=gpu), torch.rand(256, device=gpu)

    def calls(i):
        y, codes, scale = quant.matmul_int8(x[i], *w[i], want_codes=True)
        out = [y, quant.weight_grad(dy[i], codes, scale), quant.input_grad(dy[i], *w[i])]
        if i == 0:
            a, kept = quant.norm_act(x[0], g, b, 1e-3, 0.1)
            out += [a, *quant.norm_act_backward(a, kept)]
        return out
    want = [calls(0), calls(1)]
    torch.cuda.synchronize()

    def work(i):
        done = 0
        with torch.cuda.stream(torch.cuda.Stream(gpu)):
            for _ in range(50):
                done += all(torch.equal(a, c) for a, c in zip(calls(i % 2), want[i % 2]))
        return done
    with ThreadPoolExecutor(4) as pool:
        assert [f.result() for f in [pool.submit(work, i) for i in range(4)]] == [50] * 4
