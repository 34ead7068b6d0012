"""Plain statements of the row operators (yolo_tf_amd.quant) for the tests: NumPy float64 on the CPU,
and the single-precision steps that the definitions name."""
import numpy as np
import torch

U = 2.0 ** -24                                   # half a step of float32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}   # of subnormal results
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def f64(t):
    return t.detach().cpu().double().numpy()


def rows_of(x, levels=127):
    """(codes float64, scale float32) of float32 rows, by the definition."""
    x = np.asarray(x, dtype=np.float32)
    top = np.abs(x).max(axis=1) if x.shape[1] else np.zeros(len(x), np.float32)
    bad = ~np.isfinite(x).all(axis=1)
    live = ~bad & (top >= np.float32(2.0 ** -110))
    t = np.where(live, top, np.float32(1)).astype(np.float32)
    r = (np.float32(levels) / t).astype(np.float32)
    with np.errstate(invalid='ignore'):
        q = np.rint(np.where(live[:, None], x, 0).astype(np.float64) * r.astype(np.float64)[:, None])
    s = np.where(live, (t / np.float32(levels)).astype(np.float32), np.where(bad, np.float32(np.nan), np.float32(0)))
    return q, s.astype(np.float32)


def sum_bound(terms_abs, adds):
    """Error of a float32 sum whose `adds` roundings are independent: four standard deviations, each rounding at most half
    a step of a partial sum, which is at most the sum of the magnitudes; and one rounding of each term."""
    return (1 + 4 * np.sqrt(adds)) * U * terms_abs


def normed(z, gamma, beta, mean, invstd, slope, residual=None):
    """The forward pass element by element in float32, from given statistics: (a before rounding to the row's type,
    xhat, side)."""
    f = np.float32
    xhat = ((z.astype(f) - mean.astype(f)) * invstd.astype(f)).astype(f)
    u = ((xhat * gamma.astype(f)).astype(f) + beta.astype(f)).astype(f)
    side = u > 0
    a = np.where(side, u, (f(slope) * u).astype(f))
    if residual is not None:
        a = (a + residual.astype(f)).astype(f)
    return a, xhat, side
