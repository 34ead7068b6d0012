"""Measured cases of the 8-bit row operators (yolo_tf_amd.quant): the checkpoint of
a layer's input, the integer product of a pointwise convolution with its two
gradients, and batch normalisation with leaky ReLU on an 8-bit checkpoint.

A "row" is one pixel of an NHWC activation: M rows (batch * height * width) of K
or C channels.  The sizes are those of Darknet-53 / Darknet-19 and their headers
on 416 x 416 images (13, 26, 52, 104, 208 pixels a side, 32 .. 1536 channels, 255
channels in a prediction layer), for one image up to a batch of 64, and ragged
sizes around them.

`own` is set from outside: False computes the plain forms in elementary torch
operations, True makes the library's calls.

Definitions shared by both forms (all the values a rounding depends on are single
precision numbers, so that both take every decision alike):
  codes of a row   r = 127 / max|x| rounded to float32, code = round-half-even of
                   the exact product x * r, scale = max|x| / 127 in float32; a row
                   whose largest value is below 2^-110 is zero;
  norm checkpoint  the same with 63 in the place of 127 for the normalised value,
                   and the sign of the activation's input in the lowest bit."""
import math

import torch

own = False

EPS, SLOPE = 1e-3, 0.1
ROW_MIN = 2.0 ** -110
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
MOST_ELEMENTS, MOST_FLOPS = 60e6, 1.2e10


def listed():
    return [
        # checkpoint of a convolution's input, written and read again: the 3x3 convolutions keep their inputs so
        {"name": "checkpoint 52x52x64 of 128", "op": "checkpoint", "m": 173056, "k": 128, "type": "float32"},
        {"name": "checkpoint ragged bf16", "op": "checkpoint", "m": 2707, "k": 771, "type": "bfloat16"},
        # one cell's prediction: the smallest call of the serving path, where latency is all there is
        {"name": "product one row", "op": "product", "m": 1, "k": 1024, "n": 255, "type": "float32"},
        # the 13 x 13 header of a single image
        {"name": "product one image 13x13", "op": "product", "m": 169, "k": 1024, "n": 512, "type": "float32"},
        # a residual unit's 1x1 convolution, batch 64, 52 x 52
        {"name": "product 52x52x64", "op": "product", "m": 173056, "k": 256, "n": 128, "type": "float32"},
        # the widest pointwise layer of Darknet-19 in half precision: 1024 + 512 channels
        {"name": "product 26x26x64 bf16", "op": "product", "m": 43264, "k": 1536, "n": 425, "type": "bfloat16"},
        # gradients of the same layers in a training step
        {"name": "weight gradient 13x13x64", "op": "weight_grad", "m": 10816, "k": 1024, "n": 512, "type": "float32"},
        {"name": "weight gradient 104x104x64", "op": "weight_grad", "m": 692224, "k": 128, "n": 64, "type": "float32"},
        {"name": "input gradient 26x26x64", "op": "input_grad", "m": 43264, "k": 512, "n": 256, "type": "float32"},
        {"name": "input gradient 52x52 pred", "op": "input_grad", "m": 21632, "k": 128, "n": 255, "type": "float32"},
        # a whole step of normalisation, activation and shortcut: 104 x 104, batch 32, and the last layers of one image
        {"name": "norm step 104x104x32", "op": "norm", "m": 346112, "k": 128, "type": "float32", "residual": True},
        {"name": "norm step 13x13 bf16", "op": "norm", "m": 169, "k": 1024, "type": "bfloat16", "residual": False},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))))))


def draw(rng):
    """Rows from one to 700 thousand, channels from one to 1536, within the largest listed cases' elements and products."""
    op = rng.choice(["checkpoint", "product", "product", "weight_grad", "input_grad", "norm"])
    case = {"op": op, "type": rng.choice(["float32", "float32", "bfloat16", "float16"])}
    k = _spread(rng, 1, 1536)
    n = _spread(rng, 1, 1536)
    wide = max(k, n) if op in ("product", "weight_grad", "input_grad") else k
    most = min(700000, int(MOST_ELEMENTS / 2 / wide))
    if op in ("product", "weight_grad", "input_grad"):
        most = min(most, max(1, int(MOST_FLOPS / 2 / k / n)))
        case["n"] = n
    # with fewer rows than eight a batch norm's input gradient is all cancellation
    case["m"], case["k"] = _spread(rng, 8 if op == "norm" else 1, most), k
    if op == "norm":
        case["residual"] = rng.random() < 0.5
    if op in ("checkpoint", "product") and rng.random() < 0.25:
        case["pitch"] = k + rng.randint(1, 64)           # a channel slice of a wider tensor
    return case


def _codes_of(x):
    """The row codes of a float32 matrix: (whole numbers in float32, scales)."""
    top = x.abs().amax(dim=1)
    live = top >= ROW_MIN
    t64 = torch.where(live, top, torch.ones_like(top)).double()
    r = (127.0 / t64).float().double()
    q = torch.round(x.double() * r[:, None])
    q = torch.where(live[:, None], q, torch.zeros_like(q)).float()
    return q, torch.where(live, (t64 / 127.0).float(), torch.zeros_like(top))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    op, m, k, dtype = case["op"], case["m"], case["k"], TYPES[case["type"]]
    s = {"op": op, "type": dtype}
    if op == "norm":
        gain = torch.exp(0.5 * normal(k))                      # channels of different size and offset
        s["z"] = (normal(m, k) * gain + 0.3 * normal(k)).to(dtype)
        s["gamma"], s["beta"] = 1.0 + 0.1 * normal(k), 0.1 * normal(k)
        s["residual"] = normal(m, k).to(dtype) if case["residual"] else None
        s["da"] = (1e-3 * normal(m, k) * torch.exp(normal(m, 1))).to(dtype)
        return s
    x = normal(m, case.get("pitch", k))
    x = torch.where(x > 0, x, SLOPE * x).to(dtype)[:, :k]      # what a leaky ReLU leaves
    if op == "checkpoint":
        s["x"] = x
        return s
    n = case["n"]
    q, scale = _codes_of(normal(n, k) * math.sqrt(2.6 / k))    # the layer's weights, quantised once
    s["w"], s["w_scale"] = q.to(torch.int8), scale
    if op == "product":
        s["x"], s["bias"] = x, 0.1 * normal(n)
        return s
    s["dy"] = (1e-3 * normal(m, n) * torch.exp(normal(m, 1))).to(dtype)
    if op == "weight_grad":
        q, scale = _codes_of(x.float())
        s["codes"], s["scale"] = q.to(torch.int8), scale
    return s


def _plain_norm(z, gamma, beta, residual, da):
    t = z.dtype
    m = z.shape[0]
    z, da = z.float(), da.float()
    z64 = z.double()
    mean64 = z64.mean(dim=0)
    var64 = (z64 - mean64).square().mean(dim=0)
    mean, invstd = mean64.float(), (1.0 / torch.sqrt(var64 + EPS)).float()
    xhat = (z - mean) * invstd
    u = xhat * gamma + beta
    up = u > 0
    a = torch.where(up, u, SLOPE * u)
    if residual is not None:
        a = a + residual.float()
    top = xhat.abs().amax(dim=1)
    live = top >= ROW_MIN
    t64 = torch.where(live, top, torch.ones_like(top)).double()
    q = torch.round(xhat.double() * (63.0 / t64).float().double()[:, None]).float()
    kept = torch.where(live[:, None], q, torch.zeros_like(q)) * torch.where(live, (t64 / 63.0).float(), torch.zeros_like(top))[:, None]
    du = torch.where(up, da, SLOPE * da)
    dbeta = du.sum(dim=0, dtype=torch.float64)
    dgamma = (du.double() * kept).sum(dim=0)
    dz = (gamma * invstd) * (du - (dbeta / m).float() - kept * (dgamma / m).float())
    return {"a": a.to(t), "mean": mean, "invstd": invstd, "dz": dz.to(t), "dgamma": dgamma.float(), "dbeta": dbeta.float()}


def run(s):
    op = s["op"]
    if own:
        from yolo_tf_amd import quant

        if op == "checkpoint":
            codes, scale = quant.quantize_rows(s["x"])
            return quant.dequantize_rows(codes, scale, s["type"])
        if op == "product":
            return quant.matmul_int8(s["x"], s["w"], s["w_scale"], s["bias"])
        if op == "weight_grad":
            dw, db = quant.weight_grad(s["dy"], s["codes"], s["scale"], want_bias=True)
            return {"dw": dw, "db": db}
        if op == "input_grad":
            return quant.input_grad(s["dy"], s["w"], s["w_scale"])
        a, kept = quant.norm_act(s["z"], s["gamma"], s["beta"], EPS, SLOPE, residual=s["residual"])
        dz, dgamma, dbeta = quant.norm_act_backward(s["da"], kept)
        return {"a": a, "mean": kept.mean, "invstd": kept.invstd, "dz": dz, "dgamma": dgamma, "dbeta": dbeta}
    if op == "checkpoint":
        q, scale = _codes_of(s["x"].float())
        return (q * scale[:, None]).to(s["type"])
    if op == "product":
        q, scale = _codes_of(s["x"].float())
        y = (q * scale[:, None]) @ (s["w"].float() * s["w_scale"][:, None]).t()
        return (y + s["bias"]).to(s["type"])
    if op == "weight_grad":
        dy = s["dy"].float()
        return {"dw": dy.t() @ (s["codes"].float() * s["scale"][:, None]), "db": dy.sum(dim=0, dtype=torch.float64).float()}
    if op == "input_grad":
        return (s["dy"].float() @ (s["w"].float() * s["w_scale"][:, None])).to(s["type"])
    return _plain_norm(s["z"], s["gamma"], s["beta"], s["residual"], s["da"])


def work(case):
    m, k, e = case["m"], case["k"], SIZE[case["type"]]
    if case["op"] == "checkpoint":
        return {"bytes": m * k * 2 * e, "flops": 4 * m * k}
    if case["op"] == "norm":
        # forward: z (and the shortcut) in, the activation out; backward: its gradient in, z's out; per-channel vectors
        return {"bytes": m * k * e * (5 if case["residual"] else 4) + 24 * k, "flops": 24 * m * k}
    n = case["n"]
    if case["op"] == "product":
        return {"bytes": m * k * e + n * k + 8 * n + m * n * e, "flops": 2 * m * n * k}
    if case["op"] == "weight_grad":
        return {"bytes": m * n * e + m * k + 4 * m + 4 * n * k + 4 * n, "flops": 2 * m * n * k}
    return {"bytes": m * n * e + n * k + 4 * n + m * k * e, "flops": 2 * m * n * k}


def _row_codes(v, levels):
    """Codes and scales from the definition, in 64 bits but for the two float32 numbers that it names."""
    v = v.to(torch.float64)
    peak, _ = torch.max(torch.abs(v), dim=1, keepdim=True)
    dead = peak < 2.0 ** -110
    peak = torch.where(dead, torch.full_like(peak, 1.0), peak)
    factor = torch.div(float(levels), peak).to(torch.float32).to(torch.float64)
    step = torch.div(peak, float(levels)).to(torch.float32).to(torch.float64)
    whole = torch.mul(v, factor).round()
    return whole.masked_fill(dead, 0.0), step.masked_fill(dead, 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("checkpoint", "product"):
        whole, step = _row_codes(s["x"], 127)
        if op == "checkpoint":
            return whole * step
        sums = torch.mm(whole, s["w"].to(torch.float64).t().contiguous())          # whole numbers: exact
        return sums * step * s["w_scale"].to(torch.float64)[None, :] + s["bias"].to(torch.float64)[None, :]
    if op == "weight_grad":
        dy = s["dy"].to(torch.float64)
        weighted = (dy * s["scale"].to(torch.float64)[:, None]).t().contiguous()
        return {"dw": torch.mm(weighted, s["codes"].to(torch.float64)), "db": dy.sum(0)}
    if op == "input_grad":
        return torch.mm(s["dy"].to(torch.float64) * s["w_scale"].to(torch.float64)[None, :], s["w"].to(torch.float64))
    z, da = s["z"].to(torch.float64), s["da"].to(torch.float64)
    gamma, beta = s["gamma"].to(torch.float64), s["beta"].to(torch.float64)
    rows = float(z.shape[0])
    centre = z.sum(0) / rows
    spread = torch.pow(z - centre, 2).sum(0) / rows
    inv = torch.pow(spread + EPS, -0.5)
    # the decisions (which side of zero, which code) are those of single precision
    normal32 = (s["z"].to(torch.float32) - centre.to(torch.float32)) * inv.to(torch.float32)
    side = (normal32 * s["gamma"] + s["beta"]) > 0
    whole, step = _row_codes(normal32, 63)
    kept = whole * step
    lin = (z - centre) * inv * gamma + beta
    act = lin * torch.where(side, 1.0, SLOPE).to(torch.float64)
    if s["residual"] is not None:
        act = act + s["residual"].to(torch.float64)
    dlin = da * torch.where(side, 1.0, SLOPE).to(torch.float64)
    dbeta, dgamma = dlin.sum(0), (dlin * kept).sum(0)
    dz = gamma * inv * (dlin - dbeta / rows - kept * (dgamma / rows))
    return {"a": act, "mean": centre, "invstd": inv, "dz": dz, "dgamma": dgamma, "dbeta": dbeta}
