"""Layer norm, counter-based dropout and their fusion: the calls that are measured, in the
framework's own form (``own``) and in a plain form of elementary torch operations.

Definitions.

* dropout with probability p from a 64-bit seed and a 32-bit stream number ``offset``.  Element i
  (in the tensor's dense order) gets a 32-bit number u(i): the Philox-4x32-10 generator (Salmon et
  al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the seed as its key turns the
  counter (i / 8 low, i / 8 high, offset, h) into four words, i.e. eight 16-bit halves, low half
  first; half i % 8 is the upper half of u(i) for h = 0 and its lower half for h = 1.  The element
  is dropped where u(i) < round(p 2^32), otherwise scaled by 1 / (1 - p).
* layer norm of each row of ``cols`` values: y = (x - mean) rstd w + b, rstd = (var + eps)^-1/2 with
  the biased variance; its backward for dx, dw, db, from the stored x or from the stored y
  (xhat = (y - b) / w).
* dropout, residual add and layer norm in one: z = residual + dropout(x), y = layer norm(z); z is
  an output where the residual stream goes on (pre-norm), and then brings a gradient dz of its own.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one token of a decoder: latency
        _case("ln_one_token", "ln", 1, 4096, "bf16", "bf16"),
        # a short batch of tokens through a narrow transformer, master weights in fp32
        _case("ln_tokens", "ln", 4096, 1024, "bf16", "f32"),
        # whole 64x56x56 feature maps, one per image of a batch of 184
        _case("ln_feature_maps", "ln", 184, 64 * 56 * 56, "f32", "f32"),
        # training of a wide model, the largest backward
        _case("ln_bwd_wide", "ln_bwd_x", 16384, 4096, "bf16", "f32"),
        # widths that no vector divides and a ragged number of rows
        _case("ln_bwd_ragged", "ln_bwd_x", 5003, 1023, "f16", "f16"),
        # 128 channels at every position of 28x28 maps, batch 184, from the kept output
        _case("ln_bwd_channels", "ln_bwd_y", 184 * 28 * 28, 128, "f32", "f32"),
        # few rows, long: the last positions of a few sequences
        _case("ln_bwd_few_rows", "ln_bwd_y", 37, 8192, "bf16", "bf16"),
        # the classifier's dropout of VGG-16, batch 176
        _case("dropout_classifier", "dropout", 176, 4096, "f32", "f32", 0.5),
        # hidden activations of a large model, an odd number of values
        _case("dropout_hidden", "dropout", 1, 8192 * 8192 + 3, "bf16", "bf16", 0.1),
        # the end of a transformer block, forward, pre-norm: the sum goes on
        _case("block_fwd", "block", 8192, 2048, "bf16", "f32", 0.1),
        # its backward, with the gradient of the residual stream
        _case("block_bwd", "block_bwd", 8192, 2048, "bf16", "f32", 0.1),
        # post-norm block in fp32, forward and backward with nothing kept but the output
        _case("block_post_norm", "block_post", 2051, 1000, "f32", "f32", 0.2),
    ]


def _case(name, op, rows, cols, dtype, params, p=0.0):
    c = {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "params": params, "p": p}
    return c if name else {k: v for k, v in c.items() if k != "name"}


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["ln", "ln_bwd_x", "ln_bwd_y", "dropout", "block", "block_bwd", "block_post"])
    dtype = rng.choice(["f32", "bf16", "f16"]) if op != "block_post" else "f32"
    params = rng.choice(["f32", dtype])
    # whole feature maps go through plain layer norm; a row of a model is at most 16384 wide
    cols = _log(rng, 16, 250000 if op == "ln" else 16384)
    if rng.random() < 0.6:
        cols += -cols % 8
    rows = _log(rng, 1, max(2, min(150000, (1 << 25) // cols)))
    if op == "dropout":
        cols = _log(rng, 64, 1 << 25)
        rows = 1
    p = rng.choice([0.05, 0.1, 0.2, 0.5, rng.uniform(0.01, 0.9)]) if op not in ("ln", "ln_bwd_x", "ln_bwd_y") else 0.0
    return _case("", op, rows, cols, dtype, params, p)


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, rows, cols, t = case["op"], case["rows"], case["cols"], TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    s = dict(case)
    s["seed"] = torch.randint(-(1 << 62), 1 << 62, (1,), generator=g, device="cuda")
    s["offset"] = seed % 1000
    if op == "dropout":
        s["x"], s["dy"] = normal(rows, cols), normal(rows, cols, scale=1e-2)
        return s
    wt = TYPES[case["params"]]
    # trained scales lie around one and away from zero; shifts are smaller
    s["w"] = (torch.rand(cols, generator=g, device="cuda") + 0.5).to(wt)
    s["b"] = normal(cols, scale=0.2, dtype=wt)
    column = normal(cols, scale=0.5, dtype=torch.float32)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * 1.3 + column).to(t)
    if op == "ln":
        s["x"] = x
        return s
    s["dy"] = normal(rows, cols, scale=1e-2)
    if op in ("ln_bwd_x", "ln_bwd_y"):
        f = x.float()
        mean = f.mean(1)
        rstd = torch.rsqrt((f - mean[:, None]).square().mean(1) + EPS)
        if op == "ln_bwd_x":
            s["x"], s["mean"], s["rstd"] = x, mean, rstd
        else:
            y = (f - mean[:, None]) * rstd[:, None] * s["w"].float() + s["b"].float()
            s["y"], s["rstd"] = y.to(t), rstd
        return s
    s["x"], s["residual"] = normal(rows, cols, scale=0.7), x
    if op == "block_bwd":
        z = x.float()
        s["z"], s["mean"] = x, z.mean(1)
        s["rstd"] = torch.rsqrt((z - s["mean"][:, None]).square().mean(1) + EPS)
        s["dz"] = normal(rows, cols, scale=1e-2)
        del s["x"], s["residual"]
    return s


# ----------------------------------------------------------------------------- the plain form
_LOW = 0xFFFFFFFF


def _words(seed, blocks, offset, half):
    """Four Philox-4x32-10 words for the counters (block, offset, half), as int64 tensors."""
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    a, b = blocks & _LOW, (blocks >> 32) & _LOW
    c, d = torch.full_like(blocks, offset), torch.full_like(blocks, half)
    for _ in range(10):
        m, n = a * 0xD2511F53, c * 0xCD9E8D57        # the 64 bits of each product, signs aside
        a, b, c, d = ((n >> 32) & _LOW) ^ b ^ k0, n & _LOW, ((m >> 32) & _LOW) ^ d ^ k1, m & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack([a, b, c, d], 1)


def _halves(seed, n, offset, half):
    words = _words(seed, torch.arange((n + 7) // 8, device=seed.device), offset, half)
    return torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]


def _factor(s, shape):
    """0 where an element is dropped, 1 / (1 - p) where it is kept, in 32 bits."""
    n = math.prod(shape)
    u = (_halves(s["seed"], n, s["offset"], 0) << 16) | _halves(s["seed"], n, s["offset"], 1)
    kept = u >= int(round(s["p"] * 2.0 ** 32))
    return (kept.float() * (1.0 / (1.0 - s["p"]))).reshape(shape)


def _plain_forward(v, w, b):
    mean = v.sum(1, keepdim=True) / v.shape[1]
    c = v - mean
    rstd = 1.0 / torch.sqrt((c * c).sum(1, keepdim=True) / v.shape[1] + EPS)
    return c * rstd * w.float() + b.float(), mean[:, 0], rstd[:, 0]


def _plain_backward(dy, xhat, w, rstd):
    g = dy * w.float()
    a = g.sum(1, keepdim=True) / g.shape[1]
    c = (g * xhat).sum(1, keepdim=True) / g.shape[1]
    dx = (g - a - xhat * c) * rstd[:, None]
    return dx, (dy * xhat).sum(0).to(w.dtype), dy.sum(0).to(w.dtype)


def _plain(s):
    op, t = s["op"], TYPES[s["dtype"]]
    if op == "dropout":
        f = _factor(s, s["x"].shape)
        return {"y": (s["x"].float() * f).to(t), "dx": (s["dy"].float() * f).to(t)}
    w, b = s["w"], s["b"]
    if op == "ln":
        y, mean, rstd = _plain_forward(s["x"].float(), w, b)
        return {"y": y.to(t), "mean": mean, "rstd": rstd}
    if op == "ln_bwd_x":
        xhat = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        dx, dw, db = _plain_backward(s["dy"].float(), xhat, w, s["rstd"])
        return {"dx": dx.to(t), "dw": dw, "db": db}
    if op == "ln_bwd_y":
        xhat = (s["y"].float() - b.float()) / w.float()
        dx, dw, db = _plain_backward(s["dy"].float(), xhat, w, s["rstd"])
        return {"dx": dx.to(t), "dw": dw, "db": db}
    if op == "block_bwd":
        xhat = (s["z"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        d, dw, db = _plain_backward(s["dy"].float(), xhat, w, s["rstd"])
        d = d + s["dz"].float()
        return {"dx": (d * _factor(s, d.shape)).to(t), "dresidual": d.to(t), "dw": dw, "db": db}
    f = _factor(s, s["x"].shape)
    z = s["residual"].float() + s["x"].float() * f
    y, mean, rstd = _plain_forward(z, w, b)
    if op == "block":
        return {"y": y.to(t), "z": z.to(t), "mean": mean, "rstd": rstd}
    y = y.to(t)
    xhat = (y.float() - b.float()) / w.float()
    d, dw, db = _plain_backward(s["dy"].float(), xhat, w, rstd)
    return {"y": y, "dx": (d * f).to(t), "dresidual": d.to(t), "dw": dw, "db": db}


# --------------------------------------------------------------------------- the framework's
def _framework(s):
    from monet_b200 import functional as F
    op = s["op"]
    if op == "dropout":
        return {"y": F.dropout(s["x"], s["p"], s["seed"], s["offset"]),
                "dx": F.dropout_bwd(s["dy"], s["p"], s["seed"], s["offset"])}
    w, b, shape = s["w"], s["b"], (s["cols"],)
    if op == "ln":
        y, mean, rstd = F.layer_norm(s["x"], shape, w, b, EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "ln_bwd_x":
        dx, dw, db = F.layer_norm_bwd_from_input(s["dy"], s["x"], shape, w, s["mean"], s["rstd"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "ln_bwd_y":
        dx, dw, db = F.layer_norm_bwd_from_output(s["dy"], s["y"], shape, w, b, s["rstd"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "block_bwd":
        dx, dr, dw, db = F.dropout_add_layer_norm_bwd_from_sum(
            s["dy"], s["z"], shape, w, s["mean"], s["rstd"], s["p"], s["seed"], s["offset"], dz=s["dz"])
        return {"dx": dx, "dresidual": dr, "dw": dw, "db": db}
    y, z, mean, rstd = F.dropout_add_layer_norm(
        s["x"], s["residual"], shape, w, b, EPS, s["p"], s["seed"], s["offset"], want_sum=op == "block")
    if op == "block":
        return {"y": y, "z": z, "mean": mean, "rstd": rstd}
    dx, dr, dw, db = F.dropout_add_layer_norm_bwd_from_output(
        s["dy"], y, shape, w, b, rstd, s["p"], s["seed"], s["offset"])
    return {"y": y, "dx": dx, "dresidual": dr, "dw": dw, "db": db}


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------------------ what it costs
def work(case):
    op, rows, cols, e, w = case["op"], case["rows"], case["cols"], BYTES[case["dtype"]], BYTES[case["params"]]
    n = rows * cols
    # tensors of the activations' size that are read and written, parameters and their gradients,
    # 32-bit statistics, operations a value
    tensors, parameters, statistics, flops = {
        "dropout": (4, 0, 0, 4), "ln": (2, 2, 2, 8), "ln_bwd_x": (3, 3, 2, 14), "ln_bwd_y": (3, 4, 1, 14),
        "block": (4, 2, 2, 11), "block_bwd": (5, 3, 2, 17), "block_post": (6, 4, 0, 27)}[op]
    return {"bytes": n * e * tensors + cols * w * parameters + rows * 4 * statistics, "flops": n * flops}


# --------------------------------------------------------------------- the definitions, 64 bits
def _exact_kept(seed, offset, n, p):
    """Which of n elements are kept, by numpy's unsigned 64-bit arithmetic on 32-bit words."""
    key, numbers = seed % (1 << 64), None
    block = np.arange((n + 7) // 8, dtype=np.uint64)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    for half in (0, 1):
        c = [block & low, block >> shift, np.uint64(offset), np.uint64(half)]
        for r in range(10):
            k0 = np.uint64(((key & 0xFFFFFFFF) + r * 0x9E3779B9) % (1 << 32))
            k1 = np.uint64(((key >> 32) + r * 0xBB67AE85) % (1 << 32))
            first, third = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
            c = [(third >> shift) ^ c[1] ^ k0, third & low, (first >> shift) ^ c[3] ^ k1, first & low]
        words = np.empty((block.size, 4), dtype="<u4")
        for j in range(4):
            words[:, j] = c[j]
        halves = words.view("<u2").reshape(-1)[:n].astype(np.uint32)
        numbers = halves << np.uint32(16) if half == 0 else numbers | halves
    return torch.from_numpy(numbers >= round(p * 2.0 ** 32))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    keep = None
    if case["p"]:
        keep = _exact_kept(int(s["seed"]), s["offset"], case["rows"] * case["cols"], case["p"])
        keep = keep.reshape(case["rows"], case["cols"]).cuda()

    def dropped(v):
        return torch.where(keep, v / (1 - case["p"]), torch.zeros_like(v))

    def norm(v):
        var, mean = torch.var_mean(v, 1, correction=0)
        return mean, (var + EPS).rsqrt()

    def gradients(xhat, rstd):
        h = d["dy"] * d["w"]
        dv = rstd[:, None] * (h - h.mean(1, True) - xhat * (h * xhat).mean(1, True))
        return dv, torch.einsum("rc,rc->c", d["dy"], xhat), d["dy"].sum(0)

    if op == "dropout":
        return {"y": dropped(d["x"]), "dx": dropped(d["dy"])}
    if op == "ln":
        mean, rstd = norm(d["x"])
        return {"y": torch.addcmul(d["b"], (d["x"] - mean[:, None]) * rstd[:, None], d["w"]), "mean": mean, "rstd": rstd}
    if op in ("ln_bwd_x", "ln_bwd_y"):
        xhat = (d["x"] - d["mean"][:, None]) * d["rstd"][:, None] if op == "ln_bwd_x" else (d["y"] - d["b"]) / d["w"]
        dx, dw, db = gradients(xhat, d["rstd"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "block_bwd":
        dv, dw, db = gradients((d["z"] - d["mean"][:, None]) * d["rstd"][:, None], d["rstd"])
        dv = dv + d["dz"]
        return {"dx": dropped(dv), "dresidual": dv, "dw": dw, "db": db}
    z = d["residual"] + dropped(d["x"])
    mean, rstd = norm(z)
    xhat = (z - mean[:, None]) * rstd[:, None]
    y = torch.addcmul(d["b"], xhat, d["w"])
    if op == "block":
        return {"y": y, "z": z, "mean": mean, "rstd": rstd}
    dv, dw, db = gradients(xhat, rstd)
    return {"y": y, "dx": dropped(dv), "dresidual": dv, "dw": dw, "db": db}
