"""Layer norm's backward from the output at weights near both ends of fp32's range (a weight of zero alone is
undefined), on tensors that the vector kernels take and on ones that start off their boundary.

Tolerances.  As for ordinary weights, u = 2^-24 being the fp32 rounding, with xhat = (y - b) / w off by at most 4 u
of itself.  Results below 2^-126 are rounded in steps of 2^-149, so each product dy t (t = y - b) is off by 2^-150
more, which dw divides by w, and each product dy w by 2^-150.  A bfloat16 below 2^-126 has steps of 2^-133: what is
stored as one is off by 2^-134."""
import pytest
import torch

from oracle import lm_ops_oracle as oracle
from tests.test_layernorm_gpu import EPS, TYPES, U, half_step

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -150      # half a step of a subnormal fp32 result
STORED = {torch.float32: TINY, torch.bfloat16: 2.0 ** -134}
# subnormal ones, the smallest normal one, two whose reciprocal is subnormal
WEIGHTS = [2.0 ** -133, 1.5 * 2.0 ** -130, -(2.0 ** -128), 2.0 ** -126, 2.0 ** 126, -1.25 * 2.0 ** 126, 1.5 * 2.0 ** 126]


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("mix", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")], ids="-".join)
@pytest.mark.parametrize("cols", [24, 96, 520, 1000, 4096, 16376, 70000])
def test_weights_of_any_size(cuda, cols, mix, off):
    from monet_b200 import functional as F
    t, wt = TYPES[mix[0]], TYPES[mix[1]]
    rows = 3
    g = torch.Generator().manual_seed(cols)
    w, b = torch.rand(cols, generator=g) + 0.5, torch.randn(cols, generator=g) * 0.3
    at = [(7 * i + 3) * (cols // 24) % cols for i in range(len(WEIGHTS) * 3)][::3]
    xhat = torch.randn(rows, cols, generator=g, dtype=torch.float64).clamp(-1.5, 1.5)
    dy = torch.randn(rows, cols, generator=g)
    for i, value in zip(at, WEIGHTS):
        w[i], b[i] = value, 0.0
        if abs(value) > 1:
            dy[:, i] /= abs(value)      # its dy w is of the others' size
    w, b, dy = w.to(wt), b.to(wt), dy.to(t)
    y = (xhat * w.double() + b.double()).to(t)
    rstd = torch.rand(rows, generator=g) + 0.5

    def put(a):
        v = torch.empty(a.numel() + 8, dtype=a.dtype, device=cuda)[off:off + a.numel()].view(a.shape)
        return v.copy_(a)

    dx, dw, db = F.layer_norm_bwd_from_output(put(dy), put(y), (cols,), w.to(cuda), b.to(cuda), rstd.to(cuda))
    dyd, wd = dy.double(), w.double()
    h = (y.double() - b.double()) / wd
    want, ww, wb = oracle.layer_norm_backward(dyd, h, wd, rstd)
    k = cols / 256 + 56
    size, r = (dyd * wd).abs(), rstd.double()[:, None]
    m2 = (size * h.abs()).mean(1, True)
    # xhat's own error on both its uses, then the formula's roundings; what is rounded to 2^-149 before a division by w
    tol = r * ((k + 8) * U * (size + size.mean(1, True) + h.abs() * m2) + 4 * TINY + TINY * h.abs())
    tol = tol + (half_step(t) * (want.abs() + tol) if t != torch.float32 else 0) + 2 * STORED[t]
    bad = (dx.cpu().double() - want).abs() - tol
    assert bool((bad <= 0).all()), (cols, float(bad.max()), bad.argmax() % cols, at)
    tol = 168 * U * (dyd * h).abs().sum(0) + rows * (TINY / wd.abs() + TINY)
    tol = tol + (half_step(wt) * (ww.abs() + tol) if wt != torch.float32 else 0) + 2 * STORED[wt]
    bad = (dw.cpu().double() - ww).abs() - tol
    assert bool((bad <= 0).all()), (cols, float(bad.max()))
    assert bool(db.isfinite().all())
