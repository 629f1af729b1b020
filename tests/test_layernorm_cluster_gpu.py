"""Layer norm's statistics at widths that a cluster of CTAs shares, also where its last CTA holds less
than the others, on rows whose mean is many deviations away from zero.

Tolerance.  u = 2^-24, R = max|v| rstd.  A lane's sum of 32 values is a chain of at most 17 additions, a merge
of two sets of n values adds one more per step: a sum over n values is off by at most (18 + j) u n max|v| after j
steps.  The difference d of two such sums enters the squared deviations as d^2 / 2n, with |d| of the order of
sqrt(2n) deviations, so that step's error is below 1.13 (18 + j) u R / sqrt(n) of the variance; over the steps, n = 32,
64, ..., these add up to 14 u R, and merging the warps and the CTAs with their counts adds 2 u R each: rstd
moves by half of 18 u R.  16 u R leaves room for sets that differ more than random ones; a sum made in the kernel
(one rounding of a value, one of a product) adds 4 u R.  What does not grow with R is below (n / 256 + 64) u, and
what grows with its square below (64 u R)^2."""
import pytest
import torch

from oracle import lm_ops_oracle as oracle
from tests.test_layernorm_gpu import EPS, MIXES, TYPES, U, check_forward

pytestmark = pytest.mark.gpu

# widths just below those that fill a cluster's CTAs evenly, and these themselves
WIDTHS = {"f32": [16372, 16380, 16384, 32756, 32760, 32764, 32768],
          "16": [16376, 16384, 32744, 32752, 32760, 32768, 65512, 65520, 65528, 65536]}
CASES = [(c, m) for m in MIXES for c in WIDTHS["f32" if m[0] == "f32" else "16"]]


def check(got, v, w, b, t, extra, summed):
    check_forward(got, v, w, b, t, extra=extra)
    rstd = got[2].cpu().double()
    exact = oracle.layer_norm_forward(v, w, b, EPS)[2]
    r = v.abs().amax(1) * exact
    tol = U * ((20 if summed else 16) * r + v.shape[1] / 256 + 64) + (64 * U * r) ** 2
    off = (rstd - exact).abs() / exact
    assert bool((off <= tol).all()), (off / tol).tolist()


@pytest.mark.parametrize("cols,mix", CASES, ids=lambda v: v if isinstance(v, int) else "-".join(v))
def test_mean_away_from_zero(cuda, cols, mix):
    from monet_b200 import functional as F
    t, wt = TYPES[mix[0]], TYPES[mix[1]]
    g = torch.Generator().manual_seed(cols)
    means = torch.tensor([0.0, 1.0, -10.0, 100.0, 1000.0])[:, None]
    x = (torch.randn(5, cols, generator=g) + means).to(t)
    branch = torch.randn(5, cols, generator=g).to(t)
    w, b = (torch.rand(cols, generator=g) + 0.5).to(wt), torch.randn(cols, generator=g).to(wt)
    xg, bg, wg, biasg = (a.to(cuda) for a in (x, branch, w, b))
    check(F.layer_norm(xg, (cols,), wg, biasg, EPS), x.double(), w, b, t, 0.0, False)
    seed = torch.tensor([cols], device=cuda)
    for p in (0.0, 0.1):
        y, _, mean, rstd = F.dropout_add_layer_norm(bg, xg, (cols,), wg, biasg, EPS, p, seed, 3)
        keep = oracle.dropout_keep(cols, 3, 5 * cols, p).view(5, cols)
        v = x.double() + torch.where(keep, branch.double() / (1 - p), torch.zeros(5, cols, dtype=torch.float64))
        check((y, mean, rstd), v, w, b, t, 6 * U, True)
