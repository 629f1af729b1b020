"""Layer norm (forward, backward from input and from output) and its fusion with dropout and the
residual add, against the definition in 64 bits.

Tolerances.  u = 2^-24 is the fp32 rounding; a sum over a row of n values adds at most n/256 + 48
terms one after another (the rest is a tree), so its error is below (n/256 + 48) u sum|terms|, and a
sum over r rows has chains of at most r/8 + 160.  Each stored value adds half a step of its type."""
import pytest
import torch

from oracle import lm_ops_oracle as oracle

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SHAPES = [(1, 1), (3, 1), (5, 2), (4, 7), (1, 8), (2, 16), (37, 31), (64, 64), (9, 100), (33, 128), (7, 257), (130, 768),
          (50, 1000), (11, 1023), (3, 2047), (8, 2048), (5, 4096), (3, 4099), (2, 8192), (2, 12289), (3, 16384), (1, 1 << 15),
          (2, 40000), (3, 65537), (1, 200704), (2, 300000), (2000, 72), (1201, 33), (700, 1024), (500, 2501),
          (301, 20000), (299, 17001), (150, 66001), (40, 131080), (900, 8192), (640, 9999)]
MIXES = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")]


def half_step(t):
    """Half a rounding step relative to the value; subnormals of fp16 have an absolute step instead."""
    return torch.finfo(t).eps / 2


def floor_step(t):
    return 2.0 ** -25 if t == torch.float16 else 0.0


def make(rows, cols, t, wt, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + cols)
    x = (torch.randn(rows, cols, generator=g) * 1.5 + 0.5).to(t)
    dy = torch.randn(rows, cols, generator=g).to(t)
    w = (torch.rand(cols, generator=g) + 0.5).to(wt)
    b = torch.randn(cols, generator=g).mul(0.3).to(wt)
    return x, dy, w, b


def check_forward(got, v, w, b, t, eps=EPS, extra=0.0):
    """`got` = (y, mean, rstd) against the definition on v (float64 [rows, cols]); `extra`: how far v
    itself may be off, relative to its largest value."""
    y, mean, rstd = (a.detach().cpu().double() for a in got)
    n = v.shape[1]
    k = n / 256 + 48
    ey, em, er = oracle.layer_norm_forward(v, w, b, eps)
    size = v.abs().amax(1)
    off = (k * U + extra) * size + U * em.abs()
    assert bool(((mean - em).abs() <= off).all())
    # the variance is a sum of squares of values that are each off by `off` + u |v|
    std2 = (v - em[:, None]).square().mean(1)
    var_off = (k + 4) * U * std2 + 2 * (off + U * size) * std2.sqrt() + (off + U * size) ** 2
    rel = var_off / (std2 + eps) / 2 + 4 * U
    assert bool(((rstd - er).abs() <= rel * er * (1 + 2 * rel)).all())
    wv = w.double().abs() if w is not None else torch.ones(n, dtype=torch.float64)
    bv = b.double().abs() if b is not None else torch.zeros(n, dtype=torch.float64)
    xhat = (v - em[:, None]).abs() * er[:, None]
    tol = (off + 2 * U * size)[:, None] * er[:, None] * wv + xhat * wv * (rel * (1 + 2 * rel) + 4 * U)[:, None] + 2 * U * bv
    tol = tol + (half_step(t) * (ey.abs() + tol) if t != torch.float32 else 0) + floor_step(t)
    bad = (y - ey).abs() - tol
    assert bool((bad <= 0).all()), float(bad.max())


def check_backward(got, dy, xhat, xhat_off, w, rstd, t, wt, dz=None, rows_chain=None):
    """`got` = (dv, dw, db) against the formula on xhat (float64), itself known to `xhat_off`."""
    rows, n = xhat.shape
    k = n / 256 + 56
    dv, dw, db = (a.detach().cpu().double() if a is not None else None for a in got)
    ev, ew, eb = oracle.layer_norm_backward(dy, xhat, w, rstd)
    g = dy.double().abs() * (w.double().abs() if w is not None else 1.0)
    h = xhat.abs()
    r = rstd.double()[:, None]
    m1, m2 = g.mean(1, True), (g * h).mean(1, True)
    tol = r * ((k * U) * (g + m1 + h * m2) + xhat_off * m2 + h * (g * xhat_off).mean(1, True))
    if dz is not None:
        ev = ev + dz.double()
        tol = tol + 2 * U * (ev.abs() + dz.double().abs())
    tol = tol + (half_step(t) * (ev.abs() + tol) if t != torch.float32 else 0) + floor_step(t)
    bad = (dv - ev).abs() - tol
    assert bool((bad <= 0).all()), ("dv", float(bad.max()))
    chain = rows / 8 + 160
    if dw is not None:
        tol = chain * U * (dy.double().abs() * h).sum(0) + (dy.double().abs() * xhat_off).sum(0) * (1 + chain * U)
        tol = tol + (half_step(wt) * (ew.abs() + tol) if wt != torch.float32 else 0) + floor_step(wt)
        bad = (dw.flatten() - ew).abs() - tol
        assert bool((bad <= 0).all()), ("dw", float(bad.max()))
    if db is not None:
        tol = chain * U * dy.double().abs().sum(0)
        tol = tol + (half_step(wt) * (eb.abs() + tol) if wt != torch.float32 else 0) + floor_step(wt)
        bad = (db.flatten() - eb).abs() - tol
        assert bool((bad <= 0).all()), ("db", float(bad.max()))


def input_xhat(v, mean, rstd):
    """xhat from the stored tensor and the fp32 statistics, and its fp32 error."""
    m, r = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    xhat = (v.double() - m) * r
    return xhat, 3 * U * xhat.abs()      # one difference, one product: each rounds the result once


def output_xhat(y, w, b):
    wv = w.double() if w is not None else 1.0
    bv = b.double() if b is not None else 0.0
    xhat = (y.double() - bv) / wv
    return xhat, 4 * U * xhat.abs()      # a difference, then a division or a product with 1/w


@pytest.mark.parametrize("mix", MIXES, ids="-".join)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(cuda, rows, cols, mix):
    from monet_b200 import functional as F
    t, wt = TYPES[mix[0]], TYPES[mix[1]]
    x, dy, w, b = make(rows, cols, t, wt)
    xg, dyg, wg, bg = (a.to(cuda) for a in (x, dy, w, b))
    y, mean, rstd = F.layer_norm(xg, (cols,), wg, bg, EPS)
    assert y.dtype == t and mean.shape == rstd.shape == (rows,)
    check_forward((y, mean, rstd), x.double(), w, b, t)
    grads = F.layer_norm_bwd_from_input(dyg, xg, (cols,), wg, mean, rstd)
    assert grads[0].dtype == t and grads[1].dtype == grads[2].dtype == wt
    xhat, off = input_xhat(x, mean, rstd)
    check_backward(grads, dy, xhat, off, w, rstd.cpu(), t, wt)
    grads = F.layer_norm_bwd_from_output(dyg, y, (cols,), wg, bg, rstd)
    xhat, off = output_xhat(y.cpu(), w, b)
    check_backward(grads, dy, xhat, off, w, rstd.cpu(), t, wt)


@pytest.mark.parametrize("mix", MIXES, ids="-".join)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 7), (13, 64), (9, 100), (130, 768), (50, 1000), (11, 1023), (6, 4096), (3, 8200),
                                       (2, 20001), (1201, 33), (3, 70000), (150, 33001), (33, 131072)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5])
def test_dropout_add_layer_norm(cuda, rows, cols, mix, p):
    """Forward with and without the sum, backward from the sum (with a gradient of its own) and from
    the output; the mask is the oracle's, element by element."""
    from monet_b200 import functional as F
    t, wt = TYPES[mix[0]], TYPES[mix[1]]
    res, dy, w, b = make(rows, cols, t, wt)
    x, dz, _, _ = make(rows, cols, t, wt, seed=1)
    seed, offset = -987654321987654321, 5
    sg = torch.tensor([seed], device=cuda)
    keep = oracle.dropout_keep(seed, offset, rows * cols, p).view(rows, cols)
    drop = lambda a: torch.where(keep, a.double() / (1 - p), torch.zeros_like(a, dtype=torch.float64))   # noqa: E731
    v = res.double() + drop(x)
    args = (x.to(cuda), res.to(cuda), (cols,), w.to(cuda), b.to(cuda), EPS, p, sg, offset)
    y, z, mean, rstd = F.dropout_add_layer_norm(*args)
    check_forward((y, mean, rstd), v, w, b, t, extra=6 * U)
    assert z.dtype == t
    zc = z.cpu().double()
    part = res.double().abs() + drop(x).abs()
    assert bool(((zc - v).abs() <= 4 * U * part + half_step(t) * (v.abs() + 4 * U * part) + floor_step(t)).all())
    y2, none, mean2, rstd2 = F.dropout_add_layer_norm(*args, want_sum=False)
    assert none is None and torch.equal(y, y2) and torch.equal(mean, mean2) and torch.equal(rstd, rstd2)

    for from_output in (False, True):
        for with_dz in (False, True):
            kw = dict(p=p, seed=sg, offset=offset, dz=dz.to(cuda) if with_dz else None)
            if from_output:
                dx, dr, dw, db = F.dropout_add_layer_norm_bwd_from_output(dy.to(cuda), y, (cols,), w.to(cuda), b.to(cuda), rstd, **kw)
                xhat, off = output_xhat(y.cpu(), w, b)
            else:
                dx, dr, dw, db = F.dropout_add_layer_norm_bwd_from_sum(dy.to(cuda), z, (cols,), w.to(cuda), mean, rstd, **kw)
                xhat, off = input_xhat(z.cpu(), mean, rstd)
            check_backward((dr, dw, db), dy, xhat, off, w, rstd.cpu(), t, wt, dz if with_dz else None)
            if p == 0.0:
                assert dx is dr
                continue
            assert torch.equal(dx.cpu()[~keep], torch.zeros(int((~keep).sum()), dtype=t))
            # dx and dresidual are one fp32 value rounded twice: each is off by half a step
            want = dr.cpu().double() / (1 - p)
            lim = (2 * half_step(t) + 4 * U) * want.abs() * (1 + half_step(t)) + 2 * floor_step(t) / (1 - p) + 2.0 ** -126
            assert bool(((dx.cpu().double() - want).abs()[keep] <= lim[keep]).all())


def test_fused_chain_is_the_unfused_one_bit_for_bit_in_fp32(cuda):
    """In fp32 the stored intermediates are the registers of the fused kernel."""
    from monet_b200 import functional as F
    for rows, cols in ((13, 64), (50, 1000), (7, 1023), (3, 8192)):
        res, dy, w, b = (a.to(cuda) for a in make(rows, cols, torch.float32, torch.float32))
        x = make(rows, cols, torch.float32, torch.float32, seed=1)[0].to(cuda)
        seed = F.dropout_seed(cuda)
        y, z, mean, rstd = F.dropout_add_layer_norm(x, res, (cols,), w, b, EPS, 0.3, seed, 2)
        zz = F.add(res, F.dropout(x, 0.3, seed, 2))
        yy, mm, rr = F.layer_norm(zz, (cols,), w, b, EPS)
        assert torch.equal(z, zz) and torch.equal(y, yy) and torch.equal(mean, mm) and torch.equal(rstd, rr)
        dx, dr, dw, db = F.dropout_add_layer_norm_bwd_from_sum(dy, z, (cols,), w, mean, rstd, 0.3, seed, 2)
        d2, dw2, db2 = F.layer_norm_bwd_from_input(dy, zz, (cols,), w, mm, rr)
        assert torch.equal(dr, d2) and torch.equal(dw, dw2) and torch.equal(db, db2)
        assert torch.equal(dx, F.dropout_bwd(d2, 0.3, seed, 2))


@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
def test_absent_parameters(cuda, affine):
    from monet_b200 import functional as F
    for rows, cols in ((6, 96), (5, 33), (3, 20000)):
        x, dy, w, b = make(rows, cols, torch.float32, torch.float32)
        w, b = (w if affine == "weight" else None), (b if affine == "bias" else None)
        wg, bg = (a.to(cuda) if a is not None else None for a in (w, b))
        y, mean, rstd = F.layer_norm(x.to(cuda), cols, wg, bg)
        check_forward((y, mean, rstd), x.double(), w, b, torch.float32)
        for got, (xhat, off) in (
                (F.layer_norm_bwd_from_input(dy.to(cuda), x.to(cuda), cols, wg, mean, rstd, w is not None, b is not None),
                 input_xhat(x, mean, rstd)),
                (F.layer_norm_bwd_from_output(dy.to(cuda), y, cols, wg, bg, rstd, w is not None, b is not None),
                 output_xhat(y.cpu(), w, b))):
            assert (got[1] is None) == (w is None) and (got[2] is None) == (b is None)
            check_backward(got, dy, xhat, off, w, rstd.cpu(), torch.float32, torch.float32)


def test_strides_offsets_and_shapes(cuda):
    """Rows with gaps, a start off the vector boundary, a strided last axis, a repeated row, more than
    one normalised axis, channels_last: results as for the dense copy, bit for bit where the row is
    walked in the same order."""
    from monet_b200 import functional as F
    g = torch.Generator().manual_seed(3)
    big = torch.randn(40, 700, generator=g).to(cuda)
    views = [big[:, :512], big[:, 8:520], big[:, 3:515], big[:, 1:502], big[::2, :512], big[:, ::2], big.t()[:96],
             big[:1].expand(9, 700), big.flatten()[1:1 + 20 * 64].view(20, 64), big.flatten()[4:4 + 20 * 64].view(20, 64),
             big[:, :505], big[0, :1].expand(6, 50)]
    for t in (torch.float32, torch.bfloat16):
        for v in views:
            base = big.to(t)
            v = torch.as_strided(base, v.shape, v.stride(), v.storage_offset())
            n = v.shape[1]
            w, b = (torch.rand(n, generator=g) + 0.5).to(cuda), torch.randn(n, generator=g).to(cuda)
            y, mean, rstd = F.layer_norm(v, (n,), w, b)
            check_forward((y, mean, rstd), v.cpu().double(), w.cpu(), b.cpu(), t)
            assert y.is_contiguous()
            dy = v.flip(0)
            for dyv in (dy, torch.as_strided(base.flip(0), v.shape, v.stride(), v.storage_offset())):
                got = F.layer_norm_bwd_from_input(dyv, v, (n,), w, mean, rstd)
                xhat, off = input_xhat(v.cpu(), mean, rstd)
                check_backward(got, dyv.cpu(), xhat, off, w.cpu(), rstd.cpu(), t, torch.float32)
            seed = torch.tensor([7], device=cuda)
            a = F.dropout_add_layer_norm(v, v, (n,), w, b, EPS, 0.4, seed)
            c = F.dropout_add_layer_norm(v.contiguous(), v.contiguous(), (n,), w, b, EPS, 0.4, seed)
            keep = oracle.dropout_keep(7, 0, v.numel(), 0.4).view(v.shape)
            for q in (a, c):
                assert torch.equal(q[1].cpu()[~keep], v.cpu()[~keep])
    x = torch.randn(3, 4, 5, 6, generator=g).to(cuda)
    for fmt in (torch.contiguous_format, torch.channels_last):
        xf = x.contiguous(memory_format=fmt)
        w = torch.rand(4, 5, 6, generator=g).to(cuda) + 0.5
        y, mean, rstd = F.layer_norm(xf, (4, 5, 6), w, None)
        check_forward((y.view(3, -1), mean, rstd), x.cpu().double().view(3, -1), w.cpu().flatten(), None, torch.float32)
        dx, dw, _ = F.layer_norm_bwd_from_input(xf, xf, (4, 5, 6), w, mean, rstd)
        assert dx.shape == x.shape and dw.shape == (4, 5, 6)


def test_in_place(cuda):
    from monet_b200 import functional as F
    for t in (torch.float32, torch.bfloat16):
        for rows, cols in ((9, 96), (40, 33), (40, 1001), (5, 4096), (3, 70001)):
            x, dy, w, b = (a.to(cuda) for a in make(rows, cols, t, torch.float32))
            y, mean, rstd = F.layer_norm(x, (cols,), w, b)
            xi = x.clone()
            yi, mi, ri = F.layer_norm(xi, (cols,), w, b, inplace=True)
            assert yi.data_ptr() == xi.data_ptr() and torch.equal(yi, y) and torch.equal(mi, mean) and torch.equal(ri, rstd)
            seed = torch.tensor([11], device=cuda)
            a = F.dropout_add_layer_norm(x, dy, (cols,), w, b, EPS, 0.2, seed)
            xi = x.clone()
            c = F.dropout_add_layer_norm(xi, dy, (cols,), w, b, EPS, 0.2, seed, inplace=True)
            assert c[0].data_ptr() == xi.data_ptr() and all(torch.equal(p, q) for p, q in zip(a, c))


def test_backward_over_its_inputs(cuda):
    """Through the C ABI: dv over dy and dx over the kept tensor."""
    import ctypes as C
    from monet_b200 import _lib
    from monet_b200 import functional as F
    for rows, cols in ((9, 96), (40, 33), (300, 1001), (5, 4096), (3, 70001)):
        x, dy, w, b = (a.to(cuda) for a in make(rows, cols, torch.bfloat16, torch.float32))
        seed = torch.tensor([13], device=cuda)
        y, mean, rstd = F.layer_norm(x, (cols,), w, b)
        want = F.dropout_add_layer_norm_bwd_from_sum(dy, x, (cols,), w, mean, rstd, 0.2, seed, 3)
        d = _lib.LnDesc(rows, cols, cols, cols, 0, _lib.MB_BF16, _lib.MB_F32, 0.0)
        q = _lib.DropoutDesc(0.2, seed.data_ptr(), 3)
        ws = torch.empty(_lib.lib().mb_layer_norm_bwd_workspace_bytes(C.byref(d)), dtype=torch.uint8, device=cuda)
        dw, db = torch.empty(cols, device=cuda), torch.empty(cols, device=cuda)
        a, k = dy.clone(), x.clone()
        rc = _lib.lib().mb_layer_norm_bwd(a.data_ptr(), k.data_ptr(), 0, None, w.data_ptr(), None, mean.data_ptr(),
                                          rstd.data_ptr(), a.data_ptr(), k.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                          C.byref(d), C.byref(q), ws.data_ptr(), ws.numel(),
                                          torch.cuda.current_stream().cuda_stream)
        assert rc == 0, _lib.last_error()
        assert torch.equal(k, want[0]) and torch.equal(a, want[1]) and torch.equal(dw, want[2]) and torch.equal(db, want[3])


def test_no_rows(cuda):
    """No rows: empty outputs, and gradients of the parameters that are zero, not left unwritten."""
    from monet_b200 import functional as F
    x, w, b = torch.empty(0, 24, device=cuda), torch.ones(24, device=cuda), torch.zeros(24, device=cuda)
    y, mean, rstd = F.layer_norm(x, (24,), w, b)
    assert y.shape == (0, 24) and mean.numel() == rstd.numel() == 0
    for got in (F.layer_norm_bwd_from_input(x, x, (24,), w, mean, rstd), F.layer_norm_bwd_from_output(x, x, (24,), w, b, rstd)):
        assert got[0].shape == (0, 24) and not bool(got[1].any()) and not bool(got[2].any())
    y, z, _, _ = F.dropout_add_layer_norm(x, x, (24,), w, b, EPS, 0.5, torch.tensor([1], device=cuda))
    assert y.shape == z.shape == (0, 24)


def test_constant_rows_and_values_that_are_not_finite(cuda):
    """A constant row has xhat = 0, whatever its size (no cancellation between two large sums); a row
    with an infinity or NaN is NaN in its own row only; NaN under a dropped element stays out."""
    from monet_b200 import functional as F
    for cols in (7, 64, 1000, 4096, 50000):
        x = torch.randn(6, cols)
        x[0] = 3.0e4
        x[1] = -1.0
        x[2, cols // 2] = float("inf")
        x[4, 0] = float("nan")
        w, b = torch.rand(cols) + 0.5, torch.randn(cols)
        y, mean, rstd = F.layer_norm(x.to(cuda), (cols,), w.to(cuda), b.to(cuda))
        k = cols / 256 + 48
        # the mean of equal values is off by k u |x|, and 1/sqrt(eps) is the largest rstd
        assert bool(((y[0].cpu() - b).abs() <= w * (2 * k * U * 3.0e4 * EPS ** -0.5) + 2 * U * b.abs()).all())
        assert bool(((y[1].cpu() - b).abs() <= w * (2 * k * U * EPS ** -0.5) + 2 * U * b.abs()).all())
        assert bool(y[2].isnan().any()) and bool(y[4].isnan().all())
        rows = [1, 3, 5]
        check_forward((y[rows], mean[rows], rstd[rows]), x[rows].double(), w, b, torch.float32)
        seed = torch.tensor([5], device=cuda)
        keep = oracle.dropout_keep(5, 0, 6 * cols, 0.5).view(6, cols)
        poisoned = torch.where(keep, torch.zeros(6, cols), torch.full((6, cols), float("nan")))
        clean = torch.randn(6, cols)
        got = F.dropout_add_layer_norm(poisoned.to(cuda), clean.to(cuda), (cols,), w.to(cuda), b.to(cuda), EPS, 0.5, seed)
        assert torch.equal(got[1].cpu(), clean) and bool(got[0].isfinite().all())


def test_large_mean_keeps_its_digits(cuda):
    """Mean 1000 times the deviation: the two-step variance loses no more than the inputs' rounding."""
    from monet_b200 import functional as F
    for cols in (96, 1000, 4096, 30000):
        x = torch.randn(5, cols) + 1000.0
        y, mean, rstd = F.layer_norm(x.to(cuda), (cols,), None, None)
        check_forward((y, mean, rstd), x.double(), None, None, torch.float32)
        er = oracle.layer_norm_forward(x)[2]
        assert bool(((rstd.cpu().double() - er).abs() <= 1e-4 * er).all())


def test_zero_weight_from_output_is_nan_and_from_input_is_right(cuda):
    from monet_b200 import functional as F
    for cols in (40, 4096):
        x, dy, w, b = make(3, cols, torch.float32, torch.float32)
        w[5] = 0.0
        y, mean, rstd = F.layer_norm(x.to(cuda), (cols,), w.to(cuda), b.to(cuda))
        got = F.layer_norm_bwd_from_input(dy.to(cuda), x.to(cuda), (cols,), w.to(cuda), mean, rstd)
        xhat, off = input_xhat(x, mean, rstd)
        check_backward(got, dy, xhat, off, w, rstd.cpu(), torch.float32, torch.float32)
        bad = F.layer_norm_bwd_from_output(dy.to(cuda), y, (cols,), w.to(cuda), b.to(cuda), rstd)
        assert bool(bad[1][5].isnan())


def test_gradient_against_differences(cuda):
    """sum(c * y) moved by a central difference of the 64-bit forward in x, w and b."""
    from monet_b200 import functional as F
    for cols in (5, 24, 33):
        x, c, w, b = make(4, cols, torch.float32, torch.float32)
        y, mean, rstd = F.layer_norm(x.to(cuda), (cols,), w.to(cuda), b.to(cuda))
        dx, dw, db = F.layer_norm_bwd_from_input(c.to(cuda), x.to(cuda), (cols,), w.to(cuda), mean, rstd)
        d = 1e-4
        f = lambda x, w, b: float((oracle.layer_norm_forward(x, w, b)[0] * c.double()).sum())     # noqa: E731
        # the difference quotient is off by d^2/6 of the third derivative: 1e-8 times values of order ten
        for i, j in ((0, 0), (1, cols // 2), (3, cols - 1)):
            e = torch.zeros(4, cols, dtype=torch.float64)
            e[i, j] = d
            assert abs((f(x.double() + e, w, b) - f(x.double() - e, w, b)) / (2 * d) - float(dx[i, j])) < 2e-5
            assert abs((f(x, w.double() + e[i], b) - f(x, w.double() - e[i], b)) / (2 * d) - float(dw[j])) < 2e-5
            assert abs((f(x, w, b.double() + e[i]) - f(x, w, b.double() - e[i])) / (2 * d) - float(db[j])) < 2e-5


def test_many_elements(cuda):
    """Element offsets and dropout indices past 2^32."""
    from monet_b200 import functional as F
    rows, cols = (1 << 22) + 3, 1024
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda)
    x.view(-1)[: 1 << 20].normal_()
    x[1024:] = x[:1024].repeat((rows - 1024 + 1023) // 1024, 1)[: rows - 1024]
    w, b = torch.rand(cols, device=cuda) + 0.5, torch.randn(cols, device=cuda)
    y, mean, rstd = F.layer_norm(x, (cols,), w, b)
    small = F.layer_norm(x[:1024], (cols,), w, b)
    for at in (0, (1 << 21) - 1024, 1 << 21, (1 << 22) - 1024):
        assert torch.equal(y[at:at + 1024], small[0]) and torch.equal(rstd[at:at + 1024], small[2])
    assert torch.equal(y[-3:], small[0][:3])
    del y
    seed = torch.tensor([21], device=cuda)
    z = F.dropout_add_layer_norm(x, x, (cols,), w, b, EPS, 0.25, seed)[1]
    tail = z[-8:].cpu()
    first = (rows - 8) * cols // 8
    import numpy as np
    halves = oracle.philox_words([np.arange(1024, dtype=np.uint64) + np.uint64(first), 0, 0, 0], 21).view("<u2").reshape(8, cols)
    keep = torch.from_numpy((halves >= 0x4000))
    xt = x[-8:].cpu().float()
    want = torch.where(keep, xt + xt * torch.tensor(1 / 0.75), xt).to(torch.bfloat16)
    assert torch.equal(tail, want)


def test_streams_graphs_and_repeatability(cuda):
    """A side stream, a captured forward + backward replayed on new inputs and a new seed, two graphs
    that run in turn, and two runs that agree bit for bit."""
    from monet_b200 import functional as F
    rows, cols = 300, 520
    res, dy, w, b = (a.to(cuda) for a in make(rows, cols, torch.bfloat16, torch.float32))
    x = make(rows, cols, torch.bfloat16, torch.float32, seed=1)[0].to(cuda)
    seed = torch.tensor([1234], device=cuda)

    def step(seed=seed):
        y, z, mean, rstd = F.dropout_add_layer_norm(x, res, (cols,), w, b, EPS, 0.3, seed, 1)
        return (y,) + F.dropout_add_layer_norm_bwd_from_sum(dy, z, (cols,), w, mean, rstd, 0.3, seed, 1, dz=dy)

    first = [t.clone() for t in step()]
    assert all(torch.equal(p, q) for p, q in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for value in (1234, 99, -5):
        seed.fill_(value)
        x.add_(0.5)
        for g, _ in graphs:
            g.replay()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(want, out))
    x.sub_(1.5)


def test_refusals(cuda):
    from monet_b200 import functional as F
    x, w = torch.randn(4, 16, device=cuda), torch.ones(16, device=cuda)
    stat = torch.ones(4, device=cuda)
    seed = torch.tensor([1], device=cuda)
    bad = [
        lambda: F.layer_norm(x.double(), (16,)), lambda: F.layer_norm(x.to(torch.int32), (16,)), lambda: F.layer_norm(x.cpu(), (16,)),
        lambda: F.layer_norm(x, (8,)), lambda: F.layer_norm(x, ()), lambda: F.layer_norm(x, (2, 4, 16)),
        lambda: F.layer_norm(x[:, :0], (0,)), lambda: F.layer_norm(x, (16,), w[:8]), lambda: F.layer_norm(x, (16,), w.cpu()),
        lambda: F.layer_norm(x, (16,), w.half()), lambda: F.layer_norm(x.half(), (16,), w.half(), w),
        lambda: F.layer_norm(x, (16,), w, w, -1.0), lambda: F.layer_norm(x, (16,), w, w, float("nan")),
        lambda: F.layer_norm_bwd_from_input(x, x[:2], (16,), w, stat, stat),
        lambda: F.layer_norm_bwd_from_input(x.half(), x, (16,), w, stat, stat),
        lambda: F.layer_norm_bwd_from_input(x, x, (16,), w, stat[:3], stat),
        lambda: F.layer_norm_bwd_from_input(x, x, (16,), w, stat, stat.double()),
        lambda: F.dropout_add_layer_norm(x, x[:1], (16,), w, w), lambda: F.dropout_add_layer_norm(x, x.half(), (16,), w, w),
        lambda: F.dropout_add_layer_norm(x, x, (16,), w, w, EPS, 0.5), lambda: F.dropout_add_layer_norm(x, x, (16,), w, w, EPS, 1.5, seed),
        lambda: F.dropout_add_layer_norm(x, x, (16,), w, w, EPS, 0.5, seed.cpu()),
        lambda: F.dropout_add_layer_norm(x, x, (16,), w, w, EPS, 0.5, seed.int()),
        lambda: F.dropout_add_layer_norm(x, x, (16,), w, w, EPS, 0.5, seed, -1),
        lambda: F.dropout_add_layer_norm_bwd_from_sum(x, x, (16,), w, stat, stat, dz=x[:2]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was not refused")
