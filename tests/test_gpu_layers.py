"""Layer norm, dropout and their residual add on the GPU against the float64 formulas of oracle/layer_norm.py, on the same
inputs.

Bounds.  u = 2^-24 is half a step of float32, half(T) = finfo(T).eps / 2 that of an output's type.  A sum over the C
channels of a row is formed by at most 16 additions in a lane, 6 between lanes and 16 between waves, so it is off by at
most 38 u times the sum of magnitudes; with the product by 1/C: D = 40.  Then, with A the row's mean of |x|,
  mean    off by D u A                        (e_m)
  rstd    relative (D + 8) u                  (squares, their sum, root and division; the mean's error is second order)
  hat     off by rstd e_m + (D + 10) u |hat|  (e_h)
  y       off by |w| e_h + 4 u (|w hat| + |b|), then half(T) |y|
  dx      with g = dy w:  rstd ( 3 u |g| + (D + 4) u (mean|g| + |hat| mean|g hat|) + |hat| mean(|g| e_h) + e_h |mean(g hat)| )
          + (D + 12) u |dx|, then half(T) |dx|
  columns a lane adds at most n / 128 + 1 rows, then 6 + 16 joins, then float64:
          dweight off by (n / 128 + 24) u sum|dy hat| + sum(|dy| e_h), dbias by (n / 128 + 24) u sum|dy|; then half(W)
The bounds are doubled once for the second-order terms left out."""
import copy

import numpy as np
import pytest
import torch

from oracle import layer_norm as O
from segmentation_amd import layers, ops, scenes, spunet, train

pytestmark = pytest.mark.gpu

U, D = 2.0 ** -24, 40
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _half(dtype, ref):
    """Half a step of `dtype` at `ref` (below the normal range: of the smallest normal number)."""
    f = torch.finfo(dtype)
    return f.eps / 2 * ref.abs().clamp_min(f.tiny)


def _close(name, got, ref, tol):
    err = (got.detach().double().cpu() - ref).abs()
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((err / tol.clamp_min(1e-300)).max()))


def _e_hat(x, mean, rstd):
    hat = (x - mean[:, None]) * rstd[:, None]
    return hat, rstd[:, None] * (D * U * x.abs().mean(1))[:, None] + (D + 10) * U * hat.abs()


def _tol_y(x, w, b, mean, rstd):
    hat, e = _e_hat(x, mean, rstd)
    return 2 * (w.abs() * e + 4 * U * ((w * hat).abs() + b.abs()))


def _tol_dx(x, dy, w, mean, rstd, dx):
    hat, e = _e_hat(x, mean, rstd)
    g = dy * w
    mg, mgh = g.abs().mean(1, keepdim=True), (g * hat).abs().mean(1, keepdim=True)
    s = 3 * U * g.abs() + (D + 4) * U * (mg + hat.abs() * mgh) + hat.abs() * (g.abs() * e).mean(1, keepdim=True) \
        + e * (g * hat).mean(1, keepdim=True).abs()
    return 2 * (rstd[:, None] * s + (D + 12) * U * dx.abs())


def _tol_columns(x, dy, mean, rstd):
    hat, e = _e_hat(x, mean, rstd)
    k = (x.shape[0] / 128 + 24) * U
    return 2 * (k * (dy * hat).abs().sum(0) + (dy.abs() * e).sum(0)), 2 * k * dy.abs().sum(0)


def _randn(seed, *shape, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def _sliced(t, pad, device):
    """t on the device as the front columns of a wider tensor."""
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=device)
    wide[:, :t.shape[1]] = t.to(device)
    return wide[:, :t.shape[1]]


SHAPES = [(1, 1), (3, 2), (1, 7), (5, 8), (2, 33), (64, 16), (130, 32), (1000, 96), (257, 100), (33, 255), (70, 256),
          (19, 513), (41, 768), (9, 1001), (7, 1500), (6, 2048), (5, 4096), (3, 5000), (4, 8192), (2, 8200), (3, 16383),
          (2, 16384)]
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)]


@pytest.mark.parametrize("xt,wt", TYPES)
@pytest.mark.parametrize("n,c", SHAPES)
def test_layer_norm(device, n, c, xt, wt):
    x, dy = _randn(1, n, c, dtype=xt, scale=1.5, shift=0.5), _randn(2, n, c, dtype=xt)
    w, b = _randn(3, c, dtype=wt, scale=0.2, shift=1.0), _randn(4, c, dtype=wt, scale=0.3)
    X, DY, W, B = x.double(), dy.double(), w.double(), b.double()
    Y, MEAN, RSTD = O.layer_norm(X, W, B)
    DX, DW, DB = O.layer_norm_backward(X, DY, MEAN, RSTD, W)
    for pad in (0, 3):
        xg, dyg = _sliced(x, pad, device), _sliced(dy, pad, device)
        y, mean, rstd = ops.layer_norm_fwd(xg, w.to(device), b.to(device))
        assert y.dtype == xt and mean.dtype == rstd.dtype == F32
        _close("mean", mean, MEAN, 2 * D * U * X.abs().mean(1))
        _close("rstd", rstd, RSTD, 2 * (D + 8) * U * RSTD)
        ty = _tol_y(X, W, B, MEAN, RSTD)
        _close("y", y, Y, ty + _half(xt, Y.abs() + ty))
        dx, dw, db = ops.layer_norm_backward(xg, dyg, mean, rstd, w.to(device))
        assert dx.dtype == xt and dw.dtype == db.dtype == wt
        tx = _tol_dx(X, DY, W, MEAN, RSTD, DX)
        _close("dx", dx, DX, tx + _half(xt, DX.abs() + tx))
        tw, tb = _tol_columns(X, DY, MEAN, RSTD)
        _close("dw", dw, DW, tw + _half(wt, DW.abs() + tw))
        _close("db", db, DB, tb + _half(wt, DB.abs() + tb))
    again = ops.layer_norm_backward(xg, dyg, mean, rstd, w.to(device))
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("n,c", [(20011, 32), (70000, 8), (3000, 800)])
def test_layer_norm_many_rows(device, n, c):
    """More rows than one sweep of the launch covers, without an affine pair and with each half of it."""
    x, dy = _randn(5, n, c, scale=2.0, shift=-3.0), _randn(6, n, c)
    X, DY = x.double(), dy.double()
    one = torch.ones(c, dtype=torch.float64)
    Y, MEAN, RSTD = O.layer_norm(X, eps=1e-3)
    y, mean, rstd = ops.layer_norm_fwd(x.to(device), eps=1e-3)
    ty = _tol_y(X, one, 0 * one, MEAN, RSTD)
    _close("y", y, Y, ty + _half(F32, Y))
    w = _randn(7, c)
    half = ops.layer_norm_fwd(x.to(device), w.to(device), None, 1e-3)[0]
    _close("y w", half, Y * w.double(), _tol_y(X, w.double(), 0 * one, MEAN, RSTD) + _half(F32, Y * w.double()))
    half = ops.layer_norm_fwd(x.to(device), None, w.to(device), 1e-3)[0]
    _close("y b", half, Y + w.double(), _tol_y(X, one, w.double(), MEAN, RSTD) + _half(F32, Y + w.double()))
    DX, DW, DB = O.layer_norm_backward(X, DY, MEAN, RSTD)
    for want_dw, want_db in ((True, True), (True, False), (False, True), (False, False)):
        dx, dw, db = ops.layer_norm_backward(x.to(device), dy.to(device), mean, rstd, None, want_dw, want_db)
        _close("dx", dx, DX, _tol_dx(X, DY, one, MEAN, RSTD, DX) + _half(F32, DX))
        tw, tb = _tol_columns(X, DY, MEAN, RSTD)
        assert (dw is not None) == want_dw and (db is not None) == want_db
        if want_dw:
            _close("dw", dw, DW, tw + _half(F32, DW))
        if want_db:
            _close("db", db, DB, tb + _half(F32, DB))


ADD_TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16)]


@pytest.mark.parametrize("xt,rt,wt", ADD_TYPES)
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 7), (130, 32), (257, 96), (70, 250), (41, 768), (9, 1001), (5, 4096), (3, 9000),
                                 (2, 16384)])
def test_dropout_add_layer_norm(device, n, c, p, xt, rt, wt):
    """p = 0.5 doubles a value exactly, so h is known to the bit: the float32 sum, rounded to the stream's type."""
    seed, offset = 0x123456789ABCDEF, (5 << 32) + 3
    x, r = _randn(11, n, c, dtype=xt, scale=1.5), _randn(12, n, c, dtype=rt, scale=2.0, shift=0.3)
    dy, dh = _randn(13, n, c, dtype=xt), _randn(14, n, c, dtype=rt)
    w, b = _randn(15, c, dtype=wt, scale=0.2, shift=1.0), _randn(16, c, dtype=wt, scale=0.3)
    keep = O.dropout_keep(n, c, p, seed, offset)
    scale = 1.0 / (1.0 - p)
    H = (r.float() + torch.where(keep, x.float() * scale, torch.zeros(()))).to(rt)
    HD, DY, DH, W, B = H.double(), dy.double(), dh.double(), w.double(), b.double()
    Y, MEAN, RSTD = O.layer_norm(HD, W, B)
    DX, DW, DB = O.layer_norm_backward(HD, DY, MEAN, RSTD, W)
    kw = dict(p=p, seed=seed, offset=offset)
    wg, bg = w.to(device), b.to(device)
    for pad in (0, 5):
        y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(_sliced(x, pad, device), _sliced(r, pad, device), wg, bg, **kw)
        assert y.dtype == xt and h.dtype == rt and torch.equal(h.cpu(), H)
        ty = _tol_y(HD, W, B, MEAN, RSTD)
        _close("y", y, Y, ty + _half(xt, Y.abs() + ty))
        for use_dh in (True, False):
            T = DX + DH if use_dh else DX
            tt = _tol_dx(HD, DY, W, MEAN, RSTD, DX) + U * T.abs()
            dx, dr, dw, db = ops.dropout_add_layer_norm_backward(
                _sliced(H, pad, device), _sliced(dy, pad, device), _sliced(dh, pad, device) if use_dh else None, mean, rstd,
                wg, **kw)
            _close("dresidual", dr, T, tt + _half(rt, T.abs() + tt))
            TX = torch.where(keep, T * scale, torch.zeros((), dtype=torch.float64))
            tx = tt * scale + 2 * U * TX.abs()
            assert (dx.cpu()[~keep] == 0).all()
            _close("dx", dx, TX, torch.where(keep, tx + _half(xt, TX.abs() + tx), torch.zeros((), dtype=torch.float64)))
            tw, tb = _tol_columns(HD, DY, MEAN, RSTD)
            _close("dw", dw, DW, tw + _half(wt, DW.abs() + tw))
            _close("db", db, DB, tb + _half(wt, DB.abs() + tb))
    with torch.inference_mode():   # (tensors made here have no version)
        ops.dropout_next(ops.dropout_state(1, device))
    bare = ops.dropout_add_layer_norm_fwd(x.to(device), r.to(device), wg, bg, want_h=False, **kw)
    assert bare[1] is None and torch.equal(bare[0], y)
    only = ops.dropout_add_layer_norm_backward(h, dy.to(device), None, mean, rstd, wg, want_dresidual=False,
                                               want_dweight=False, want_dbias=False, **kw)
    assert torch.equal(only[0], dx) and only[1] is None and only[2] is None and only[3] is None


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (5,), (1, 1), (3, 7), (1000, 3), (333, 96), (17, 1001), (4, 5, 64), (2, 70001)])
def test_dropout_values(device, shape, dtype):
    """Kept values are x / (1 - p) within half a float32 step for the factor, one for the product, half(T) for the
    result; the others are exactly 0.  The mask is the oracle's to the last value, and the same for every type."""
    x = _randn(21, *shape, dtype=dtype, scale=2.0)
    n, c = x.numel() // shape[-1], shape[-1]
    for p, seed, offset in ((0.1, 1, 0), (0.5, 2 ** 64 - 3, 2 ** 63 + 7), (0.9, 0, 2 ** 32), (1.0, 4, 4), (0.0, 4, 4)):
        keep = O.dropout_keep(n, c, p, seed, offset)
        ref = O.dropout(x.double().reshape(n, c), p, seed, offset)
        y = ops.dropout(x.to(device), p, seed, offset)
        assert y.shape == x.shape and y.dtype == dtype
        y = y.reshape(n, c)
        assert torch.equal(y.cpu() != 0, keep & (x.reshape(n, c) != 0))
        _close("y", y, ref, 2 * U * ref.abs() + _half(dtype, ref * (1 + 2 * U)))
    if len(shape) == 2:
        assert torch.equal(ops.dropout(_sliced(x, 9, device), 0.3, 5, 6), ops.dropout(x.to(device), 0.3, 5, 6))
        cols = x.to(device).t()   # column-major: the mask goes by the logical position
        assert torch.equal(ops.dropout(cols, 0.3, 5, 6), ops.dropout(cols.contiguous(), 0.3, 5, 6))


def test_dropped_values_hide_what_they_held(device):
    """A dropped value is 0 whatever it was, a kept NaN or infinity stays one; a row of the norm that holds one is NaN,
    and its neighbours are not touched."""
    n, c, p, seed, offset = 64, 40, 0.5, 3, 9
    keep = O.dropout_keep(n, c, p, seed, offset)
    x = _randn(31, n, c)
    x[~keep] = float("nan")
    x[5, :] = torch.where(keep[5], x[5], torch.full((), float("-inf")))
    y = ops.dropout(x.to(device), p, seed, offset).cpu()
    assert torch.equal(y, torch.where(keep, x * 2, torch.zeros(())))
    r = _randn(32, n, c)
    out, h, mean, rstd = ops.dropout_add_layer_norm_fwd(x.to(device), r.to(device), p=p, seed=seed, offset=offset)
    assert torch.isfinite(out).all() and torch.isfinite(h).all()
    clean = ops.dropout_add_layer_norm_fwd(torch.where(keep, x, torch.zeros(())).to(device), r.to(device), p=p, seed=seed,
                                           offset=offset)
    assert torch.equal(out, clean[0])
    r[7, 3], r[9, 4] = float("inf"), float("nan")
    bad = ops.dropout_add_layer_norm_fwd(x.to(device), r.to(device), p=p, seed=seed, offset=offset)[0]
    rows = torch.isnan(bad).any(1).nonzero().flatten().tolist()
    assert rows == [7, 9] and torch.isnan(bad[[7, 9]]).sum() >= 2 * (c - 1)
    others = [i for i in range(n) if i not in rows]
    assert torch.equal(bad[others], out[others])


def test_constant_rows_and_large_means(device):
    """Variance 0: y is the bias (eps keeps 1 / 0 away), dx is rstd (g - mean g).  A mean far above the deviation: the
    deviations are taken from the mean, not from a difference of squares."""
    c = 256
    x = torch.full((4, c), 3.0)
    x[1] = 0.0
    b = _randn(41, c)
    y, mean, rstd = ops.layer_norm_fwd(x.to(device), None, b.to(device))
    assert torch.equal(y.cpu(), b.expand(4, c)) and torch.equal(mean.cpu(), x[:, 0])
    assert torch.allclose(rstd.cpu(), torch.full((4,), 1e-5).rsqrt(), rtol=4 * U)
    dy = _randn(42, 4, c)
    dx, dw, _ = ops.layer_norm_backward(x.to(device), dy.to(device), mean, rstd)
    X = x.double()
    _, M, R = O.layer_norm(X)
    DX, _, _ = O.layer_norm_backward(X, dy.double(), M, R)
    _close("dx", dx, DX, _tol_dx(X, dy.double(), torch.ones(c, dtype=torch.float64), M, R, DX) + _half(F32, DX))
    assert (dw == 0).all()
    for shift in (1e3, -1e5):
        x = _randn(43, 50, c, shift=shift)
        X = x.double()
        Y, M, R = O.layer_norm(X)
        y, _, _ = ops.layer_norm_fwd(x.to(device))
        one = torch.ones(c, dtype=torch.float64)
        _close("y", y, Y, _tol_y(X, one, 0 * one, M, R) + _half(F32, Y))


def test_no_rows_and_other_shapes(device):
    w = torch.ones(16, device=device)
    x = torch.empty(0, 16, device=device)
    y, mean, rstd = ops.layer_norm_fwd(x, w, w)
    assert y.shape == (0, 16) and mean.shape == rstd.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all() and dw.shape == (16,)
    y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(x, x, w, w, p=0.3)
    dx, dr, dw, db = ops.dropout_add_layer_norm_backward(h, x, x, mean, rstd, w, p=0.3)
    assert dx.shape == dr.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    assert ops.dropout(x, 0.5).shape == (0, 16) and ops.dropout(torch.empty(3, 0, device=device), 0.5).shape == (3, 0)
    assert ops.dropout(torch.ones((), device=device), 0.0).item() == 1.0
    t = _randn(51, 3, 5, 24).to(device)
    flat = ops.layer_norm_fwd(t.reshape(15, 24))[0]
    assert torch.equal(ops.layer_norm_fwd(t)[0], flat.reshape(3, 5, 24))
    assert torch.equal(ops.layer_norm_fwd(t[:, 1])[0], flat.reshape(3, 5, 24)[:, 1])
    assert torch.equal(ops.layer_norm_fwd(t[0, 0])[0], flat[0])
    row = t[0, :1].expand(6, 24)   # the same row six times, stride 0
    assert torch.equal(ops.layer_norm_fwd(row)[0], flat[:1].expand(6, 24))
    turned = t[0].t().contiguous().t()   # column-major
    assert torch.equal(ops.layer_norm_fwd(turned)[0], flat[:5])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_addresses_off_the_16_byte_grid(device, dtype):
    """Slices that start at any element, and rows so far apart that the kernels do not address them (copied)."""
    for c in (8, 24, 40, 77):
        wide = _randn(52, 37, c + 8, dtype=dtype).to(device)
        for s in range(8):
            x, r = wide[:, s:s + c], wide[:, 8 - s:8 - s + c]
            xc, rc = x.contiguous(), r.contiguous()
            y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(x, r, p=0.25, seed=s)
            want = ops.dropout_add_layer_norm_fwd(xc, rc, p=0.25, seed=s)
            assert all(torch.equal(a, b) for a, b in zip((y, h, mean, rstd), want))
            got = ops.dropout_add_layer_norm_backward(h, x, r, mean, rstd, p=0.25, seed=s)
            assert all(torch.equal(a, b) for a, b in zip(got, ops.dropout_add_layer_norm_backward(h, xc, rc, mean, rstd,
                                                                                                  p=0.25, seed=s)))
            assert torch.equal(ops.layer_norm_fwd(x)[0], ops.layer_norm_fwd(xc)[0])
            assert torch.equal(ops.dropout(x, 0.25, s), ops.dropout(xc, 0.25, s))
            w = wide.flatten()[s:s + c]   # a weight off the grid
            assert torch.equal(ops.layer_norm_fwd(xc, w, w)[0], ops.layer_norm_fwd(xc, w.clone(), w.clone())[0])
    far = torch.zeros(3, (1 << 20) + 40, dtype=dtype, device=device)
    far[:, :77] = wide[:3, :77]
    assert torch.equal(ops.layer_norm_fwd(far[:, :77])[0], ops.layer_norm_fwd(wide[:3, :77].contiguous())[0])
    assert torch.equal(ops.dropout(far[:, :77], 0.5, 3), ops.dropout(wide[:3, :77].contiguous(), 0.5, 3))


def test_rows_behind_the_last_are_left_alone(device):
    """The kernels write their own rows and channels, nothing behind them."""
    import ctypes
    from segmentation_amd import _lib
    lib = _lib.load()
    for n, c in ((5, 33), (3, 7), (1, 1001), (9, 4)):
        x = _randn(61, n, c).to(device)
        out = torch.full((n * c + 64,), 7.0, device=device)
        stats = torch.full((2, n + 8), 7.0, device=device)
        p = lambda t: ctypes.c_void_p(t.data_ptr())
        s = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        null = ctypes.c_void_p(0)
        assert lib.m3d_layer_norm_fwd(p(x), c, 0, n, c, null, null, 0, 1e-5, p(out), p(stats[0]), p(stats[1]), s) == 0
        assert torch.equal(out[:n * c].reshape(n, c), ops.layer_norm_fwd(x)[0])
        assert (out[n * c:] == 7.0).all() and (stats[:, n:] == 7.0).all()
        dx, dw = torch.full_like(out, 7.0), torch.full((c + 8,), 7.0, device=device)
        nb = lib.m3d_layer_norm_workspace_bytes(n, c, 0)
        ws = torch.full((nb + 64,), 9, dtype=torch.uint8, device=device)
        assert lib.m3d_layer_norm_backward(p(x), c, p(x), c, 0, n, c, p(stats[0]), p(stats[1]), null, 0, p(dx), p(dw), null,
                                           p(ws), nb, s) == 0
        assert (dx[n * c:] == 7.0).all() and (dw[c:] == 7.0).all() and (ws[nb:] == 9).all()
        y = torch.full_like(out, 7.0)
        assert lib.m3d_dropout(p(x), c, 0, n, c, 0.5, 1, 2, null, p(y), s) == 0
        assert (y[n * c:] == 7.0).all()


# ---------------------------------------------------------------- derivatives
def test_gradients_against_differences(device):
    """<dx, v> of the kernels against a central difference of the float64 formula along v: truncation below
    step^2 * 1e2 (third derivatives of a layer norm of unit-variance rows), gradients within the bounds above."""
    n, c, step = 6, 48, 1e-4
    x, r, w, b = _randn(71, n, c), _randn(72, n, c), _randn(73, c, shift=1.0), _randn(74, c)
    dy, dh = _randn(75, n, c).double(), _randn(76, n, c).double()
    p, seed, offset = 0.5, 17, 23
    args = [t.to(device).requires_grad_() for t in (x, r, w, b)]
    y, h = layers.dropout_add_layer_norm(*args, p=p, seed=seed, offset=offset)
    grads = torch.autograd.grad((y, h), args, (dy.float().to(device), dh.float().to(device)))

    def value(x, r, w, b):
        H = r + O.dropout(x, p, seed, offset)
        return (O.layer_norm(H, w, b)[0] * dy).sum() + (H * dh).sum()

    at = [t.double() for t in (x, r, w, b)]
    for k, g in enumerate(grads):
        v = _randn(80 + k, *at[k].shape).double()
        up, down = [list(at), list(at)]
        up[k], down[k] = at[k] + step * v, at[k] - step * v
        ref = (value(*up) - value(*down)) / (2 * step)
        got = (g.double().cpu() * v).sum()
        # every gradient is within 200 u of its value plus 200 u (the bounds above for rows of unit scale)
        tol = (200 * U * (g.double().cpu().abs() + 1) * v.abs()).sum() + 100 * step ** 2
        assert abs(float(got - ref)) <= float(tol), (k, float(got), float(ref), float(tol))


def test_autograd_matches_the_operators(device):
    n, c = 50, 96
    x, r = _randn(91, n, c, dtype=BF16).to(device), _randn(92, n, c).to(device)
    w, b = _randn(93, c).to(device), _randn(94, c).to(device)
    kw = dict(p=0.3, seed=5, offset=6)
    dy, dh = _randn(95, n, c, dtype=BF16).to(device), _randn(96, n, c).to(device)
    xs = [t.clone().requires_grad_() for t in (x, r, w, b)]
    y, h = layers.dropout_add_layer_norm(*xs, **kw)
    y0, h0, mean, rstd = ops.dropout_add_layer_norm_fwd(x, r, w, b, **kw)
    assert torch.equal(y, y0) and torch.equal(h, h0)
    full = ops.dropout_add_layer_norm_backward(h0, dy, dh, mean, rstd, w, **kw)
    got = torch.autograd.grad((y, h), xs, (dy, dh), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, full))
    # only one of the outputs used
    only_y = torch.autograd.grad(y, xs, dy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(only_y, ops.dropout_add_layer_norm_backward(h0, dy, None, mean, rstd, w, **kw)))
    only_h = torch.autograd.grad(h, xs, dh, retain_graph=True, allow_unused=True)
    assert torch.equal(only_h[1], dh) and torch.equal(only_h[0], ops.dropout(dh, **kw).to(BF16))
    assert (only_h[2] == 0).all() and (only_h[3] == 0).all()
    # a gradient that is broadcast, and inputs that need none
    y1, _ = layers.dropout_add_layer_norm(x, xs[1], w, b, **kw)
    g = torch.autograd.grad(y1.float().sum(), xs[1])[0]
    assert torch.equal(g, ops.dropout_add_layer_norm_backward(h0, torch.ones_like(x), None, mean, rstd, w, **kw)[1])
    z = layers.layer_norm(xs[0], xs[2], xs[3])
    gz = torch.autograd.grad(z, (xs[0], xs[2], xs[3]), dy)
    _, m2, r2 = ops.layer_norm_fwd(x, w, b)
    assert all(torch.equal(p, q) for p, q in zip(gz, ops.layer_norm_backward(x, dy, m2, r2, w)))
    d = layers.dropout(xs[0], **kw)
    assert torch.equal(torch.autograd.grad(d, xs[0], dy)[0], ops.dropout(dy, **kw))
    # without dropout the gradients of x and residual are one tensor; as leaves they are filled independently
    f = [_randn(97, n, c).to(device).requires_grad_(), _randn(98, n, c).to(device).requires_grad_()]
    for _ in range(2):
        layers.dropout_add_layer_norm(f[0], f[1], w, b)[0].float().pow(2).sum().backward()
        f[0].grad.zero_()
    assert (f[0].grad == 0).all() and f[1].grad.abs().sum() > 0
    # the same tensor as x and as residual
    s = _randn(99, n, c).to(device).requires_grad_()
    ys, hs = layers.dropout_add_layer_norm(s, s, w, b)
    assert torch.equal(hs, 2 * s)
    gs = torch.autograd.grad(hs.sum(), s)[0]
    assert (gs == 2).all()
    with pytest.raises(RuntimeError, match="once_differentiable"):
        t = _randn(90, 4, c).to(device).requires_grad_()
        (g1,) = torch.autograd.grad(layers.layer_norm(t, w, b).pow(2).sum(), t, create_graph=True)
        g1.sum().backward()


# ---------------------------------------------------------------- streams, graphs, workspaces, state
def test_generator_state(device):
    x = _randn(101, 30, 50).to(device)
    st = ops.dropout_state(77, device, offset=5)
    a, b = ops.dropout_next(st), ops.dropout_next(st, step=3)
    assert a.tolist() == [77, 5] and b.tolist() == [77, 6] and st.tolist() == [77, 9]
    assert torch.equal(ops.dropout(x, 0.4, state=a), ops.dropout(x, 0.4, 77, 5))
    assert torch.equal(ops.dropout(x, 0.4, offset=2, state=b), ops.dropout(x, 0.4, 77, 8))
    m = layers.Dropout(0.4, seed=77).to(device)
    y0, y1 = m(x), m(x)
    assert torch.equal(y0, ops.dropout(x, 0.4, 77, 0)) and torch.equal(y1, ops.dropout(x, 0.4, 77, 1))
    m2 = layers.Dropout(0.4, seed=1).to(device)
    m2.load_state_dict(m.state_dict())
    assert torch.equal(m2(x), m(x))
    assert m.eval()(x) is x


def test_a_state_that_moved_on_is_refused(device):
    """A backward pass whose mask can no longer be formed says so; a drawn state is the caller's to keep, and serves a
    forward that is computed twice (activation checkpointing)."""
    from torch.utils.checkpoint import checkpoint
    x = _randn(102, 40, 24).to(device).requires_grad_()
    st = ops.dropout_state(5, device)
    for y in (layers.dropout(x, 0.5, state=st), layers.dropout_add_layer_norm(x, x, p=0.5, state=st)[0]):
        ops.dropout_next(st)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    block = layers.DropoutAddLayerNorm(24, 0.5, seed=9).to(device)
    gy = _randn(103, 40, 24).to(device)
    st = block.drop.draw()
    direct = torch.autograd.grad((block(x, x, st)[0] * gy).sum(), x)[0]
    again = torch.autograd.grad((checkpoint(lambda t: block(t, t, st)[0], x, use_reentrant=False) * gy).sum(), x)[0]
    assert torch.equal(direct, again) and block.drop.rng.tolist() == [9, 1]


def test_block_in_a_captured_graph(device):
    """A block's forward and backward, captured: every replay draws masks of its own from the state on the device and
    gives what eager calls with those masks give; eager work runs in between on the same stream's workspace."""
    n, c, p = 300, 128, 0.3
    block = layers.DropoutAddLayerNorm(c, p, seed=11).to(device)
    block.norm.weight.data.normal_(1.0, 0.2)
    x, r = _randn(111, n, c).to(device), _randn(112, n, c).to(device)
    dy, dh = _randn(113, n, c).to(device), _randn(114, n, c).to(device)
    w, b = block.norm.weight.detach(), block.norm.bias.detach()
    sx, sr = x.clone(), r.clone()

    def step():
        st = ops.dropout_next(block.drop.rng)
        y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(sx, sr, w, b, p=p, state=st)
        return (y, h) + ops.dropout_add_layer_norm_backward(h, dy, dh, mean, rstd, w, p=p, state=st)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    block.drop.rng.copy_(ops.dropout_state(11, device))
    seen = []
    for k in range(4):
        g, out = graphs[k % 2]
        sx.copy_(x * (k + 1))
        g.replay()
        torch.cuda.synchronize()
        kw = dict(p=p, seed=11, offset=k)
        y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(sx, sr, w, b, **kw)
        want = (y, h) + ops.dropout_add_layer_norm_backward(h, dy, dh, mean, rstd, w, **kw)
        assert all(torch.equal(a, e) for a, e in zip(out, want)), k
        seen.append(out[1].clone())
    assert block.drop.rng.tolist() == [11, 4]
    assert not torch.equal(seen[0], seen[2])
    # two graphs captured on one stream, replayed side by side on two: their workspaces are their own
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    st = block.drop.rng.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        graphs[0][0].replay()
    torch.cuda.synchronize()
    ref0 = [t.clone() for t in graphs[0][1][4:]]
    block.drop.rng.copy_(st)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        graphs[0][0].replay()
    with torch.cuda.stream(s2):
        layers.layer_norm(x.clone().requires_grad_(), w.clone().requires_grad_(), b).sum().backward()
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(graphs[0][1][4:], ref0))


def test_training_step_captured_through_autograd(device):
    """Forward and backward of a module under capture, after the usual warm-up on a side stream."""
    n, c = 200, 64
    block = layers.DropoutAddLayerNorm(c, 0.2, seed=3).to(device)
    x = _randn(121, n, c).to(device)
    gy, gh = _randn(122, n, c).to(device), _randn(123, n, c).to(device)
    params = list(block.parameters())

    def step():
        return torch.autograd.grad(block(x, x), params, (gy, gh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    block.drop.rng.copy_(ops.dropout_state(3, device))
    twin = copy.deepcopy(block)
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(twin(x, x), list(twin.parameters()), (gy, gh))
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, want)), k


def test_other_streams_and_side_by_side_calls(device):
    """Calls on two streams have workspaces of their own and give the bits of the default stream."""
    n, c = 5000, 256
    x, dy = _randn(131, n, c).to(device), _randn(132, n, c).to(device)
    _, mean, rstd = ops.layer_norm_fwd(x)
    want = ops.layer_norm_backward(x, dy, mean, rstd)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.layer_norm_backward(x, dy, mean, rstd))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, e) for a, e in zip(g, want))


def test_offsets_beyond_32_bits(device):
    """More than 2^32 bytes and 2^31 values in one tensor, and rows whose slices lie far apart."""
    n, c = 140000, 16384   # 2.3e9 values, 4.6 GB
    x = torch.zeros(n, c, dtype=BF16, device=device)
    rows = [0, 131071, 131072, n - 1]
    tail = _randn(141, len(rows), c, dtype=BF16).to(device)
    x[rows] = tail
    y, mean, rstd = ops.layer_norm_fwd(x)
    small, m2, r2 = ops.layer_norm_fwd(tail)
    assert torch.equal(y[rows], small) and torch.equal(mean[rows], m2) and torch.equal(rstd[rows], r2)
    assert (y[5] == 0).all()
    dx, dw, _ = ops.layer_norm_backward(x, y, mean, rstd)
    assert torch.equal(dx[rows], ops.layer_norm_backward(tail, small, m2, r2)[0])
    del dx, dw, y
    z = ops.dropout(x, 0.5, 3, 4)
    keep = O.dropout_keep(1, c, 0.5, 3, 4)
    assert torch.equal(z[0].cpu() != 0, keep[0] & (tail[0].cpu() != 0))
    # row n - 1 alone, through the generator's definition
    words = O.philox4x32((np.arange(c // 4), np.full(c // 4, n - 1), 4, 0), (3, 0), 7)
    last = torch.from_numpy(np.stack(words, -1).reshape(-1).astype(np.int64) >= 2 ** 31)
    assert torch.equal(z[-1].cpu() != 0, last & (tail[-1].cpu() != 0))


def test_more_rows_than_31_bits(device):
    """2^31 + 100 rows of one channel: several launches of the dropout, 64-bit rows in the norm."""
    n = 2 ** 31 + 100
    x = torch.ones(n, 1, dtype=BF16, device=device)
    y = ops.dropout(x, 0.5, 7, 8)
    for lo in (0, 0x7fff0000 - 50, n - 100):
        words = O.philox4x32((0, np.arange(lo, lo + 100), 8, 0), (7, 0), 7)[0]
        keep = torch.from_numpy(words.astype(np.int64) >= 2 ** 31)
        assert torch.equal(y[lo:lo + 100, 0].cpu() == 2, keep) and torch.equal(y[lo:lo + 100, 0].cpu() == 0, ~keep)
    x[-1] = 5
    b = torch.full((1,), 0.25, dtype=BF16, device=device)
    del y
    y, mean, rstd = ops.layer_norm_fwd(x, None, b)
    assert mean[-2:].tolist() == [1.0, 5.0] and y[-1].item() == 0.25 and y[2 ** 30].item() == 0.25
    del y, rstd


def test_tensors_of_a_wrong_place_are_refused(device):
    x = torch.zeros(4, 8, device=device)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.layer_norm_fwd(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.dropout(x, 0.5, state=ops.dropout_state(1, "cpu"))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.dropout_add_layer_norm_fwd(x, torch.zeros(4, 8))


# ---------------------------------------------------------------- the backbone
def _batch(device):
    sc = scenes.make_scene(seed=3, target_voxels=1500)
    n = sc["coord"].shape[0]
    return dict(coord=torch.from_numpy(sc["coord"]).to(device), feat=torch.from_numpy(sc["feat"]).to(device),
                offset=torch.tensor([0, n]), grid_size=0.02, condition=["ScanNet"])


def test_backbone_with_layer_norms(device):
    """SpUNet(norm="layer"): in evaluation mode deterministic; in training mode every block drops values of its own and
    moves its generator on; the gradient of every used parameter is finite and there; and a block's norm equals the
    oracle's on what it was given."""
    torch.manual_seed(5)
    net = spunet.PPT(spunet.SpUNet(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32, norm="layer",
                                   dropout=0.2)).to(device)
    batch = _batch(device)
    seen = []
    block = net.backbone.enc[0].block0
    handle = block.bn2.register_forward_hook(lambda m, args, kwargs, out: seen.append((args, kwargs, out)), with_kwargs=True)
    net.eval()
    with torch.no_grad():
        a, b = net(dict(batch))["feat"], net(dict(batch))["feat"]
    assert torch.equal(a, b) and torch.isfinite(a).all()
    args, kwargs, out = seen[0]
    H = (kwargs["residual"] + args[0]).double().cpu()
    ln = block.bn2.pick("ScanNet")
    Y, M, R = O.layer_norm(H, ln.weight.double().cpu().detach(), ln.bias.double().cpu().detach(), ln.eps)
    one = torch.ones(H.shape[1], dtype=torch.float64)
    # (zero-initialised modulation: weight 1, bias 0)
    _close("block", out, Y.clamp_min(0), _tol_y(H, one, 0 * one, M, R) + _half(F32, Y))
    handle.remove()
    net.train()
    c = net(dict(batch))["feat"]
    d = net(dict(batch))["feat"]
    assert not torch.equal(c, d) and not torch.equal(c, a)
    assert block.bn2.drop.rng[1].item() == 2 and block.bn1.drop.rng[1].item() == 0
    d.square().mean().backward()
    used = [(k, p) for k, p in net.named_parameters() if ".bns." not in k or ".bns.0." in k]
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for _, p in used)


@pytest.mark.parametrize("decouple,adaptive,affine", [(True, True, True), (True, True, False), (False, False, True),
                                                      (False, True, True), (True, False, False)])
@pytest.mark.parametrize("with_res,relu", [(False, False), (True, True)])
def test_pd_layer_norm_matches_float64(device, decouple, adaptive, affine, with_res, relu):
    """relu?(layer norm(residual + x) (1 + scale) + shift) with its gradients, every combination of the options.  Bars as
    for the batch norms: relative 2-norm 1e-5 of outputs and input gradients, 1e-4 of parameters."""
    torch.manual_seed(8)
    m = spunet.PDLayerNorm(48, 32, decouple=decouple, adaptive=adaptive, affine=affine)
    for p in m.parameters():
        p.data.normal_(0.0, 0.3)
    ref = copy.deepcopy(m).double()
    m = m.to(device)
    x, res, ctx, gy = _randn(151, 90, 48), _randn(152, 90, 48), _randn(153, 1, 32), _randn(154, 90, 48)
    ins = [t.to(device).requires_grad_() for t in (x, res, ctx)]
    y = m(ins[0], "Matterport3D", ins[2], residual=ins[1] if with_res else None, relu=relu)
    X, R, C = (t.double().requires_grad_() for t in (x, res, ctx))
    H = X + R if with_res else X
    D = H - H.mean(1, keepdim=True)
    Y = D * (D.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    ln = ref.bns[2] if decouple else ref.bn
    if affine:
        Y = Y * ln.weight + ln.bias
    if adaptive:
        shift, scale = ref.modulation(C).chunk(2, dim=1)
        Y = Y * (1.0 + scale) + shift
    if relu:
        gy = gy * (Y.detach().abs() > 1e-4).float()   # no gradient within rounding distance of the kink
        Y = Y.clamp_min(0)
    y.backward(gy.to(device))
    Y.backward(gy.double())
    rel = lambda a, b: float((a.detach().double().cpu() - b).norm() / b.norm())
    assert rel(y, Y.detach()) < 1e-5 and rel(ins[0].grad, X.grad) < 1e-5
    assert not with_res or rel(ins[1].grad, R.grad) < 1e-5
    for (k, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        assert (p.grad is None) == (q.grad is None), k
        assert q.grad is None or rel(p.grad, q.grad) < 1e-4, k
    assert not adaptive or rel(ins[2].grad, C.grad) < 1e-4


def test_optimisation_step_with_layer_norms(device):
    """train.TrainStep on the layer-norm backbone: parameters of the used condition move, and stay finite."""
    torch.manual_seed(6)
    net = spunet.PPT(spunet.SpUNet(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=64, norm="layer",
                                   dropout=0.1)).to(device)
    batch = _batch(device)
    n = batch["coord"].shape[0]
    emb = [[torch.nn.functional.normalize(_randn(150 + i, 64), dim=0).to(device) for i in range(4)]]
    idx = [[torch.arange(i * 50, i * 50 + 200) % n for i in range(4)]]
    pi, co, cnt = train.flatten_caption_indices(idx, torch.tensor([0, n]))
    batch["caption_data"] = dict(embedding=emb, point_indices=pi, caption_offsets=co, num_points_per_caption=cnt)
    before = {k: p.detach().clone() for k, p in net.named_parameters()}
    step = train.TrainStep(net, total_steps=100)
    losses = [step(dict(batch)) for _ in range(2)]
    assert np.isfinite(losses).all()
    moved = [k for k, p in net.named_parameters() if not torch.equal(p, before[k])]
    assert all(torch.isfinite(p).all() for p in net.parameters())
    assert any(".bns.0.weight" in k for k in moved) and any("conv2.weight" in k for k in moved)


def test_checkpointed_backbone_with_dropout(device):
    """The whole network under activation checkpointing: refused where its blocks draw for themselves, and with states
    that were drawn in front of it the gradients of the plain call with those states (bar: the order of the sums of the
    convolutions' gradients, relative 2-norm 1e-4 as for parameters above)."""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(9)
    net = spunet.PPT(spunet.SpUNet(channels=(32, 64, 64, 32), layers=(1, 1, 1, 1), out_channels=32, norm="layer",
                                   dropout=0.3)).to(device)
    batch = _batch(device)
    params = [p for k, p in net.named_parameters() if "conv2.weight" in k]
    feat = batch.pop("feat").requires_grad_()
    run = lambda f, **kw: net(dict(batch, feat=f, **kw))["feat"].square().mean()
    with pytest.raises(RuntimeError, match="inside a backward pass"):
        checkpoint(run, feat, use_reentrant=False).backward()
    states = net.backbone.draw_dropout()
    want = torch.autograd.grad(run(feat, dropout_states=states), params)
    other = torch.autograd.grad(run(feat), params)   # masks of its own
    counts = [m.drop.rng[1].item() for m in net.backbone._dropping_norms()]
    got = torch.autograd.grad(checkpoint(lambda f: run(f, dropout_states=states), feat, use_reentrant=False), params)
    assert counts == [m.drop.rng[1].item() for m in net.backbone._dropping_norms()]
    rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())
    assert all(rel(a, b) < 1e-4 for a, b in zip(got, want))
    assert any(rel(a, b) > 1e-2 for a, b in zip(other, want))


def test_a_captured_call_names_its_mask(device):
    """Functions that would draw a seed on the host are refused under capture, and run outside."""
    x = _randn(161, 8, 16).to(device)
    torch.manual_seed(0)
    a, b = layers.dropout(x, 0.5), layers.dropout(x, 0.5)
    torch.manual_seed(0)
    assert not torch.equal(a, b) and torch.equal(a, layers.dropout(x, 0.5))
    st = ops.dropout_state(4, device)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="captured call"):
            layers.dropout(x, 0.5)
        with pytest.raises(RuntimeError, match="captured call"):
            layers.dropout_add_layer_norm(x, x, p=0.5)
        y = layers.dropout(x, 0.5, state=ops.dropout_next(st))
    for k in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.dropout(x, 0.5, 4, k))


def test_modules_made_on_the_device(device):
    """Under a default device the generator lies where the parameters do."""
    with torch.device(device):
        block = layers.DropoutAddLayerNorm(16, 0.5, seed=2)
        drawn = layers.Dropout(0.5)
    assert block.drop.rng.device == block.norm.weight.device == drawn.rng.device
    x = _randn(171, 4, 16).to(device)
    assert torch.equal(block(x, x)[1], ops.dropout_add_layer_norm_fwd(x, x, p=0.5, seed=2)[1])
    assert drawn(x).shape == x.shape


@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("n,c", [(5, 3), (4, 7), (9, 33), (6, 96), (7, 100), (5, 768), (3, 1001), (2, 5000), (2, 16383)])
def test_rows_far_from_zero(device, n, c, xt):
    """Rows whose values lie far from zero against their deviations (equal values among them): y must not depend on where
    they lie.  The first mean m is off by at most d = D u A; the deviations from it are exact up to u of themselves (they
    are small against the values), so with E the row's mean of |x - mean| the corrected mean is off by D u (E + d).  The
    variance is off by (D + 8) u (var + 2 d^2), of which rstd has half relative to var + eps."""
    for scale, shift in ((0.0, 1234.567), (0.0, -77.7), (0.0, 98765.4), (1.0, 1000.3), (0.1, -1e4), (1.0, 1e5)):
        x = _randn(181, n, c, scale=scale, shift=shift).to(xt)
        X = x.double()
        w, b = _randn(182, c, shift=1.0), _randn(183, c)
        W, B = w.double(), b.double()
        Y, MEAN, RSTD = O.layer_norm(X, W, B)
        d = D * U * X.abs().mean(1)
        e = (X - MEAN[:, None]).abs().mean(1)
        rel = (D + 8) * U * (1 / RSTD ** 2 + 2 * d ** 2) * RSTD ** 2
        hat = (X - MEAN[:, None]) * RSTD[:, None]
        eh = RSTD[:, None] * (D * U * (e + d))[:, None] + (rel[:, None] + 10 * U) * hat.abs()
        ty = 2 * (W.abs() * eh + 4 * U * ((W * hat).abs() + B.abs()))
        wg, bg = w.to(device), b.to(device)
        if xt == F32:
            y, mean, rstd = ops.layer_norm_fwd(x.to(device), wg, bg)
            _close("y", y, Y, ty + _half(F32, Y.abs() + ty))
        else:   # behind the add, whose stream is f32: 16-bit rows lie too far apart to be told from their mean
            zero = torch.zeros(n, c, dtype=xt, device=device)
            y, _, mean, rstd = ops.dropout_add_layer_norm_fwd(zero, x.float().to(device), wg, bg)
            _close("y", y, Y, ty + _half(xt, Y.abs() + ty))
        _close("mean", mean, MEAN, U * MEAN.abs() + 2 * D * U * (e + d))   # one rounding of the mean itself
        _close("rstd", rstd, RSTD, 2 * rel * RSTD)
        if scale == 0.0:
            assert torch.equal(mean.cpu(), x[:, 0].float())
            dy = _randn(184, n, c, dtype=xt).to(device)
            back = ops.layer_norm_backward(x.to(device), dy, mean, rstd, wg)
            assert (back[1] == 0).all()


def test_overflowing_squares_leave_the_bias(device):
    """Values whose squares leave float32: rstd is 0 and y the bias, also where all values are equal."""
    b = _randn(191, 33).to(device)
    for x in (torch.full((3, 33), 1e36), _randn(192, 3, 33, scale=1e25)):
        y, _, rstd = ops.layer_norm_fwd(x.to(device), None, b)
        assert torch.isfinite(y).all()
    assert torch.equal(y, b.expand(3, 33)) and (rstd == 0).all()


# ---------------------------------------------------------------- more rows than one sweep of the launch covers
@pytest.mark.parametrize("n,c,xt,rt,wt", [
    (40011, 96, F32, F32, F32), (40001, 64, BF16, F32, F32), (70001, 33, F32, F32, F32), (17001, 333, F16, F16, F16),
    (70003, 77, BF16, BF16, F32),                                  # f32 weights on a 16-bit stream
    (1101, 4096, BF16, BF16, BF16), (601, 3000, F32, F32, F32),    # rows of 256 lanes: workgroups of 512 in the backward pass
    (701, 7000, BF16, F32, F32),                                   # rows of 512 lanes
    (300, 9000, F32, F32, F32), (301, 13001, BF16, BF16, F32)])    # rows of 1024 lanes
def test_add_over_several_tiles(device, n, c, xt, rt, wt):
    """Every workgroup walks over several tiles: the next tile's rows, the mask's row index, dh beside the tile in flight
    and the column sums over all of them.  p = 0.5 doubles exactly, so h is known to the bit."""
    p, seed, offset = 0.5, 77, 5
    x, r = _randn(201, n, c, dtype=xt, scale=1.5), _randn(202, n, c, dtype=rt, scale=2.0, shift=0.3)
    dy, dh = _randn(203, n, c, dtype=xt), _randn(204, n, c, dtype=rt)
    w, b = _randn(205, c, dtype=wt, scale=0.2, shift=1.0), _randn(206, c, dtype=wt, scale=0.3)
    keep = O.dropout_keep(n, c, p, seed, offset)
    H = (r.float() + torch.where(keep, x.float() * 2, torch.zeros(()))).to(rt)
    HD, DY, W, B = H.double(), dy.double(), w.double(), b.double()
    Y, MEAN, RSTD = O.layer_norm(HD, W, B)
    DX, DW, DB = O.layer_norm_backward(HD, DY, MEAN, RSTD, W)
    kw = dict(p=p, seed=seed, offset=offset)
    wg, dyg = w.to(device), dy.to(device)
    y, h, mean, rstd = ops.dropout_add_layer_norm_fwd(x.to(device), r.to(device), wg, b.to(device), **kw)
    assert torch.equal(h.cpu(), H)
    ty = _tol_y(HD, W, B, MEAN, RSTD)
    _close("y", y, Y, ty + _half(xt, Y.abs() + ty))
    T = DX + dh.double()
    tt = _tol_dx(HD, DY, W, MEAN, RSTD, DX) + U * T.abs()
    dx, dr, dw, db = ops.dropout_add_layer_norm_backward(h, dyg, dh.to(device), mean, rstd, wg, **kw)
    _close("dresidual", dr, T, tt + _half(rt, T.abs() + tt))
    TX, tx = 2 * T, 2 * tt + 4 * U * T.abs()
    zero = torch.zeros((), dtype=torch.float64)
    _close("dx", dx, torch.where(keep, TX, zero), torch.where(keep, tx + _half(xt, TX.abs() + tx), zero))
    tw, tb = _tol_columns(HD, DY, MEAN, RSTD)
    _close("dw", dw, DW, tw + _half(wt, DW.abs() + tw))
    _close("db", db, DB, tb + _half(wt, DB.abs() + tb))
    if xt == rt:   # the norm alone over as many tiles
        dx, dw, db = ops.layer_norm_backward(h, dyg, mean, rstd, wg)
        tx = _tol_dx(HD, DY, W, MEAN, RSTD, DX)
        _close("dx alone", dx, DX, tx + _half(xt, DX.abs() + tx))
        _close("dw alone", dw, DW, tw + _half(wt, DW.abs() + tw))
        _close("db alone", db, DB, tb + _half(wt, DB.abs() + tb))


def test_captured_graphs_have_workspaces_of_their_own(device, monkeypatch):
    """Two backward passes captured on one stream, of different inputs: their workspaces differ from each other and from
    every eager one, and replayed side by side on two streams, beside eager work, each gives its own result."""
    n, c = 4000, 512
    ins = [(_randn(211 + k, n, c).to(device), _randn(213 + k, n, c).to(device)) for k in range(2)]
    stats = [ops.layer_norm_fwd(x)[1:] for x, _ in ins]
    want = [ops.layer_norm_backward(x, dy, *st) for (x, dy), st in zip(ins, stats)]
    torch.cuda.synchronize()
    real, spans, graphs = ops._scratch, [], []

    def recorded(nbytes, dev):
        ws = real(nbytes, dev)
        spans.append((ws.data_ptr(), ws.data_ptr() + ws.numel()))
        return ws

    side = torch.cuda.Stream()
    monkeypatch.setattr(ops, "_scratch", recorded)
    for (x, dy), st in zip(ins, stats):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.layer_norm_backward(x, dy, *st)
        graphs.append((g, out))
    monkeypatch.setattr(ops, "_scratch", real)
    assert len(spans) == 2
    spans += [(t.data_ptr(), t.data_ptr() + t.numel()) for t in ops._workspaces.values()]
    spans.sort()
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), spans
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side):
            ops.layer_norm_backward(*ins[1], *stats[1])
        torch.cuda.synchronize()
        for (_, out), ref in zip(graphs, want):
            assert all(torch.equal(a, e) for a, e in zip(out, ref))
            for t in out:
                t.zero_()


@pytest.mark.parametrize("decouple,adaptive,affine", [(True, True, True), (True, True, False), (False, False, True)])
@pytest.mark.parametrize("given", [False, True])
def test_pd_layer_norm_with_dropout_matches_float64(device, decouple, adaptive, affine, given):
    """A training block: relu(layer norm(residual + dropout(x)) (1 + scale) + shift) and its gradients, with the mask of the
    module's generator, drawn by the call or handed in.  Bars as in test_pd_layer_norm_matches_float64."""
    torch.manual_seed(12)
    p, n, c = 0.5, 90, 48
    m = spunet.PDLayerNorm(c, 32, decouple=decouple, adaptive=adaptive, affine=affine, dropout=p, seed=21)
    for q in m.parameters():
        q.data.normal_(0.0, 0.3)
    ref = copy.deepcopy(m).double()
    m = m.to(device)
    x, res, ctx, gy = _randn(221, n, c), _randn(222, n, c), _randn(223, 1, 32), _randn(224, n, c)
    for call in range(2):
        ins = [t.to(device).requires_grad_() for t in (x, res, ctx)]
        X, R, C = (t.double().requires_grad_() for t in (x, res, ctx))
        m.zero_grad(), ref.zero_grad()
        y = m(ins[0], "Matterport3D", ins[2], residual=ins[1], relu=True, **(dict(state=m.drop.draw()) if given else {}))
        assert m.drop.rng.tolist() == [21, call + 1]
        H = R + torch.where(O.dropout_keep(n, c, p, 21, call), X * 2, torch.zeros((), dtype=torch.float64))
        D = H - H.mean(1, keepdim=True)
        Y = D * (D.square().mean(1, keepdim=True) + 1e-5).rsqrt()
        ln = ref.bns[2] if decouple else ref.bn
        if affine:
            Y = Y * ln.weight + ln.bias
        if adaptive:
            shift, scale = ref.modulation(C).chunk(2, dim=1)
            Y = Y * (1.0 + scale) + shift
        g = gy * (Y.detach().abs() > 1e-4).float()   # no gradient within rounding distance of the kink
        Y = Y.clamp_min(0)
        y.backward(g.to(device))
        Y.backward(g.double())
        rel = lambda a, e: float((a.detach().double().cpu() - e).norm() / e.norm())
        assert rel(y, Y.detach()) < 1e-5 and rel(ins[0].grad, X.grad) < 1e-5 and rel(ins[1].grad, R.grad) < 1e-5
        assert not adaptive or rel(ins[2].grad, C.grad) < 1e-4
        for (k, q), (_, e) in zip(m.named_parameters(), ref.named_parameters()):
            assert (q.grad is None) == (e.grad is None), k
            assert e.grad is None or rel(q.grad, e.grad) < 1e-4, k
