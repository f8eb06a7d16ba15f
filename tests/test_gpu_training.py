"""GPU: the training operators against their formulas in 64 bits.

Tolerances are bounds, not observations.  u is half a step of a type (2^-24 fp32, 2^-8 bf16).  A fp32 sum of n terms is off
by at most n u32 sum|terms|; the kernels' sums are trees, so n is a lane's run of additions and the tree's height.  A value
rounded to its type at the end adds u |value|.  What a rounded intermediate (the stored row mean, the logits' gradient in
bf16) does is carried through the formula with absolute values."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def _u(dt):
    return torch.finfo(dt).eps / 2


def _ok(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst error / bound "
                           f"{float((err / tol)[bad].max()):.2f}")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------ LayerNorm
NORM_SIZES = [(1, 1), (3, 7), (2, 16), (5, 100), (130, 128), (9, 129), (33, 512), (17, 777), (6, 1024), (3, 1025), (3, 2047),
              (5, 2048), (2, 4096), (2, 5000), (3, 8192), (2, 8200), (2, 16384), (2, 20000), (2, 32769), (3, 40001), (2000, 64),
              (4100, 256),
              (3, 200), (301, 250), (70, 12300), (601, 10001), (40, 16384), (65, 16385), (2, 1000003),
              (5, 8), (5, 9), (40, 20), (33, 500), (700, 1501), (2500, 1290)]


def norm_reference(x, w, b, dy, eps=1e-5):
    """values and bounds (without the final rounding) of y, dx, dw, db"""
    x, dy = x.double(), dy.double()
    d, rows = x.shape[1], x.shape[0]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((x - mu).square().mean(1, keepdim=True) + eps)
    h = (x - mu) * r
    # a lane adds up to 32 elements, the tree is at most 11 high (a long row: d / 1024 + 19); the same again for the variance
    k = 64 + d / 512
    hh = h.abs() + (x.abs() + mu.abs()) * r                       # h and what its subtraction cancelled
    y, ty = h * w + b, U32 * k * (hh * w.abs() + b.abs())
    g = dy * w
    m0, m1 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = r * (g - m0 - h * m1)
    tdx = U32 * k * r * (g.abs() + g.abs().mean(1, keepdim=True) + hh * (g.abs() * hh).mean(1, keepdim=True))
    kr = 128 + rows / 256                                         # rows a group walks, the wave, the partial rows
    return y, ty, dx, tdx, (dy * h).sum(0), U32 * (k + kr) * (dy.abs() * hh).sum(0), dy.sum(0), U32 * kr * dy.abs().sum(0)


def _norm_case(rows, d, xt, wt, yt, seed=0):
    g = _gen(seed)
    x = (torch.randn(rows, d, generator=g, device="cuda") * 1.5 + 0.4).to(xt)
    w = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(wt)
    b = (0.2 * torch.randn(d, generator=g, device="cuda")).to(wt)
    dy = torch.randn(rows, d, generator=g, device="cuda").to(yt)
    return x, w, b, dy


def _norm_check(x, w, b, dy, y, dx, dw, db, what=""):
    ry, ty, rdx, tdx, rdw, tdw, rdb, tdb = norm_reference(x, w, b, dy)
    _ok(y, ry, ty + _u(y.dtype) * ry.abs(), what + " y")
    _ok(dx, rdx, tdx + _u(dx.dtype) * rdx.abs(), what + " dx")
    _ok(dw, rdw, tdw + _u(dw.dtype) * rdw.abs(), what + " dw")
    _ok(db, rdb, tdb + _u(db.dtype) * rdb.abs(), what + " db")


@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (F32, F32, BF16), (BF16, F32, F32)],
                         ids=lambda t: "-".join("f32" if v == F32 else "bf16" for v in t))
@pytest.mark.parametrize("rows,d", NORM_SIZES)
def test_layer_norm(gpu, rows, d, types):
    from video_asl_recognition_amd import training as T
    x, w, b, dy = _norm_case(rows, d, *types)
    y, mean, rstd = T.layer_norm_fwd(x, w, b, out_dtype=types[2])
    dx, dw, db = T.layer_norm_bwd(dy, x, w, mean, rstd)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (types[2], types[0], types[1], types[1])
    _norm_check(x, w, b, dy, y, dx, dw, db)


def test_layer_norm_without_weight_or_rows(gpu):
    from video_asl_recognition_amd import training as T
    x, w, b, dy = _norm_case(7, 130, F32, F32, F32)
    for ww, bb in ((None, None), (w, None), (None, b)):
        y, mean, rstd = T.layer_norm_fwd(x, ww, bb)
        dx, dw, db = T.layer_norm_bwd(dy, x, ww, mean, rstd)
        _norm_check(x, ww, bb, dy, y, dx, dw, db)
    e = torch.empty(0, 130, device="cuda")
    y, mean, rstd = T.layer_norm_fwd(e, w, b)
    dx, dw, db = T.layer_norm_bwd(e, e, w, mean, rstd)
    assert y.shape == (0, 130) and dx.shape == (0, 130) and not dw.any() and not db.any()


def test_layer_norm_strides_and_leading_dimensions(gpu):
    from video_asl_recognition_amd import training as T
    g = _gen(3)
    big = torch.randn(6, 5, 301, generator=g, device="cuda").to(BF16)
    w, b = torch.randn(100, generator=g, device="cuda"), torch.randn(100, generator=g, device="cuda")
    for x in (big[:, :, 1:101], big[:, :, 7:107], big[::2, 1:3, :100], big[:, :, :300:3], big[:5, :, :100].transpose(0, 1)):
        dy = torch.randn(x.shape, generator=g, device="cuda").to(BF16)
        y, mean, rstd = T.layer_norm_fwd(x, w, b)
        assert y.shape == x.shape and mean.shape == x.shape[:-1]
        for dyv in (dy, dy.transpose(0, 1).contiguous().transpose(0, 1), dy[:1, :1, :1].expand(x.shape)):
            dx, dw, db = T.layer_norm_bwd(dyv, x, w, mean, rstd)
            _norm_check(x.reshape(-1, 100), w, b, dyv.reshape(-1, 100), y.reshape(-1, 100), dx.reshape(-1, 100), dw, db)
    v = torch.randn(64, generator=g, device="cuda")                   # a single vector
    y, mean, rstd = T.layer_norm_fwd(v, None, None)
    assert y.shape == (64,) and mean.shape == ()


def test_layer_norm_writes_no_further_than_its_rows(gpu):
    """row strides wider than d at the C boundary: the places between stay as they were"""
    from video_asl_recognition_amd import _lib as L
    for d, ld in ((5, 8), (129, 131), (1000, 1003)):
        x, w, b, dy = _norm_case(9, d, BF16, F32, BF16)
        y = torch.full((10, ld), 7.0, dtype=BF16, device="cuda")
        dx = torch.full((10, ld), 7.0, dtype=BF16, device="cuda")
        mean, rstd = torch.empty(9, device="cuda"), torch.empty(9, device="cuda")
        dw, db = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
        p = L.LayerNormParams(9, d, d, ld, ld, L.BF16, L.F32, L.BF16, 1e-5)
        a = lambda t: t.data_ptr()
        L.check(L.lib.asl_layernorm_fwd(C.byref(p), a(x), a(w), a(b), a(y), a(mean), a(rstd), None))
        dyp = torch.zeros(9, ld, dtype=BF16, device="cuda")
        dyp[:, :d] = dy
        ws = torch.empty(L.lib.asl_layernorm_bwd_workspace(C.byref(p)), dtype=torch.uint8, device="cuda")
        L.check(L.lib.asl_layernorm_bwd(C.byref(p), a(dyp), a(x), a(w), a(mean), a(rstd), a(dx), a(dw), a(db), a(ws), None))
        torch.cuda.synchronize()
        for t in (y, dx):
            assert (t[:, d:] == 7.0).all() and (t[9] == 7.0).all()
        _norm_check(x, w, b, dy, y[:9, :d], dx[:9, :d], dw, db)


def test_layer_norm_hard_rows(gpu):
    """equal values far from nought have variance nought; a NaN or an infinity stays in its row"""
    from video_asl_recognition_amd import training as T
    for d in (96, 777, 3000, 9000):
        x = torch.full((4, d), 12345.678, device="cuda")
        x[1] = 3e4 + torch.arange(d, device="cuda") % 2
        w, b = torch.ones(d, device="cuda"), torch.full((d,), 0.5, device="cuda")
        y, mean, rstd = T.layer_norm_fwd(x, w, b)
        # the first mean is off by less than a value's last bit, 2^-10, and what is left of that by 64 u32 of it; rstd is 317
        _ok(y[0], b.double(), 64 * U32 * 2.0 ** -10 * 317 + U32, "equal values")
        assert abs(float(rstd[0]) * 1e-5 ** 0.5 - 1) < 1e-6
        ry = norm_reference(x, w, b, x)[0]
        _ok(y[1], ry[1], 1e-5 * ry[1].abs(), "offset row")        # 3e4 and 3e4 + 1 are exact, their mean and deviations too
        x[2, 5], x[3, 7] = float("nan"), float("inf")
        y2, mean, rstd = T.layer_norm_fwd(x, w, b)
        assert torch.equal(y2[:2], y[:2]) and y2[2].isnan().all() and y2[3].isnan().all()
        dy = torch.ones_like(x)
        dx, dw, db = T.layer_norm_bwd(dy, x, w, mean, rstd)
        assert dx[:2].isfinite().all() and dx[2:].isnan().all() and db.isfinite().all()


def test_layer_norm_autograd_and_differences(gpu):
    from video_asl_recognition_amd import training as T
    g = _gen(5)
    x0, w0, b0, c = (torch.randn(s, generator=g, device="cuda") for s in ((6, 40), (40,), (40,), (6, 40)))
    x, w, b = (t.clone().requires_grad_() for t in (x0, w0, b0))
    (T.layer_norm(x, w, b) * c).sum().backward()

    def f(xv, wv, bv):                                           # 64-bit oracle
        mu = xv.mean(1, keepdim=True)
        return (((xv - mu) / ((xv - mu).square().mean(1, keepdim=True) + 1e-5).sqrt() * wv + bv) * c.double()).sum()
    for i, (leaf, base) in enumerate(((x, x0), (w, w0), (b, b0))):
        v = torch.randn(base.shape, generator=g, device="cuda").double()
        at = [t.double() for t in (x0, w0, b0)]
        hi, lo = list(at), list(at)
        hi[i], lo[i] = at[i] + 1e-6 * v, at[i] - 1e-6 * v
        num = float(f(*hi) - f(*lo)) / 2e-6
        ana = float((leaf.grad.double() * v).sum())
        # central differences: 1e-12 of the third derivative, 1e-16 |f| / 1e-6; the gradient's own fp32 errors
        assert abs(num - ana) <= 64 * U32 * float((leaf.grad.double().abs() * v.abs()).sum()) + 1e-6
    xb = x0.to(BF16).requires_grad_()
    wf = w0.clone().requires_grad_()
    y = T.layer_norm(xb, wf, None, out_dtype=F32)
    y.sum().backward()
    assert y.dtype == F32 and xb.grad.dtype == BF16 and wf.grad.dtype == F32


# ------------------------------------------------------------------------------------------------ Linear + cross entropy
XENT_SIZES = [(1, 1, 1), (1, 2, 3), (2, 31, 5), (16, 2000, 512), (17, 33, 65), (32, 1000, 130), (33, 1000, 130), (3, 16384, 70), (3, 16385, 20),
              (20, 4500, 300), (8, 2000, 512), (5, 100, 64), (65, 63, 33), (64, 64, 64), (130, 257, 100), (300, 1000, 70),
              (257, 129, 513), (16, 5003, 129),
              (40, 1, 1), (40, 3, 2), (5000, 2, 3), (300, 130, 9), (12000, 70, 31)]


def xent_reference(x, w, b, t, up, ignore, smooth, reduction, bf16):
    """values and bounds (without the final rounding) of the rows' losses, dx, dw, db.  up: the loss's gradient, one value or
    one a row."""
    x, w = x.double(), w.double()
    n, v, d = x.shape[0], w.shape[0], x.shape[1]
    l = x @ w.t()
    bound = (d + 2) * U32 * (x.abs() @ w.abs().t())               # of a logit
    if b is not None:
        l, bound = l + b.double(), bound + U32 * (l.abs() + b.double().abs())
    bound = torch.nan_to_num(bound, posinf=0.0, nan=0.0)          # a masked class is exactly -inf
    lse = torch.logsumexp(l, 1)
    keep = (t != ignore) & True
    at = torch.where(keep, t, 0)[:, None]
    lt = l.gather(1, at)[:, 0]
    rows = lse - (1 - smooth) * lt
    if smooth:
        rows = rows - smooth * l.mean(1)
    rows = torch.where(keep, rows, 0.0)
    # the logits' bounds, once in lse and once in what is subtracted; the exponentials (the fast one is good to
    # (2 + |l - max|) 2^-23, weighted by p, whose |l - max| averages below 2 log v + 8) and their sum (64 a tile, then tiles)
    lg = torch.log(torch.tensor(float(v), dtype=torch.float64))
    rel = 2 * U32 * (10 + 2 * float(lg)) + U32 * (40 + v / 4096)
    trow = 2 * bound.max(1).values + rel + 4 * U32 * (lse.abs() + torch.nan_to_num(lt, neginf=0.0).abs())
    if smooth:
        trow = trow + U32 * (64 + v / 64) * smooth * torch.nan_to_num(l, neginf=0.0).abs().mean(1)
    count = keep.sum()
    gr = torch.as_tensor(up, dtype=torch.float64, device=x.device).expand(n).clone()
    if reduction == "mean":
        gr = gr / count
    gr = torch.where(keep, gr, 0.0)[:, None]
    p = torch.exp(l - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    G = gr * (p - (1 - smooth) * hot - smooth / v)
    G = torch.where(keep[:, None], G, 0.0)
    # a logit's bound and lse's move p by as much of itself; rounded on the way for bf16: the exponential to fp16 of 2^15 its
    # ratio to the tile's largest (fp16 has 11 significant bits, half a step is 2^-11 of the value; below 2^-14 its steps are
    # 2^-24, half of one 2^-25, which over 2^15 is 2^-40 of the largest), then G to bf16
    tG = gr.abs() * p * (bound + trow[:, None] + rel + 4 * U32) + 4 * U32 * (gr.abs() * (p + hot + smooth / v))
    tG32 = tG + (gr.abs() * (1 - hot) * (2.0 ** -11 * p + 2.0 ** -40 * p.max(1, keepdim=True).values) if bf16 else 0.0)
    tG = tG32 + (2.0 ** -8 * G.abs() * (1 + 2.0 ** -8) if bf16 else 0.0)
    tG, tG32 = (torch.where(keep[:, None], q, 0.0) for q in (tG, tG32))
    dx, tdx = G @ w, tG @ w.abs() + (v + 40) * U32 * (G.abs() @ w.abs())
    dw, tdw = G.t() @ x, tG.t() @ x.abs() + (n + 40) * U32 * (G.t().abs() @ x.abs())
    db, tdb = G.sum(0), tG32.sum(0) + (n + 40) * U32 * G.abs().sum(0)
    return rows, trow, lse, dx, tdx, dw, tdw, db, tdb, count


def _xent_case(n, v, d, dt, bias, ignored, seed=0):
    g = _gen(seed)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    w = torch.randn(v, d, generator=g, device="cuda") * (2.0 / d ** 0.5)
    x = torch.randn(n, d, generator=g, device="cuda") + 2.5 * torch.rand(n, 1, generator=g, device="cuda") * w[t]
    drop = torch.rand(n, generator=g, device="cuda") < ignored
    drop[0] = False
    t[drop] = -100
    return x.to(dt), w.to(dt), (0.3 * torch.randn(v, generator=g, device="cuda")).to(bias) if bias else None, t


def _xent_check(x, w, b, t, ignore=-100, smooth=0.0, reduction="mean", what=""):
    from video_asl_recognition_amd import training as T
    kw = dict(ignore_index=ignore, label_smoothing=smooth, reduction=reduction)
    loss, lse = T.linear_cross_entropy_fwd(x, w, t, b, **kw)
    loss2, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b, **kw)
    rows, trow, rlse, rdx, tdx, rdw, tdw, rdb, tdb, count = xent_reference(x, w, b, t, 1.0, ignore, smooth, reduction, x.dtype == BF16)
    _ok(lse, rlse, trow, what + " lse")
    if reduction == "none":
        r, tr = rows, trow
    else:
        c = count.double() if reduction == "mean" else 1.0
        r, tr = rows.sum() / c, (trow.sum() + (len(rows) / 256 + 16) * U32 * rows.abs().sum()) / c
    _ok(loss, r, tr, what + " loss")
    _ok(loss2, r, tr, what + " loss with gradients")
    assert dx.dtype == dw.dtype == x.dtype and dx.shape == x.shape and dw.shape == w.shape
    _ok(dx, rdx, tdx + _u(x.dtype) * (rdx.abs() + tdx) + 1e-38, what + " dx")
    _ok(dw, rdw, tdw + _u(x.dtype) * (rdw.abs() + tdw) + 1e-38, what + " dw")
    if b is not None:
        assert db.dtype == b.dtype
        _ok(db, rdb, tdb + _u(b.dtype) * (rdb.abs() + tdb) + 1e-38, what + " db")


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,v,d", XENT_SIZES)
def test_linear_cross_entropy(gpu, n, v, d, dt):
    x, w, b, t = _xent_case(n, v, d, dt, None, 0.0)
    _xent_check(x, w, b, t, what="plain")
    x, w, b, t = _xent_case(n, v, d, dt, dt, 0.3, 1)
    _xent_check(x, w, b, t, smooth=0.1, what="smoothed")
    _xent_check(x, w, b, t, reduction="sum", what="sum")
    _xent_check(x, w, b, t, reduction="none", what="none")


@pytest.mark.parametrize("n,v,d", [(256, 32768, 64), (300, 33001, 72), (257, 32769, 8), (513, 22000, 520), (1000, 8200, 256),
                                   (8200, 1100, 192), (4100, 2049, 1032), (2000, 8100, 1032), (1990, 8190, 1024)])
def test_linear_cross_entropy_large_tiles(gpu, n, v, d):
    """sizes that take the 256 x 256 tiles: whole ones, cut ones, k that ends inside a step"""
    x, w, b, t = _xent_case(n, v, d, BF16, F32, 0.1)
    b[v // 3: v // 2] = float("-inf")
    t = torch.where((t >= v // 3) & (t < v // 2), 0, t)
    _xent_check(x, w, b, t, what="large")
    x, w, b, t = _xent_case(n, v, d, BF16, None, 0.1)
    _xent_check(x, w, b, t, smooth=0.1, reduction="sum", what="large, smoothed")


@pytest.mark.parametrize("n,v,d", [(256, 8192, 64), (300, 8211, 72), (1100, 1003, 200), (2100, 6000, 33), (64, 70000, 64), (256, 33000, 72),
                                   (1100, 1003, 520), (2100, 6000, 63), (300, 8211, 264), (2000, 8100, 520)])
def test_linear_cross_entropy_large_fp32(gpu, n, v, d):
    """sizes that take fp32 apart into bf16 planes: held to the bounds of fp32 products"""
    x, w, b, t = _xent_case(n, v, d, F32, F32, 0.1)
    b[v // 3: v // 2] = float("-inf")
    t = torch.where((t >= v // 3) & (t < v // 2), 0, t)
    _xent_check(x, w, b, t, what="large fp32")
    # wide ranges: rows of very different size, weights that differ by 2^20
    x *= torch.exp2(torch.randint(-12, 1, (n, 1), generator=_gen(1), device="cuda").float())
    w *= torch.exp2(torch.randint(-20, 1, (v, 1), generator=_gen(2), device="cuda").float())
    _xent_check(x, w, b, t, smooth=0.1 if not b.isinf().any() else 0.0, reduction="sum", what="large fp32, wide range")


def test_linear_cross_entropy_bias_types_and_strides(gpu):
    g = _gen(9)
    x, w, b, t = _xent_case(70, 150, 96, BF16, F32, 0.2)
    _xent_check(x, w, b, t)
    x, w, b, t = _xent_case(70, 150, 96, F32, BF16, 0.2)
    _xent_check(x, w, b, t)
    for n, v in ((9, 150), (9, 2500), (30, 400)):
        for dt, bt in ((BF16, F32), (F32, BF16)):
            x, w, b, t = _xent_case(n, v, 96, dt, bt, 0.2)
            _xent_check(x, w, b, t, smooth=0.1)
    for dt in (F32, BF16):
        x, w, b, t = _xent_case(70, 150, 96, dt, dt, 0.2)
        xb, wb = torch.zeros(70, 131, dtype=dt, device="cuda"), torch.zeros(300, 99, dtype=dt, device="cuda")
        xs, ws = xb[:, 3:99], wb[::2, 1:97]
        xs.copy_(x), ws.copy_(w)
        _xent_check(xs, ws, b, t, what="strided")
        _xent_check(x.t().contiguous().t(), w.t().contiguous().t(), b, t, what="transposed")


def test_linear_cross_entropy_leading_dimensions(gpu):
    from video_asl_recognition_amd import training as T
    x, w, b, t = _xent_case(24, 40, 32, F32, F32, 0.2)
    loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b, reduction="none")
    l3, dx3, dw3, db3 = T.linear_cross_entropy_grad(x.view(2, 3, 4, 32), w, t.view(2, 3, 4), b, reduction="none")
    assert l3.shape == (2, 3, 4) and torch.equal(l3.flatten(), loss) and torch.equal(dx3.view(24, 32), dx)
    assert torch.equal(dw3, dw) and torch.equal(db3, db)


def test_linear_cross_entropy_pieces(gpu):
    """more rows than one piece of exponentials holds"""
    for dt, v, n, d in ((BF16, 65536, 8192 + 300, 24), (F32, 65530, 4096 + 4100, 24), (BF16, 65600, 8192 + 300, 40), (F32, 70000, 3000, 40),
                        (BF16, 70, 140000, 40), (F32, 70, 140000, 40), (BF16, 600, 140000, 64), (F32, 100, 140000, 64)):
        x, w, b, t = _xent_case(n, v, d, dt, F32, 0.1)
        _xent_check(x, w, b, t, smooth=0.1)


def test_linear_cross_entropy_masks_and_labels(gpu):
    from video_asl_recognition_amd import training as T
    for dt in (F32, BF16):
        x, w, b, t = _xent_case(80, 300, 64, dt, F32, 0.0)
        # classes masked by a bias of -inf, whole tiles of them, none of them anyone's label
        b[64:256] = float("-inf")
        t = torch.where((t >= 64) & (t < 256), t % 64, t)
        _xent_check(x, w, b, t, what="masked")
        dw, db = T.linear_cross_entropy_grad(x, w, t, b)[2:]
        assert not dw[64:256].any() and not db[64:256].any()
        # by the type's lowest value
        b[64:256] = torch.finfo(dt).min / 2
        assert T.linear_cross_entropy_fwd(x, w, t, b)[0].isfinite() and not T.linear_cross_entropy_grad(x, w, t, b)[3][64:256].any()
        # another ignored label, one inside the vocabulary; then every row ignored
        x, w, b, t = _xent_case(80, 300, 64, dt, F32, 0.0)
        t[::3] = 7
        _xent_check(x, w, b, t, ignore=7, smooth=0.1)
        t[:] = 7
        loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b, ignore_index=7)
        assert loss.isnan() and not dx.any() and not dw.any() and not db.any()
        loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b, ignore_index=7, reduction="sum")
        assert loss == 0 and not dx.any() and not dw.any() and not db.any()
        # NaN and infinities in ignored rows do not get out of them
        t = torch.randint(0, 300, (80,), generator=_gen(1), device="cuda")
        t[10:30] = -100
        clean = T.linear_cross_entropy_grad(x, w, t, b)
        xn = x.clone()
        xn[10:20], xn[20:30] = float("nan"), float("inf")
        dirty = T.linear_cross_entropy_grad(xn, w, t, b)
        assert torch.equal(dirty[0], clean[0]) and torch.equal(dirty[1], clean[1]) and torch.equal(dirty[3], clean[3])
        # ... where 0 x NaN of their features in dW is the formula's own
        # a label outside the vocabulary is loud, whichever side
        for wrong in (-1, 300, 1 << 40, -(1 << 40)):
            tw = t.clone()
            tw[3] = wrong
            loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, tw, b, reduction="none")
            assert loss[3].isnan() and loss[4:].isfinite().all() and dx[3].isnan().all() and dx[:3].isfinite().all()
            assert dw.isnan().all()


# sizes for each way the products are computed: few rows, fp32 on 64 x 64 tiles, 128 x 128 and 256 x 256, fp32 as bf16 planes
PATHS = [(12, 300, 40, BF16), (20, 300, 40, F32), (20, 4500, 40, F32), (9, 2100, 30, BF16), (80, 60, 64, BF16), (80, 300, 20, BF16), (80, 300, 64, F32), (70, 4000, 90, F32), (600, 1100, 260, F32),
         (20, 300, 40, BF16), (80, 300, 64, BF16), (400, 1000, 128, BF16), (400, 1003, 77, BF16), (1000, 8200, 256, BF16),
         (520, 9001, 136, BF16), (600, 4100, 260, F32), (1100, 8200, 65, F32), (9000, 250, 64, BF16), (2000, 8100, 1024, BF16), (2000, 8100, 520, F32)]
PATH_IDS = [f"{n}x{v}x{d}-{'f32' if dt == F32 else 'bf16'}" for n, v, d, dt in PATHS]


@pytest.mark.parametrize("n,v,d,dt", PATHS, ids=PATH_IDS)
def test_linear_cross_entropy_every_path_hard_cases(gpu, n, v, d, dt):
    from video_asl_recognition_amd import training as T
    x, w, b, t = _xent_case(n, v, d, dt, F32, 0.0)
    lo, hi = v // 4, v - 5                                        # most classes masked, whole tiles and the last one's all but five
    b[lo:hi] = float("-inf")
    t = torch.where((t >= lo) & (t < hi), t % lo, t)
    t[n // 2:] = -100
    _xent_check(x, w, b, t, what="masked")
    clean = T.linear_cross_entropy_grad(x, w, t, b)
    assert not clean[2][lo:hi].any() and not clean[3][lo:hi].any()
    # what ignored rows hold stays out of every other row
    xn = x.clone()
    xn[n // 2:n // 2 + 3], xn[n // 2 + 3:] = float("nan"), float("inf")
    dirty = T.linear_cross_entropy_grad(xn, w, t, b)
    assert torch.equal(dirty[0], clean[0]) and torch.equal(dirty[1], clean[1]) and torch.equal(dirty[3], clean[3])
    # masked by the type's lowest value
    b[lo:hi] = torch.finfo(dt).min
    low = T.linear_cross_entropy_grad(x, w, t, b)
    assert low[0].isfinite() and not low[3][lo:hi].any()
    # a label outside the vocabulary
    for wrong in (-1, v, 1 << 40):
        tw = t.clone()
        tw[1] = wrong
        loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, tw, b, reduction="none")
        assert loss[1].isnan() and loss[2:].isfinite().all() and dx[1].isnan().all() and dx[2:].isfinite().all() and dw.isnan().all()
    # every row ignored; labels all smoothing
    x, w, b, t = _xent_case(n, v, d, dt, dt, 0.1)
    _xent_check(x, w, b, t, smooth=1.0, what="smoothed away")
    t[:] = -100
    loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b)
    assert loss.isnan() and not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize("n,v,d,dt", PATHS, ids=PATH_IDS)
def test_linear_cross_entropy_every_path_upstream_and_slices(gpu, n, v, d, dt):
    """a gradient for every row, through autograd; x and w as slices of larger tensors off any alignment; memory that held
    NaN before"""
    from video_asl_recognition_amd import training as T
    x, w, b, t = _xent_case(n, v, d, dt, dt, 0.1)
    up = torch.rand(n, generator=_gen(3), device="cuda") * 2 - 0.5
    xb, wb = torch.zeros(n, d + 9, dtype=dt, device="cuda"), torch.zeros(2 * v, d + 5, dtype=dt, device="cuda")
    xs, ws = xb[:, 3:d + 3], wb[::2, 1:d + 1]
    xs.copy_(x), ws.copy_(w)
    del wb, xb
    junk = torch.full((1 << 28,), float("nan"), device="cuda")    # 1 GiB for the outputs and workspaces to come from
    del junk
    grads = []
    for a, c in ((x, w), (xs, ws)):
        leaves = [q.detach().requires_grad_() for q in (a, c, b)]
        loss = T.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
        grads.append([loss] + list(torch.autograd.grad((loss * up).sum(), leaves)))
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    ref = xent_reference(x, w, b, t, up.double(), -100, 0.0, "none", dt == BF16)
    for got, r, tol in zip(grads[0][1:], (ref[3], ref[5], ref[7]), (ref[4], ref[6], ref[8])):
        _ok(got, r, tol + _u(dt) * (r.abs() + tol) + 1e-38, "gradient")


@pytest.mark.parametrize("n,v,d,dt", PATHS, ids=PATH_IDS)
def test_linear_cross_entropy_writes_no_further_than_its_outputs(gpu, n, v, d, dt):
    """the C entry point with outputs at their types' own alignment inside larger buffers, and with each of them left out"""
    from video_asl_recognition_amd import _lib as L, training as T
    x, w, b, t = _xent_case(n, v, d, dt, dt, 0.1)
    want = T.linear_cross_entropy_grad(x, w, t, b)
    code = T._TYPES[dt]
    p = L.XentParams(n, v, d, code, code, L.REDUCE_MEAN, d, d, -100, 0.0, 0)
    room = L.lib.asl_linear_xent_workspace(C.byref(p), x.data_ptr(), w.data_ptr(), 1)
    s = torch.cuda.current_stream().cuda_stream
    for left_out in (None, 0, 1, 2):
        ws = torch.full((room + 512,), 0x5a, dtype=torch.uint8, device="cuda")
        at = -ws.data_ptr() % 256
        outs = [torch.full((q.numel() + 6,), 7.0, dtype=dt, device="cuda") for q in want[1:]]
        loss, lse = torch.full((3,), 7.0, device="cuda"), torch.full((n + 2,), 7.0, device="cuda")
        size = outs[0].element_size()
        ptr = [None if i == left_out else o.data_ptr() + 3 * size for i, o in enumerate(outs)]
        L.check(L.lib.asl_linear_xent_grad(C.byref(p), x.data_ptr(), w.data_ptr(), b.data_ptr(), t.data_ptr(), None, loss.data_ptr() + 4,
                                           lse.data_ptr() + 4, *ptr, ws.data_ptr() + at, s), "grad")
        assert loss[1] == want[0] and (loss[::2] == 7).all() and (lse[0] == 7) and (lse[-1] == 7) and lse[1:-1].isfinite().all()
        for i, (o, q) in enumerate(zip(outs, want[1:])):
            assert (o[:3] == 7).all() and (o[-3:] == 7).all()
            assert (o == 7).all() if i == left_out else torch.equal(o[3:-3], q.flatten())
        assert (ws[:at] == 0x5a).all() and (ws[at + room:] == 0x5a).all()


def test_linear_cross_entropy_pieces_of_a_large_vocabulary(gpu):
    """more exponentials than a piece holds, against the formula taken a thousand rows at a time"""
    from video_asl_recognition_amd import training as T
    n, v, d = 33600, 65530, 32
    x, w, b, t = _xent_case(n, v, d, BF16, F32, 0.1)
    loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b, reduction="sum")
    sums = [0.0] * 6
    for i in range(0, n, 1000):
        part = slice(i, i + 1000)
        rows, trow, _, rdx, tdx, *rest = xent_reference(x[part], w, b, t[part], 1.0, -100, 0.0, "sum", True)[:9]
        _ok(dx[part], rdx, tdx + 2.0 ** -8 * (rdx.abs() + tdx) + 1e-38, "dx")
        sums = [p + q for p, q in zip(sums, [rows.sum(), trow.sum() + 30 * U32 * rows.abs().sum()] + rest)]
    _ok(loss, sums[0], sums[1] + (n / 256 + 16) * U32 * sums[0], "loss")
    # the bounds of a part's sums, and as many 32-bit additions as there are rows over all of them
    over = 2 * n * U32
    _ok(dw, sums[2], sums[3] * (1 + over) + over * sums[2].abs() + 2.0 ** -8 * (sums[2].abs() + sums[3]) + 1e-38, "dw")
    _ok(db, sums[4], sums[5] * (1 + over) + over * sums[4].abs() + 1e-38, "db")


def test_linear_cross_entropy_one_row_without_dimensions(gpu):
    from video_asl_recognition_amd import training as T
    x, w, b, t = _xent_case(1, 30, 20, F32, F32, 0.0)
    for red in ("mean", "none"):
        want = T.linear_cross_entropy_grad(x, w, t, b, reduction=red)
        got = T.linear_cross_entropy_grad(x[0], w, t[0], b, reduction=red)
        assert got[0].shape == () and got[1].shape == (20,)
        assert all(torch.equal(p.flatten(), q.flatten()) for p, q in zip(got, want))
    y, mean, rstd = T.layer_norm_fwd(x[0], None, None)
    assert y.shape == (20,) and mean.shape == () and torch.equal(y, T.layer_norm_fwd(x, None, None)[0][0])


def test_rows_far_apart(gpu):
    """rows of larger tensors, 2^20 elements and more from one to the next: the places pass 2^32 bytes and 2^31 elements"""
    from video_asl_recognition_amd import training as T
    for dt, ld in ((BF16, 1 << 20), (BF16, (1 << 20) + 8), (F32, 1 << 20)):
        n, v, d = 2200, 2600, 64
        x, w, b, t = _xent_case(n, v, d, dt, F32, 0.1)
        xs, ws = torch.empty(n, ld, dtype=dt, device="cuda")[:, 8:d + 8], torch.empty(v, ld, dtype=dt, device="cuda")[:, -d:]
        xs.copy_(x), ws.copy_(w)
        for p, q in zip(T.linear_cross_entropy_grad(xs, ws, t, b), T.linear_cross_entropy_grad(x, w, t, b)):
            assert torch.equal(p, q)
        far, near = T.layer_norm_fwd(xs, b[:d], None), T.layer_norm_fwd(x, b[:d], None)
        assert all(torch.equal(p, q) for p, q in zip(far, near))
        dy = far[0]
        assert all(torch.equal(p, q) for p, q in zip(T.layer_norm_bwd(xs, xs, b[:d], *far[1:]), T.layer_norm_bwd(x, x, b[:d], *near[1:])))
        del xs, ws


def test_linear_cross_entropy_weight_of_more_than_32_bits(gpu):
    from video_asl_recognition_amd import training as T
    n, v, d = 40, (1 << 21) - 3, 1032
    g = _gen(5)
    w = torch.empty(v, d, dtype=BF16, device="cuda").normal_(std=2 / d ** 0.5, generator=g)
    x = torch.randn(n, d, generator=g, device="cuda").to(BF16)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    t[:4] = torch.arange(v - 4, v, device="cuda")
    loss, dx, dw, _ = T.linear_cross_entropy_grad(x, w, t, reduction="sum")
    l = torch.cat([x.double() @ w[i:i + (1 << 18)].double().t() for i in range(0, v, 1 << 18)], 1)
    lse = torch.logsumexp(l, 1, keepdim=True)
    G = torch.exp(l - lse)
    G.scatter_add_(1, t[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
    rows = (lse - l.gather(1, t[:, None]))[:, 0]
    # a logit: d additions of products below |x| |w|, some 60 in all, to 32 bits; lse and the loss by as much
    tol = 2 * (d + 2) * U32 * float((x.double().abs() @ w[:1000].double().abs().t()).max()) * 1.5 + 100 * U32
    _ok(loss, rows.sum(), torch.tensor(n * tol, device="cuda"), "loss")
    for part in (slice(0, 100), slice(v - 100, v)):
        ref = G[:, part].t() @ x.double()
        # G to bf16, the exponential under it to fp16, the sum to bf16
        bound = (tol + 2 * 2.0 ** -8 + 2.0 ** -11) * (G[:, part].abs().t() @ x.double().abs()) + 2.0 ** -8 * ref.abs() + 1e-12
        _ok(dw[part], ref, bound, "dw")


def test_linear_cross_entropy_pieces_without_gradients(gpu):
    """so many classes that the rows' maxima and sums are taken in pieces: the rows' results are those of calls of their own"""
    from video_asl_recognition_amd import training as T
    v, n, d = 1 << 21, 2500, 8
    x, w, b, t = _xent_case(n, v, d, BF16, BF16, 0.1)
    loss, lse = T.linear_cross_entropy_fwd(x, w, t, b, reduction="none")
    for part in (slice(0, 500), slice(1900, 2500)):
        l, e = T.linear_cross_entropy_fwd(x[part], w, t[part], b, reduction="none")
        assert torch.equal(l, loss[part]) and torch.equal(e, lse[part])
    rows = slice(2040, 2060)
    ref = xent_reference(x[rows], w, b, t[rows], 1.0, -100, 0.0, "none", True)
    _ok(loss[rows], ref[0], ref[1], "loss")
    _ok(lse[rows], ref[2], ref[1], "lse")


def test_linear_cross_entropy_no_rows(gpu):
    from video_asl_recognition_amd import training as T
    x, w, b, t = (torch.empty(0, 16, device="cuda"), torch.randn(9, 16, device="cuda"), torch.randn(9, device="cuda"),
                  torch.empty(0, dtype=torch.int64, device="cuda"))
    for red, want in (("mean", "nan"), ("sum", 0.0), ("none", None)):
        loss, dx, dw, db = T.linear_cross_entropy_grad(x, w, t, b, reduction=red)
        lf, lse = T.linear_cross_entropy_fwd(x, w, t, b, reduction=red)
        assert dx.shape == (0, 16) and not dw.any() and not db.any() and lse.shape == (0,)
        if want == "nan":
            assert loss.isnan() and lf.isnan()
        elif want is not None:
            assert loss == want and lf == want
        else:
            assert loss.shape == (0,) and lf.shape == (0,)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_linear_cross_entropy_autograd_and_differences(gpu, reduction):
    from video_asl_recognition_amd import training as T
    g = _gen(6)
    x0, w0, b0, t = _xent_case(20, 33, 24, F32, F32, 0.2)
    up = torch.rand(20, generator=g, device="cuda") + 0.5 if reduction == "none" else torch.tensor(1.7, device="cuda")
    leaves = [v.clone().requires_grad_() for v in (x0, w0, b0)]
    loss = T.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1, reduction=reduction)
    (loss * up).sum().backward()
    ref = xent_reference(x0, w0, b0, t, up.double(), -100, 0.1, reduction, False)
    for leaf, r, tol in zip(leaves, (ref[3], ref[5], ref[7]), (ref[4], ref[6], ref[8])):
        _ok(leaf.grad, r, tol + U32 * (r.abs() + tol), "gradient")

    def f(x, w, b):                                              # 64-bit oracle
        l = x @ w.t() + b
        lp = l - torch.logsumexp(l, 1, keepdim=True)
        k = t != -100
        rows = torch.where(k, -0.9 * lp.gather(1, torch.where(k, t, 0)[:, None])[:, 0] - 0.1 * lp.mean(1), 0.0)
        return (rows * up).sum() / (k.sum() if reduction == "mean" else 1)
    at = [v.double() for v in (x0, w0, b0)]
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=g, device="cuda").double()
        hi, lo = list(at), list(at)
        hi[i], lo[i] = at[i] + 1e-6 * v, at[i] - 1e-6 * v
        num = float(f(*hi) - f(*lo)) / 2e-6
        tol = ref[(4, 6, 8)[i]]
        assert abs(num - float((leaf.grad.double() * v).sum())) <= float((tol * v.abs()).sum()) * 2 + 1e-6
    # only what is asked for
    w = w0.clone().requires_grad_()
    T.linear_cross_entropy(x0, w, t).backward()
    assert w.grad is not None


# ------------------------------------------------------------------------------------------------ norm and clipping
def _tensors(sizes, types, seed=0):
    g = _gen(seed)
    return [(torch.randn(s, generator=g, device="cuda") * 4.0 ** (i % 5 - 2)).to(types[i % len(types)]) for i, s in enumerate(sizes)]


CLIP_SETS = {"one": [(1,)], "scalars": [()] * 3, "odd": [(3,), (0,), (8191,), (8192,), (8193,), (77, 5), (1, 1)],
             "many": [((i * 37) % 501,) for i in range(250)], "one launch": [(51200,), (100,), (513,), (7, 73)], "just": [(65536,)],
             "just not": [(65536,), (1,)], "slots": [(i % 3 + 1,) for i in range(64)], "slots and more": [(i % 3 + 1,) for i in range(65)], "large": [(3000, 4001), (5,), (1 << 24,)]}


@pytest.mark.parametrize("kinds", [(F32,), (BF16,), (F32, BF16)], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("name", list(CLIP_SETS))
def test_clip_grads(gpu, name, kinds):
    from video_asl_recognition_amd import training as T
    gs = _tensors(CLIP_SETS[name], kinds)
    total = sum(float(g.double().square().sum()) for g in gs) ** 0.5
    big = max((float(g.double().abs().max()) for g in gs if g.numel()), default=0.0)
    for norm_type, n in ((2.0, total), (float("inf"), big)):
        # the sum is held in 64 bits; the norm is rounded once
        assert abs(float(T.grad_norm(gs, norm_type)) - n) <= 2 * U32 * n
        for max_norm in (0.3 * n, 3.0 * n + 1.0):
            c = min(1.0, max_norm / (n + 1e-6))
            want = [g.double() * c for g in gs]
            # the factor: max_norm, norm, their quotient and 1e-6 rounded to fp32; the product; the type
            for out in ([torch.empty_like(g) for g in gs], [torch.empty(g.shape, device="cuda") for g in gs]):
                keep = [g.clone() for g in gs]
                assert abs(float(T.clip_grads(gs, max_norm, norm_type, out=out)) - n) <= 2 * U32 * n
                for o, w, g, k in zip(out, want, gs, keep):
                    _ok(o, w, (_u(o.dtype) + 8 * U32) * w.abs(), name)
                    assert torch.equal(g, k)
            mine = [g.clone() for g in gs]
            T.clip_grads(mine, max_norm, norm_type)
            for o, w, g in zip(mine, want, gs):
                _ok(o, w, (_u(o.dtype) + 8 * U32) * w.abs(), name)
                if c == 1.0:
                    assert torch.equal(o, g)


def test_clip_grads_extremes(gpu):
    from video_asl_recognition_amd import training as T
    # squares that overflow fp32, and that underflow it
    for s in (1e30, 1e-30):
        g = torch.full((5000,), s, device="cuda")
        n = s * 5000 ** 0.5
        norm = T.clip_grads([g], 0.5 * n if s > 1 else 1.0)
        assert abs(float(norm) / n - 1) < 1e-6
        if s > 1:
            assert abs(float(g[17]) / (0.5 * s) - 1) < 1e-6
    for bad in (float("nan"), float("inf")):
        for nt in (2.0, float("inf")):
            a, b = torch.ones(10000, device="cuda"), torch.ones(3, device="cuda", dtype=BF16)
            a[9000] = bad
            norm = T.clip_grads([a, b], 1.0, nt)
            if bad != bad:
                assert norm.isnan() and a.isnan().all() and b.isnan().all()
            else:                                             # torch's own: a factor of nought, and inf * 0
                assert norm.isinf() and a[9000].isnan() and not a[:9000].any() and not b.any()
    z = [torch.zeros(7, device="cuda"), torch.empty(0, device="cuda")]
    assert T.clip_grads(z, 1.0) == 0 and not z[0].any()
    assert T.grad_norm([torch.empty(0, device="cuda")]) == 0 and T.clip_grads([torch.empty(0, device="cuda")], 1.0) == 0
    g = torch.ones(9, device="cuda")
    T.clip_grads([g], 0.0)
    assert not g.any()


def test_clip_grads_layouts_and_refusals(gpu):
    from video_asl_recognition_amd import training as T
    g = torch.randn(8, 6, 5, 5, device="cuda").to(memory_format=torch.channels_last)
    k, n = g.clone(memory_format=torch.preserve_format), float(g.double().norm())
    T.clip_grads([g, g.new_zeros(4).t()], 0.5 * n)
    _ok(g, k.double() * (0.5 * n / (n + 1e-6)), 16 * U32 * k.double().abs(), "channels last")
    base = torch.randn(101, device="cuda").to(BF16)
    v = base[1:100]                                            # two bytes off any vector's alignment
    keep = base.clone()
    T.clip_grads([v], 0.1)
    assert base[0] == keep[0] and base[100] == keep[100]
    flat = torch.randn(40, device="cuda")
    with pytest.raises(ValueError, match="dense"):
        T.clip_grads([flat.view(8, 5)[:, :3]], 1.0)
    with pytest.raises(RuntimeError, match="invalid"):
        T.clip_grads([flat, flat], 1.0)
    with pytest.raises(RuntimeError, match="invalid"):
        T.clip_grads([flat[:30], flat[20:]], 1.0)
    assert T.grad_norm([flat, flat]).isfinite()               # read only: nothing races
    with pytest.raises(ValueError, match="strides"):
        T.clip_grads([flat.view(8, 5)], 1.0, out=[torch.empty(5, 8, device="cuda").t()])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        T.clip_grads([flat.half()], 1.0)


def test_clip_grad_norm_of_parameters(gpu):
    from video_asl_recognition_amd import training as T
    ps = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((30, 7), (7,), (100,))]
    for p in ps[:2]:
        p.grad = torch.randn_like(p)
    ref = [p.grad.clone() for p in ps[:2]]
    n = T.clip_grad_norm_(ps, 0.25)
    want = sum(float(r.double().square().sum()) for r in ref) ** 0.5
    assert abs(float(n) - want) <= 2 * U32 * want and ps[2].grad is None
    for p, r in zip(ps, ref):
        w = r.double() * (0.25 / (want + 1e-6))
        _ok(p.grad, w, 8 * U32 * w.abs(), "parameter")
    assert T.clip_grad_norm_(ps[2], 1.0) == 0


# ------------------------------------------------------------------------------------------------ graphs, streams, together
def _step(T, s, out):
    y, mean, rstd = T.layer_norm_fwd(s["x"], s["g"], s["b"])
    loss, dy, dw, db = T.linear_cross_entropy_grad(y, s["w"], s["t"], s["c"], label_smoothing=0.1)
    dx, dg, dbeta = T.layer_norm_bwd(dy, s["x"], s["g"], mean, rstd)
    norm = T.clip_grads([dw, db, dg, dbeta], 0.05, out=out)
    return [y, loss, dx, dw, norm] + out


def _step_state(dt, n, v, d, seed):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return dict(x=r(n, d).to(dt), g=(1 + 0.1 * r(d)).to(dt), b=(0.1 * r(d)).to(dt), w=(r(v, d) * 2 / d ** 0.5).to(dt),
                c=(0.1 * r(v)).to(dt), t=torch.randint(0, v, (n,), generator=g, device="cuda"))


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,v,d", [(8, 100, 512), (1100, 300, 96)])
def test_step_in_a_graph(gpu, dt, n, v, d):
    """norm, loss, gradients and clipping as one step, captured and replayed on new inputs between eager steps: the same
    bits every time"""
    from video_asl_recognition_amd import training as T
    states = [_step_state(dt, n, v, d, 20 + i) for i in range(4)]
    new = lambda: [torch.empty(s, device="cuda") for s in ((v, d), (v,), (d,), (d,))]
    eager = [[o.clone() for o in _step(T, s, new())] for s in states]
    static, out = {k: q.clone() for k, q in states[0].items()}, new()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(T, static, out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(T, static, out)
    for round_ in range(3):
        for s, want in zip(states, eager):
            for k in static:
                static[k].copy_(s[k])
            graph.replay()
            again = _step(T, s, new())
            torch.cuda.synchronize()
            for a, b, c in zip(captured, want, again):
                assert torch.equal(a, b) and torch.equal(c, b)


def test_steps_on_two_streams(gpu):
    from video_asl_recognition_amd import training as T
    states = [_step_state(BF16, 700, 500, 128, 40 + i) for i in range(2)]
    new = lambda: [torch.empty(s, device="cuda") for s in ((500, 128), (500,), (128,), (128,))]
    want = [[o.clone() for o in _step(T, s, new())] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        got = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                got.append(_step(T, s, new()))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dt", [F32, BF16], ids=["f32", "bf16"])
def test_autograd_in_a_graph(gpu, dt):
    """forward and backward through autograd, captured: gradients are taken as values, so nothing of an eager graph is met"""
    from video_asl_recognition_amd import training as T
    states = [_step_state(dt, 300, 500, 96, 60 + i) for i in range(3)]
    keys = ("x", "g", "b", "w", "c")

    def run(s):
        leaves = [s[k].detach().requires_grad_() for k in keys]
        y = T.layer_norm(leaves[0], leaves[1], leaves[2])
        loss = T.linear_cross_entropy(y, leaves[3], s["t"], leaves[4], label_smoothing=0.1)
        grads = list(torch.autograd.grad(loss, leaves))
        return [loss.detach(), T.clip_grads(grads, 0.05)] + grads
    eager = [[o.clone() for o in run(s)] for s in states]
    static = {k: q.clone() for k, q in states[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(static)
    for _ in range(3):
        for s, want in zip(states, eager):
            for k in static:
                static[k].copy_(s[k])
            graph.replay()
            again = run(s)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) and torch.equal(r, q) for p, q, r in zip(captured, want, again))


@pytest.mark.parametrize("n,v,d,dt", [(12, 300, 40, F32), (80, 300, 64, F32), (400, 1003, 77, BF16), (9000, 250, 64, BF16)])
def test_two_graphs_share_a_workspace(gpu, n, v, d, dt):
    """the C entry points: two captured calls on one workspace, replayed in turn on one stream"""
    from video_asl_recognition_amd import _lib as L, training as T
    code = T._TYPES[dt]
    p = L.XentParams(n, v, d, code, code, L.REDUCE_MEAN, d, d, -100, 0.0, 0)
    q = L.LayerNormParams(n, d, d, d, d, code, code, code, 0.0)
    cases = [_xent_case(n, v, d, dt, dt, 0.1, seed) for seed in (1, 2)]
    room = max(L.lib.asl_linear_xent_workspace(C.byref(p), cases[0][0].data_ptr(), cases[0][1].data_ptr(), 1),
               L.lib.asl_layernorm_bwd_workspace(C.byref(q)))
    ws = torch.empty(room + 256, dtype=torch.uint8, device="cuda")
    at = ws.data_ptr() + -ws.data_ptr() % 256
    graphs, got, want = [], [], []
    for x, w, b, t in cases:
        y, mean, rstd = T.layer_norm_fwd(x, None, None)
        want.append([o.clone() for o in T.linear_cross_entropy_grad(x, w, t, b) + T.layer_norm_bwd(x, x, b.new_ones(d), mean, rstd)])
        ones = b.new_ones(d)
        out = [torch.empty_like(o) for o in want[-1]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s = torch.cuda.current_stream().cuda_stream
            L.check(L.lib.asl_linear_xent_grad(C.byref(p), x.data_ptr(), w.data_ptr(), b.data_ptr(), t.data_ptr(), None, out[0].data_ptr(),
                                               None, *(o.data_ptr() for o in out[1:4]), at, s), "xent")
            L.check(L.lib.asl_layernorm_bwd(C.byref(q), x.data_ptr(), x.data_ptr(), ones.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                            *(o.data_ptr() for o in out[4:]), at, s), "norm")
        graphs.append((graph, ones, mean, rstd))
        got.append(out)
    for turn in (0, 1, 1, 0, 1, 0):
        for o in got[turn]:
            o.fill_(3.0)
        ws.fill_(0xff)
        graphs[turn][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got[turn], want[turn]))


# ------------------------------------------------------------------------------------------------ rows that are nearly certain
@pytest.mark.parametrize("offset", [0.0, 60.0, -60.0, 4000.0])
@pytest.mark.parametrize("n,v,d,dt", PATHS, ids=PATH_IDS)
def test_linear_cross_entropy_of_nearly_certain_rows(gpu, n, v, d, dt, offset):
    """How unsure a row is (1 - p of some 2^-18) has the error of numbers near 1, however far all its logits lie from nought.

    Every logit is exact: features are rows of the unit matrix, W's entries and the offset are numbers of few bits.  A row has its
    target at the offset, two classes e^-12.75 and less below it, and the others at -200, whose exponentials are nought.  So the
    sum, 1 + u, takes two additions that round, each by half a step of a number in [1, 2), u32; the logarithm and the exponential
    minus one are small numbers with relative errors of a few u32 (a third u32 covers them many times); u itself is a sum of two
    exponentials, good to 2^-15 of themselves (the fast one: its argument times log2 e, rounded below 32, is off by 2^-20)."""
    from video_asl_recognition_amd import training as T
    P = min(d, v // 3, 16)
    step = v // (3 * P)
    at = torch.arange(P, device="cuda")
    gap = 12.75 + 0.25 * (at % 8)
    w = torch.zeros(v, d, device="cuda")
    w[:, :P] = -200.0
    w[3 * at * step, at] = 0.0
    w[(3 * at + 1) * step, at] = -gap
    w[(3 * at + 2) * step, at] = -gap - 0.75
    row = torch.arange(n, device="cuda") % P
    x = torch.zeros(n, d, device="cuda")
    x[torch.arange(n, device="cuda"), row] = 1.0
    t = 3 * row * step
    x, w, b = x.to(dt), w.to(dt), torch.full((v,), offset, device="cuda")
    first, second = torch.exp(-gap.double()), torch.exp(-gap.double() - 0.75)
    u = first + second
    tol = 3 * U32 + 2.0 ** -15 * u
    for loss, lse in (T.linear_cross_entropy_fwd(x, w, t, b, reduction="none"), (T.linear_cross_entropy_grad(x, w, t, b, reduction="none")[0], None)):
        _ok(loss, torch.log1p(u)[row], tol[row], "loss")
        if lse is not None:
            _ok(lse, offset + torch.log1p(u)[row], tol[row] + U32 * abs(offset), "lse")
    db = T.linear_cross_entropy_grad(x, w, t, b, reduction="sum")[3]
    rows = torch.bincount(row, minlength=P).double()
    for classes, grad, off in ((3 * at * step, -u / (1 + u), tol), ((3 * at + 1) * step, first / (1 + u), first), ((3 * at + 2) * step, second / (1 + u), second)):
        if off is not tol:                                        # p: its exponential, and for bf16 operands that held as fp16
            off = off * (2.0 ** -15 + (2.0 ** -11 if dt == BF16 else 0.0)) + off * tol
        _ok(db[classes], rows * grad, rows * off + (n + 40) * U32 * rows * grad.abs(), "db")


# ------------------------------------------------------------------------------------------------ what autograd sees of clipping
def test_clipping_raises_the_versions_of_what_it_writes(gpu):
    """a tensor that some backward still needs cannot be clipped unseen, as with torch's own in-place product"""
    from video_asl_recognition_amd import training as T
    for sizes in (((40,), (7, 9)), ((3000, 40), (7, 9))):         # one launch, and two
        leaf = [torch.randn(s, device="cuda", requires_grad=True) for s in sizes]
        for how in ("grads", "out", "parameters"):
            saved = [torch.randn(s, device="cuda") for s in sizes]
            other = [torch.randn(s, device="cuda") for s in sizes]
            y = sum((a * s).sum() for a, s in zip(leaf, saved))    # its backward needs `saved`
            before = [t._version for t in saved + other]
            T.grad_norm(saved)                                    # reads only
            assert before == [t._version for t in saved + other]
            if how == "grads":
                T.clip_grads(saved, 0.01)
            elif how == "out":
                T.clip_grads(other, 0.01, out=saved)
            else:
                ps = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in sizes]
                for p, s in zip(ps, saved):
                    p.grad = s
                T.clip_grad_norm_(ps, 0.01)
            assert all(t._version > v for t, v in zip(saved, before)) and [t._version for t in other] == before[len(sizes):]
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
    # second gradients: the first ones are part of the graph
    w = torch.randn(50, device="cuda", requires_grad=True)
    first, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    penalty = first.square().sum()
    T.clip_grads([first], 0.01)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()
    # tensors without a version counter are clipped as before
    with torch.inference_mode():
        g = torch.ones(9, device="cuda")
        T.clip_grads([g], 0.5)
    T.clip_grads([g], 0.25)
    assert abs(float(g.norm()) - 0.25) < 1e-6


@pytest.mark.parametrize("n,v,d,dt", PATHS, ids=PATH_IDS)
def test_linear_cross_entropy_infinite_weights(gpu, n, v, d, dt):
    """a weight of -inf against positive features makes its class's logits -inf, as a bias of -inf does, on every path; NaN
    weights and +inf are loud; only rows that meet them are touched"""
    from video_asl_recognition_amd import training as T
    x, w, b, t = _xent_case(n, v, d, dt, F32, 0.1)
    k, lo, hi = d - 1, v // 4, v - 5
    x[:, k] = x[:, k].abs() + 0.25
    t = torch.where((t >= lo) & (t < hi), t % lo, t)
    masked = b.clone()
    masked[lo:hi] = float("-inf")
    winf = w.clone()
    winf[lo:hi, k] = float("-inf")
    for reduction in ("none", "mean"):
        loss, lse = T.linear_cross_entropy_fwd(x, winf, t, b, reduction=reduction, label_smoothing=0.0)
        want, want_lse = T.linear_cross_entropy_fwd(x, w, t, masked, reduction=reduction, label_smoothing=0.0)
        assert want.isfinite().all() and torch.equal(loss, want) and torch.equal(lse, want_lse)
    for bad in (float("nan"), float("inf")):
        wb = w.clone()
        wb[lo, k] = bad
        loss, lse = T.linear_cross_entropy_fwd(x, wb, t, b, reduction="none")
        kept = t != -100
        assert not loss[kept].isfinite().any() and not loss[~kept].any() and not lse.isfinite().any()
    # an infinite feature concerns its own row
    xi = x.clone()
    xi[0, k] = float("inf")
    loss, lse = T.linear_cross_entropy_fwd(xi, w, t, b, reduction="none")
    want, want_lse = T.linear_cross_entropy_fwd(x, w, t, b, reduction="none")
    assert not lse[0].isfinite() and torch.equal(loss[1:], want[1:]) and torch.equal(lse[1:], want_lse[1:])
