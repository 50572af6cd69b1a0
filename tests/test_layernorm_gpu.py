"""Layer norm, its two backward passes and dropout through the C ABI, against 64-bit references with derived bounds."""
import itertools

import pytest
import torch

import ln_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SEED, OFFSET = 0x9E3779B97F4A7C15, (1 << 32) - 3      # both words of the key, a block counter that carries


def make(rows, cols, dtype, seed=0, pad=0, scale=1.5, shift=0.4):
    g = torch.Generator().manual_seed(seed * 7919 + rows * 31 + cols)
    t = (torch.randn(rows, cols + pad, generator=g) * scale + shift).to(dtype)
    return t


def case(dev, rows, cols, dtype, pdtype=F32, seed=0, pad=0):
    """Device tensors (rows cut out of wider ones if ``pad``) and their float64 copies."""
    t = {k: make(rows, cols, dtype, seed + i, pad, *s).to(dev)[:, :cols]
         for i, (k, s) in enumerate((("x", (1.5, 0.4)), ("gy", (1.0, 0.0)), ("ggx", (1.0, 0.1)), ("residual", (1.0, 0.0))))}
    g = torch.Generator().manual_seed(seed + 17)
    t["gamma"] = (1 + 0.2 * torch.randn(cols, generator=g)).to(pdtype).to(dev)
    t["beta"] = (0.2 * torch.randn(cols, generator=g)).to(pdtype).to(dev)
    return t, {k: v.double().cpu() for k, v in t.items()}


def mask_of(rows, cols, p):
    return R.keep_mask(rows, cols, p, SEED, OFFSET) if p else None


def run_all(dev, rows, cols, dtype, code, p, pdtype=F32, pad=0, residual=False, seed=0):
    """Forward, backward and backward of the backward of one case, each against its reference."""
    from fcd_amd import ops
    t, d = case(dev, rows, cols, dtype, pdtype, seed, pad)
    kw = dict(act_slope=code, p=p, rng=(SEED, OFFSET) if p else None)
    m = mask_of(rows, cols, p)
    y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], residual=t["residual"] if residual else None, **kw)
    wy, wm, wr = R.forward(d["x"], d["gamma"], d["beta"], ops.LN_EPS, code, m, d["residual"] if residual else None)
    R.check(mean, wm, what="mean")
    R.check(rstd, wr, what="rstd")
    R.check(y, wy, dtype, "y")
    md, rd = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    dx, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    wx, wg, wb = R.backward(d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, m)
    R.check(dx, wx, dtype, "dx")
    R.check(dg, wg, pdtype, "dgamma")
    R.check(db, wb, pdtype, "dbeta")
    ggy, gx, dg2, db2 = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    vy, vx, vg, vb = R.backward2(d["ggx"], d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, m)
    R.check(ggy, vy, dtype, "ggy")
    R.check(gx, vx, dtype, "gx")
    R.check(dg2, vg, pdtype, "dgamma of the second backward")
    R.check(db2, vb, pdtype, "dbeta of the second backward")


COLS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 500, 512, 513, 1001, 1024, 1025, 2048,
        2049, 4095, 4096, 4104, 8192, 8193, 16384, 20000, 33000]


@pytest.mark.parametrize("cols", COLS)
def test_every_width(dev, cols):
    for i, (dtype, rows) in enumerate(itertools.product((F32, BF16, F16), (1, 3, 37))):
        run_all(dev, rows, cols, dtype, (1.0, 2.0, 0.01)[i % 3], (0.0, 0.3)[i % 2], seed=i)


@pytest.mark.parametrize("rows", [1, 2, 5, 63, 64, 65, 255, 256, 257, 1000, 4099])
@pytest.mark.parametrize("cols", [8, 24, 72, 200])
def test_row_counts(dev, rows, cols):
    run_all(dev, rows, cols, F32, 2.0, 0.25)
    run_all(dev, rows, cols, BF16, 1.0, 0.0, pad=5)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("code", [1.0, 0.0, 0.01, 2.0, 3.0])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_types_activations_dropout(dev, dtype, code, p):
    run_all(dev, 33, 320, dtype, code, p, pdtype=dtype, residual=True)
    run_all(dev, 9, 1537, dtype, code, p, pdtype=F32, pad=7, residual=True, seed=3)


def test_no_rows(dev):
    from fcd_amd import ops
    x = torch.empty(0, 24, device=dev)
    w, b = torch.ones(24, device=dev), torch.zeros(24, device=dev)
    y, mean, rstd = ops.layernorm_fwd(x, w, b)
    assert y.shape == (0, 24) and mean.shape == (0,)
    dx, dg, db = ops.layernorm_bwd(x, x, mean, rstd, w, b)
    assert dx.shape == (0, 24) and not dg.any() and not db.any() and not torch.isnan(dg).any()
    keep = torch.full((24,), 3.0, device=dev)
    _, dg, _ = ops.layernorm_bwd(x, x, mean, rstd, w, b, dgamma=keep, accumulate=True)
    assert bool((dg == 3.0).all())
    ggy, gx, dg, db = ops.layernorm_bwd2(x, x, x, mean, rstd, w, b)
    assert ggy.shape == gx.shape == (0, 24) and not dg.any() and not db.any()
    assert ops.dropout(x, 0.5, (1, 2)).shape == (0, 24)
    assert ops.dropout(torch.empty(3, 0, device=dev), 0.5, (1, 2)).shape == (3, 0)


def test_parameters_left_out(dev):
    """gamma or beta None: 1 or 0; a gradient that is not asked for is not computed."""
    from fcd_amd import ops
    t, d = case(dev, 12, 200, F32)
    one, zero = torch.ones(200, device=dev), torch.zeros(200, device=dev)
    for g, b in ((None, None), ("gamma", None), (None, "beta")):
        gt, bt = t[g] if g else None, t[b] if b else None
        full = (gt if g else one, bt if b else zero)
        y, mean, rstd = ops.layernorm_fwd(t["x"], gt, bt, act_slope=2.0)
        assert torch.equal(y, ops.layernorm_fwd(t["x"], *full, act_slope=2.0)[0])
        dx, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, gt, bt, act_slope=2.0)
        fx, fg, fb = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, *full, act_slope=2.0)
        assert torch.equal(dx, fx) and (dg is None) == (g is None) and (db is None) == (b is None)
        assert dg is None or torch.equal(dg, fg)
        assert db is None or torch.equal(db, fb)
        o2 = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, gt, bt, act_slope=2.0)
        f2 = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, *full, act_slope=2.0)
        assert torch.equal(o2[0], f2[0]) and torch.equal(o2[1], f2[1])
        dx, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, gt, bt, act_slope=2.0, want_affine=False)
        assert torch.equal(dx, fx) and dg is None and db is None


@pytest.mark.parametrize("pdtype", [F32, BF16])
def test_accumulating_gradients(dev, pdtype):
    from fcd_amd import ops
    t, d = case(dev, 70, 136, BF16, pdtype)
    _, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"])
    md, rd = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    start = torch.full((136,), 0.75, dtype=pdtype, device=dev)
    _, wg, wb = R.backward(d["x"], d["gy"], md, rd, d["gamma"], d["beta"], 1.0, None)
    g, b = start.clone(), start.clone()
    ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], dgamma=g, dbeta=b, accumulate=True)
    R.check(g, wg + 0.75, pdtype)
    R.check(b, wb + 0.75, pdtype)
    only = start.clone()
    _, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], dbeta=only)
    assert dg is None and db is only
    R.check(only, wb, pdtype)
    _, _, vg, vb = R.backward2(d["ggx"], d["x"], d["gy"], md, rd, d["gamma"], d["beta"], 1.0, None)
    g = start.clone()
    b = start.clone()
    ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], dgamma=g, dbeta=b, accumulate=True)
    R.check(g, vg + 0.75, pdtype)
    R.check(b, vb + 0.75, pdtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [5, 64, 1000, 8200])
def test_row_strides_alignment_and_neighbours(dev, dtype, cols):
    """Rows at odd addresses inside wider tensors: same bits as contiguous copies, and nothing beside the rows is written."""
    from fcd_amd import ops
    rows = 11
    t, _ = case(dev, rows, cols, dtype, seed=5)
    for lead, tail in ((1, 2), (3, 0), (0, 5), (8, 8)):
        w = {k: torch.full((rows, lead + cols + tail), 7.0, dtype=dtype, device=dev) for k in ("x", "gy", "ggx", "residual", "out")}
        for k in ("x", "gy", "ggx", "residual"):
            w[k][:, lead:lead + cols] = t[k]
        s = {k: v[:, lead:lead + cols] for k, v in w.items()}
        kw = dict(act_slope=2.0, p=0.25, rng=(5, 6))
        y0, m0, r0 = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], residual=t["residual"], **kw)
        y1, m1, r1 = ops.layernorm_fwd(s["x"], t["gamma"], t["beta"], residual=s["residual"], out=s["out"], **kw)
        assert torch.equal(y0, y1) and torch.equal(m0, m1) and torch.equal(r0, r1)
        assert bool((w["out"][:, :lead] == 7).all()) and bool((w["out"][:, lead + cols:] == 7).all())
        a = ops.layernorm_bwd(t["gy"], t["x"], m0, r0, t["gamma"], t["beta"], **kw)
        b = ops.layernorm_bwd(s["gy"], s["x"], m0, r0, t["gamma"], t["beta"], out=s["out"], **kw)
        assert all(torch.equal(i, j) for i, j in zip(a, b))
        assert bool((w["out"][:, :lead] == 7).all()) and bool((w["out"][:, lead + cols:] == 7).all())
        a = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], m0, r0, t["gamma"], t["beta"], **kw)
        b = ops.layernorm_bwd2(s["ggx"], s["gy"], s["x"], m0, r0, t["gamma"], t["beta"], **kw)
        assert all(torch.equal(i, j) for i, j in zip(a, b))
        a = ops.dropout(t["x"], 0.25, (5, 6), residual=t["residual"])
        b = ops.dropout(s["x"], 0.25, (5, 6), residual=s["residual"], out=s["out"])
        assert torch.equal(a, b)
        assert bool((w["out"][:, :lead] == 7).all()) and bool((w["out"][:, lead + cols:] == 7).all())


def test_leading_axes_and_repeated_rows(dev):
    from fcd_amd import ops
    t, _ = case(dev, 2 * 3 * 5, 48, F32)
    x = t["x"].reshape(2, 3, 5, 48)
    y, mean, rstd = ops.layernorm_fwd(x, t["gamma"], t["beta"])
    assert y.shape == x.shape and mean.shape == (2, 3, 5)
    assert torch.equal(y.reshape(30, 48), ops.layernorm_fwd(t["x"], t["gamma"], t["beta"])[0])
    v = t["x"][0]
    y1, m1, _ = ops.layernorm_fwd(v, t["gamma"], t["beta"])
    assert y1.shape == (48,) and m1.shape == () and torch.equal(y1, y.reshape(30, 48)[0])
    ye, _, _ = ops.layernorm_fwd(v.expand(6, 48), t["gamma"], t["beta"])
    assert all(torch.equal(r, y1) for r in ye)
    every = t["x"][::3]                                   # every third row
    assert torch.equal(ops.layernorm_fwd(every, t["gamma"], t["beta"])[0], y.reshape(30, 48)[::3])


@pytest.mark.parametrize("rows,cols", [(9, 40), (128, 40), (9, 1000), (120, 2048), (500, 4096), (300, 8192), (9, 8200), (40, 20000)])
def test_in_place(dev, rows, cols):
    """Outputs in the place of inputs.  (The affine sums of a few rows are computed beside dx: not when dx overwrites what they
    read.)"""
    from fcd_amd import ops
    t, _ = case(dev, rows, cols, BF16)
    kw = dict(act_slope=2.0, p=0.3, rng=(1, 9))
    y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], residual=t["residual"], **kw)
    x = t["x"].clone()
    assert torch.equal(ops.layernorm_fwd(x, t["gamma"], t["beta"], residual=t["residual"], out=x, **kw)[0], y)
    r = t["residual"].clone()
    assert torch.equal(ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], residual=r, out=r, **kw)[0], y)
    dx, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    for name in ("gy", "x"):
        o = dict(gy=t["gy"].clone(), x=t["x"].clone())
        got = ops.layernorm_bwd(o["gy"], o["x"], mean, rstd, t["gamma"], t["beta"], out=o[name], **kw)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dg) and torch.equal(got[2], db)
    two = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    for names in (("gy", "x"), ("ggx", "gy"), ("x", "ggx")):
        o = {k: t[k].clone() for k in ("x", "gy", "ggx")}
        got = ops.layernorm_bwd2(o["ggx"], o["gy"], o["x"], mean, rstd, t["gamma"], t["beta"], outs=tuple(o[k] for k in names), **kw)
        assert all(torch.equal(i, j) for i, j in zip(got, two))
    d = ops.dropout(t["x"], 0.3, (1, 9), residual=t["residual"])
    x = t["x"].clone()
    assert torch.equal(ops.dropout(x, 0.3, (1, 9), residual=t["residual"], out=x), d)


# ---- values that spread ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cols", [24, 300, 4096, 8200])
def test_non_finite_rows_stay_alone(dev, cols):
    from fcd_amd import ops
    t, _ = case(dev, 16, cols, F32)
    y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"])
    x = t["x"].clone()
    x[3, cols // 2] = float("nan")
    x[7, 0] = float("inf")
    y1, m1, r1 = ops.layernorm_fwd(x, t["gamma"], t["beta"])
    rest = [i for i in range(16) if i not in (3, 7)]
    assert torch.equal(y1[rest], y[rest]) and torch.equal(r1[rest], rstd[rest])
    assert bool(torch.isnan(y1[3]).all()) and bool(torch.isnan(y1[7]).any())
    assert bool(torch.isnan(m1[3])) and float(m1[7]) == float("inf")
    dx, _, _ = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"])
    dx1, _, _ = ops.layernorm_bwd(t["gy"], x, m1, r1, t["gamma"], t["beta"])
    assert torch.equal(dx1[rest], dx[rest]) and bool(torch.isnan(dx1[3]).all())
    o = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"])
    o1 = ops.layernorm_bwd2(t["ggx"], t["gy"], x, m1, r1, t["gamma"], t["beta"])
    assert torch.equal(o1[0][rest], o[0][rest]) and torch.equal(o1[1][rest], o[1][rest])


@pytest.mark.parametrize("cols", [8, 65, 1024, 9000])
def test_rows_without_spread(dev, cols):
    """A constant row: xhat is 0 and rstd 1 / sqrt(eps), whatever the constant; large means keep their digits."""
    from fcd_amd import ops
    x = torch.tensor([0.0, 1.0, -3.0, 1024.0], device=dev)[:, None].expand(4, cols).contiguous()
    b = torch.randn(cols, device=dev)
    y, mean, rstd = ops.layernorm_fwd(x, None, b)
    assert torch.equal(mean, x[:, 0]) and torch.equal(y, b.expand(4, cols))
    assert bool(((rstd - 1e-5 ** -0.5).abs() <= 4 * R.U * 1e-5 ** -0.5 + 1e-4).all())
    far = (torch.randn(5, cols, device=dev) * 0.5 + 3000.0)
    wy, wm, wr = R.forward(far.double().cpu(), torch.ones(cols).double(), torch.zeros(cols).double(), 1e-5, 1.0, None, None)
    y, mean, rstd = ops.layernorm_fwd(far)
    R.check(mean, wm)
    R.check(rstd, wr)
    R.check(y, wy)


@pytest.mark.parametrize("cols", [5, 64, 200, 1001, 8192, 20000])
def test_tiny_variance_without_eps(dev, cols):
    """eps 0 and rows whose variance is a subnormal number (about 2^-128).  A square added to a partial sum, and the sum over
    the length, are off by up to half a step of the subnormal numbers each, 2^-150: the mean of the squares by 2^-149."""
    from fcd_amd import ops
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(7, cols, generator=g) * 2.0 ** -64).to(dev)
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(dev)
    y, mean, rstd = ops.layernorm_fwd(x, w, None, eps=0.0)
    d = x.double().cpu()
    var = ((d - d.mean(1, keepdim=True)) ** 2).mean(1, keepdim=True)
    assert bool((var < 2.0 ** -126).all()) and bool((var > 2.0 ** -132).all())
    more = 0.5 * 2.0 ** -149 / var
    wy, _, wr = R.forward(d, w.double().cpu(), torch.zeros(cols, dtype=torch.float64), 0.0, 1.0, None, None)
    R.check(rstd, R.V(wr.v, wr.e + more * wr.v), what="rstd")
    R.check(y, R.V(wy.v, wy.e + more * wy.v.abs()), what="y")


def test_dropped_elements_are_zero_whatever_they_held(dev):
    from fcd_amd import ops
    rows, cols, p = 6, 104, 0.5
    m = mask_of(rows, cols, p)
    rng = (SEED, OFFSET)
    bad = torch.full((rows, cols), float("nan"), device=dev)
    ones = torch.ones(rows, cols, device=dev)
    holes = torch.where(m.to(dev) > 0, ones, bad)
    assert torch.equal(ops.dropout(holes, p, rng), m.float().to(dev))
    t, _ = case(dev, rows, cols, F32)
    _, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"])
    gy = torch.where(m.to(dev) > 0, t["gy"], bad)
    a = ops.layernorm_bwd(gy, t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=2.0, p=p, rng=rng)
    b = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=2.0, p=p, rng=rng)
    assert all(torch.equal(i, j) for i, j in zip(a, b))


# ---- dropout --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 8), (5, 9), (2, 1023), (17, 64), (1000, 33), (3, 70001)])
def test_dropout_draws_the_published_generator(dev, shape, dtype):
    from fcd_amd import ops
    for i, p in enumerate((0.1, 0.5, 1.0 / 65536, 0.999)):
        seed, offset = SEED + i, OFFSET + 8 * i if i < 3 else (1 << 64) - 2      # the last one's counter wraps around
        x = make(*shape, dtype, seed=i).to(dev)
        m = R.keep_mask(*shape, p, seed, offset)
        want = (x.double().cpu() * m)
        got = ops.dropout(x, p, (seed, offset))
        assert torch.equal((got == 0).cpu(), (want == 0))
        R.check(got, R.V(want, 2 * R.U * want.abs()), dtype)
        assert torch.equal(ops.dropout(x, p, ops.dropout_state(seed, dev, offset)), got)
        r = make(*shape, dtype, seed=i + 9).to(dev)
        both = R.V(want, 2 * R.U * want.abs()) + r.double().cpu()
        R.check(ops.dropout(x, p, (seed, offset), residual=r), both, dtype)


def test_dropout_extremes(dev):
    from fcd_amd import ops
    x = torch.randn(40, 50, device=dev)
    assert torch.equal(ops.dropout(x, 0.0, None), x)
    assert torch.equal(ops.dropout(x, 1e-6, (1, 1)), x)              # resolved to 2^-16: nothing dropped, nothing scaled
    assert not ops.dropout(x, 1.0, (1, 1)).any()
    assert torch.equal(ops.dropout(x, 1.0, (1, 1), residual=x), x)
    y = ops.dropout(x.view(-1), 0.3, (4, 4))
    assert torch.equal(y, ops.dropout(x, 0.3, (4, 4)).view(-1))      # the index is the row-major one, whatever the shape
    z = ops.dropout(x.view(-1)[80:], 0.3, (4, 4 + 10))               # ... and offset counts blocks of eight
    assert torch.equal(z, y[80:])


def test_dropout_keeps_the_promised_share(dev):
    """Kept share of 2^24 draws within 6 standard deviations, and the mean preserved through the scale."""
    from fcd_amd import ops
    n = 1 << 24
    for p in (0.1, 0.5, 0.9):
        y = ops.dropout(torch.ones(n, device=dev), p, (77, 0))
        t = round(p * 65536) / 65536
        kept = float((y != 0).double().mean())
        assert abs(kept - (1 - t)) <= 6 * (t * (1 - t) / n) ** 0.5
        assert abs(float(y.double().mean()) - 1.0) <= 6 * (t / (1 - t) / n) ** 0.5 + 2 * R.U


def test_dropout_in_the_norm_is_dropout_behind_it(dev):
    from fcd_amd import ops
    for rows, cols in ((7, 100), (4, 1001), (3, 9001), (300, 65)):
        t, _ = case(dev, rows, cols, F32)
        y = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], act_slope=2.0)[0]
        a = ops.dropout(y, 0.4, (3, 8))
        b = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], act_slope=2.0, p=0.4, rng=(3, 8))[0]
        assert torch.equal(a, b)


def test_taking_ranges(dev):
    from fcd_amd import ops
    st = ops.dropout_state(-5, dev, offset=(1 << 64) - 1)
    a = ops.dropout_take(st, 17)
    b = ops.dropout_take(st, 8)
    c = ops.dropout_take(st, 0)
    assert [v & (2 ** 64 - 1) for v in a.tolist()] == [2 ** 64 - 5, 2 ** 64 - 1]
    assert b.tolist() == [-5, 2] and c.tolist() == [-5, 3] and st.tolist() == [-5, 3]
    x = torch.randn(10, 10, device=dev)
    assert torch.equal(ops.dropout(x, 0.5, b), ops.dropout(x, 0.5, (-5, 2)))


# ---- streams, graphs, sizes -------------------------------------------------------------------------------------------------

def _step(ops, t, rng, gb):
    y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], act_slope=2.0, p=0.2, rng=rng, residual=t["residual"])
    dx, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=2.0, p=0.2, rng=rng)
    o2 = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=2.0, p=0.2, rng=rng)
    z = ops.dropout(y, 0.2, rng)
    ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=2.0, dgamma=gb[0], dbeta=gb[1], accumulate=True)
    return [y, mean, rstd, dx, dg, db, *o2, z]


def test_taking_ranges_on_two_streams(dev):
    """Every block is handed out once, whichever stream asks first."""
    from fcd_amd import ops
    state = ops.dropout_state(11, dev)
    streams = [torch.cuda.Stream() for _ in range(2)]
    taken = []
    torch.cuda.synchronize()
    for i in range(200):
        with torch.cuda.stream(streams[i % 2]):
            taken.append(ops.dropout_take(state, 24))
    torch.cuda.synchronize()
    assert sorted(int(t[1]) for t in taken) == [3 * i for i in range(200)]
    assert all(int(t[0]) == 11 for t in taken) and state.tolist() == [11, 600]


def test_statistics_between_rows(dev):
    """mean and rstd may lie in the gap behind a row of a wider tensor."""
    import ctypes as C
    from fcd_amd import _lib, ops
    t, _ = case(dev, 4, 40, F32)
    wide = torch.zeros(4, 56, device=dev)
    wide[:, :40] = t["x"]
    y = torch.empty(4, 40, device=dev)
    d = _lib.LayerNormDesc()
    for k, v in dict(rows=4, cols=40, ld_x=56, ld_out=40, eps=ops.LN_EPS, act=1.0).items():
        setattr(d, k, v)
    at = wide.data_ptr() + (56 + 40) * 4
    rc = _lib.load().fcd_layernorm_fwd(C.byref(d), wide.data_ptr(), t["gamma"].data_ptr(), t["beta"].data_ptr(), None, y.data_ptr(),
                                       at, at + 16, None, 0, _lib.stream())
    _lib.check(rc, "layernorm_fwd")
    wy, wm, wr = ops.layernorm_fwd(t["x"].contiguous(), t["gamma"], t["beta"])
    assert torch.equal(y, wy) and torch.equal(wide[1, 40:44], wm) and torch.equal(wide[1, 44:48], wr)
    assert torch.equal(wide[:, :40], t["x"])


@pytest.mark.parametrize("rows,cols", [(700, 64), (300, 1000), (40, 9000)])
def test_captured_graphs(dev, rows, cols):
    """Two graphs of the same step, replayed in turn with eager work between: every replay draws the next masks and gives the
    eager bits; the graphs share no scratch."""
    from fcd_amd import ops
    t, _ = case(dev, rows, cols, BF16)
    state = ops.dropout_state(11, dev)
    gbs = [[torch.zeros(cols, device=dev) for _ in range(2)] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ops, t, ops.dropout_take(state, rows * cols), gbs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            taken = ops.dropout_take(state, rows * cols)
            outs.append(_step(ops, t, taken, gbs[k]))
        graphs.append(g)
    for gb in gbs:
        for b in gb:
            b.zero_()
    state.copy_(ops.dropout_state(11, dev, offset=100))
    eager_state = ops.dropout_state(11, dev, offset=100)
    egbs = [[torch.zeros(cols, device=dev) for _ in range(2)] for _ in range(2)]
    for i in (0, 1, 1, 0, 0, 1):
        graphs[i].replay()
        want = _step(ops, t, ops.dropout_take(eager_state, rows * cols), egbs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want))
        assert all(torch.equal(a, b) for a, b in zip(gbs[i], egbs[i]))


@pytest.mark.parametrize("rows,cols", [(700, 64), (3000, 1000), (40, 9000)])
def test_two_graphs_at_once(dev, rows, cols):
    """Two graphs captured one after the other and replayed at the same time on two streams: neither's sums run through
    the other's scratch."""
    from fcd_amd import ops
    ts = [case(dev, rows, cols, BF16, seed=k)[0] for k in range(2)]
    stats = [ops.layernorm_fwd(t["x"])[1:] for t in ts]
    want = [ops.layernorm_bwd(t["gy"], t["x"], *st, t["gamma"], t["beta"], act_slope=2.0) for t, st in zip(ts, stats)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for t, st in zip(ts, stats):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([ops.layernorm_bwd(t["gy"], t["x"], *st, t["gamma"], t["beta"], act_slope=2.0) for _ in range(8)])
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(i, j) for one in o for i, j in zip(one, w))


def test_same_bits_every_time_and_on_other_streams(dev):
    from fcd_amd import ops
    for rows, cols in ((3000, 64), (500, 1537), (20, 12000)):
        t, _ = case(dev, rows, cols, F32)
        gb = [torch.zeros(cols, device=dev), torch.zeros(cols, device=dev)]
        first = _step(ops, t, (8, 8), gb)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = _step(ops, t, (8, 8), gb)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_more_than_32_bits_of_elements(dev):
    """Tensors of 2.3e9 elements: the first, a middle and the last rows against the same rows by themselves."""
    from fcd_amd import ops
    rows, cols = 70001, 32776
    x = torch.empty(rows, cols, dtype=BF16, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    for i in range(0, rows, 4096):
        x[i:i + 4096].normal_(generator=g)
    y, mean, rstd = ops.layernorm_fwd(x, p=0.25, rng=(3, 4), act_slope=2.0)
    dx, _, _ = ops.layernorm_bwd(y, x, mean, rstd, p=0.25, rng=(3, 4), act_slope=2.0)
    z = ops.dropout(x, 0.25, (3, 4))
    one, zero = torch.ones(cols).double(), torch.zeros(cols).double()
    for i in (0, 40000, rows - 1):
        assert i * cols % 8 == 0
        m = R.keep_mask(1, cols, 0.25, 3, 4 + i * cols // 8)
        xd = x[i:i + 1].double().cpu()
        wy, wm, wr = R.forward(xd, one, zero, ops.LN_EPS, 2.0, m, None)
        R.check(y[i], wy, BF16, "y")
        R.check(mean[i], wm)
        md, rd = mean[i].double().cpu(), rstd[i].double().cpu()
        wx, _, _ = R.backward(xd, y[i:i + 1].double().cpu(), md, rd, one, zero, 2.0, m)
        R.check(dx[i], wx, BF16, "dx")
        R.check(z[i], R.V(xd * m, 2 * R.U * (xd * m).abs()), BF16, "dropout")


@pytest.mark.parametrize("rows,cols", [(1, 65536), (2, 300007), (3, 131080), (5, 8193), (300, 16385), (700, 8200)])
def test_split_rows(dev, rows, cols):
    """Rows longer than a workgroup's registers, with one chunk of the row nearly empty and with ragged ends."""
    run_all(dev, rows, cols, F32, 2.0, 0.1)
    run_all(dev, rows, cols, BF16, 1.0, 0.0, pad=3, residual=True)
    run_all(dev, rows, cols, F16, 0.01, 0.4, seed=2)


# ---- the second backward around its means -----------------------------------------------------------------------------------

def offset_case(dev, rows, cols, dtype, offset, code, p, seed=0):
    """First and second backward with gradients whose mean is ``offset`` times their spread, against bounds that grow with the
    offset, not with its square."""
    from fcd_amd import ops
    t, _ = case(dev, rows, cols, dtype, seed=seed)
    # (gamma's spread shrinks with the offset: that of gamma gy stays the noise's)
    t["gamma"] = (1 + (t["gamma"].double() - 1) / offset).float()
    t["gy"] = (t["gy"].double() + offset).to(dtype)
    t["ggx"] = (t["ggx"].double() + offset).to(dtype)
    d = {k: v.double() for k, v in t.items()}
    m = mask_of(rows, cols, p)
    m = None if m is None else m.to(dev)
    kw = dict(act_slope=code, p=p, rng=(SEED, OFFSET) if p else None)
    mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"])[1:]
    md, rd = mean.double()[:, None], rstd.double()[:, None]
    got = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    for g, w, dt, name in zip(got, R.backward(d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, m), (dtype, F32, F32),
                              ("dx", "dgamma", "dbeta")):
        R.check(g, w, dt, name)
    got = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    for g, w, dt, name in zip(got, R.second(d["ggx"], d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, m), (dtype, dtype, F32, F32),
                              ("ggy", "gx", "dgamma of the second backward", "dbeta of the second backward")):
        R.check(g, w, dt, name)


@pytest.mark.parametrize("offset", [10.0, 100.0, 1000.0])
@pytest.mark.parametrize("cols", [7, 24, 60, 100, 255, 500, 1001, 1537, 4096, 8192, 8195, 20000, 65541])
def test_gradients_far_from_zero(dev, cols, offset):
    for i, (code, p) in enumerate(((1.0, 0.0), (2.0, 0.0), (0.01, 0.3), (1.0, 0.3))):
        offset_case(dev, 37 if cols < 9000 else 5, cols, F32, offset, code, p, seed=i)
    offset_case(dev, 9, cols, BF16, offset, 1.0, 0.0)


# ---- activations far out ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("code", [2.0, 3.0])
@pytest.mark.parametrize("far", [60.0, 1e4, 1e8, 1e12, 1e16, 1e20, 3e30])
def test_smooth_activations_far_from_zero(dev, code, far):
    """Pre-activations of +-far (through beta): act is u or 0, act' 1 or 0, act'' 0, within four steps of fp32 however large u
    is.  (|u| > 50: the exact ones are within 50 e^-50 < 1e-15 of these.)"""
    from fcd_amd import ops
    for rows, cols in ((3, 24), (700, 64), (5, 1000), (300, 1537), (3, 9001)):
        t, d = case(dev, rows, cols, F32)
        up = torch.rand(cols, generator=torch.Generator().manual_seed(cols)) < 0.5
        t["beta"] = torch.where(up, far, -far).to(dev)
        d["beta"] = t["beta"].double().cpu()
        y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], act_slope=code)
        wy, _, _ = R.forward(d["x"], d["gamma"], d["beta"], ops.LN_EPS, 1.0, None, None)
        R.check(y, R.V(wy.v * up, (wy.e + 4 * R.U * wy.v.abs()) * up + 1e-15), what="y")
        md, rd = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
        one = R.V(up.double().expand(rows, cols), 4 * R.U)
        flat = R.V(torch.zeros(rows, cols, dtype=torch.float64), 1e-15)
        got = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=code)
        for g, w, name in zip(got, R.first(d["x"], d["gy"], md, rd, d["gamma"], one), ("dx", "dgamma", "dbeta")):
            R.check(g, w, what=name)
        got = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], act_slope=code)
        want = R.second(d["ggx"], d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, None, (one, flat))
        for g, w, name in zip(got, want, ("ggy", "gx", "dgamma", "dbeta")):
            R.check(g, w, what="second " + name)
