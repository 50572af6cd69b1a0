"""Layer norm and dropout over more rows than one turn of the grid, and written over their inputs with ragged rows: every
register-resident shape against 64-bit references (computed on the device)."""
import pytest
import torch

import ln_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SEED, OFFSET = 0x9E3779B97F4A7C15, (1 << 32) - 3


def operands(dev, rows, cols, dtype, seed=0, pad=0):
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + rows * 31 + cols)
    t = {k: (torch.randn(rows, cols + pad, generator=g, device=dev) * a + b).to(dtype)[:, :cols]
         for k, a, b in (("x", 1.5, 0.4), ("gy", 1.0, 0.0), ("ggx", 1.0, 0.1), ("residual", 1.0, 0.0))}
    t["gamma"] = 1 + 0.2 * torch.randn(cols, generator=g, device=dev)
    t["beta"] = 0.2 * torch.randn(cols, generator=g, device=dev)
    return t


def compare(dev, rows, cols, dtype, code, p, passes, pad=0, seed=0):
    """The given passes against the 64-bit formulas, element by element."""
    from fcd_amd import ops
    t = operands(dev, rows, cols, dtype, seed, pad)
    d = {k: v.double() for k, v in t.items()}
    m = R.keep_mask(rows, cols, p, SEED, OFFSET).to(dev) if p else None
    kw = dict(act_slope=code, p=p, rng=(SEED, OFFSET) if p else None)
    y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], residual=t["residual"], **kw)
    if "fwd" in passes:
        for g, w, dt, name in zip((y, mean, rstd), R.forward(d["x"], d["gamma"], d["beta"], ops.LN_EPS, code, m, d["residual"]),
                                  (dtype, F32, F32), ("y", "mean", "rstd")):
            R.check(g, w, dt, name)
    md, rd = mean.double()[:, None], rstd.double()[:, None]
    if "bwd" in passes:
        got = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
        for g, w, dt, name in zip(got, R.backward(d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, m), (dtype, F32, F32),
                                  ("dx", "dgamma", "dbeta")):
            R.check(g, w, dt, name)
    if "bwd2" in passes:
        got = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
        for g, w, dt, name in zip(got, R.second(d["ggx"], d["x"], d["gy"], md, rd, d["gamma"], d["beta"], code, m),
                                  (dtype, dtype, F32, F32), ("ggy", "gx", "second dgamma", "second dbeta")):
            R.check(g, w, dt, name)


EPILOGUES = [(F32, 1.0, 0.0), (BF16, 1.0, 0.3), (F16, 2.0, 0.0), (F32, 0.01, 0.25), (BF16, 3.0, 0.1)]

# One turn of the forward grid: 2048 workgroups of 256 threads (1024 of 512, 256 of 1024), each with 256 / G rows of up to 64
# lanes or one longer row.  Widths: one per shape, most of them ragged, some with waves that hold no element.
FWD = [(7, 131072), (30, 131072), (61, 65536), (120, 32768), (251, 16384), (500, 8192), (1001, 8192), (1537, 2048), (2048, 2048),
       (4095, 2048), (5000, 1024), (8191, 1024), (9001, 256), (16383, 256)]


@pytest.mark.parametrize("i", range(len(FWD)))
def test_forward_over_several_turns(dev, i):
    """Between two and three turns, so that a workgroup's two buffers and its prefetch are both used again."""
    cols, turn = FWD[i]
    dtype, code, p = EPILOGUES[i % len(EPILOGUES)]
    compare(dev, 2 * turn + turn // 3 + 5, cols, dtype, code, p, ("fwd",), pad=i % 3)
    compare(dev, 2 * turn + turn // 3 + 5, cols, F16, 1.0, 0.0, ("fwd",))


# One turn of the backward grids: 512 workgroups of 256 threads, 1024 of 128, 256 of 512 or 1024.
BWD = [(7, 32768), (30, 32768), (61, 16384), (120, 8192), (251, 4096), (505, 2048), (601, 1024), (1024, 1024), (1200, 512), (1537, 512),
       (2048, 512), (2500, 256), (4095, 256), (5001, 256), (8192, 256)]


@pytest.mark.parametrize("e", range(len(EPILOGUES)))
@pytest.mark.parametrize("cols,turn", BWD)
def test_both_backward_passes_over_several_turns(dev, cols, turn, e):
    dtype, code, p = EPILOGUES[e]
    compare(dev, 2 * turn + turn // 3 + 5, cols, dtype, code, p, ("bwd", "bwd2"), pad=e % 2, seed=e)


@pytest.mark.parametrize("rows,cols", [(700, 1023), (600, 8200), (520, 20001)])
def test_gradients_far_from_zero_over_several_turns(dev, rows, cols):
    """Offsets of a hundred times the spread, in rows that a workgroup takes one after another."""
    from fcd_amd import ops
    t = operands(dev, rows, cols, F32)
    t["gamma"] = 1 + (t["gamma"] - 1) / 100
    t["gy"], t["ggx"] = t["gy"] + 100, t["ggx"] - 100
    d = {k: v.double() for k, v in t.items()}
    mean, rstd = ops.layernorm_fwd(t["x"])[1:]
    got = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"])
    want = R.second(d["ggx"], d["x"], d["gy"], mean.double()[:, None], rstd.double()[:, None], d["gamma"], d["beta"], 1.0, None)
    for g, w, name in zip(got, want, ("ggy", "gx", "dgamma", "dbeta")):
        R.check(g, w, what=name)


# Widths whose last unit is ragged and begins a wave (513, 1027, 1539) or, in split rows, a workgroup (8195, 18433 = 9 * 2048 + 1):
# that unit's load covers columns which another wave may already have written.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cols", [13, 65, 513, 1027, 1539, 2051, 4099, 8195, 18433])
@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("pad", [0, 3])
def test_in_place_with_ragged_rows(dev, rows, cols, pad, dtype):
    from fcd_amd import ops
    t = operands(dev, rows, cols, dtype, seed=1, pad=pad)
    kw = dict(act_slope=2.0, p=0.3, rng=(1, 9))

    def fresh(*names):
        """copies with the same strides"""
        out = {}
        for k in names:
            wide = torch.full((rows, cols + pad), 7.0, dtype=dtype, device=dev)
            out[k] = wide[:, :cols].copy_(t[k])
        return out

    def gaps(o):
        return all(bool((v.as_strided((rows, cols + pad), (cols + pad, 1))[:, cols:] == 7).all()) for v in o.values())

    y, mean, rstd = ops.layernorm_fwd(t["x"], t["gamma"], t["beta"], residual=t["residual"], **kw)
    dx, dg, db = ops.layernorm_bwd(t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    two = ops.layernorm_bwd2(t["ggx"], t["gy"], t["x"], mean, rstd, t["gamma"], t["beta"], **kw)
    drop = ops.dropout(t["x"], 0.3, (1, 9), residual=t["residual"])
    for name in ("x", "residual"):
        o = fresh("x", "residual")
        got = ops.layernorm_fwd(o["x"], t["gamma"], t["beta"], residual=o["residual"], out=o[name], **kw)
        assert torch.equal(got[0], y) and torch.equal(got[1], mean) and torch.equal(got[2], rstd) and gaps(o)
        o = fresh("x", "residual")
        assert torch.equal(ops.dropout(o["x"], 0.3, (1, 9), residual=o["residual"], out=o[name]), drop) and gaps(o)
    for name in ("gy", "x"):
        o = fresh("gy", "x")
        got = ops.layernorm_bwd(o["gy"], o["x"], mean, rstd, t["gamma"], t["beta"], out=o[name], **kw)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dg) and torch.equal(got[2], db) and gaps(o)
    for names in (("gy", "x"), ("ggx", "gy"), ("x", "ggx")):
        o = fresh("x", "gy", "ggx")
        got = ops.layernorm_bwd2(o["ggx"], o["gy"], o["x"], mean, rstd, t["gamma"], t["beta"], outs=tuple(o[k] for k in names), **kw)
        assert all(torch.equal(i, j) for i, j in zip(got, two)) and gaps(o)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(33000, 7), (300, 1021), (70000, 13), (5, 100003)])
def test_dropout_in_place_with_rows_inside_a_block(dev, rows, cols, dtype):
    """Rows that begin inside a generator block, strided, written over themselves, more of them than one turn of the grid."""
    from fcd_amd import ops
    wide = torch.randn(rows, cols + 5, device=dev, generator=torch.Generator(device=dev).manual_seed(cols)).to(dtype)
    m = R.keep_mask(rows, cols, 0.3, SEED, OFFSET).to(dev)
    want = wide[:, :cols].double() * m
    tail = wide[:, cols:].clone()
    got = ops.dropout(wide[:, :cols], 0.3, (SEED, OFFSET), out=wide[:, :cols])
    R.check(got, R.V(want, 2 * R.U * want.abs()), dtype)
    assert torch.equal(got == 0, want == 0) and torch.equal(wide[:, cols:], tail)


@pytest.mark.parametrize("rows,cols", [(525000, 8192), (67200000, 64), (140000, 32768)])
def test_more_than_4_billion_elements(dev, rows, cols):
    """Register-resident and split rows beyond 2^32 elements: the first, a middle and the last rows have the bits that the same rows
    have by themselves, in all three directions and in dropout, written over their inputs to keep the memory small."""
    from fcd_amd import ops
    g = torch.Generator(device=dev).manual_seed(1)
    few = 24
    at = [0, rows // 2 // 8 * 8, rows - few]
    tile = [torch.randn(few, cols, generator=g, device=dev).to(BF16) for _ in range(3)]
    x, gy, v = (t.repeat((rows + few - 1) // few, 1)[:rows] for t in tile)
    samples = [[t[i:i + few].clone() for i in at] for t in (x, gy, v)]
    kw = dict(act_slope=2.0, p=0.25)
    y = torch.empty_like(x)
    _, mean, rstd = ops.layernorm_fwd(x, out=y, rng=(3, 4), **kw)
    want = [ops.layernorm_fwd(s, rng=(3, 4 + i * cols // 8), **kw) for s, i in zip(samples[0], at)]
    for i, w in zip(at, want):
        assert torch.equal(y[i:i + few], w[0]) and torch.equal(mean[i:i + few], w[1]) and torch.equal(rstd[i:i + few], w[2])
    ops.layernorm_bwd(gy, x, mean, rstd, out=y, rng=(3, 4), **kw)
    for k, i in enumerate(at):
        w = ops.layernorm_bwd(samples[1][k], samples[0][k], *want[k][1:], rng=(3, 4 + i * cols // 8), **kw)[0]
        assert torch.equal(y[i:i + few], w)
    del y
    ops.layernorm_bwd2(v, gy, x, mean, rstd, outs=(gy, v), rng=(3, 4), **kw)
    for k, i in enumerate(at):
        w = ops.layernorm_bwd2(samples[2][k], samples[1][k], samples[0][k], *want[k][1:], rng=(3, 4 + i * cols // 8), **kw)
        assert torch.equal(gy[i:i + few], w[0]) and torch.equal(v[i:i + few], w[1])
    ops.dropout(x, 0.25, (3, 4), out=x)
    for k, i in enumerate(at):
        assert torch.equal(x[i:i + few], ops.dropout(samples[0][k], 0.25, (3, 4 + i * cols // 8)))
