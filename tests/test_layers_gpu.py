"""Layer norm and dropout as modules and inside the critic: gradients against formulas, differences and a 64-bit critic."""
import pytest
import torch
import torch.nn.functional as F

import ln_reference as R
from conftest import relerr

pytestmark = pytest.mark.gpu

CODES = {None: 1.0, "relu": 0.0, "lrelu": 0.01, "silu": 2.0, "mish": 3.0}


def tensors(dev, rows, cols, dtype, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(rows, cols, generator=g)).to(dtype).to(dev) for _ in range(n)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("activation", [None, "lrelu", "silu", "mish"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_layer_norm_function_and_both_backwards(dev, dtype, activation, p):
    from fcd_amd import layers
    x, gy, v, res = tensors(dev, 19, 136, dtype, 4, seed=3)
    w = (1 + 0.1 * torch.arange(136, device=dev) / 136).requires_grad_(True)
    b = (0.2 - torch.arange(136, device=dev) / 400).requires_grad_(True)
    x.requires_grad_(True)
    gy.requires_grad_(True)
    res.requires_grad_(True)
    rng = (21, 22)
    y = layers.layer_norm(x, w, b, activation=activation, p=p, rng=rng if p else None, residual=res)
    d = [t.detach().double().cpu() for t in (x, gy, v, res, w, b)]
    m = R.keep_mask(19, 136, p, 21, 22) if p else None
    code = CODES[activation]
    wy, wm, wr = R.forward(d[0], d[4], d[5], 1e-5, code, m, d[3])
    R.check(y, wy, dtype, "y")
    dx, dw, db, dres = torch.autograd.grad(y, (x, w, b, res), gy, create_graph=True)
    assert torch.equal(dres, gy)
    # the kernels' statistics are rounded; the formulas take the exact ones with that rounding as their error
    mean, rstd = R.V(wm.v, wm.e), R.V(wr.v, wr.e)
    x1, w1, b1 = R.backward(d[0], d[1], mean, rstd, d[4], d[5], code, m)
    R.check(dx, x1, dtype, "dx")
    R.check(dw, w1, what="dweight")
    R.check(db, b1, what="dbias")
    gg = torch.autograd.grad(dx, (gy, x, w, b), v)
    g2 = R.backward2(d[2], d[0], d[1], mean, rstd, d[4], d[5], code, m)
    for got, want, t, name in zip(gg, g2, (dtype, dtype, torch.float32, torch.float32), ("ggy", "gx", "dweight", "dbias")):
        R.check(got, want, t, "second " + name)


def test_gradients_against_differences(dev):
    """Directional derivatives of the definition in 64 bits (central differences, h = 1e-4: error h^2 times the third
    derivative, far below the bound) against the kernels' gradients and second gradients."""
    from fcd_amd import layers
    x, gy, v, dirn = tensors(dev, 5, 40, torch.float32, 4, seed=8)
    w = torch.linspace(0.8, 1.2, 40, device=dev)
    b = torch.linspace(-0.3, 0.3, 40, device=dev)
    xd, gd, vd, dd, wd, bd = (t.double().cpu() for t in (x, gy, v, dirn, w, b))
    m = R.keep_mask(5, 40, 0.25, 3, 4)

    def value(t):
        mean = t.mean(1, keepdim=True)
        u = (t - mean) / ((t - mean).square().mean(1, keepdim=True) + 1e-5).sqrt() * wd + bd
        return u * torch.sigmoid(u) * m

    def grad(t):
        t = t.clone().requires_grad_(True)
        return torch.autograd.grad(value(t), t, gd)[0]

    x.requires_grad_(True)
    y = layers.layer_norm(x, w, b, activation="silu", p=0.25, rng=(3, 4))
    dx, = torch.autograd.grad(y, x, gy, create_graph=True)
    gx, = torch.autograd.grad(dx, x, v)
    h = 1e-4
    mean = R.forward(xd, wd, bd, 1e-5, 2.0, m, None)
    b1 = R.backward(xd, gd, mean[1], mean[2], wd, bd, 2.0, m)[0]
    b2 = R.backward2(vd, xd, gd, mean[1], mean[2], wd, bd, 2.0, m)[1]
    for got, num, bound in ((dx, ((value(xd + h * dd) - value(xd - h * dd)) * gd).sum() / (2 * h), b1),
                            (gx, ((grad(xd + h * dd) - grad(xd - h * dd)) * vd).sum() / (2 * h), b2)):
        tol = float((R.rounded(bound, torch.float32) * dd.abs()).sum()) + 1e-5 * float((bound.v.abs() * dd.abs()).sum())
        assert abs(float((got.detach().double().cpu() * dd).sum()) - float(num)) <= tol


def test_dropout_module(dev):
    from fcd_amd import Dropout, ops
    m = Dropout(0.4, seed=9).to(dev)
    x = torch.randn(7, 33, device=dev, requires_grad=True)
    res = torch.randn(7, 33, device=dev, requires_grad=True)
    y = m(x, res)
    y2 = m(x, res)
    assert not torch.equal(y, y2)                       # the state moved on
    assert m.dropout_state.tolist() == [9, 2 * ((7 * 33 + 7) // 8)]
    keep = R.keep_mask(7, 33, 0.4, 9, 0)
    g = torch.randn(7, 33, device=dev)
    gx, gr = torch.autograd.grad(y, (x, res), g)
    assert torch.equal(gr, g)
    want = R.V(g.double().cpu() * keep, 2 * R.U * (g.double().cpu() * keep).abs())
    R.check(gx, want)
    # linear, so its gradient can be differentiated again
    z, = torch.autograd.grad(m(x), x, g.requires_grad_(True), create_graph=True)
    gg, = torch.autograd.grad(z, g, torch.ones_like(z))
    assert torch.equal(gg, ops.dropout(torch.ones_like(x), 0.4, (9, 2 * 29)))
    m.eval()
    assert m(x) is x and torch.equal(m(x, res), x + res)
    assert list(m.state_dict()) == ["dropout_state"] and not Dropout(0.0).state_dict()
    m.train()
    again = Dropout(0.4, seed=1).to(dev)
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(x), m(x))


def test_layer_norm_module(dev):
    from fcd_amd import LayerNorm
    m = LayerNorm(50, activation="mish", dropout=0.2, seed=5).to(dev)
    x = torch.randn(2, 3, 50, device=dev, requires_grad=True)
    y = m(x)
    keep = R.keep_mask(6, 50, 0.2, 5, 0).reshape(2, 3, 50)
    assert torch.equal((y == 0).cpu(), keep == 0)
    y.square().sum().backward()
    assert m.weight.grad.shape == (50,) and x.grad.shape == x.shape
    m.eval()
    ref = F.mish(F.layer_norm(x.double().cpu(), (50,)))
    assert relerr(m(x), ref) <= 1e-6
    # gradients that arrive expanded or transposed are taken as they come
    z = m(x)
    a, = torch.autograd.grad(z.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(z, x, torch.ones_like(z), retain_graph=True)
    assert torch.equal(a, b)
    t = torch.randn(50, 6, device=dev)
    a, = torch.autograd.grad(z, x, t.t().reshape(2, 3, 50))
    assert a.shape == x.shape
    plain = LayerNorm(50, affine=False).to(dev)
    assert not list(plain.parameters()) and relerr(plain(x), F.layer_norm(x.double().cpu(), (50,))) <= 1e-6
    with pytest.raises(RuntimeError, match="last axis"):
        plain(torch.zeros(2, 49, device=dev))
    with pytest.raises(NotImplementedError):
        LayerNorm(8, activation="gelu")
    with pytest.raises(ValueError):
        LayerNorm(8, dropout=1.5)


@pytest.mark.parametrize("layout", ["transposed", "every second column", "expanded"])
def test_inputs_without_even_rows(dev, layout):
    """Layouts the kernels do not take are copied; first and second gradients still reach the tensor that was given."""
    from fcd_amd import layers
    g = torch.Generator().manual_seed(2)
    base = {"transposed": torch.randn(24, 10, generator=g), "every second column": torch.randn(10, 48, generator=g),
            "expanded": torch.randn(10, 1, generator=g)}[layout].to(dev).requires_grad_(True)
    view = {"transposed": lambda t: t.t(), "every second column": lambda t: t[:, ::2], "expanded": lambda t: t.expand(10, 24)}[layout]
    w = torch.linspace(0.5, 1.5, 24, device=dev)
    gy, v = torch.randn(10, 24, generator=g).to(dev), torch.randn(base.shape, generator=g).to(dev)
    res = []
    for x in (view(base), view(base).contiguous()):
        y = layers.layer_norm(x, w, activation="silu", residual=x)
        dx, = torch.autograd.grad(y, base, gy, create_graph=True)
        res.append((y, dx, torch.autograd.grad(dx, base, v)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    y = layers.dropout(view(base), 0.5, (1, 2))
    assert torch.equal(y, layers.dropout(view(base).contiguous(), 0.5, (1, 2)))


def test_parameter_gradients_are_not_differentiable(dev):
    from fcd_amd import layers
    x = torch.randn(4, 16, device=dev, requires_grad=True)
    w = torch.ones(16, device=dev, requires_grad=True)
    y = layers.layer_norm(x, w)
    dw, = torch.autograd.grad(y, w, torch.ones_like(y), create_graph=True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(dw.sum(), x)


def test_module_in_a_captured_graph(dev):
    """A module's training pass (forward, both backward passes) captured once: every replay draws new masks and equals the
    eager pass from the same state."""
    from fcd_amd import LayerNorm
    m = LayerNorm(96, activation="silu", dropout=0.3, seed=4).to(dev)
    x = torch.randn(40, 96, device=dev, requires_grad=True)
    gy, v = torch.randn(40, 96, device=dev), torch.randn(40, 96, device=dev)

    def run():
        y = m(x)
        dx, = torch.autograd.grad(y, x, gy, create_graph=True)
        return [y.detach(), dx.detach(), *torch.autograd.grad(dx, (x, m.weight, m.bias), v)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    start = m.dropout_state.clone()
    got = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got.append([t.clone() for t in outs])
    assert not torch.equal(got[0][0], got[1][0])
    m.dropout_state.copy_(start)
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, run()))


# ---- the critic -------------------------------------------------------------------------------------------------------------

def critic64(params, x, act, norm, p, seed, offset, repeat):
    """The critic in 64 bits on the host: (out_src, out_cls, features of every layer, next offset)."""
    f = {"lrelu": lambda u: torch.where(u > 0, u, 0.01 * u), "silu": F.silu, "mish": F.mish}[act]
    a = x
    for i in range(repeat):
        a = F.conv2d(a, params[f"{i}.weight"], params[f"{i}.bias"], 2, 1)
        n, c, h, w = a.shape
        if norm:
            z = a.permute(0, 2, 3, 1)
            mean = z.mean(-1, keepdim=True)
            z = (z - mean) / ((z - mean).square().mean(-1, keepdim=True) + 1e-5).sqrt()
            a = (z * params[f"{i}.gamma"] + params[f"{i}.beta"]).permute(0, 3, 1, 2)
        a = f(a)
        if p:
            keep = R.keep_mask(n * h * w, c, p, seed, offset).reshape(n, h, w, c).permute(0, 3, 1, 2)
            offset += (n * h * w * c + 7) // 8
            a = a * keep
    return F.conv2d(a, params["conv1"], None, 1, 1), F.conv2d(a, params["conv2"]), a, offset


def critic_params(D):
    out = {}
    for i, cv in enumerate(D._convs):
        out[f"{i}.weight"], out[f"{i}.bias"] = cv.weight, cv.bias
    for i, nm in enumerate(D._norms):
        out[f"{i}.gamma"], out[f"{i}.beta"] = nm.weight, nm.bias
    out["conv1"], out["conv2"] = D.conv1.weight, D.conv2.weight
    return out


@pytest.mark.parametrize("arena", [False, True])
@pytest.mark.parametrize("act,norm,p,conv_dim", [("silu", "layer", 0.25, 8), ("lrelu", "layer", 0.0, 8), ("mish", "layer", 0.0, 6),
                                                ("lrelu", "none", 0.25, 8), ("silu", "none", 0.25, 6), ("lrelu", "layer", 0.5, 16)])
def test_critic_step_with_gradient_penalty(dev, act, norm, p, conv_dim, arena):
    """Losses and all gradients of a critic's step with the gradient penalty against the 64-bit critic (the bar of the
    framework's fp32 path, 1e-4 relative), with gradients carried by autograd and accumulated in an arena."""
    from fcd_amd import Discriminator
    from fcd_amd.arena import ParamArena
    from fcd_amd.discriminator import input_grad_only
    from fcd_amd import losses
    torch.manual_seed(7)
    D = Discriminator(32, conv_dim, 1, 3, 10, activation=act, n_feature_layers=2, norm=norm, dropout=p, dropout_seed=77)
    for nm in D._norms:
        with torch.no_grad():
            nm.weight.uniform_(0.7, 1.3)
            nm.bias.uniform_(-0.3, 0.3)
    x, xh = torch.rand(3, 10, 32, 32) * 2 - 1, torch.rand(2, 10, 32, 32) * 2 - 1
    ref = {k: t.detach().double().requires_grad_(True) for k, t in critic_params(D).items()}
    D = D.to(dev)
    ar = ParamArena(D.parameters()) if arena else None

    def total(src, cls, gp):
        return -src.mean() + (cls * torch.linspace(0.5, 1.0, 3, dtype=cls.dtype, device=cls.device)[:, None]).sum() + 10 * gp

    src, cls, _ = D(x.to(dev))
    xg = xh.to(dev).requires_grad_(True)
    s2, _, _ = D(xg)
    with input_grad_only(D):
        dydx, = torch.autograd.grad(s2, xg, torch.ones_like(s2), create_graph=True)
    loss = total(src, cls, losses.gp_loss(dydx.reshape(2, -1)))
    if arena:
        with ar.accumulating():
            loss.backward()
    else:
        loss.backward()

    rs, rc, _, off = critic64(ref, x.double(), act, norm == "layer", p, 77, 0, 3)
    xr = xh.double().requires_grad_(True)
    r2, _, _, off = critic64(ref, xr, act, norm == "layer", p, 77, off, 3)
    rdx, = torch.autograd.grad(r2, xr, torch.ones_like(r2), create_graph=True)
    rl = total(rs, rc.reshape(3, 1), ((rdx.reshape(2, -1).norm(2, 1) - 1) ** 2).mean())
    rl.backward()
    if p:
        assert D.dropout_state.tolist() == [77, off]
    assert relerr(src, rs) <= 1e-4 and relerr(cls, rc.reshape(3, 1)) <= 1e-4 and relerr(dydx, rdx) <= 1e-4
    assert abs(float(loss.detach()) - float(rl.detach())) <= 1e-4 * max(1.0, abs(float(rl.detach())))
    # a bias in front of a norm over channels still matters (the norm takes the mean over channels, not pixels)
    for k, t in critic_params(D).items():
        assert t.grad is not None and relerr(t.grad, ref[k].grad) <= 1e-4, k


@pytest.mark.parametrize("precision", ["fp32", "fp32x2"])
def test_training_steps_with_norm_and_dropout(dev, precision):
    """Whole training steps of the solver: finite losses, every critic parameter moves, the same run gives the same bits, and
    evaluation does not draw."""
    from fcd_amd import FCDSolver
    from oracle import fcd_oracle as O

    def run():
        torch.manual_seed(3)
        s = FCDSolver(None, c_dim=1, image_size=32, g_conv_dim=8, d_conv_dim=8, g_repeat_num=2, d_repeat_num=3, num_channels=10,
                      batch_size=2, n_critic=1, norm_D="layer", dropout_D=0.25, precision=precision)
        s.to(dev)
        batch, alpha = O.synth_batch(2, 32, 10)
        s.alpha_override = alpha
        before = [t.detach().clone() for t in s.D.parameters()]
        for _ in range(3):
            s.train_step(tuple(t.to(dev) for t in batch))
        assert all(bool(torch.isfinite(v).all()) for v in s.loss_dict.values())
        moved = [not torch.equal(a, b) for a, b in zip(before, s.D.parameters())]
        assert all(moved)
        return s, [t.detach().clone() for t in list(s.D.parameters()) + list(s.G.parameters())]

    s, a = run()
    _, b = run()
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    s.D.eval()
    state = s.D.dropout_state.clone()
    x = torch.rand(2, 10, 32, 32, device=dev)
    assert torch.equal(s.D(x)[0], s.D(x)[0]) and torch.equal(state, s.D.dropout_state)


def test_modules_without_a_seed_drop_other_elements(dev):
    """Three modules of one model on one shape: each pair of masks agrees where two independent draws would (share 1/2 of 2^16
    elements within 6 standard deviations), at the first step and at the next."""
    from fcd_amd import Dropout, LayerNorm
    torch.manual_seed(3)
    mods = [Dropout(0.5).to(dev), Dropout(0.5).to(dev), LayerNorm(64, dropout=0.5).to(dev)]
    x = torch.randn(1024, 64, device=dev) + 5
    for _ in range(2):
        kept = [m(x) != 0 for m in mods]
        for i in range(3):
            for k in range(i):
                assert abs(float((kept[i] == kept[k]).double().mean()) - 0.5) <= 6 * (0.25 / x.numel()) ** 0.5


def test_rng_that_changed_since_the_forward_pass(dev):
    """The backward passes draw the forward's mask again: an rng tensor that moved on meanwhile (a generator's own state, or words
    written over) is refused as any saved tensor is, not used for another mask."""
    from fcd_amd import layers, ops
    x = torch.randn(16, 64, device=dev, requires_grad=True)
    moves = {"state": lambda t: ops.dropout_take(t, x.numel()), "words": lambda t: t.add_(1)}
    for move in moves.values():
        for wrap in (lambda t: t, lambda t: (t, 5)):
            for run in (lambda rng: layers.dropout(x, 0.5, rng), lambda rng: layers.layer_norm(x, activation="silu", p=0.5, rng=rng)):
                rng = ops.dropout_state(3, dev)
                y = run(wrap(rng))
                want, = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)       # (unchanged: taken)
                assert torch.equal(want, torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)[0])
                move(rng)
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(y, x, torch.ones_like(y))
                gy = torch.ones_like(y).requires_grad_(True)
                rng = ops.dropout_state(3, dev)
                dx, = torch.autograd.grad(run(wrap(rng)), x, gy, create_graph=True)
                move(rng)
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(dx, gy, torch.ones_like(dx))
