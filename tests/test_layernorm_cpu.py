"""Layer norm and dropout: the published generator's test vectors, the formulas against autograd, and every refusal (none of
these calls reaches a GPU)."""
import ctypes as C

import numpy as np
import pytest
import torch

import ln_reference as R


def test_generator_matches_its_published_vectors():
    """Known answers distributed with the Philox4x32-10 paper's library."""
    for counter, key, want in (
            ([0, 0, 0, 0], [0, 0], [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
             [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])):
        assert R.philox(np.array([counter], np.uint64), key)[0].tolist() == want


@pytest.mark.parametrize("code", [1.0, 0.01, 2.0, 3.0])
def test_formulas_against_autograd(code):
    """The backward formulas (first and second) are the derivatives of the definition."""
    g = torch.Generator().manual_seed(4)
    x, gy, v = (torch.randn(6, 23, generator=g, dtype=torch.float64) for _ in range(3))
    ga, be = 1 + 0.2 * torch.randn(23, generator=g, dtype=torch.float64), 0.2 * torch.randn(23, generator=g, dtype=torch.float64)
    m = R.keep_mask(6, 23, 0.4, 5, 6)
    f = {1.0: lambda u: u, 0.01: lambda u: torch.where(u > 0, u, 0.01 * u), 2.0: lambda u: u * torch.sigmoid(u),
         3.0: lambda u: u * torch.tanh(torch.log1p(torch.exp(u)))}[code]
    leaves = [t.clone().requires_grad_(True) for t in (x, gy, ga, be)]
    mean = leaves[0].mean(1, keepdim=True)
    rstd = (((leaves[0] - mean) ** 2).mean(1, keepdim=True) + 1e-5) ** -0.5
    y = f((leaves[0] - mean) * rstd * leaves[2] + leaves[3]) * m
    wy, _, _ = R.forward(x, ga, be, 1e-5, code, m, None)
    assert torch.allclose(wy.v, y, rtol=1e-12, atol=1e-12)
    grads = torch.autograd.grad(y, (leaves[0], leaves[2], leaves[3]), leaves[1], create_graph=True)
    md, rd = mean.detach(), rstd.detach()
    for got, want in zip(R.backward(x, gy, md, rd, ga, be, code, m), grads):
        assert torch.allclose(got.v, want, rtol=1e-10, atol=1e-10)
    second = torch.autograd.grad(grads[0], (leaves[1], leaves[0], leaves[2], leaves[3]), v, allow_unused=True)
    for got, want in zip(R.backward2(v, x, gy, md, rd, ga, be, code, m), second):
        assert torch.allclose(got.v, torch.zeros_like(got.v) if want is None else want, rtol=1e-9, atol=1e-9)


# ---- refusals of the C entries: the pointers are made up, no call may get as far as a launch ------------------------------

P = 1 << 20


def desc(**over):
    from fcd_amd import _lib
    d = _lib.LayerNormDesc()
    base = dict(rows=4, cols=16, ld_x=16, ld_res=16, ld_gy=16, ld_ggx=16, ld_out=16, ld_ggy=16, eps=1e-5, act=1.0)
    for k, v in {**base, **over}.items():
        setattr(d, k, v)
    return d


def refused(rc, text, code=-1):
    from fcd_amd import _lib
    msg = _lib.load().fcd_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


BAD = [
    (dict(dtype=3), "element type"), (dict(dtype=-1), "element type"), (dict(dtype=1, param_dtype=2), "parameters must be"),
    (dict(rows=-1), "negative number of rows"), (dict(cols=0), "columns"), (dict(cols=-3), "columns"),
    (dict(cols=1 << 31, ld_x=1 << 31, ld_out=1 << 31, ld_gy=1 << 31, ld_ggx=1 << 31, ld_ggy=1 << 31), "columns"),
    (dict(rows=1 << 60), "too many"), (dict(rows=1 << 40, cols=1 << 20), "too many"),
    (dict(act=-0.1), "activation"), (dict(act=1.5), "activation"), (dict(act=4.0), "activation"),
    (dict(act=float("nan")), "activation"), (dict(drop_p=-0.1), "probability"), (dict(drop_p=1.1), "probability"),
    (dict(drop_p=float("nan")), "probability"), (dict(drop_p=0.1, rng=P + 4), "8-byte"),
    (dict(ld_x=-1), "row stride"), (dict(ld_out=15), "row stride"), (dict(ld_x=1 << 57), "too large"),
]


@pytest.mark.parametrize("over,text", BAD)
def test_descriptors_refused(over, text):
    from fcd_amd import _lib
    lib, d = _lib.load(), C.byref(desc(**over))
    f = lambda i: P * 64 * i
    refused(lib.fcd_layernorm_fwd(d, f(1), None, None, None, f(2), f(3), f(4), None, 0, None), text)
    refused(lib.fcd_layernorm_bwd(d, f(1), f(2), f(3), f(4), None, None, f(5), None, None, 0, None, 0, None), text)
    refused(lib.fcd_layernorm_bwd2(d, f(1), f(2), f(3), f(4), f(5), None, None, f(6), f(7), None, None, 0, None, 0, None), text)


@pytest.mark.parametrize("eps", [-1e-5, float("nan"), float("inf")])
def test_eps_refused(eps):
    from fcd_amd import _lib
    refused(_lib.load().fcd_layernorm_fwd(C.byref(desc(eps=eps)), P, None, None, None, 2 * P, None, None, None, 0, None), "eps")


def test_forward_operands_refused():
    from fcd_amd import _lib
    lib = _lib.load()
    fwd = lambda *a: lib.fcd_layernorm_fwd(*a[:-1], None, 0, a[-1])
    d = C.byref(desc())
    refused(fwd(None, P, None, None, None, 2 * P, None, None, None), "NULL descriptor")
    refused(fwd(d, None, None, None, None, P, None, None, None), "x is NULL")
    refused(fwd(d, P, None, None, None, None, None, None, None), "y is NULL")
    refused(fwd(d, P + 2, None, None, None, 2 * P, None, None, None), "x is not aligned")
    refused(fwd(d, P, P + 1, None, None, 2 * P, None, None, None), "gamma / beta")
    refused(fwd(d, P, None, None, None, 2 * P, 3 * P + 1, 4 * P, None), "mean / rstd")
    refused(fwd(d, P, None, None, None, 2 * P, 3 * P, None, None), "go together")
    refused(fwd(d, P, None, None, None, P + 4, None, None, None), "overlaps x")
    refused(fwd(d, P, None, None, 2 * P, 2 * P + 16 * 4 * 3, None, None, None), "overlaps residual")
    # the same address with another row stride; columns of a wider tensor that meet; rows written over one another
    refused(fwd(C.byref(desc(ld_x=20)), P, None, None, None, P, None, None, None), "overlaps x")
    refused(fwd(C.byref(desc(ld_x=40, ld_out=40)), P, None, None, None, P + 15 * 4, None, None, None), "overlaps x")
    refused(fwd(C.byref(desc(ld_x=40, ld_out=40)), P, None, None, None, P + 25 * 4, None, None, None), "overlaps x")
    refused(fwd(C.byref(desc(ld_out=8)), P, None, None, None, 2 * P, None, None, None), "row stride 8 of y")


def test_backward_operands_refused():
    from fcd_amd import _lib
    lib = _lib.load()
    d = desc(rows=400)
    need = lib.fcd_layernorm_workspace_bytes(C.byref(d), 1, 1)
    assert need >= 2 * 16 * 4
    f = lambda i: P * i
    call = lambda **k: lib.fcd_layernorm_bwd(C.byref(d), *[{**dict(gy=f(1), x=f(2), mean=f(3), rstd=f(4), ga=None, be=None, dx=f(5),
                                                            dg=f(6), db=f(7), acc=0, ws=f(8), n=need, st=None), **k}[n]
                                                           for n in ("gy", "x", "mean", "rstd", "ga", "be", "dx", "dg", "db", "acc", "ws", "n", "st")])
    refused(call(gy=None), "gy is NULL")
    refused(call(mean=None), "mean / rstd are NULL")
    refused(call(n=need - 1), "workspace", -2)
    refused(call(ws=None), "workspace")
    refused(call(ws=f(8) + 4), "workspace")
    refused(call(dg=f(6) + 2), "gamma / beta")
    refused(call(dx=f(1) + 4), "overlaps gy")
    d2 = lambda *a: lib.fcd_layernorm_bwd2(C.byref(d), *a)
    refused(d2(f(1), f(2), f(3), f(4), f(5), None, None, f(6), f(6), None, None, 0, None, 0, None), "overlaps ggy")
    refused(d2(f(1), f(2), f(3), f(4), f(5), None, None, f(6), f(1) + 8, None, None, 0, None, 0, None), "overlaps ggx")
    refused(d2(None, f(2), f(3), f(4), f(5), None, None, f(6), f(7), None, None, 0, None, 0, None), "ggx is NULL")
    refused(d2(f(1), f(2), f(3), f(4), f(5), None, None, f(6), f(7), f(8), None, 0, f(9), 8, None), "workspace", -2)
    for which in (0, 1, 2):
        assert lib.fcd_layernorm_workspace_bytes(None, which, 1) == 0
        assert lib.fcd_layernorm_workspace_bytes(C.byref(desc(rows=0)), which, 1) == 0
    small = C.byref(desc(rows=4))
    assert lib.fcd_layernorm_workspace_bytes(small, 0, 1) == 0            # the forward pass and few rows need none
    assert lib.fcd_layernorm_workspace_bytes(small, 1, 1) == 0
    assert lib.fcd_layernorm_workspace_bytes(small, 2, 1) >= 2 * 16 * 4
    assert lib.fcd_layernorm_workspace_bytes(small, 2, 0) == 0
    # split rows need some in every pass, with or without affine gradients
    n = 40000
    wide = desc(rows=4, cols=n, ld_x=n, ld_gy=n, ld_ggx=n, ld_out=n, ld_ggy=n)
    for which in (0, 1, 2):
        assert lib.fcd_layernorm_workspace_bytes(C.byref(wide), which, 0) > 0
    refused(lib.fcd_layernorm_fwd(C.byref(wide), f(1), None, None, None, f(2), None, None, None, 0, None), "workspace", -2)
    refused(lib.fcd_layernorm_bwd(C.byref(wide), f(1), f(2), f(3), f(4), None, None, f(5), None, None, 0, None, 0, None),
            "workspace", -2)


def test_vectors_that_share_memory_refused():
    """A vector or workspace that a call writes shares no byte with anything else of it; gaps between rows are free."""
    from fcd_amd import _lib
    lib = _lib.load()
    f = lambda i: P * 64 * i
    d = C.byref(desc())                                                  # 4 rows of 16 fp32
    def fwd(**k):
        at = {**dict(x=f(1), gamma=f(2), beta=f(3), res=f(4), y=f(5), mean=f(6), rstd=f(7)), **k}
        return lib.fcd_layernorm_fwd(d, *at.values(), None, 0, None)

    def bwd(d=d, **k):
        at = {**dict(gy=f(1), x=f(2), mean=f(3), rstd=f(4), gamma=f(5), beta=f(6), dx=f(7), dgamma=f(8), dbeta=f(9)), **k}
        return lib.fcd_layernorm_bwd(d, *at.values(), 0, None, 0, None)

    def bwd2(**k):
        at = {**dict(ggx=f(10), gy=f(1), x=f(2), mean=f(3), rstd=f(4), gamma=f(5), beta=f(6), ggy=f(7), gx=f(11), dgamma=f(8),
                     dbeta=f(9)), **k}
        return lib.fcd_layernorm_bwd2(d, *at.values(), 0, f(12), lib.fcd_layernorm_workspace_bytes(d, 2, 1), None)

    refused(fwd(rstd=f(6)), "mean overlaps rstd")
    refused(fwd(rstd=f(6) + 12), "mean overlaps rstd")
    refused(fwd(mean=f(2) + 60), "mean overlaps gamma")
    refused(fwd(rstd=f(3) - 12), "rstd overlaps beta")
    refused(fwd(mean=f(1)), "mean overlaps x")
    refused(fwd(rstd=f(4) + 255 // 4 * 4), "rstd overlaps residual")
    refused(fwd(mean=f(5) - 4), "mean overlaps y")
    refused(fwd(gamma=f(5)), "gamma overlaps y")
    wide = C.byref(desc(ld_x=24, ld_out=16))
    refused(lib.fcd_layernorm_fwd(wide, f(1), None, None, None, f(5), f(1) + 64 + 20, f(7), None, 0, None), "mean overlaps x")

    refused(bwd(dgamma=f(9)), "dgamma overlaps dbeta")
    refused(bwd(dgamma=f(5)), "dgamma overlaps gamma")
    refused(bwd(dbeta=f(6) + 60), "dbeta overlaps beta")
    refused(bwd(dbeta=f(3)), "dbeta overlaps mean")
    refused(bwd(dgamma=f(7)), "dgamma overlaps dx")
    refused(bwd(dgamma=f(1)), "dgamma overlaps gy")
    refused(bwd(mean=f(7)), "mean overlaps dx")
    many = desc(rows=400)
    need = lib.fcd_layernorm_workspace_bytes(C.byref(many), 1, 1)
    refused(lib.fcd_layernorm_bwd(C.byref(many), f(1), f(2), f(3), f(4), f(5), f(6), f(7), f(8), f(9), 0, f(8) - 64, need, None),
            "dgamma overlaps workspace")
    refused(bwd2(dbeta=f(10)), "dbeta overlaps ggx")
    refused(bwd2(dgamma=f(11)), "dgamma overlaps gx")
    refused(bwd2(rstd=f(7) + 4), "rstd overlaps ggy")
    rng = C.byref(desc(drop_p=0.5, rng=f(7) + 8))
    refused(bwd(d=rng), "rng overlaps dx")
    refused(lib.fcd_dropout(f(1), None, f(2), 4, 16, 16, 0, 16, 0, 0.5, 0, 0, f(2) + 248, None), "rng overlaps y")


def test_dropout_refused():
    from fcd_amd import _lib
    lib = _lib.load()
    call = lambda **k: lib.fcd_dropout(*[{**dict(x=P, r=None, y=2 * P, rows=4, cols=16, lx=16, lr=16, ly=16, dt=0, p=0.5, seed=1,
                                                 off=2, rng=None, st=None), **k}[n]
                                         for n in ("x", "r", "y", "rows", "cols", "lx", "lr", "ly", "dt", "p", "seed", "off", "rng", "st")])
    refused(call(dt=7), "element type")
    refused(call(rows=-1), "negative size")
    refused(call(cols=-1), "negative size")
    refused(call(p=-1e-9), "probability")
    refused(call(p=float("nan")), "probability")
    refused(call(rng=P + 2), "8-byte")
    refused(call(x=None), "x is NULL")
    refused(call(y=None), "y is NULL")
    refused(call(y=P + 4), "overlaps x")
    refused(call(r=3 * P + 1), "residual is not aligned")
    refused(call(ly=15), "row stride")
    refused(call(rows=1 << 50, lx=1 << 20, ly=1 << 20), "too large")
    refused(lib.fcd_dropout_take(None, P, 1, None), "NULL")
    refused(lib.fcd_dropout_take(P, P + 8, 1, None), "overlaps")
    refused(lib.fcd_dropout_take(P + 4, 2 * P, 1, None), "8-byte")


def test_python_operands_refused():
    from fcd_amd import ops
    x = torch.zeros(4, 16)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        ops.layernorm_fwd(x)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        ops.dropout(x, 0.5, (1, 2))
    with pytest.raises(RuntimeError, match="on the GPU"):
        ops.dropout_take(torch.zeros(2, dtype=torch.int64), 4)
    # the layout rules are host logic
    assert ops._rows(x, "x") == (4, 16, 16)
    assert ops._rows(x[:, 3:10], "x") == (4, 7, 16)
    assert ops._rows(x[::2], "x") == (2, 16, 32)
    assert ops._rows(x[0], "x") == (1, 16, 16)
    assert ops._rows(x[0].expand(5, 16), "x") == (5, 16, 0)
    assert ops._rows(torch.zeros(2, 3, 5, 8)[..., 1:4], "x") == (30, 3, 8)
    assert ops._rows(torch.zeros(0, 8), "x") == (0, 8, 8)
    assert ops._rows(torch.zeros(3, 0), "x")[:2] == (3, 0)
    for bad in (x.t(), torch.zeros(4, 6, 8)[:, ::4], torch.zeros(4, 6, 8).transpose(0, 1), torch.tensor(1.0), x[:, ::2]):
        if bad.dim() == 3 and bad.shape[1] == 2:
            bad = bad[:, :, :4].transpose(0, 1)
        with pytest.raises(RuntimeError):
            ops._rows(bad, "x")
    with pytest.raises(RuntimeError, match="expected"):
        ops._row_operand(torch.zeros(4, 8), "gy", x)
    with pytest.raises(RuntimeError, match="expected"):
        ops._row_operand(torch.zeros(4, 16, dtype=torch.float16), "gy", x)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(RuntimeError, match="probability"):
            ops._rng_words(p, (1, 2), 0)
    with pytest.raises(RuntimeError, match="needs rng"):
        ops._rng_words(0.5, None, 0)
    with pytest.raises(RuntimeError, match="int64"):
        ops._rng_words(0.5, torch.zeros(2), 0)
    assert ops._rng_words(0.5, (-1, 2), 0) == (2 ** 64 - 1, 2, None)
    assert ops.dropout_state(-5, "cpu", offset=(1 << 64) - 1).tolist() == [-5, -1]


def test_critic_keys_and_refusals():
    from fcd_amd import Discriminator
    D = Discriminator(32, 8, 1, 3, 10, n_feature_layers=2, norm="layer", dropout=0.1, dropout_seed=3)
    keys = set(D.state_dict())
    assert {"features.0.0.weight", "features.0.1.weight", "features.0.1.bias", "main.0.1.weight", "dropout_state"} <= keys
    assert "features.0.1.weight" not in Discriminator(32, 8, 1, 3, 10).state_dict()
    with pytest.raises(NotImplementedError):
        Discriminator(32, 8, 1, 3, 10, norm="batch")
    with pytest.raises(NotImplementedError):
        Discriminator(32, 8, 1, 3, 10, norm="layer", interm_non_act=True)
    with pytest.raises(ValueError):
        Discriminator(32, 8, 1, 3, 10, dropout=-0.5)


def test_modules_refuse_the_cpu_and_bad_arguments():
    from fcd_amd import Dropout, LayerNorm
    with pytest.raises(RuntimeError, match="GPU"):
        LayerNorm(8)(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        Dropout(0.5)(torch.zeros(2, 8))
    assert Dropout(0.5).eval()(torch.zeros(2, 8)).shape == (2, 8)      # the identity launches nothing
    with pytest.raises(ValueError):
        Dropout(-0.1)
    with pytest.raises(NotImplementedError):
        LayerNorm(8, activation="tanh")


def test_modules_without_a_seed_draw_apart():
    """Modules whose seed is left out get generators of their own, the same ones again under the same ``manual_seed``; a given
    seed is taken as it is; parameters come out as without dropout."""
    from fcd_amd import Discriminator, Dropout, LayerNorm

    def build():
        torch.manual_seed(12)
        return [Dropout(0.5), Dropout(0.5), LayerNorm(8, dropout=0.5), LayerNorm(8, dropout=0.5),
                Discriminator(32, 8, 1, 3, 10, n_feature_layers=2, dropout=0.5)]

    first, again = build(), build()
    states = [tuple(m.dropout_state.tolist()) for m in first]
    assert len({s for s, _ in states}) == len(states) and all(o == 0 for _, o in states)
    assert states == [tuple(m.dropout_state.tolist()) for m in again]
    assert Dropout(0.5, seed=7).dropout_state.tolist() == LayerNorm(8, dropout=0.1, seed=7).dropout_state.tolist() == [7, 0]
    torch.manual_seed(5)
    with_dropout = Discriminator(32, 8, 1, 3, 10, n_feature_layers=2, dropout=0.5)
    torch.manual_seed(5)
    without = Discriminator(32, 8, 1, 3, 10, n_feature_layers=2)
    assert all(torch.equal(a, b) for a, b in zip(with_dropout.parameters(), without.parameters()))
    before = torch.get_rng_state()
    Dropout(0.0), LayerNorm(8), Dropout(0.5, seed=1)                # nothing to draw: torch's generator stays where it is
    assert torch.equal(before, torch.get_rng_state())


@pytest.mark.parametrize("code", [1.0, 0.01, 2.0, 3.0])
@pytest.mark.parametrize("offset", [0.0, 100.0])
def test_centred_second_backward_is_the_same_function(code, offset):
    """The second backward's formula around the means equals the one that is checked against autograd."""
    g = torch.Generator().manual_seed(6)
    x, gy, v = (torch.randn(6, 23, generator=g, dtype=torch.float64) + s for s in (0.0, offset, offset))
    ga, be = 1 + 0.2 * torch.randn(23, generator=g, dtype=torch.float64), 0.2 * torch.randn(23, generator=g, dtype=torch.float64)
    m = R.keep_mask(6, 23, 0.4, 5, 6)
    mean = x.mean(1, keepdim=True)
    rstd = (((x - mean) ** 2).mean(1, keepdim=True) + 1e-5) ** -0.5
    for got, want in zip(R.second(v, x, gy, mean, rstd, ga, be, code, m), R.backward2(v, x, gy, mean, rstd, ga, be, code, m)):
        assert torch.allclose(got.v, want.v, rtol=1e-9, atol=1e-9 * max(1.0, offset ** 2))
    one = R.V(torch.full((6, 23), 0.5, dtype=torch.float64))
    for got, want in zip(R.first(x, gy, mean, rstd, ga, one), R.backward(x, gy * 0.5, mean, rstd, ga, be, 1.0, None)):
        assert torch.allclose(got.v, want.v, rtol=1e-12, atol=1e-10)
