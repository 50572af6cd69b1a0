"""Plain 64-bit layer norm, dropout and their gradients with running error bounds.

Every quantity is a pair (value in 64 bits, bound on the error an fp32 evaluation of the same expression may have), to
first order: an operation passes on its operands' errors and adds half a step of its result.  The bounds are what the
tests compare the kernels with; nothing in them is measured."""
import numpy as np
import torch

U = 2.0 ** -24            # half a step of fp32, relative
# Additions on the longest path of one row sum: 8 elements of a lane's unit, up to 64 units or chunks one after another at the
# tested lengths, 6 stages in the wave, up to 16 waves, and the division by the length.
CHAIN = 8 + 64 + 6 + 16 + 1
# ... of a column sum: up to 80 rows kept by a thread and the wave's threads of that column, up to 16 wave sums one after another,
# then up to 512 workgroups' sums in at most 32 strands of 16, joined in order (48).
COLUMN = 80 + 64 + 64 + 4
FUNC = 16                 # an activation or its derivatives: a few roundings around an exp2 and reciprocals of a step each


class V:
    """value, error bound"""

    def __init__(self, v, e=0.0):
        self.v = v
        self.e = e if torch.is_tensor(e) else torch.full_like(v, e)

    def __add__(self, o):
        o = wrap(o, self.v)
        v = self.v + o.v
        return V(v, self.e + o.e + U * v.abs())

    def __sub__(self, o):
        o = wrap(o, self.v)
        v = self.v - o.v
        return V(v, self.e + o.e + U * v.abs())

    def __mul__(self, o):
        o = wrap(o, self.v)
        v = self.v * o.v
        return V(v, self.e * o.v.abs() + o.e * self.v.abs() + U * v.abs())

    def mean(self, chain=CHAIN):
        v = self.v.mean(-1, keepdim=True)
        return V(v, self.e.mean(-1, keepdim=True) + chain * U * self.v.abs().mean(-1, keepdim=True))

    def colsum(self, chain=COLUMN):
        return V(self.v.sum(0), self.e.sum(0) + chain * U * self.v.abs().sum(0))


def wrap(o, like):
    return o if isinstance(o, V) else V(torch.as_tensor(o, dtype=like.dtype, device=like.device))


def act(u, code, order):
    """The activation of a V or its first / second derivative; the error passes through the next derivative."""
    if code <= 1.0:
        s = torch.where(u.v > 0, torch.ones_like(u.v), torch.full_like(u.v, code))
        if order == 0:           # (the slope is a rounded number itself)
            return V(u.v * s, u.e + 2 * U * u.v.abs())
        if order == 1:           # a u within its error of zero may take either side
            return V(s, torch.where(u.v.abs() <= u.e, torch.full_like(u.v, 1.0 - code), U * s))
        return V(torch.zeros_like(u.v))
    x = u.v.clone().requires_grad_(True)
    with torch.enable_grad():
        f = x * torch.sigmoid(x) if code == 2.0 else x * torch.tanh(torch.log1p(torch.exp(x)))
        d = [f]
        for _ in range(order + 1):
            d.append(torch.autograd.grad(d[-1].sum(), x, create_graph=True)[0])
    val, nxt = d[order].detach(), d[order + 1].detach()
    return V(val, nxt.abs() * u.e + FUNC * U * (1.0 + u.v.abs()))


def rounded(v, dtype):
    """Tolerance of a V stored in ``dtype``: its error, half a step of the type, half its smallest number."""
    if dtype == torch.float32:
        return v.e + 1e-37
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    return v.e + torch.finfo(dtype).eps / 2 * (v.v.abs() + v.e) + tiny


def check(got, want, dtype=torch.float32, what=""):
    """``got`` (any shape) against the V ``want``, element by element."""
    assert got.dtype == dtype, (what, got.dtype)
    diff = (got.double().cpu().reshape(want.v.shape) - want.v.cpu()).abs()
    tol = rounded(V(want.v.cpu(), want.e.cpu()), dtype)
    bad = ~(diff <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((diff / tol).nan_to_num(1e30).max()), bad.nonzero()[:4].tolist())


# ---- dropout ------------------------------------------------------------------------------------------------------------

def philox(counter, key, rounds=10):
    """Philox4x32 of 64-bit unsigned arrays of words: counter (n, 4), key (2) -> (n, 4)."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    m = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def keep_mask(rows, cols, p, seed, offset):
    """(rows, cols) of 0 and the scale."""
    total = rows * cols
    blocks = (np.arange((total + 7) // 8, dtype=np.uint64) + np.uint64(offset & (2 ** 64 - 1)))
    counter = np.zeros((len(blocks), 4), np.uint64)
    counter[:, 0], counter[:, 1] = blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32)
    w = philox(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    bits = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], 2).reshape(-1)[:total]
    t = int(np.rint(p * 65536))
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return torch.from_numpy(np.where(bits >= t, scale, 0.0)).reshape(rows, cols)


# ---- layer norm -----------------------------------------------------------------------------------------------------------

def forward(x, gamma, beta, eps, code, mask, residual):
    """(y, mean, rstd) of float64 tensors."""
    x = V(x)
    n = x.v.shape[-1]
    mean = x.mean()
    d = x - mean
    # the sum of squares taken around the rounded mean: its shift adds (error of the mean)^2, below first order, but for
    # rows without spread it is all there is
    var = (d * d).mean()
    var = V(var.v, var.e + mean.e ** 2)
    s = var + eps
    rstd = V(s.v ** -0.5, 0.5 * s.v ** -1.5 * s.e + 4 * U * s.v ** -0.5)
    u = d * rstd * gamma + beta
    y = act(u, code, 0)
    y = y * V(mask, U * mask) if mask is not None else y
    if residual is not None:
        y = y + residual
    return y, mean, rstd


def parts(x, gy, mean, rstd, gamma, beta, code, mask):
    """What both backward passes share, given the statistics the forward pass left: exact operands, or Vs."""
    xh = (V(x) - mean) * rstd
    u = xh * gamma + beta
    g = V(gy) * V(mask, U * mask) if mask is not None else V(gy)
    g1 = g * act(u, code, 1)
    return xh, u, g, g1, g1 * gamma


def backward(x, gy, mean, rstd, gamma, beta, code, mask):
    xh, u, g, g1, a = parts(x, gy, mean, rstd, gamma, beta, code, mask)
    dx = (a - a.mean() - xh * (a * xh).mean()) * rstd
    return dx, (g1 * xh).colsum(), g1.colsum()


def backward2(ggx, x, gy, mean, rstd, gamma, beta, code, mask):
    xh, u, g, g1, a = parts(x, gy, mean, rstd, gamma, beta, code, mask)
    v = V(ggx)
    am, ax, vm, vx = a.mean(), (a * xh).mean(), v.mean(), (v * xh).mean()
    s = (v * a).mean() - vm * am - vx * ax
    t = (v - vm - xh * vx) * rstd
    ggy = act(u, code, 1) * gamma * t
    ggy = ggy * V(mask, U * mask) if mask is not None else ggy
    q = g * act(u, code, 2) * gamma * t
    qg = q * gamma
    h = qg - (v * ax + a * vx) * rstd
    # the means of h and h xhat from those of their parts (mean xhat = 0 and mean xhat^2 = 1 are not used)
    hm = qg.mean() - (vm * ax + am * vx) * rstd
    hx = (qg * xh).mean() - vx * ax * rstd * 2.0
    gx = (h - hm - xh * hx) * rstd - s * rstd * rstd * xh
    return ggy, gx, (g1 * t + q * xh).colsum(), q.colsum()


def second(ggx, x, gy, mean, rstd, gamma, beta, code, mask, derivatives=None):
    """:func:`backward2` with every product taken around its means, so that the bounds grow with the operands' offsets and not
    with their square.  ``derivatives``: act'(u) and act''(u) in place of those of ``code``."""
    xh = (V(x) - mean) * rstd
    u = xh * gamma + beta
    m = V(mask, U * mask) if mask is not None else None
    g = V(gy) * m if mask is not None else V(gy)
    d1, d2 = derivatives or (act(u, code, 1), act(u, code, 2))
    g1 = g * d1
    a, v = g1 * gamma, V(ggx)
    am, ax, vm, vx = a.mean(), (a * xh).mean(), v.mean(), (v * xh).mean()
    ac, w = a - am, v - vm - xh * vx
    s = (w * ac).mean()
    t = w * rstd
    ggy = d1 * gamma * t
    ggy = ggy * m if mask is not None else ggy
    q = g * d2 * gamma * t
    qg = q * gamma
    # h - mean h - xh mean(h xh) with h = q gamma - rstd (v A + a B) written in w and in a around its mean
    gx = (qg - qg.mean() - xh * (qg * xh).mean()) * rstd - (w * ax + ac * vx - xh * (ax * vx)) * rstd * rstd - s * rstd * rstd * xh
    return ggy, gx, (g1 * t + q * xh).colsum(), q.colsum()


def first(x, gy, mean, rstd, gamma, d1):
    """:func:`backward` for a given act'(u)."""
    xh = (V(x) - mean) * rstd
    g1 = V(gy) * d1
    a = g1 * gamma
    return (a - a.mean() - xh * (a * xh).mean()) * rstd, (g1 * xh).colsum(), g1.colsum()
