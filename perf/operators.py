"""Timed cases of the layer norm (forward, backward, backward of the backward) and the counter-based dropout.

A case names the direction (``op``), the matrix (``rows`` x ``cols``: the norm runs over ``cols``), the element type and
the fused epilogue: ``act`` (the activation code's name), ``p`` (dropout), ``residual``, ``pad`` (extra elements per row of
the input tensors, i.e. rows cut out of a wider tensor).  ``run`` computes the plain form unless ``own`` is set.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SLOPES = {"none": 1.0, "relu": 0.0, "lrelu": 0.01, "silu": 2.0, "mish": 3.0}      # the framework's activation codes


def _case(name, op, rows, cols, dtype, act="none", p=0.0, residual=False, pad=0):
    return dict(name=name, op=op, rows=rows, cols=cols, dtype=dtype, act=act, p=p, residual=residual, pad=pad)


# The leaky activations' slope is a step at u = 0, where either side is a right answer for a u within a rounding of zero:
# the forward cases take them (the value is continuous there), the gradient cases take smooth ones or none.
def listed():
    return [
        # one row of a wide model: what a call costs when there is nothing to do
        _case("fwd one row", "fwd", 1, 4096, "bf16"),
        # the critic's first layer, 16 images of 128 x 128 (64 x 64 pixels of 64 channels), leaky activation, dropout
        _case("fwd critic first layer", "fwd", 65536, 64, "f32", act="lrelu", p=0.25),
        # a wide block: norm, dropout, residual in one pass over 256 MB
        _case("fwd wide", "fwd", 16384, 8192, "bf16", p=0.1, residual=True),
        # odd width, odd row count, rows cut out of a wider tensor
        _case("fwd ragged", "fwd", 4099, 1001, "f16", act="silu", pad=23),
        # the critic's last layer, 16 images (2 x 2 pixels of 2048 channels): few rows, latency
        _case("bwd critic last layer", "bwd", 64, 2048, "f32", act="silu", p=0.25),
        # a wide block's gradient
        _case("bwd wide", "bwd", 16384, 8192, "bf16", p=0.1),
        _case("bwd ragged", "bwd", 3001, 1537, "f16", act="silu", pad=7),
        # the gradient penalty's second backward: the critic's first layer, and a block of ordinary width
        _case("bwd2 critic first layer", "bwd2", 65536, 64, "f32", act="mish"),
        _case("bwd2 block", "bwd2", 4096, 4096, "bf16", act="silu", p=0.1),
        # dropout by itself: in front of a head, over odd rows of a wider tensor, over 256 MB with the residual add
        _case("dropout head", "dropout", 16, 2048, "f32", p=0.5),
        _case("dropout ragged", "dropout", 1003, 4097, "f16", p=0.3, pad=3),
        _case("dropout wide", "dropout", 16384, 8192, "bf16", p=0.1, residual=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    op = rng.choice(["fwd", "bwd", "bwd2", "dropout"])
    cols = log_int(16, 8192)
    most = {"fwd": 1 << 27, "bwd": 1 << 27, "bwd2": 1 << 24, "dropout": 1 << 27}[op]
    rows = log_int(1, max(1, min(65536, most // cols)))
    if rng.random() < 0.3:                      # ordinary models have even widths
        cols = max(16, cols // 16 * 16)
    smooth = ["none", "none", "silu", "mish"]
    act = "none" if op == "dropout" else rng.choice(smooth + ["relu", "lrelu"] if op == "fwd" else smooth)
    p = rng.uniform(0.05, 0.6) if op == "dropout" or rng.random() < 0.5 else 0.0
    residual = op in ("fwd", "dropout") and rng.random() < 0.4
    pad = rng.choice([0, 0, 0, rng.randint(1, 64)])
    return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["f32", "bf16", "f16"]), act=act, p=p, residual=residual,
                pad=pad)


def work(case):
    n, c = case["rows"] * case["cols"], case["cols"]
    e = 4 if case["dtype"] == "f32" else 2
    op = case["op"]
    tensors = {"fwd": 2, "bwd": 3, "bwd2": 5, "dropout": 2}[op] + bool(case["residual"])
    params = {"fwd": 2, "bwd": 3 if case["act"] == "none" else 4, "bwd2": 3 if case["act"] == "none" else 4, "dropout": 0}[op]
    stats = 0 if op == "dropout" else 8 * case["rows"]
    flops = {"fwd": 8, "bwd": 16, "bwd2": 35, "dropout": 1}[op] + (2 if case["p"] and op != "dropout" else 0)
    return {"bytes": n * e * tensors + 4 * c * params + stats, "flops": n * flops}


def _wide(case, gen, scale, shift, dev):
    """rows x cols with ``pad`` more elements between the rows."""
    r, c, pad = case["rows"], case["cols"], case["pad"]
    t = torch.empty((r, c + pad), dtype=TYPES[case["dtype"]], device=dev)
    step = max(1, (1 << 26) // (c + pad))
    for i in range(0, r, step):                 # in pieces: no second copy in 32 bits of a large matrix
        k = min(step, r - i)
        t[i:i + k] = torch.randn((k, c + pad), generator=gen, device=dev) * scale + shift
    return t[:, :c]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c = case["cols"]
    st = {"case": case}
    st["x"] = _wide(case, gen, 1.5, 0.4, dev)
    if case["op"] != "dropout":
        st["gamma"] = 1.0 + 0.2 * torch.randn(c, generator=gen, device=dev)
        st["beta"] = 0.2 * torch.randn(c, generator=gen, device=dev)
    if case["residual"]:
        st["residual"] = _wide(case, gen, 1.0, 0.0, dev)
    if case["op"] in ("bwd", "bwd2"):
        st["gy"] = _wide(case, gen, 1.0, 0.0, dev)
        # what the forward pass left
        mean = torch.empty(case["rows"], device=dev)
        rstd = torch.empty(case["rows"], device=dev)
        step = max(1, (1 << 25) // c)
        for i in range(0, case["rows"], step):
            xd = st["x"][i:i + step].double()
            mean[i:i + step] = xd.mean(1)
            rstd[i:i + step] = (xd.var(1, unbiased=False) + EPS).rsqrt()
        st["mean"], st["rstd"] = mean, rstd
    if case["op"] == "bwd2":
        st["ggx"] = _wide(case, gen, 1.0, 0.0, dev)
    # dropout's seed and first block: beyond 32 bits, as after a long run
    st["rng"] = (0x1234567 * (seed + 1) & (2**63 - 1), (1 << 33) + 977 * seed)
    return st


# ---- the plain form ---------------------------------------------------------------------------------------------------

M32 = 0xFFFFFFFF


def _mask(rows, cols, p, rng, dev):
    """Scaled keep mask (fp32): element i takes 16 bits of block ``offset + i // 8`` of Philox4x32-10 (Salmon, Moraes, Dror,
    Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011) and is dropped where they are below ``65536 p``."""
    seed, offset = rng
    total = rows * cols
    ctr = torch.arange((total + 7) // 8, device=dev) + offset
    c = [ctr & M32, (ctr >> 32) & M32, torch.zeros_like(ctr), torch.zeros_like(ctr)]
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & M32) ^ c[1] ^ k0, p1 & M32, ((p0 >> 32) & M32) ^ c[3] ^ k1, p0 & M32]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    bits = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], 1).to(torch.int32).view(-1)[:total]
    t = round(p * 65536)
    scale = 65536.0 / (65536 - t) if t < 65536 else 0.0
    return ((bits >= t).float() * scale).view(rows, cols)


def _act(u, name, order):
    """The activation (order 0) or its first / second derivative at ``u``."""
    if name == "none":
        return u if order == 0 else torch.full_like(u, 1.0 if order == 1 else 0.0)
    if name in ("relu", "lrelu"):
        s = torch.where(u > 0, 1.0, SLOPES[name]).to(u.dtype)
        return u * s if order == 0 else (s if order == 1 else torch.zeros_like(u))
    sg = 1 / (1 + torch.exp(-u))
    if name == "silu":
        return [lambda: u * sg, lambda: sg * (1 + u * (1 - sg)), lambda: sg * (1 - sg) * (2 + u * (1 - 2 * sg))][order]()
    th = torch.tanh(torch.where(u > 20, u, torch.log1p(torch.exp(u.clamp(max=20)))))
    w = (1 - th * th) * sg
    return [lambda: u * th, lambda: th + u * w, lambda: 2 * w + u * w * ((1 - sg) - 2 * th * sg)][order]()


def _plain(st):
    case = st["case"]
    op, p, act = case["op"], case["p"], case["act"]
    dt = TYPES[case["dtype"]]
    x = st["x"].float()
    m = _mask(case["rows"], case["cols"], p, st["rng"], x.device) if p else 1.0
    if op == "dropout":
        y = x * m
        return (y + st["residual"].float() if case["residual"] else y).to(dt)
    gamma, beta = st["gamma"], st["beta"]
    if op == "fwd":
        mean = x.mean(1, keepdim=True)
        xc = x - mean
        rstd = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
        y = _act(xc * rstd * gamma + beta, act, 0) * m
        if case["residual"]:
            y = y + st["residual"].float()
        return y.to(dt), mean[:, 0], rstd[:, 0]
    r = st["rstd"][:, None]
    xh = (x - st["mean"][:, None]) * r
    u = xh * gamma + beta
    gy = st["gy"].float() * m
    g1 = gy * _act(u, act, 1)
    a = g1 * gamma
    bm, bx = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    if op == "bwd":
        dx = r * (a - bm - xh * bx)
        return dx.to(dt), (g1 * xh).sum(0), g1.sum(0)
    v = st["ggx"].float()
    vm, vx = v.mean(1, keepdim=True), (v * xh).mean(1, keepdim=True)
    s = (v * a).mean(1, keepdim=True) - vm * bm - vx * bx
    t = r * (v - vm - xh * vx)
    ggy = _act(u, act, 1) * gamma * t * m
    q = gy * _act(u, act, 2) * gamma * t
    h = q * gamma - r * (v * bx + a * vx)
    gx = r * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True)) - s * r * r * xh
    return ggy.to(dt), gx.to(dt), (g1 * t + q * xh).sum(0), q.sum(0)


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _own(st):
    from fcd_amd import ops
    case = st["case"]
    if case["op"] == "dropout":
        return ops.dropout(st["x"], case["p"], st["rng"], residual=st.get("residual"))
    kw = dict(act_slope=SLOPES[case["act"]], p=case["p"], rng=st["rng"] if case["p"] else None)
    if case["op"] == "fwd":
        return ops.layernorm_fwd(st["x"], st["gamma"], st["beta"], eps=EPS, residual=st.get("residual"), **kw)
    if case["op"] == "bwd":
        return ops.layernorm_bwd(st["gy"], st["x"], st["mean"], st["rstd"], st["gamma"], st["beta"], **kw)
    return ops.layernorm_bwd2(st["ggx"], st["gy"], st["x"], st["mean"], st["rstd"], st["gamma"], st["beta"], **kw)


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def _exact_mask(rows, cols, p, rng):
    """The generator again, on the host: 64-bit unsigned products, one 32-bit word of the block at a time."""
    total = rows * cols
    out = np.empty(total, np.float64)
    t = int(np.rint(p * 65536))
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    with np.errstate(over="ignore"):
        for lo in range(0, (total + 7) // 8, 1 << 20):
            hi = min((total + 7) // 8, lo + (1 << 20))
            n = np.arange(lo, hi, dtype=np.uint64) + np.uint64(rng[1])
            w = np.stack([n.astype(np.uint32), (n >> np.uint64(32)).astype(np.uint32), np.zeros_like(n, np.uint32),
                          np.zeros_like(n, np.uint32)])
            key = np.array([rng[0] & M32, rng[0] >> 32], np.uint32)
            for _ in range(10):
                left = w[0].astype(np.uint64) * np.uint64(0xD2511F53)
                right = w[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
                w = np.stack([(right >> np.uint64(32)).astype(np.uint32) ^ w[1] ^ key[0], right.astype(np.uint32),
                              (left >> np.uint64(32)).astype(np.uint32) ^ w[3] ^ key[1], left.astype(np.uint32)])
                key = key + np.array([0x9E3779B9, 0xBB67AE85], np.uint32)
            half = np.ascontiguousarray(w.T).view(np.uint16).reshape(-1)        # little endian: low half first
            part = out[lo * 8:hi * 8]
            part[:] = np.where(half[:part.size] < t, 0.0, scale)
    return torch.from_numpy(out).view(rows, cols)


def exact(case, seed):
    st = prepare(case, seed)
    f = {"none": lambda u: u, "relu": lambda u: torch.clamp(u, min=0), "lrelu": lambda u: torch.where(u > 0, u, 0.01 * u),
         "silu": lambda u: u * torch.sigmoid(u), "mish": lambda u: u * torch.tanh(torch.log1p(torch.exp(u)))}[case["act"]]
    rows, op = case["rows"], case["op"]
    keep = _exact_mask(rows, case["cols"], case["p"], st["rng"]) if case["p"] else None
    outs, sums = [], None
    step = max(1, (1 << 24) // case["cols"])
    for i in range(0, rows, step):
        x = st["x"][i:i + step].double()
        m = 1.0 if keep is None else keep[i:i + step].to(x.device)
        res = st["residual"][i:i + step].double() if case["residual"] else 0.0
        if op == "dropout":
            outs.append((x * m + res,))
            continue
        grads = op != "fwd"
        x.requires_grad_(grads)
        gamma = st["gamma"].double().requires_grad_(grads)
        beta = st["beta"].double().requires_grad_(grads)
        mean = x.mean(1, keepdim=True)
        rstd = ((x - mean) ** 2).mean(1, keepdim=True).add(EPS) ** -0.5
        y = f((x - mean) * rstd * gamma + beta) * m
        if op == "fwd":
            outs.append((y + res, mean[:, 0], rstd[:, 0]))
            continue
        gy = st["gy"][i:i + step].double()
        if op == "bwd":
            dx, dg, db = torch.autograd.grad(y, (x, gamma, beta), gy)
            outs.append((dx,))
        else:
            gy.requires_grad_(True)
            dx, = torch.autograd.grad(y, (x,), gy, create_graph=True)
            v = st["ggx"][i:i + step].double()
            ggy, gx, dg, db = torch.autograd.grad(dx, (gy, x, gamma, beta), v, allow_unused=True)
            outs.append((ggy, gx))
            db = torch.zeros_like(beta) if db is None else db
        sums = (dg, db) if sums is None else (sums[0] + dg, sums[1] + db)
        del y, x
    whole = tuple(torch.cat(parts).detach() for parts in zip(*outs))
    if op == "dropout":
        return whole[0]
    return whole + tuple(t.detach() for t in sums) if sums is not None else whole
