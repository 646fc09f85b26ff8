"""The measured cases of the training-step operators: dropout without a stored
mask, layer norm with its backward pass (alone and behind dropout and a residual
add), and the linear layer on microscaled 4-bit floating-point operands.

Plain forms (``own`` false) are elementary torch operations in float32; with
``own`` true the same passes go through the package's public functions.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-5


def _actcomp():
    path = os.path.join(os.getcwd(), "triton-kernel-test_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import actcomp

    return actcomp


# ---------------------------------------------------------------------- the cases
def listed():
    return [
        # an odd-sized activation of a small float32 model under attention dropout rates
        {"name": "dropout f32 1023x1155", "op": "dropout", "rows": 1023, "cols": 1155, "dtype": "f32", "p": 0.5},
        # a long batch's hidden states: one call moves 1.3 GB
        {"name": "dropout bf16 32768x5120", "op": "dropout", "rows": 32768, "cols": 5120, "dtype": "bf16", "p": 0.1},
        # single tokens of eight sequences being served: latency
        {"name": "ln fwd bf16 8x4096", "op": "ln_fwd", "rows": 8, "cols": 4096, "dtype": "bf16", "wide": False},
        # a training batch's hidden states
        {"name": "ln fwd bf16 16384x4096", "op": "ln_fwd", "rows": 16384, "cols": 4096, "dtype": "bf16", "wide": False},
        # odd rows and channels, half precision with float32 weights
        {"name": "ln bwd f16 2049x1001", "op": "ln_bwd", "rows": 2049, "cols": 1001, "dtype": "f16", "wide": True},
        # a training batch's gradient
        {"name": "ln bwd bf16 16384x4096", "op": "ln_bwd", "rows": 16384, "cols": 4096, "dtype": "bf16", "wide": False},
        # the end of a residual branch and the next block's norm, forward
        {"name": "branch fwd bf16 16384x4096", "op": "branch_fwd", "rows": 16384, "cols": 4096, "dtype": "bf16",
         "p": 0.1},
        # the same place on the way back, with the residual stream's own gradient
        {"name": "branch bwd bf16 8192x5120", "op": "branch_bwd", "rows": 8192, "cols": 5120, "dtype": "bf16",
         "p": 0.1},
        # a saved activation stored in 4 bits and read back
        {"name": "mx4 round trip 16384x11008", "op": "mx4_trip", "rows": 16384, "cols": 11008, "dtype": "bf16",
         "turn": False},
        # the same by columns, sizes that end inside a block of 32
        {"name": "mx4 columns 2050x1338", "op": "mx4_trip", "rows": 2050, "cols": 1338, "dtype": "bf16", "turn": True},
        # one token through a projection: latency and the weight's bytes
        {"name": "mx4 linear 1 token", "op": "mx4_linear", "tokens": 1, "k": 4096, "n": 11008, "dtype": "bf16"},
        # a training step of the projection: output, input gradient, weight gradient
        {"name": "mx4 step 16384 tokens", "op": "mx4_step", "tokens": 16384, "k": 4096, "n": 11008, "dtype": "bf16"},
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi], often odd; sometimes rounded to a multiple of 8 or 64 as model widths are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    m = rng.choice([1, 1, 8, 64])
    return min(hi, max(lo, -(-v // m) * m))


def draw(rng):
    op = rng.choice(["dropout", "ln_fwd", "ln_bwd", "branch_fwd", "branch_bwd", "mx4_trip", "mx4_linear", "mx4_step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("mx4_linear", "mx4_step"):
        dtype = rng.choice(["bf16", "f16"])
        while True:
            t, k, n = _size(rng, 1 if op == "mx4_linear" else 64, 16384), _size(rng, 64, 16384), _size(rng, 64, 16384)
            if 1 << 18 <= t * k * n <= (1 << 38 if op == "mx4_step" else 1 << 39):
                return {"op": op, "tokens": t, "k": k, "n": n, "dtype": dtype}
    while True:
        rows, cols = _size(rng, 1, 65536), _size(rng, 16, 20000)
        if 1 << 10 <= rows * cols <= 1 << 26:
            break
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
    if op in ("dropout", "branch_fwd", "branch_bwd"):
        case["p"] = rng.choice([0.0, 0.05, 0.1, 0.2, 0.5, round(rng.uniform(0, 0.95), 3)])
    if op in ("ln_fwd", "ln_bwd"):
        case["wide"] = rng.random() < 0.4
    if op == "mx4_trip":
        case["turn"] = rng.random() < 0.5
    return case


def work(case):
    op, s = case["op"], 4 if case["dtype"] == "f32" else 2
    if op.startswith("mx4_") and op != "mx4_trip":
        t, k, n = case["tokens"], case["k"], case["n"]
        q = 17 / 32  # bytes of a 4-bit value with its share of a block's scale
        if op == "mx4_linear":
            return {"bytes": s * t * k + q * n * k + s * t * n, "flops": 2 * t * k * n}
        # x, dy in; both layouts of the weight in; y, dx, dw out
        return {"bytes": s * (t * k + t * n) + 2 * q * n * k + s * (t * n + t * k + n * k), "flops": 6 * t * k * n}
    rows, cols = case["rows"], case["cols"]
    e = rows * cols
    if op == "dropout":
        return {"bytes": 2 * s * e, "flops": e}
    if op == "mx4_trip":  # x in, 4-bit values out, values out
        return {"bytes": 2 * s * e + 17 / 32 * e, "flops": 2 * e}
    v = (4 if case.get("wide") else s) * cols
    if op == "ln_fwd":
        return {"bytes": 2 * s * e + 2 * v + 8 * rows, "flops": 8 * e}
    if op == "ln_bwd":
        return {"bytes": 3 * s * e + 3 * v + 8 * rows, "flops": 14 * e}
    if op == "branch_fwd":
        return {"bytes": 4 * s * e + 2 * v + 8 * rows, "flops": 10 * e}
    return {"bytes": 5 * s * e + 3 * v + 8 * rows, "flops": 16 * e}


# ---------------------------------------------------------------------- inputs
def _hidden(rows, cols, gen):
    """Hidden states: unit normal with a row level and a few channels of much larger spread, in float32."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x += 0.3 * torch.randn(rows, 1, generator=gen, device="cuda")
    big = torch.rand(cols, generator=gen, device="cuda") < 0.004
    return x * torch.where(big, 20.0, 1.0)


def _inputs(case, seed):
    """What both forms and the 64-bit one are given."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]
    rand = random.Random(seed)
    s = {"case": dict(case), "seed": rand.getrandbits(63), "row_offset": rand.getrandbits(20)}
    if op in ("mx4_linear", "mx4_step"):
        t, k, n = case["tokens"], case["k"], case["n"]
        s["x"] = _hidden(t, k, gen).to(dt)
        s["w"] = (torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)).to(dt)
        if op == "mx4_step":
            s["dy"] = (0.01 * torch.randn(t, n, generator=gen, device="cuda")).to(dt)
        return s
    rows, cols = case["rows"], case["cols"]
    x = _hidden(rows, cols, gen)
    s["x"] = x.to(dt)
    if op in ("dropout", "mx4_trip"):
        return s
    wt = torch.float32 if case.get("wide") else dt
    s["w"] = (1 + 0.2 * torch.randn(cols, generator=gen, device="cuda")).to(wt)
    s["b"] = (0.1 * torch.randn(cols, generator=gen, device="cuda")).to(wt)
    if op == "branch_fwd":
        s["residual"] = _hidden(rows, cols, gen).to(dt)
    if op in ("ln_bwd", "branch_bwd"):
        xs = s["x"].float()
        s["mean"] = xs.mean(1)
        s["rstd"] = torch.rsqrt((xs - s["mean"][:, None]).square().mean(1) + EPS)
        s["dy"] = torch.randn(rows, cols, generator=gen, device="cuda").to(dt)
    if op == "branch_bwd":
        s["dh"] = torch.randn(rows, cols, generator=gen, device="cuda").to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("mx4_linear", "mx4_step"):  # the weight is kept in the form that the products read
        w = s.pop("w")
        if own:
            mx4 = _actcomp().mx4
            if case["op"] == "mx4_step":
                s["wq"], s["wtq"] = mx4.quantize_pair(w)
            else:
                s["wq"] = mx4.quantize(w)
        else:
            s["wq"] = _plain_mx4(w.float())
            if case["op"] == "mx4_step":
                s["wtq"] = _plain_mx4(w.float().t())
    return s


# ---------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    A, op, case = _actcomp(), s["case"]["op"], s["case"]
    if op == "dropout":
        return A.dropout(s["x"], case["p"], s["seed"], s["row_offset"])
    if op == "ln_fwd":
        return A.layer_norm(s["x"], s["w"], s["b"], EPS)
    if op == "ln_bwd":
        return A.layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"])
    if op == "branch_fwd":
        return A.dropout_add_layer_norm(s["x"], s["residual"], s["w"], s["b"], case["p"], s["seed"], s["row_offset"],
                                        EPS)
    if op == "branch_bwd":
        return A.dropout_add_layer_norm_backward(s["dy"], s["x"], s["w"], s["mean"], s["rstd"], case["p"], s["seed"],
                                                 s["row_offset"], dh=s["dh"])
    if op == "mx4_trip":
        return A.mx4.dequantize(A.mx4.quantize(s["x"], transpose=case["turn"]), s["x"].dtype)
    if op == "mx4_linear":
        return A.mx4.linear(s["x"], s["wq"])
    y, saved = A.mx4.linear_forward(s["x"], s["wq"])
    return (y,) + A.mx4.linear_backward(s["dy"], saved, s["wtq"])


def _plain_keep(s, rows, cols, p):
    """The dropout mask: Philox4x32-10 (Salmon et al., 2011) at counter (column / 8, 0, row), keyed by the seed; a
    value's 16-bit half of the result against round(p 2^16)."""
    m32 = 0xFFFFFFFF
    row = torch.arange(rows, device="cuda", dtype=torch.int64)[:, None] + s["row_offset"]
    blk = torch.arange((cols + 7) // 8, device="cuda", dtype=torch.int64)[None, :]
    c0, c1 = blk.expand(rows, -1), torch.zeros_like(blk)
    c2, c3 = row & m32, (row >> 32) & m32
    k0, k1 = s["seed"] & m32, (s["seed"] >> 32) & m32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products, modulo 2^64
        c0, c1, c2, c3 = ((b >> 32) & m32) ^ c1 ^ k0, b & m32, ((a >> 32) & m32) ^ c3 ^ k1, a & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    words = torch.stack([w.expand(rows, blk.shape[1]) for w in (c0, c1, c2, c3)], -1)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, -1)[:, :cols]
    return halves >= round(p * 65536)


def _plain_scale(p):
    t = round(p * 65536)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def _plain_mx4(v):
    """Rows of float32 values as the microscaled 4-bit format holds them."""
    rows, cols = v.shape
    b = torch.nn.functional.pad(v, (0, -cols % 32)).reshape(rows, -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = ((amax.view(torch.int32) >> 23) - 127 - 2).clamp_min(-127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    a = torch.ldexp(b.abs(), -e)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = ((a / step).round() * step).clamp_max(6.0)
    q = torch.ldexp(torch.where(b < 0, -q, q), e)
    q = torch.where(torch.isfinite(amax), q, torch.full_like(q, float("nan")))
    return q.reshape(rows, -1)[:, :cols].contiguous()


def _run_plain(s):
    op, case = s["case"]["op"], s["case"]
    dt = DTYPES[case["dtype"]]
    x = s["x"].float()
    if op == "dropout":
        keep = _plain_keep(s, case["rows"], case["cols"], case["p"])
        return torch.where(keep, x * _plain_scale(case["p"]), 0.0).to(dt)
    if op == "mx4_trip":
        return _plain_mx4(x.t() if case["turn"] else x).to(dt)
    if op == "mx4_linear":
        return (_plain_mx4(x) @ s["wq"].t()).to(dt)
    if op == "mx4_step":
        dy = s["dy"].float()
        y = (_plain_mx4(x) @ s["wq"].t()).to(dt)
        dx = (_plain_mx4(dy) @ s["wtq"].t()).to(dt)
        dw = (_plain_mx4(dy.t()) @ _plain_mx4(x.t()).t()).to(dt)
        return y, dx, dw
    w, b = s["w"].float(), s["b"].float()
    if op in ("ln_fwd", "branch_fwd"):
        if op == "branch_fwd":
            keep = _plain_keep(s, case["rows"], case["cols"], case["p"])
            x = s["residual"].float() + torch.where(keep, x * _plain_scale(case["p"]), 0.0)
        mean = x.mean(1)
        xc = x - mean[:, None]
        rstd = 1 / torch.sqrt(xc.square().mean(1) + EPS)
        y = (xc * rstd[:, None] * w + b).to(dt)
        return (y, x.to(dt), mean, rstd) if op == "branch_fwd" else (y, mean, rstd)
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh = (x - s["mean"][:, None]) * rstd
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    dw, db = (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)
    if op == "ln_bwd":
        return dx.to(dt), dw, db
    dr = dx + s["dh"].float()
    keep = _plain_keep(s, case["rows"], case["cols"], case["p"])
    return torch.where(keep, dr * _plain_scale(case["p"]), 0.0).to(dt), dr.to(dt), dw, db


# ---------------------------------------------------------------------- the definition in 64 bits
def _exact_keep(s, rows, cols, p):
    """The mask again, its 32 x 32-bit products from 16-bit pieces."""
    def mulhilo(m, v):
        mh, ml, vh, vl = m >> 16, m & 0xFFFF, v >> 16, v & 0xFFFF
        ll, lh, hl, hh = ml * vl, ml * vh, mh * vl, mh * vh
        mid = (ll >> 16) + (lh & 0xFFFF) + (hl & 0xFFFF)
        return hh + (lh >> 16) + (hl >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (ll & 0xFFFF)

    nb, full = (cols + 7) // 8, 2 ** 32
    ctr = [torch.zeros(rows, nb, dtype=torch.int64, device="cuda") for _ in range(4)]
    ctr[0] += torch.arange(nb, device="cuda")
    r = s["row_offset"] + torch.arange(rows, device="cuda")
    ctr[2] += (r % full)[:, None]
    ctr[3] += (r // full)[:, None]
    key = [s["seed"] % full, s["seed"] // full]
    for i in range(10):
        h0, l0 = mulhilo(0xD2511F53, ctr[0])
        h1, l1 = mulhilo(0xCD9E8D57, ctr[2])
        ka, kb = (key[0] + i * 0x9E3779B9) % full, (key[1] + i * 0xBB67AE85) % full
        ctr = [h1 ^ ctr[1] ^ ka, l1, h0 ^ ctr[3] ^ kb, l0]
    keep = torch.empty(rows, nb, 8, dtype=torch.bool, device="cuda")
    t = math.floor(p * 65536 + 0.5) if (p * 65536) % 1 != 0.5 else round(p * 65536)
    for j in range(8):
        keep[:, :, j] = ((ctr[j // 2] >> (16 * (j % 2))) % 65536) >= t
    return keep.reshape(rows, nb * 8)[:, :cols], (0.0 if t == 65536 else 1.0 / (1.0 - t / 65536))


def _exact_mx4(v):
    """Rows of float64 values: exponents from frexp, codes by counting the midpoints that a value is past."""
    rows, cols = v.shape
    pad = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device="cuda")
    pad[:, :cols] = v
    b = pad.view(rows, -1, 32)
    amax = b.abs().max(-1, keepdim=True).values
    e = torch.frexp(amax).exponent.to(torch.int64) - 3  # floor(log2) - 2
    e = torch.where(amax > 0, e, -127).clamp_min(-127).to(torch.float64)
    a = b.abs() * torch.exp2(-e)
    q = torch.zeros_like(a)
    value = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    for i in range(7):  # from value[i] to value[i + 1]: past the midpoint, or on it where value[i + 1] is the even one
        mid = (value[i] + value[i + 1]) / 2
        past = a >= mid if i % 2 else a > mid
        q += torch.where(past, value[i + 1] - value[i], 0.0)
    q = torch.copysign(q, b) * torch.exp2(e)
    q = q.masked_fill(~torch.isfinite(amax), float("nan"))
    return q.reshape(rows, -1)[:, :cols]


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    x = s["x"].double()
    if op == "dropout":
        keep, scale = _exact_keep(s, *x.shape, case["p"])
        return (x * scale).masked_fill(~keep, 0.0)
    if op == "mx4_trip":
        return _exact_mx4(x.t() if case["turn"] else x)
    if op == "mx4_linear":
        return torch.einsum("tk,nk->tn", _exact_mx4(x), _exact_mx4(s["w"].double()))
    if op == "mx4_step":
        w, dy = s["w"].double(), s["dy"].double()
        return (torch.einsum("tk,nk->tn", _exact_mx4(x), _exact_mx4(w)),
                torch.einsum("tn,kn->tk", _exact_mx4(dy), _exact_mx4(w.t())),
                torch.einsum("nt,kt->nk", _exact_mx4(dy.t()), _exact_mx4(x.t())))
    w, b, n = s["w"].double(), s["b"].double(), x.shape[1]
    if op in ("ln_fwd", "branch_fwd"):
        if op == "branch_fwd":
            keep, scale = _exact_keep(s, *x.shape, case["p"])
            x = (x * scale).masked_fill(~keep, 0.0) + s["residual"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + EPS).rsqrt()
        y = torch.addcmul(b, (x - mean[:, None]) * rstd[:, None], w)
        return (y, x, mean, rstd) if op == "branch_fwd" else (y, mean, rstd)
    mean, rstd, dy = s["mean"].double(), s["rstd"].double(), s["dy"].double()
    xh = rstd[:, None] * (x - mean[:, None])
    s1 = dy @ w / n
    s2 = (dy * xh) @ w / n
    dx = rstd[:, None] * (dy * w - s1[:, None] - xh * s2[:, None])
    dw, db = torch.einsum("rc,rc->c", dy, xh), dy.sum(0)
    if op == "ln_bwd":
        return dx, dw, db
    dr = s["dh"].double() + dx
    keep, scale = _exact_keep(s, *x.shape, case["p"])
    return (dr * scale).masked_fill(~keep, 0.0), dr, dw, db
