"""The measured cases of the operators at a model's ends and between its 8-bit
linear layers: root-mean-square norm with the residual's addition (forward,
backward, and with an 8-bit output), 8-bit floating point with a scale per block
of 128 (quantisation, linear layer, its gradients), and the cross entropy of a
linear layer over a large vocabulary, whose logits are not kept.

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
IGNORE = -100


def _actcomp():
    path = os.path.join(os.getcwd(), "triton-kernel-test_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import actcomp

    return actcomp


# ---------------------------------------------------------------------- the cases
def listed():
    return [
        # single tokens of eight sequences being served: latency
        {"name": "rms fwd bf16 8x4096", "op": "rms_fwd", "rows": 8, "cols": 4096, "dtype": "bf16", "wide": False,
         "add": False},
        # a training batch's residual stream into an 8-bit linear layer's input
        {"name": "rms add fp8 bf16 16384x4096", "op": "rms_fp8", "rows": 16384, "cols": 4096, "dtype": "bf16",
         "add": True},
        # odd rows and channels, half precision with float32 weights
        {"name": "rms bwd f16 2049x1001", "op": "rms_bwd", "rows": 2049, "cols": 1001, "dtype": "f16", "wide": True,
         "add": False},
        # a training batch's gradient, with the residual stream's own
        {"name": "rms bwd bf16 16384x4096", "op": "rms_bwd", "rows": 16384, "cols": 4096, "dtype": "bf16",
         "wide": False, "add": True},
        # a saved activation in 8 bits, by rows and by columns, read back
        {"name": "fp8 pair 16384x11008", "op": "fp8_pair", "rows": 16384, "cols": 11008, "dtype": "bf16",
         "fmt": "e4m3"},
        # a weight by tiles, sizes that end inside a tile
        {"name": "fp8 tiles f32 2050x1338", "op": "fp8_tiles", "rows": 2050, "cols": 1338, "dtype": "f32",
         "fmt": "e4m3"},
        # one token being served: the norm in 8 bits, then a projection: latency and the weight's bytes
        {"name": "fp8 norm and linear 1 token", "op": "fp8_serve", "tokens": 1, "k": 4096, "n": 11008,
         "dtype": "bf16"},
        # a batch of sequences being served, one token each
        {"name": "fp8 linear 200 tokens", "op": "fp8_linear", "tokens": 200, "k": 4096, "n": 11008, "dtype": "bf16"},
        # a training step of the projection: output, input gradient, weight gradient
        {"name": "fp8 step 16384 tokens", "op": "fp8_step", "tokens": 16384, "k": 4096, "n": 11008, "dtype": "bf16"},
        # the loss of a validation batch of a small model, an odd vocabulary
        {"name": "xent fwd f16 1000x1024x50257", "op": "xent_fwd", "tokens": 1000, "k": 1024, "vocab": 50257,
         "dtype": "f16"},
        # the gradient of a short batch, with the normaliser's own
        {"name": "xent bwd bf16 511x1024x32000", "op": "xent_bwd", "tokens": 511, "k": 1024, "vocab": 32000,
         "dtype": "bf16", "dlse": True},
        # a training batch against a large vocabulary: loss, input gradient, weight gradient
        {"name": "xent step bf16 8192x4096x128000", "op": "xent_step", "tokens": 8192, "k": 4096, "vocab": 128000,
         "dtype": "bf16", "dlse": False},
    ]


def _size(rng, lo, hi):
    """Log-uniform in [lo, hi], often odd; sometimes rounded to a multiple of 8 or 64 as model widths are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    m = rng.choice([1, 1, 8, 64])
    return min(hi, max(lo, -(-v // m) * m))


def draw(rng):
    op = rng.choice(["rms_fwd", "rms_fp8", "rms_bwd", "fp8_pair", "fp8_tiles", "fp8_serve", "fp8_linear", "fp8_step",
                     "xent_fwd", "xent_bwd", "xent_step"])
    if op.startswith("xent"):
        case = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16"])}
        while True:
            t, k, v = _size(rng, 1, 16384), _size(rng, 64, 8192), _size(rng, 1000, 200000)
            if 1 << 24 <= t * k * v <= 1 << 40:
                break
        case.update(tokens=t, k=k, vocab=v)
        if op != "xent_fwd":
            case["dlse"] = rng.random() < 0.4
        return case
    if op in ("fp8_serve", "fp8_linear", "fp8_step"):
        lo, hi = {"fp8_serve": (1, 64), "fp8_linear": (1, 16384), "fp8_step": (64, 16384)}[op]
        dtype = rng.choice(["bf16", "f16"] if op == "fp8_serve" else ["bf16", "bf16", "f16", "f32"])
        while True:
            t, k, n = _size(rng, lo, hi), _size(rng, 64, 16384), _size(rng, 64, 16384)
            if 1 << 18 <= t * k * n <= (1 << 38 if op == "fp8_step" else 1 << 39):
                return {"op": op, "tokens": t, "k": k, "n": n, "dtype": dtype}
    while True:
        rows, cols = _size(rng, 1, 65536), _size(rng, 16, 20000)
        if 1 << 10 <= rows * cols <= 1 << 26:
            break
    dtype = rng.choice(["bf16", "f16"] if op == "rms_fp8" else ["bf16", "bf16", "f16", "f32"])
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
    if op in ("rms_fwd", "rms_bwd"):
        case["wide"] = rng.random() < 0.4
    if op.startswith("rms"):
        case["add"] = rng.random() < 0.6
    else:
        case["fmt"] = rng.choice(["e4m3", "e4m3", "e5m2"])
    return case


def work(case):
    op, s = case["op"], 4 if case["dtype"] == "f32" else 2
    q = 129 / 128  # bytes of an 8-bit value with its share of a block's scale
    if op.startswith("xent"):
        t, k, v = case["tokens"], case["k"], case["vocab"]
        one = 2 * t * k * v  # the logits; each gradient is as much again
        if op == "xent_fwd":
            return {"bytes": s * (t * k + v * k) + 16 * t, "flops": one}
        more = 4 * t if case["dlse"] else 0
        if op == "xent_bwd":
            return {"bytes": 2 * s * (t * k + v * k) + 16 * t + more, "flops": 3 * one}
        return {"bytes": 2 * s * (t * k + v * k) + 20 * t + more, "flops": 3 * one}
    if op in ("fp8_serve", "fp8_linear", "fp8_step"):
        t, k, n = case["tokens"], case["k"], case["n"]
        if op == "fp8_serve":
            return {"bytes": 3 * s * t * k + s * k + 4 * t + q * n * k + s * t * n, "flops": 2 * t * k * n}
        if op == "fp8_linear":
            return {"bytes": s * t * k + q * n * k + s * t * n, "flops": 2 * t * k * n}
        return {"bytes": s * (t * k + t * n) + q * n * k + s * (t * n + t * k + n * k), "flops": 6 * t * k * n}
    rows, cols = case["rows"], case["cols"]
    e, add = rows * cols, 1 if case.get("add") else 0
    if op == "fp8_pair":  # x in, both forms' codes out, both forms' values out
        return {"bytes": 3 * s * e + 2 * q * e, "flops": 4 * e}
    if op == "fp8_tiles":
        return {"bytes": 2 * s * e + e, "flops": 2 * e}
    v = (4 if case.get("wide") else s) * cols
    if op == "rms_fwd":
        return {"bytes": (2 + 2 * add) * s * e + v + 4 * rows, "flops": 5 * e}
    if op == "rms_fp8":  # the codes, and the values that they stand for
        return {"bytes": (2 + 2 * add) * s * e + q * e + v + 4 * rows, "flops": 7 * e}
    return {"bytes": (3 + add) * s * e + 2 * v + 4 * rows, "flops": 10 * e}


# ---------------------------------------------------------------------- inputs
def _hidden(rows, cols, gen):
    """Hidden states: unit normal with a few channels of much larger spread, in float32."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    big = torch.rand(cols, generator=gen, device="cuda") < 0.004
    return x * torch.where(big, 20.0, 1.0)


def _inputs(case, seed):
    """What both forms and the 64-bit one are given."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, op = DTYPES[case["dtype"]], case["op"]
    rand = random.Random(seed)
    s = {"case": dict(case)}
    if op.startswith("xent"):
        t, k, v = case["tokens"], case["k"], case["vocab"]
        w = torch.randn(v, k, generator=gen, device="cuda") / math.sqrt(k)
        s["w"] = w.to(dt)
        s["target"] = torch.randint(0, v, (t,), generator=gen, device="cuda")
        # a model that has learned something: the target's logit is raised, by a different amount for each token
        lift = 12 * torch.rand(t, 1, generator=gen, device="cuda")
        s["x"] = (2 * torch.randn(t, k, generator=gen, device="cuda") + lift * w[s["target"]]).to(dt)
        gone = torch.rand(t, generator=gen, device="cuda") < 0.1
        gone[rand.randrange(t)] = False
        s["target"][gone] = IGNORE
        if op != "xent_fwd":
            live = (~gone).sum()
            s["dloss"] = (0.5 + torch.rand(t, generator=gen, device="cuda")) / live  # a weighted mean's gradient
            s["dlse"] = 1e-3 * torch.rand(t, generator=gen, device="cuda") / live if case["dlse"] else None
        if op == "xent_bwd":
            step = max(1, (1 << 28) // v)
            s["lse"] = torch.cat([torch.logsumexp(c.float() @ s["w"].float().t(), 1) for c in s["x"].split(step)])
        return s
    if op in ("fp8_serve", "fp8_linear", "fp8_step"):
        t, k, n = case["tokens"], case["k"], case["n"]
        s["x"] = _hidden(t, k, gen).to(dt)
        s["w"] = (torch.randn(n, k, generator=gen, device="cuda") / math.sqrt(k)).to(dt)
        if op == "fp8_serve":
            s["residual"] = _hidden(t, k, gen).to(dt)
            s["scale"] = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dt)
        if op == "fp8_step":
            s["dy"] = (0.01 * torch.randn(t, n, generator=gen, device="cuda")).to(dt)
        return s
    rows, cols = case["rows"], case["cols"]
    s["x"] = _hidden(rows, cols, gen).to(dt)
    if op.startswith("fp8"):
        return s
    wt = torch.float32 if case.get("wide") else dt
    s["w"] = (1 + 0.2 * torch.randn(cols, generator=gen, device="cuda")).to(wt)
    if op != "rms_bwd":
        s["residual"] = _hidden(rows, cols, gen).to(dt) if case["add"] else None
        return s
    s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
    s["dy"] = torch.randn(rows, cols, generator=gen, device="cuda").to(dt)
    s["dh"] = torch.randn(rows, cols, generator=gen, device="cuda").to(dt) if case["add"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("fp8_serve", "fp8_linear", "fp8_step"):  # the weight is kept in the form that the products read
        w = s.pop("w")
        if own:
            s["wq"] = _actcomp().fp8.quantize_weight(w)
        else:
            s["wq"] = _plain_fp8(w.float(), "tiles")
    return s


# ---------------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    A, op, case = _actcomp(), s["case"]["op"], s["case"]
    if op == "rms_fwd":
        if s["residual"] is None:
            return A.rms_norm(s["x"], s["w"], EPS)
        return A.add_rms_norm(s["x"], s["residual"], s["w"], EPS)
    if op == "rms_fp8":
        if s["residual"] is None:
            q, rstd = A.fp8.rms_norm(s["x"], s["w"], EPS)
            return A.fp8.dequantize(q), rstd
        q, h, rstd = A.fp8.add_rms_norm(s["x"], s["residual"], s["w"], EPS)
        return A.fp8.dequantize(q), h, rstd
    if op == "rms_bwd":
        return A.rms_norm_backward(s["dy"], s["x"], s["w"], s["rstd"], dh=s["dh"])
    if op == "fp8_pair":
        q, qt = A.fp8.quantize_pair(s["x"], format=case["fmt"])
        return A.fp8.dequantize(q), A.fp8.dequantize(qt).t()
    if op == "fp8_tiles":
        return A.fp8.dequantize(A.fp8.quantize_weight(s["x"], format=case["fmt"]))
    if op == "fp8_serve":
        q, h, rstd = A.fp8.add_rms_norm(s["x"], s["residual"], s["scale"], EPS)
        return A.fp8.matmul(q, s["wq"]), h, rstd
    if op == "fp8_linear":
        return A.fp8.linear(s["x"], s["wq"])
    if op == "fp8_step":
        y, saved = A.fp8.linear_forward(s["x"], s["wq"])
        return (y,) + A.fp8.linear_backward(s["dy"], saved, s["wq"])
    if op == "xent_fwd":
        return A.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE)
    if op == "xent_bwd":
        return A.linear_cross_entropy_backward(s["dloss"], s["x"], s["w"], s["target"], s["lse"], dlse=s["dlse"],
                                               ignore_index=IGNORE)
    loss, lse = A.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE)
    return (loss, lse) + A.linear_cross_entropy_backward(s["dloss"], s["x"], s["w"], s["target"], lse,
                                                         dlse=s["dlse"], ignore_index=IGNORE)


# mantissa bits, smallest normal exponent, largest exponent and largest value
FORMATS = {"e4m3": (3, -6, 8, 448.0), "e5m2": (2, -14, 15, 57344.0)}


def _plain_fp8(v, by, fmt="e4m3"):
    """float32 values as 8-bit floating point holds them, a power-of-two scale per 128 values of a row ("rows"), of a
    column ("cols") or per 128 x 128 ("tiles"): the smallest scale under which the block's largest magnitude fits."""
    bits, low, top, most = FORMATS[fmt]
    rows, cols = v.shape
    br, bc = (1 if by == "rows" else 128), (1 if by == "cols" else 128)
    b = torch.nn.functional.pad(v, (0, -cols % bc, 0, -rows % br))
    b = b.reshape(b.shape[0] // br, br, b.shape[1] // bc, bc)
    amax = b.abs().amax((1, 3), keepdim=True)
    word = amax.view(torch.int32)
    e = (word >> 23) - 127 - top + ((word & 0x7FFFFF) > 0x600000).int()
    e = torch.where(amax == 0, torch.full_like(e, -127), e.clamp_min(-127))
    a = torch.ldexp(b.abs(), -e)
    step = torch.ldexp(torch.ones_like(a), ((a.view(torch.int32) >> 23) - 127).clamp_min(low) - bits)
    q = ((a / step).round() * step).clamp_max(most)
    q = torch.ldexp(torch.where(b < 0, -q, q), e)
    q = torch.where(torch.isfinite(amax), q, torch.full_like(q, float("nan")))
    return q.reshape(q.shape[0] * br, -1)[:rows, :cols].contiguous()


def _plain_rms(x, residual, w):
    h = x if residual is None else x + residual
    rstd = 1 / torch.sqrt(h.square().mean(1) + EPS)
    return h * rstd[:, None] * w, h, rstd


def _plain_grads(s, z, lse, x, w):
    """dx and dw of the loss from the logits."""
    dt = s["x"].dtype
    live = s["target"] != IGNORE
    d = torch.where(live, s["dloss"], 0.0)
    a = d if s["dlse"] is None else d + s["dlse"]
    g = torch.exp(z - lse[:, None]) * a[:, None]
    rows = torch.arange(z.shape[0], device=z.device)
    g[rows, s["target"].clamp_min(0)] -= d
    return (g @ w).to(dt), (g.t() @ x).to(dt)


def _run_plain(s):
    op, case = s["case"]["op"], s["case"]
    dt = DTYPES[case["dtype"]]
    x = s["x"].float()
    if op.startswith("xent"):
        w = s["w"].float()
        z = x @ w.t()
        if op == "xent_bwd":
            return _plain_grads(s, z, s["lse"], x, w)
        top = z.amax(1)
        lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
        at = z.gather(1, s["target"].clamp_min(0)[:, None])[:, 0]
        loss = torch.where(s["target"] != IGNORE, lse - at, 0.0)
        return (loss, lse) + (_plain_grads(s, z, lse, x, w) if op == "xent_step" else ())
    if op == "fp8_pair":
        return _plain_fp8(x, "rows", case["fmt"]).to(dt), _plain_fp8(x, "cols", case["fmt"]).to(dt)
    if op == "fp8_tiles":
        return _plain_fp8(x, "tiles", case["fmt"]).to(dt)
    if op == "fp8_linear":
        return (_plain_fp8(x, "rows") @ s["wq"].t()).to(dt)
    if op == "fp8_step":
        dy = s["dy"].float()
        y = (_plain_fp8(x, "rows") @ s["wq"].t()).to(dt)
        dx = (_plain_fp8(dy, "rows") @ s["wq"]).to(dt)
        dw = (_plain_fp8(dy, "cols").t() @ _plain_fp8(x, "cols")).to(dt)
        return y, dx, dw
    if op == "fp8_serve":
        y, h, rstd = _plain_rms(x, s["residual"].float(), s["scale"].float())
        return (_plain_fp8(y, "rows") @ s["wq"].t()).to(dt), h.to(dt), rstd
    w = s["w"].float()
    if op != "rms_bwd":
        y, h, rstd = _plain_rms(x, None if s["residual"] is None else s["residual"].float(), w)
        y = _plain_fp8(y, "rows") if op == "rms_fp8" else y
        return (y.to(dt), rstd) if s["residual"] is None else (y.to(dt), h.to(dt), rstd)
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh, g = x * rstd, dy * w
    dx = rstd * (g - xh * (g * xh).mean(1, keepdim=True))
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return dx.to(dt), (dy * xh).sum(0).to(s["w"].dtype)


# ---------------------------------------------------------------------- the definition in 64 bits
def _exact_fp8(v, by, fmt="e4m3"):
    """float64 values: exponents from frexp, each value to the nearest of its binade's grid, halves to the even."""
    bits, low, top, most = FORMATS[fmt]
    if by == "cols":
        return _exact_fp8(v.t(), "rows", fmt).t()
    rows, cols = v.shape
    tall = 128 if by == "tiles" else 1
    pad = torch.zeros(-(-rows // tall) * tall, -(-cols // 128) * 128, dtype=torch.float64, device=v.device)
    pad[:rows, :cols] = v
    b = pad.view(-1, tall, pad.shape[1] // 128, 128)
    amax = b.abs().amax(dim=(1, 3), keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    e = e.to(torch.int64) - 1 - top
    e = e + (2 * m > most / 2.0 ** top).to(torch.int64)
    e = torch.where(amax > 0, e, -127).clamp_min(-127).to(torch.float64)
    a = b * torch.exp2(-e)
    grid = torch.exp2((torch.frexp(a).exponent.to(torch.float64) - 1).clamp_min(low) - bits)
    q = torch.round(a / grid) * grid * torch.exp2(e)
    q = q.masked_fill(~torch.isfinite(amax), float("nan"))
    return q.reshape(pad.shape)[:rows, :cols]


def _exact_xent(s):
    """Loss, normaliser and gradients, some tokens at a time."""
    op, t = s["case"]["op"], s["case"]["tokens"]
    w = s["w"].double()
    loss, lse, dx, dw = [], [], [], torch.zeros_like(w) if op != "xent_fwd" else None
    step = max(1, (1 << 28) // w.shape[0])
    for i in range(0, t, step):
        x, target = s["x"][i:i + step].double(), s["target"][i:i + step]
        z = torch.einsum("tk,vk->tv", x, w)
        n = torch.logsumexp(z, 1)
        gone = target == IGNORE
        hit = torch.nn.functional.one_hot(target.masked_fill(gone, 0), w.shape[0]).to(torch.float64)
        hit = hit.masked_fill(gone[:, None], 0.0)
        lse.append(n)
        loss.append((n - (z * hit).sum(1)).masked_fill(gone, 0.0))
        if op == "xent_fwd":
            continue
        at = s["lse"][i:i + step].double() if op == "xent_bwd" else n
        p = (z - at[:, None]).exp()
        d = s["dloss"][i:i + step].double().masked_fill(gone, 0.0)[:, None]
        g = (p - hit) * d
        if s["dlse"] is not None:
            g = g + p * s["dlse"][i:i + step].double()[:, None]
        dx.append(torch.einsum("tv,vk->tk", g, w))
        dw += torch.einsum("tv,tk->vk", g, x)
    if op == "xent_fwd":
        return torch.cat(loss), torch.cat(lse)
    if op == "xent_bwd":
        return torch.cat(dx), dw
    return torch.cat(loss), torch.cat(lse), torch.cat(dx), dw


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op.startswith("xent"):
        return _exact_xent(s)
    x = s["x"].double()
    if op == "fp8_pair":
        return _exact_fp8(x, "rows", case["fmt"]), _exact_fp8(x, "cols", case["fmt"])
    if op == "fp8_tiles":
        return _exact_fp8(x, "tiles", case["fmt"])
    if op == "fp8_linear":
        return torch.einsum("tk,nk->tn", _exact_fp8(x, "rows"), _exact_fp8(s["w"].double(), "tiles"))
    if op == "fp8_step":
        w, dy = _exact_fp8(s["w"].double(), "tiles"), s["dy"].double()
        return (torch.einsum("tk,nk->tn", _exact_fp8(x, "rows"), w), torch.einsum("tn,nk->tk", _exact_fp8(dy, "rows"), w),
                torch.einsum("tn,tk->nk", _exact_fp8(dy, "cols"), _exact_fp8(x, "cols")))
    n = x.shape[1]
    if op != "rms_bwd":
        if s["residual"] is not None:
            x = s["residual"].double() + x
        rstd = ((x * x).sum(1) / n + EPS).rsqrt()
        y = x * (s["scale"] if op == "fp8_serve" else s["w"]).double() * rstd[:, None]
        if op != "rms_fwd":
            y = _exact_fp8(y, "rows")
        if op == "fp8_serve":
            y = torch.einsum("tk,nk->tn", y, _exact_fp8(s["w"].double(), "tiles"))
        return (y, rstd) if s["residual"] is None else (y, x, rstd)
    w, dy, rstd = s["w"].double(), s["dy"].double(), s["rstd"].double()
    xh = x * rstd[:, None]
    c = torch.einsum("rc,rc,c->r", dy, xh, w) / n
    dx = rstd[:, None] * (dy * w - xh * c[:, None])
    if s["dh"] is not None:
        dx = dx + s["dh"].double()
    return dx, torch.einsum("rc,rc->c", dy, xh)
