"""Performance cases of what stands around the layers in a training step: the norm in front of them, the
loss over a vocabulary behind them, and the optimizer's step over all tensors.

norm    y = (x - mean) / sqrt(var + eps) * w + b over a row's features; the backward gives dx, dw, db
loss    logits = x w^T + b; -log softmax(logits)[target], rows whose target is -100 left out; the backward
        gives dx, dw, db
adamw   m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
        p = p (1 - lr wd) - lr (m / c1) / (sqrt(v / c2) + eps) over a list of tensors.  The moments are fp32,
        bf16, or 8 bits: blocks of 256 elements share fp32 scales, m = s c |c| with c in [-127, 127] and
        s = max |m| / 127^2, v = (r c^2)^2 with c in [0, 255] (1 at least where v > 0) and
        r = sqrt(max v) / 255^2, the maxima rounded to fp32; c is the nearest by its root
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4, "int8": 1}
IGNORED = -100
EPS = 1e-5
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
STEP = 100  # steps that the optimizer has done

# norm: out and par are the types of y and of w and b; pitch: elements between rows of x past its width
NORM = dict(kind="norm", train=True, dtype="bf16", out="bf16", par="bf16", pitch=0)
# loss: ignored is the share of rows without a target
LOSS = dict(kind="loss", train=True, dtype="bf16", bias=False, ignored=0.0, reduction="mean")
# adamw: total elements in count tensors; gradients in the parameters' type, or (main) in fp32 buffers that the step clears
ADAMW = dict(kind="adamw", dtype="bf16", moments="fp32", main=False)


def listed():
    return [
        # one token being served: latency
        dict(NORM, name="norm_one", train=False, M=1, D=4096),
        # nothing a multiple of anything, columns of a wider tensor
        dict(NORM, name="norm_odd", M=777, D=1001, dtype="fp32", out="fp32", par="fp32", pitch=23),
        # a training batch, from an fp32 residual stream to a bf16 product's input
        dict(NORM, name="norm_train", M=8192, D=4096, dtype="fp32"),
        # a wide model over a long batch
        dict(NORM, name="norm_large", M=32768, D=8192),
        # a few tokens scored against a vocabulary, no gradients
        dict(LOSS, name="loss_score", train=False, M=16, K=1024, V=32768, reduction="none"),
        # a ragged batch with prompts left out, over an odd number of classes
        dict(LOSS, name="loss_odd", M=777, K=1001, V=12553, bias=True, ignored=0.3),
        # a classifier's head in full precision
        dict(LOSS, name="loss_fp32", M=1024, K=1024, V=8192, dtype="fp32", bias=True),
        # an ordinary training step's head
        dict(LOSS, name="loss_train", M=4096, K=1024, V=50000),
        # a long batch over a large vocabulary
        dict(LOSS, name="loss_large", M=8192, K=4096, V=131072, ignored=0.1),
        # many small tensors, as biases and norms are: latency
        dict(ADAMW, name="adamw_small", total=400_000, count=48),
        # a sparse layer and the dense tensors around it with moments in 8 bits
        dict(ADAMW, name="adamw_8bit", total=150_000_000, count=12, moments="int8"),
        # a large layer in full precision whose gradients were accumulated in fp32 buffers
        dict(ADAMW, name="adamw_large", total=400_000_000, count=8, dtype="fp32", main=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "loss", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "norm":
        d = _log(rng, 8, 16384)  # of two features nothing but rounding is left in dx
        m = _log(rng, 1, min(65536, 32768 * 8192 // d // (1 if dtype == "bf16" else 2)))
        return dict(NORM, M=m, D=d, dtype=dtype, out=rng.choice(["bf16", "fp32"]) if dtype == "fp32" else "bf16",
                    par=rng.choice(["bf16", "fp32"]), train=rng.random() < 0.7, pitch=rng.choice([0, 0, 1, 8]))
    if kind == "loss":
        k, v = _log(rng, 16, 8192), _log(rng, 16, 131072)
        m = _log(rng, 1, min(16384, 8192 * 4096 * 131072 // (k * v) // (1 if dtype == "bf16" else 16), 2 ** 30 // v))
        return dict(LOSS, M=m, K=k, V=v, dtype=dtype, bias=rng.random() < 0.5, ignored=rng.choice([0.0, 0.0, 0.5]),
                    train=rng.random() < 0.7, reduction=rng.choice(["mean", "sum", "none"]))
    moments = rng.choice(["int8", "bf16", "fp32"])
    total = _log(rng, 1, 100_000_000)
    return dict(ADAMW, total=total, count=min(total, _log(rng, 1, 24 if moments == "int8" else 64)), dtype=dtype,
                moments=moments, main=rng.random() < 0.3)


# ---------------------------------------------------------------------------- inputs
def _sizes(total, count):
    """``count`` tensors of very different sizes, ``total`` elements in all."""
    rng = random.Random(total * 1009 + count)
    parts = [math.exp(rng.uniform(0, 6)) for _ in range(count)]
    left = total - count
    sizes = [1 + int(left * p / sum(parts)) for p in parts]
    sizes[0] += total - sum(sizes)
    return sizes


def _inputs(c, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    def uniform(*shape):
        return torch.rand(*shape, device=DEVICE, generator=gen)

    if c["kind"] == "norm":
        M, D, p = c["M"], c["D"], c["pitch"]
        # features of a residual stream differ in scale and place
        x = normal(M, D + p).mul_(torch.exp(0.5 * normal(1, D + p))).add_(0.5 * normal(1, D + p)).to(dt)[:, :D]
        par = DTYPES[c["par"]]
        t = dict(x=x, w=(1 + 0.2 * normal(D)).to(par), b=(0.1 * normal(D)).to(par))
        if c["train"]:
            t["dy"] = normal(M, D).to(DTYPES[c["out"]])
        return t
    if c["kind"] == "loss":
        M, K, V = c["M"], c["K"], c["V"]
        t = dict(x=normal(M, K).to(dt), w=normal(V, K).mul_(2 / math.sqrt(K)).to(dt))
        if c["bias"]:
            t["b"] = (0.5 * normal(V)).to(dt)
        # some classes are far more frequent than others
        target = (torch.exp(uniform(M).double() * math.log(V)).long() - 1).clamp(0, V - 1)
        t["target"] = torch.where(uniform(M) < c["ignored"], IGNORED, target)
        if c["train"] and c["reduction"] == "none":
            t["dy"] = uniform(M) / M
        return t
    sizes = _sizes(c["total"], c["count"])
    at, places = 0, []
    for n in sizes:  # every tensor at a multiple of 256 elements of one buffer
        places.append((at, n))
        at += -(-n // 256) * 256
    used = torch.zeros(at, device=DEVICE, dtype=torch.bool)
    for a, n in places:
        used[a:a + n] = True

    def buffer(v, dtype):
        return torch.where(used, v, 0.0).to(dtype)

    scale = torch.exp(normal(at // 256, 1)).expand(-1, 256).reshape(-1)  # of the gradients, by region
    t = dict(places=places, p=buffer(0.02 * normal(at), dt))
    t["g"] = buffer(1e-3 * scale * normal(at), torch.float32 if c["main"] else dt)
    m, v = buffer(3e-4 * scale * normal(at), torch.float32), buffer((1e-3 * scale).square() * (0.2 + uniform(at)), torch.float32)
    if c["moments"] == "int8":
        t["m"], t["m_scale"], t["v"], t["v_scale"] = _to_8bit(m, v)
    else:
        t["m"], t["v"] = m.to(DTYPES[c["moments"]]), v.to(DTYPES[c["moments"]])
    return t


def prepare(case, seed):
    c, t = dict(case), _inputs(case, seed)
    if c["kind"] == "adamw":
        if own:
            _optimizer(c, t)
    elif c["train"]:
        for name in ("x", "w", "b"):
            if name in t:
                t[name] = t[name].requires_grad_(True)
    return c, t


def work(case):
    c, s = case, SIZE[case["dtype"]]
    if c["kind"] == "norm":
        M, D, o, par = c["M"], c["D"], SIZE[c["out"]], SIZE[c["par"]]
        if c["train"]:
            return {"bytes": 2 * M * D * (s + o) + 4 * D * par, "flops": 20 * M * D}
        return {"bytes": M * D * (s + o) + 2 * D * par, "flops": 8 * M * D}
    if c["kind"] == "loss":
        M, K, V = c["M"], c["K"], c["V"]
        once = s * (M * K + V * K + (V if c["bias"] else 0)) + 8 * M
        return {"bytes": 2 * once if c["train"] else once, "flops": (6 if c["train"] else 2) * M * K * V}
    n, m = c["total"], SIZE[c["moments"]]
    moments = 4 * m if c["moments"] != "int8" else 4 * m + 8  # their values are an output too
    return {"bytes": n * (2 * s + moments + (8 if c["main"] else s)), "flops": 16 * n}


# ---------------------------------------------------------------------------- the framework's calls
def _optimizer(c, t):
    """The optimizer of a program that has done ``STEP`` steps, over views of the buffers."""
    from granulelayer_amd import FusedAdamW

    params = [torch.nn.Parameter(t["p"][a:a + n]) for a, n in t["places"]]
    opt = FusedAdamW(params, moments=c["moments"], stochastic_rounding=False, **HYPER)
    for p, (a, n) in zip(params, t["places"]):
        opt.state[p] = dict(step=STEP, m=t["m"][a:a + n], v=t["v"][a:a + n])
        if c["moments"] == "int8":
            k = slice(a // 256, (a + n + 255) // 256)
            opt.state[p].update(m_scale=t["m_scale"][k], v_scale=t["v_scale"][k])
        g = t["g"][a:a + n]
        if c["main"]:
            p.main_grad = g
    t["params"], t["opt"] = params, opt
    t["grads"] = None if c["main"] else [t["g"][a:a + n] for a, n in t["places"]]


def _own(c, t):
    import granulelayer_amd as gl

    if c["kind"] == "adamw":
        if t["grads"] is not None:
            for p, g in zip(t["params"], t["grads"]):
                p.grad = g
        t["opt"].step()
        if c["moments"] == "int8":
            values = t["opt"].moment_values()
            return dict(p=t["p"], m=[m for m, v in values], v=[v for m, v in values])
        return dict(p=t["p"], m=t["m"], v=t["v"])
    names = [n for n in ("x", "w", "b") if n in t]
    if c["kind"] == "norm":
        y = gl.layer_norm(t["x"], t["w"], t["b"], EPS, DTYPES[c["out"]])
        if not c["train"]:
            return y
        grads = torch.autograd.grad(y, [t[n] for n in names], t["dy"])
        return dict({"d" + n: g for n, g in zip(names, grads)}, y=y.detach())
    loss = gl.dense_cross_entropy(t["x"], t["w"], t["target"], t.get("b"), c["reduction"], IGNORED)
    if not c["train"]:
        return loss
    grads = torch.autograd.grad(loss, [t[n] for n in names], t.get("dy"))
    return dict({"d" + n: g for n, g in zip(names, grads)}, loss=loss.detach())


# ---------------------------------------------------------------------------- the plain form, in 32 bits
def _to_8bit(m, v):
    """Codes and scales.  A quotient next to a border decides a code: in 64 bits."""
    m, v = m.double().reshape(-1, 256), v.double().reshape(-1, 256)
    top, vtop = m.abs().amax(1, keepdim=True).float(), v.amax(1, keepdim=True).float()
    sm = torch.where(top >= 2.0 ** -100, top.double() / 127 ** 2, 0.0).float()
    sv = torch.where(vtop >= 2.0 ** -126, vtop.double().sqrt() / 255 ** 2, 0.0).float()
    # without a scale the quotients are 0 / 1
    cm = torch.floor(torch.where(sm > 0, m.abs(), 0.0).div(torch.where(sm > 0, sm, 1.0)).sqrt() + 0.5)
    cv = torch.floor(torch.where(sv > 0, v, 0.0).sqrt().div(torch.where(sv > 0, sv, 1.0)).sqrt() + 0.5)
    cv = torch.where((sv > 0) & (v > 0), cv.clamp(min=1), cv)
    cm = torch.copysign(cm, m)
    return cm.to(torch.int8).reshape(-1), sm.reshape(-1), cv.to(torch.uint8).reshape(-1), sv.reshape(-1)


def _from_8bit(t):
    cm, cv = t["m"].double().reshape(-1, 256), t["v"].double().reshape(-1, 256)
    m = cm * cm.abs() * t["m_scale"][:, None]
    return m.reshape(-1), (cv * cv * t["v_scale"][:, None]).square().reshape(-1)


def _plain_adamw(c, t):
    lr, (b1, b2), eps, wd = HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    step = t["step"] = t.get("step", STEP) + 1
    p, g = t["p"].float(), t["g"].float()
    if c["moments"] == "int8":
        m, v = _from_8bit(t)
        m64, v64 = m * b1 + g.double() * (1 - b1), v * b2 + g.double().square() * (1 - b2)
        m, v = m64.float(), v64.float()
    else:
        m, v = t["m"].float() * b1 + g * (1 - b1), t["v"].float() * b2 + g * g * (1 - b2)
    p = p * (1 - lr * wd) - lr * (m / (1 - b1 ** step)) / ((v / (1 - b2 ** step)).sqrt() + eps)
    t["p"].copy_(p)
    if c["main"]:
        t["g"].zero_()
    if c["moments"] != "int8":
        t["m"].copy_(m)
        t["v"].copy_(v)
        return dict(p=t["p"], m=t["m"], v=t["v"])
    t["m"], t["m_scale"], t["v"], t["v_scale"] = _to_8bit(m64, v64)
    m, v = (u.float() for u in _from_8bit(t))
    return dict(p=t["p"], m=[m[a:a + n] for a, n in t["places"]], v=[v[a:a + n] for a, n in t["places"]])


def _plain_norm(c, t):
    x, w, b = t["x"].detach().float(), t["w"].detach().float(), t["b"].detach().float()
    d = x - x.mean(1, keepdim=True)
    r = 1 / (d.square().mean(1, keepdim=True) + EPS).sqrt()
    h = d * r
    y = (h * w + b).to(DTYPES[c["out"]])
    if not c["train"]:
        return y
    dy = t["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dict(y=y, dx=dx.to(t["x"].dtype), dw=(dy * h).sum(0).to(t["w"].dtype), db=dy.sum(0).to(t["b"].dtype))


def _plain_loss(c, t):
    x, w, target = t["x"].detach().float(), t["w"].detach().float(), t["target"]
    z = x @ w.t()
    if "b" in t:
        z = z + t["b"].detach().float()
    counts = target != IGNORED
    z = z - z.amax(1, keepdim=True)
    at = torch.where(counts, target, 0)[:, None]
    picked = z.gather(1, at)[:, 0]
    z = z.exp()
    total = z.sum(1)
    loss = torch.where(counts, total.log() - picked, 0.0)
    n = counts.sum().clamp(min=1)
    share = t["dy"] if "dy" in t else 1.0 / n if c["reduction"] == "mean" else 1.0
    loss = loss if c["reduction"] == "none" else loss.sum() / n if c["reduction"] == "mean" else loss.sum()
    if not c["train"]:
        return loss
    share = torch.where(counts, share, 0.0)
    z = z * (share / total)[:, None]
    z = z.scatter_add(1, at, -share[:, None])
    dt = t["x"].dtype
    out = dict(loss=loss, dx=(z @ w).to(dt), dw=(z.t() @ x).to(dt))
    if "b" in t:
        out["db"] = z.sum(0).to(dt)
    return out


def run(state):
    c, t = state
    if own:
        return _own(c, t)
    return {"norm": _plain_norm, "loss": _plain_loss, "adamw": _plain_adamw}[c["kind"]](c, t)


# ---------------------------------------------------------------------------- the definition, in 64 bits
def _kept64(a, top, most):
    """a >= 0 at the nearest of unit i^2, most i to the top: the unit is kept in fp32."""
    unit = (top / most ** 2).float().double().clamp(min=1e-300)
    i = torch.round((a / unit).sqrt())
    return unit * i.square(), unit


def _exact_adamw(c, t):
    out = dict(p=t["p"].double(), m=[], v=[])
    if c["moments"] != "int8":
        out.update(m=t["m"].double(), v=t["v"].double())
    b1, b2 = HYPER["betas"]
    for a, n in t["places"]:
        k = slice(a, a + n)
        g, p = t["g"][k].double(), out["p"][k]
        m, v = t["m"][k].double(), t["v"][k].double()
        if c["moments"] == "int8":
            of = torch.arange(a, a + n, device=DEVICE) // 256
            m = m * m.abs() * t["m_scale"].double()[of]
            v = v.pow(4) * t["v_scale"].double()[of].square()
        m = torch.lerp(g, m, b1)
        v = torch.lerp(g.square(), v, b2)
        hat = m / (1 - b1 ** (STEP + 1)) / (v.div(1 - b2 ** (STEP + 1)).sqrt() + HYPER["eps"])
        p.copy_(p - HYPER["lr"] * (hat + HYPER["weight_decay"] * p))
        if c["moments"] != "int8":
            out["m"][k], out["v"][k] = m, v
            continue
        first = torch.arange(n, device=DEVICE) // 256
        tops = torch.zeros(2, int(first[-1]) + 1, device=DEVICE, dtype=torch.float64)
        tops[0].scatter_reduce_(0, first, m.abs(), "amax")
        tops[1].scatter_reduce_(0, first, v, "amax")
        tops = tops.float().double()
        out["m"].append(torch.sign(m) * _kept64(m.abs(), tops[0][first], 127)[0])
        root, unit = _kept64(v.sqrt(), tops[1].sqrt()[first], 255)
        out["v"].append(torch.where(v > 0, torch.maximum(root, unit), root).square())
    return out


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["kind"] == "adamw":
        return _exact_adamw(c, t)
    x, w = t["x"].double(), t["w"].double()
    if c["kind"] == "norm":
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        scale = torch.rsqrt(var + EPS)
        hat = (x - mean) * scale
        y = torch.addcmul(t["b"].double(), hat, w)
        if not c["train"]:
            return y
        dy = t["dy"].double()
        dh = dy * w
        dx = scale * (dh - hat * torch.mean(dh * hat, 1, keepdim=True) - torch.mean(dh, 1, keepdim=True))
        return {"y": y, "dx": dx, "dw": torch.sum(dy * hat, 0), "db": torch.sum(dy, 0)}
    M, target = c["M"], t["target"]
    z = torch.mm(x, w.t())
    if "b" in t:
        z += t["b"].double()
    norm = torch.logsumexp(z, 1)
    rows = torch.nonzero(target >= 0)[:, 0]
    loss = torch.zeros(M, device=DEVICE, dtype=torch.float64)
    loss[rows] = norm[rows] - z[rows, target[rows]]
    g = torch.zeros_like(loss)
    g[rows] = {"none": t["dy"].double()[rows] if "dy" in t else 0.0, "sum": 1.0, "mean": 1.0 / max(1, len(rows))}[c["reduction"]]
    if c["reduction"] != "none":
        loss = loss.sum() / (max(1, len(rows)) if c["reduction"] == "mean" else 1)
    if not c["train"]:
        return loss
    z = z.sub_(norm[:, None]).exp_()
    z[rows, target[rows]] -= 1
    z *= g[:, None]
    out = {"loss": loss, "dx": torch.mm(z, w), "dw": torch.mm(z.t(), x)}
    if "b" in t:
        out["db"] = z.sum(0)
    return out
