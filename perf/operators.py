"""Performance cases of the dense projection and of activations kept in 8 bits.

The dense projection maps a model's width into a sparse layer's inputs, or its pooled outputs back
onto a residual stream:

    z = x W^T + b,   y = act(z) + residual

and its backward takes what the forward kept: x and, for GELU, z, either in the operands' type
(``ckpt`` "exact") or in 8 bits ("int8"); for ReLU the sign of z.  The 8-bit form gives every
block of 32 features of a row a common power of two and every value an integer in [-127, 127].

Three kinds of passes: ``infer`` (the forward, no gradients), ``train`` (forward, backward; returns
y and every gradient) and ``keep`` (a tensor put into 8 bits and read back).
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
# res: type of the residual ("" without one); pitch: elements between rows of x past its width
BASE = dict(kind="infer", act="gelu", dtype="bf16", res="", ckpt="exact", pitch=0)


def listed():
    return [
        # one token through a square projection with a residual: latency, W is read once
        dict(name="serve_one", M=1, K=4096, N=4096, act="relu", res="bf16"),
        # a small batch of tokens being served
        dict(name="serve_batch", M=48, K=1024, N=4096),
        # nothing a multiple of anything, as with a pruned or feature-selected model
        dict(name="infer_odd", M=777, K=1001, N=1255),
        # a large batch onto an fp32 residual stream
        dict(name="infer_large", M=8192, K=4096, N=8192, res="fp32"),
        # full-precision scoring of a medium batch
        dict(name="infer_fp32", M=512, K=1024, N=4096, dtype="fp32", act="relu"),
        # a ragged training batch with its inputs in 8 bits
        dict(name="train_odd", kind="train", M=1000, K=1001, N=1255, act="relu", ckpt="int8"),
        # an ordinary training step's projection, activations kept as they are
        dict(name="train_1k", kind="train", M=4096, K=1024, N=4096),
        # the same in full precision, with a residual
        dict(name="train_fp32", kind="train", M=2048, K=1024, N=4096, dtype="fp32", res="fp32"),
        # a long batch whose activations are kept in 8 bits
        dict(name="train_large", kind="train", M=16384, K=4096, N=4096, res="bf16", ckpt="int8"),
        # the inputs of a small layer put away and read back: latency
        dict(name="keep_small", kind="keep", M=64, K=1024),
        # columns of a wider fp32 tensor, an odd number of them
        dict(name="keep_odd", kind="keep", M=5000, K=1001, dtype="fp32", pitch=23),
        # the inputs of a wide layer over a long batch
        dict(name="keep_large", kind="keep", M=32768, K=8192),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["infer", "infer", "train", "train", "keep"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "keep":
        k = _log(rng, 1, 16384)
        return dict(kind=kind, M=_log(rng, 1, min(65536, 32768 * 8192 // k // (1 if dtype == "bf16" else 2))), K=k,
                    dtype=dtype, pitch=rng.choice([0, 0, 1, 24]))
    k, n = _log(rng, 16, 8192), _log(rng, 16, 8192)
    m = _log(rng, 1, min(16384, 16384 * 4096 * 4096 // (k * n)))
    case = dict(kind=kind, M=m, K=k, N=n, dtype=dtype, res=rng.choice(["", dtype]), pitch=rng.choice([0, 0, 8]))
    if kind == "infer":
        return dict(case, act=rng.choice(["identity", "relu", "gelu"]))
    if dtype == "bf16":
        return dict(case, act=rng.choice(["identity", "relu", "gelu"]), ckpt=rng.choice(["exact", "int8"]))
    # in fp32 a sign or an 8-bit rounding of z that falls the other way shows in single gradients
    return dict(case, **rng.choice([dict(act="gelu", ckpt="exact"), dict(act="identity", ckpt="int8")]))


def _inputs(case, seed):
    c = dict(BASE, **case)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    M, K = c["M"], c["K"]
    # features differ in scale, as activations do
    x = normal(M, K + c["pitch"])
    x = (x * torch.exp(0.5 * normal(1, K + c["pitch"]))).to(dt)[:, :K]
    if c["kind"] == "keep":
        return c, dict(x=x)
    N = c["N"]
    t = dict(x=x, w=(normal(N, K) / math.sqrt(K)).to(dt), b=(0.1 * normal(N)).to(dt))
    if c["res"]:
        t["res"] = normal(M, N).to(DTYPES[c["res"]])
    if c["kind"] == "train":
        t["dy"] = normal(M, N).to(torch.promote_types(dt, DTYPES[c["res"] or c["dtype"]]))
    return c, t


def prepare(case, seed):
    c, t = _inputs(case, seed)
    if c["kind"] == "train":
        for name in ("x", "w", "b", "res"):
            if name in t:
                t[name] = t[name].requires_grad_(True)
    return c, t


def work(case):
    c = dict(BASE, **case)
    M, K = c["M"], c["K"]
    size = {"bf16": 2, "fp32": 4, "": 0}
    s = size[c["dtype"]]
    if c["kind"] == "keep":
        return {"bytes": 2 * s * M * K, "flops": 4 * M * K}
    N, r = c["N"], size[c["res"]]
    y = max(s, r)
    read, product = s * (M * K + N * K + N) + r * M * N, 2 * M * N * K
    if c["kind"] == "infer":
        return {"bytes": read + y * M * N, "flops": product}
    return {"bytes": read + 2 * y * M * N + s * (M * K + N * K + N), "flops": 3 * product}


# ---------------------------------------------------------------------------- the framework's calls
def _own(c, t):
    from granulelayer_amd import dense_projection, pack_activation

    if c["kind"] == "keep":
        return pack_activation(t["x"]).unpack()
    if c["kind"] == "infer":
        with torch.no_grad():
            return dense_projection(t["x"], t["w"], t["b"], t.get("res"), c["act"])
    y = dense_projection(t["x"], t["w"], t["b"], t.get("res"), c["act"], activation_checkpoint=c["ckpt"])
    names = [n for n in ("x", "w", "b", "res") if n in t]
    grads = torch.autograd.grad(y, [t[n] for n in names], t["dy"])
    return dict({"d" + n: g for n, g in zip(names, grads)}, y=y.detach())


# ---------------------------------------------------------------------------- the plain form, in 32 bits
def _eight_bits(x):
    """x [M, K] fp32 as the values its 8-bit form stands for."""
    M, K = x.shape
    blocks = torch.nn.functional.pad(x, (0, -K % 32)).reshape(M, -1, 32)
    a = blocks.abs().amax(-1, keepdim=True)
    e = (((a.view(torch.int32) + 0x10000) >> 23) - 6).clamp(min=1)
    step = (e << 23).view(torch.float32)
    q = torch.round(blocks * ((254 - e) << 23).view(torch.float32))
    return (q * step).reshape(M, -1)[:, :K]


def _plain(c, t):
    x = t["x"].detach().float()
    if c["kind"] == "keep":
        return _eight_bits(x).to(t["x"].dtype)
    w, b = t["w"].detach().float(), t["b"].detach().float()
    act, dt = c["act"], t["x"].dtype
    z = x @ w.t() + b
    y = z if act == "identity" else z.clamp(min=0) if act == "relu" else 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if "res" in t:
        y = y + t["res"].detach().float()
        y = y.to(torch.promote_types(dt, t["res"].dtype))
    else:
        y = y.to(dt)
    if c["kind"] == "infer":
        return y
    dz = t["dy"].float()
    if act == "relu":
        dz = dz * (z > 0)
    elif act == "gelu":
        z = _eight_bits(z) if c["ckpt"] == "int8" else z.to(dt).float()
        dz = dz * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    kept = _eight_bits(x) if c["ckpt"] == "int8" else x
    out = dict(y=y, dx=(dz @ w).to(dt), dw=(dz.t() @ kept).to(dt), db=dz.sum(0).to(dt))
    if "res" in t:
        out["dres"] = t["dy"].to(t["res"].dtype)
    return out


def run(state):
    c, t = state
    return _own(c, t) if own else _plain(c, t)


# ---------------------------------------------------------------------------- the definition, in 64 bits
def _kept64(v):
    """8-bit form of v (64 bits): per row and 32 columns the smallest power of two, of 2^-126 or more,
    that the block's values round to integers of magnitude 127 or less in."""
    cols = []
    for c0 in range(0, v.shape[1], 32):
        part = v[:, c0:c0 + 32]
        top = part.abs().max(dim=1, keepdim=True).values
        p = torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 6
        p = torch.where(top >= 127.5 * torch.exp2(p), p + 1, p).clamp(min=-126)
        cols.append(torch.round(part / torch.exp2(p)) * torch.exp2(p))
    return torch.cat(cols, 1)


def exact(case, seed):
    c, t = _inputs(case, seed)
    x = t["x"].double()
    if c["kind"] == "keep":
        return _kept64(x)
    w = t["w"].double()
    z = torch.addmm(t["b"].double(), x, w.t())
    half = 1 / math.sqrt(2)
    y = {"identity": lambda: z, "relu": lambda: torch.relu(z), "gelu": lambda: z * torch.special.erfc(-z * half) / 2}[c["act"]]()
    if "res" in t:
        y = y + t["res"].double()
    if c["kind"] == "infer":
        return y
    g = t["dy"].double()
    if c["act"] == "relu":
        g = torch.where(z > 0, g, torch.zeros_like(g))
    elif c["act"] == "gelu":
        z = _kept64(z) if c["ckpt"] == "int8" else z.to(t["x"].dtype).double()
        g = g * (torch.special.erfc(-z * half) / 2 + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi))
    out = {"y": y, "dx": torch.mm(g, w), "dw": torch.mm(g.t(), _kept64(x) if c["ckpt"] == "int8" else x), "db": g.sum(0)}
    if "res" in t:
        out["dres"] = t["dy"].double()
    return out
