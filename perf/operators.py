"""Cases of the feed-forward operators: the linear layer with its epilogue,
the gated linear layer, and activations kept in 8 bits for the backward pass.

``run`` computes a case either in elementary torch operations in 32 bits
(``own`` false) or with the framework's operators (``own`` true); ``exact``
gives the same results in 64 bits.

    linear   y = act(x W^T + b) + r             rocps.ops.linear.linear_act
    gated    y = act(x Wg^T + bg) * (x Wu^T + bu), W = [Wg; Wu]
                                                rocps.ops.gated.gated_linear
    pack     x in 8 bits and back               rocps.ops.act8

A training case returns y and every gradient.  With ``keep8`` the layer
keeps its input and its pre-activations in 8 bits between the forward and the
backward pass, so the gradients are those of the kept values.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(op, rows, k, n, act, dtype, bias=True, res=False, train=False,
          keep8=False):
    return {"op": op, "rows": rows, "k": k, "n": n, "act": act,
            "dtype": dtype, "bias": bias, "res": res, "train": train,
            "keep8": keep8}


def listed():
    c = []

    def add(name, *a, **kw):
        c.append({"name": name, **_case(*a, **kw)})

    # one token through the attention's output projection at BERT-base's
    # width: nothing but latency
    add("linear one token", "linear", 1, 768, 768, "none", "bf16", res=True)
    # a few sequences answered together at a large model's width: the weights
    # have to be read once
    add("linear few tokens", "linear", 24, 4096, 4096, "gelu", "bf16")
    # evaluation of a batch of 64 x 128 tokens: the output projection with the
    # residual stream added
    add("linear batch", "linear", 8192, 768, 768, "none", "bf16", res=True)
    # a classifier's odd sizes and a ragged batch, with mixed-precision types
    add("linear odd train", "linear", 1531, 1001, 515, "relu", "fp16",
        train=True)
    # a large model's dense layer in training
    add("linear large train", "linear", 8192, 4096, 4096, "gelu", "bf16",
        res=True, train=True)
    # one token through a large model's gated block
    add("gated one token", "gated", 1, 4096, 8192, "silu", "bf16",
        bias=False)
    # BERT-base's width with a gated block of the usual two thirds of 4 x 768,
    # 64 x 128 tokens, in training
    add("gated base train", "gated", 8192, 768, 2048, "gelu", "bf16",
        train=True)
    # a mid-sized model's gated block in training
    add("gated mid train", "gated", 4096, 2048, 5632, "silu", "fp16",
        bias=False, train=True)
    # a batch's activations at BERT-base's width kept in 8 bits
    add("pack base", "pack", 8192, 768, 768, "none", "bf16")
    # a large model's activations kept in 8 bits
    add("pack large", "pack", 16384, 8192, 8192, "none", "fp16")
    # the first product of BERT-base's feed-forward at a batch of 64 x 128,
    # its checkpoints in 8 bits
    add("linear keep8 train", "linear", 8192, 768, 2048, "gelu", "bf16",
        train=True, keep8=True)
    # the mid-sized gated block with its checkpoints in 8 bits
    add("gated keep8 train", "gated", 4096, 2048, 5632, "silu", "bf16",
        bias=False, train=True, keep8=True)
    return c


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: mostly whole tiles, sometimes whole vectors, now and
    then odd."""
    v = _spread(rng, lo, hi)
    step = rng.choice((128, 64, 64, 8, 1))
    return max(lo, v // step * step)


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(("linear", "linear", "gated", "gated", "pack"))
        dtype = rng.choice(("bf16", "bf16", "fp16"))
        train = op != "pack" and rng.random() < 0.6
        rows = _spread(rng, 64 if train else 1, 16384)
        k = _width(rng, 256, 8192)
        n = k if op == "pack" else _width(rng, 256, 8192)
        act = ("none" if op == "pack" else
               rng.choice(("none", "relu", "gelu", "silu")) if op == "linear"
               else rng.choice(("gelu", "silu")))
        if op == "pack":
            rows = max(rows, 64)
        c = _case(op, rows, k, n, act, dtype, bias=rng.random() < 0.6,
                  res=op == "linear" and rng.random() < 0.5, train=train,
                  keep8=train and rng.random() < 0.4)
        if work(c)["flops"] <= most:
            return c


def prepare(case, seed):
    """Tensors of one layer: normal inputs with a few strong channels, weights
    of unit gain, gradients of a mean loss's size."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = _TYPES[case["dtype"]]
    m, k, n = case["rows"], case["k"], case["n"]
    outs = 2 * n if case["op"] == "gated" else n

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = {"case": dict(case)}
    s["x"] = (normal(m, k) * (0.4 * normal(k)).exp()).to(t)
    if case["op"] == "pack":
        return s
    s["w"] = (normal(outs, k) / math.sqrt(k)).to(t)
    s["b"] = (0.1 * normal(outs)).to(t) if case["bias"] else None
    s["r"] = normal(m, n).to(t) if case["res"] else None
    if case["train"]:
        s["dy"] = (normal(m, n) / 64).to(t)
        for name in ("x", "w", "b", "r"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# -- the framework's operators -------------------------------------------------


def _run_own(s):
    case = s["case"]
    if case["op"] == "pack":
        from rocps.ops.act8 import pack_activation, unpack_activation
        return {"x": unpack_activation(pack_activation(s["x"]))}
    act = None if case["act"] == "none" else case["act"]
    keep = "8bit" if case["keep8"] else None
    if case["op"] == "linear":
        from rocps.ops.linear import linear_act
        y = linear_act(s["x"], s["w"], s["b"], s["r"], activation=act,
                       checkpoint=keep)
    else:
        from rocps.ops.gated import gated_linear
        y = gated_linear(s["x"], s["w"], s["b"], activation=act,
                         checkpoint=keep)
    out = {"y": y.detach()}
    if case["train"]:
        names = [p for p in ("x", "w", "b", "r") if s[p] is not None]
        grads = torch.autograd.grad(y, [s[p] for p in names], s["dy"])
        out.update({"d" + p: v for p, v in zip(names, grads)})
    return out


# -- the plain form ------------------------------------------------------------

_C = 0.7978845608028654  # sqrt(2 / pi)
_A = 0.044715


def _act(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.tanh(_C * (v + _A * v * v * v)))
    return v


def _slope(v, name):
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name == "silu":
        z = torch.sigmoid(v)
        return z * (1 + v * (1 - z))
    if name == "gelu":
        z = torch.tanh(_C * (v + _A * v * v * v))
        return (0.5 * (1 + z)
                + 0.5 * v * (1 - z * z) * _C * (1 + 3 * _A * v * v))
    return torch.ones_like(v)


def _kept8(v):
    """v as 8 bits hold it: for each 32 values along the last axis a power of
    two s, the smallest that brings them to 448 at most, and v / s in e4m3."""
    m, k = v.shape
    pad = -k % 32
    if pad:
        v = torch.cat([v, v.new_zeros(m, pad)], dim=1)
    u = v.reshape(m, -1, 32)
    frac, exp = torch.frexp(u.abs().amax(-1, keepdim=True))
    exp = (exp - 9 + (frac > 0.875).to(exp.dtype)).clamp(-118, 120)
    up, down = (((127 + e) << 23).view(torch.float32) for e in (exp, -exp))
    q = (u * down).to(torch.float8_e4m3fn).to(v.dtype)
    return (q * up).reshape(m, -1)[:, :k]


def _rounded(v, t):
    """To type t, values past its largest finite one held there."""
    most = torch.finfo(t).max
    return v.clamp(-most, most).to(t)


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    t = _TYPES[case["dtype"]]
    x = s["x"].float()
    if case["op"] == "pack":
        return {"x": _rounded(_kept8(x), t)}
    act, n = case["act"], case["n"]
    w = s["w"].float()
    pre = x @ w.t()
    if s["b"] is not None:
        pre = pre + s["b"].float()
    if case["op"] == "linear":
        y = _act(pre, act)
        if s["r"] is not None:
            y = y + s["r"].float()
    else:
        y = _act(pre[:, :n], act) * pre[:, n:]
    out = {"y": y.to(t)}
    if not case["train"]:
        return out
    dy = s["dy"].float()
    if case["keep8"]:
        x = _kept8(x)
        if case["op"] == "gated":  # the groups of each half begin at its start
            pre = torch.cat([_kept8(pre[:, :n]), _kept8(pre[:, n:])], dim=1)
        elif act != "none":
            pre = _kept8(pre)
    if case["op"] == "linear":
        dpre = dy * _slope(pre, act)
    else:
        gate, up = pre[:, :n], pre[:, n:]
        dpre = torch.cat([dy * up * _slope(gate, act), dy * _act(gate, act)],
                         dim=1)
    out["dx"] = (dpre @ w).to(t)
    out["dw"] = (dpre.t() @ x).to(t)
    if s["b"] is not None:
        out["db"] = dpre.sum(0).to(t)
    if s["r"] is not None:
        out["dr"] = s["dy"]
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -- the definition in 64 bits -------------------------------------------------


def _two(e):
    """2 to the whole number e, from its bits: a library's power may be off."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """Nearest e4m3 value, ties to even, of |v| at most 448."""
    e = torch.frexp(v)[1].clamp(min=-5) - 1
    step = _two(e - 3)
    return torch.round(v / step) * step


def _hold8(v):
    parts = []
    for a in range(0, v.shape[1], 4096):  # whole groups of 32
        u = v[:, a:a + 4096].double()
        groups = torch.nn.functional.pad(u, (0, -u.shape[1] % 32))
        groups = groups.unflatten(1, (-1, 32))
        top = groups.abs().amax(2)
        e = torch.ceil(torch.log2(top / 448)).nan_to_num(neginf=-118)
        e = e.clamp(-200, 200)  # and now to the very border
        e = torch.where(_two(e - 1) * 448 >= top, e - 1, e)
        e = torch.where(_two(e) * 448 < top, e + 1, e)
        scale = _two(e.clamp(-118, 120)).unsqueeze(2)
        held = (_e4m3(groups / scale) * scale).flatten(1)[:, :u.shape[1]]
        parts.append(held)
    return torch.cat(parts, 1)


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"]
    if case["op"] == "pack":
        most = torch.finfo(x.dtype).max
        held = torch.empty(x.shape, dtype=torch.float32, device=x.device)
        for a in range(0, x.shape[0], 1024):  # all held values are exact here
            held[a:a + 1024] = _hold8(x[a:a + 1024]).clamp(-most, most)
        return {"x": held}
    n, name = case["n"], case["act"]

    def f(v):
        if name == "gelu":
            return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi)
                                      * (v + 0.044715 * v.pow(3))))
        if name == "silu":
            return v / (1 + torch.exp(-v))
        return torch.where(v > 0, v, torch.zeros_like(v)) \
            if name == "relu" else v

    def df(v):
        if name == "none":
            return torch.ones_like(v)
        if name == "relu":
            return torch.where(v > 0, 1.0, 0.0).to(v)
        if name == "silu":
            z = 1 / (1 + torch.exp(-v))
            return z + v * z * (1 - z)
        r = math.sqrt(2 / math.pi)
        z = 1 / (1 + torch.exp(-2 * r * (v + 0.044715 * v.pow(3))))
        return z + 2 * r * v * z * (1 - z) * (1 + 3 * 0.044715 * v.pow(2))

    x, w = x.double(), s["w"].double()
    a = torch.mm(x, w.t().contiguous())
    if s["b"] is not None:
        a += s["b"].double()
    out = {}
    if case["op"] == "linear":
        out["y"] = f(a)
        if s["r"] is not None:
            out["y"] = out["y"] + s["r"].double()
    else:
        out["y"] = f(a[:, :n]) * a[:, n:]
    if not case["train"]:
        return out
    dy = s["dy"].double()
    if case["keep8"]:
        x = _hold8(x)
        if case["op"] == "gated":
            a[:, :n] = _hold8(a[:, :n])
            a[:, n:] = _hold8(a[:, n:])
        elif name != "none":
            a = _hold8(a)
    if case["op"] == "linear":
        da = dy * df(a)
    else:
        da = torch.empty_like(a)
        da[:, :n] = dy * a[:, n:] * df(a[:, :n])
        da[:, n:] = dy * f(a[:, :n])
    out["dx"] = torch.mm(da, w)
    out["dw"] = torch.mm(da.t().contiguous(), x)
    if s["b"] is not None:
        out["db"] = da.sum(0)
    if s["r"] is not None:
        out["dr"] = dy
    return out


def work(case):
    m, k, n = case["rows"], case["k"], case["n"]
    if case["op"] == "pack":
        # in and out in 16 bits; the kept form, written and read: a byte a
        # value and one a group of 32
        groups = m * ((k + 31) // 32)
        return {"bytes": 4 * m * k + 2 * (m * k + groups), "flops": 4 * m * k}
    outs = 2 * n if case["op"] == "gated" else n
    nbytes = m * k + outs * k + m * n
    nbytes += outs if case["bias"] else 0
    nbytes += m * n if case["res"] else 0
    flops = 2 * m * outs * k
    if case["train"]:
        nbytes += m * n + m * k + outs * k + (outs if case["bias"] else 0)
        flops *= 3
    return {"bytes": 2 * nbytes, "flops": flops}
