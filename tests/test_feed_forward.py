"""The feed-forward operators against their formulas in float64: linear_act,
gated_linear, and activations in 8 bits.

Bounds are derived, not tuned.  u = eps / 2 is the type's rounding, h = 2**-24
float32's.  A sum of n products in float32 is off by at most (n + 8) h times
the sum of the products' magnitudes, whatever its order (n h to first order,
8 h for the bias, the activation's own arithmetic and the residual); a value
rounded to the type is off by u of itself, or by the type's smallest step.
Errors go on through |act'| <= 1.13 and |act''| <= 1.
"""

import math

import pytest
import torch

from rocps.ops.act8 import pack_activation, unpack_activation
from rocps.ops.gated import gated_linear
from rocps.ops.linear import linear_act

BF16, FP16 = torch.bfloat16, torch.float16
_H = 2.0 ** -24


def _devices():
    return ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _act(v, a):
    if a == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if a == "gelu":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi)
                                 * (v + 0.044715 * v ** 3))
    if a == "silu":
        return v * torch.sigmoid(v)
    return v


def _slope(v, a):
    if a is None:
        return torch.ones_like(v)
    with torch.enable_grad():
        u = v.detach().requires_grad_()
        return torch.autograd.grad(_act(u, a).sum(), u)[0]


def _tiny(t):
    """Half the smallest step, or the smallest normal where the GPU flushes
    what is below."""
    return 2.0 ** -25 if t == FP16 else 2.0 ** -126


def _round(v, t):
    """How far v may move when it is rounded to t."""
    return v.abs() * torch.finfo(t).eps / 2 + _tiny(t)


def _kept8(v):
    """The definition of activations in 8 bits, for finite v in float64."""
    m, n = v.shape
    g = torch.nn.functional.pad(v.double(), (0, -n % 32))
    g = g.reshape(m, g.shape[1] // 32, 32)
    top = g.abs().amax(2, keepdim=True)
    e = torch.full_like(top, -118.0)
    for k in range(-118, 121):  # the smallest that fits
        e = torch.where(top > 448 * 2.0 ** (k - 1), float(min(k, 120)), e)
    s = torch.pow(2.0, e)
    q = g / s
    low = torch.frexp(q)[1].clamp(min=-5).double() - 1
    step = torch.pow(2.0, low - 3)
    return (torch.round(q / step) * step * s).reshape(m, -1)[:, :n], \
        s.expand_as(g).reshape(m, -1)[:, :n]


def _kept_error(v):
    s = _kept8(v)[1]
    return v.abs() * 2.0 ** -4 + s * 2.0 ** -10


def _make(m, k, n, t, device, seed, gated=False, bias=True, res=False,
          scale=1.0):
    g = torch.Generator().manual_seed(seed)
    outs = 2 * n if gated else n

    def normal(*s):
        return torch.randn(*s, generator=g)

    x = (normal(m, k) * scale).to(t).to(device)
    w = (normal(outs, k) / math.sqrt(k)).to(t).to(device)
    b = (normal(outs) / 4).to(t).to(device) if bias else None
    r = normal(m, n).to(t).to(device) if res else None
    dy = normal(m, n).to(t).to(device)
    return x, w, b, r, dy


def _within(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.cpu()
    bound = bound.cpu()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0
    assert worst <= 1, f"{what}: {worst:.3g} times its bound"


def _check(x, w, b, r, dy, act, gated, eight=False, which="xwbr"):
    """Output and gradients of one layer against float64."""
    t = x.dtype
    leaves = {"x": x, "w": w, "b": b, "r": r}
    leaves = {p: v.detach().requires_grad_(p in which)
              for p, v in leaves.items() if v is not None}
    lx, lw, lb, lr = (leaves.get(p) for p in "xwbr")
    keep = "8bit" if eight else None
    if gated:
        y = gated_linear(lx, lw, lb, activation=act, checkpoint=keep)
    else:
        y = linear_act(lx, lw, lb, lr, activation=act, checkpoint=keep)
    assert y.dtype == t and y.is_contiguous()

    X, W, D = (v.detach().cpu().double() for v in (x, w, dy))
    X = X.reshape(-1, X.shape[-1])
    D = D.reshape(-1, D.shape[-1])
    n, k, m = D.shape[1], X.shape[1], X.shape[0]
    P = X @ W.t()
    mag = X.abs() @ W.abs().t()
    if b is not None:
        P = P + b.detach().cpu().double()
        mag = mag + b.detach().cpu().double().abs()
    ep = (k + 8) * _H * mag  # of the float32 pre-activations
    if gated:
        A, U, ea, eu = P[:, :n], P[:, n:], ep[:, :n], ep[:, n:]
        Y = _act(A, act) * U
        ey = 1.13 * ea * (U.abs() + eu) + _act(A, act).abs() * eu \
            + 8 * _H * Y.abs()
    else:
        Y = _act(P, act)
        ey = 1.13 * ep + 8 * _H * Y.abs()
        if r is not None:
            R = r.detach().cpu().double().reshape(-1, n)
            Y = Y + R
            ey = ey + 2 * _H * (R.abs() + Y.abs())
    _within(y.reshape(-1, n), Y, 1.001 * ey + _round(Y, t), "y")

    names = [p for p in "xwbr" if p in which and leaves.get(p) is not None]
    if not names:
        return
    grads = dict(zip(names, torch.autograd.grad(
        y, [leaves[p] for p in names], dy)))
    # the kept pre-activations
    ex = torch.zeros_like(X)
    if eight:
        if act is not None:
            ep = ep * 1.07 + (torch.cat([_kept_error(A), _kept_error(U)], 1)
                              if gated else _kept_error(P))
        ex = _kept_error(X)
    elif act is not None:
        ep = ep + _round(P, t)
    if gated:
        ea, eu = ep[:, :n], ep[:, n:]
        sa, fa = _slope(A, act), _act(A, act)
        es = ea + 8 * _H
        if act == "relu":
            es = (A.abs() <= ea).double()
        G = torch.cat([D * U * sa, D * fa], 1)
        eg = torch.cat([D.abs() * (eu * (sa.abs() + es) + U.abs() * es),
                        D.abs() * (1.13 * ea + 8 * _H * fa.abs())], 1)
    else:
        s = _slope(P, act)
        es = torch.zeros_like(P) if act is None else ep + 8 * _H
        if act == "relu":
            es = (P.abs() <= ep).double()
        G, eg = D * s, D.abs() * es
    eg = eg + 4 * _H * G.abs()
    er = eg + (0 if act is None else _round(G, t) * 1.01)  # as the products see it
    GM = G.abs() + er
    if "x" in grads:
        o = W.shape[0]
        dX = G @ W
        _within(grads["x"].reshape(-1, k), dX,
                1.001 * (er @ W.abs() + (o + 8) * _H * (GM @ W.abs()))
                + _round(dX, t), "dx")
    if "w" in grads:
        dW = G.t() @ X
        XM = X.abs() + ex
        _within(grads["w"], dW,
                1.001 * (er.t() @ XM + G.abs().t() @ ex
                         + (m + 8) * _H * (GM.t() @ XM)) + _round(dW, t),
                "dw")
    if "b" in grads:
        dB = G.sum(0)
        _within(grads["b"], dB,
                1.001 * (eg.sum(0) + (m + 8) * _H * (G.abs() + eg).sum(0))
                + _round(dB, t), "db")
    if "r" in grads:
        assert torch.equal(grads["r"], dy)


SIZES = [  # rows, k, n: one, odd, whole and broken tiles, steps of k
    (1, 64, 64), (1, 1, 1), (3, 5, 7), (17, 33, 130), (64, 128, 128),
    (65, 72, 136), (100, 768, 40), (127, 200, 257), (128, 64, 384),
    (130, 129, 96), (200, 1000, 100),
]


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_sizes(m, k, n, t, device):
    act = (None, "relu", "gelu", "silu")[(m + k + n) % 4]
    _check(*_make(m, k, n, t, device, m + k, res=n % 2 == 0), act, False)


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gated_sizes(m, k, n, t, device):
    act = ("relu", "gelu", "silu")[(m + k + n) % 3]
    _check(*_make(m, k, n, t, device, m + k, gated=True, bias=k % 2 == 0),
           act, True)


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("act", [None, "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias,res", [(True, True), (False, True),
                                      (True, False), (False, False)])
def test_linear_epilogues(act, bias, res, device):
    _check(*_make(70, 96, 80, BF16, device, 3, bias=bias, res=res), act,
           False)


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("which", ["x", "w", "b", "r", "xw", "wb", "xb"])
def test_only_the_gradients_asked_for(which, device):
    for act in (None, "gelu"):
        _check(*_make(33, 48, 56, BF16, device, 4, res=True), act, False,
               which=which)
        _check(*_make(33, 48, 51, BF16, device, 4, res=True), act, False,
               which=which)
    if which != "r":
        _check(*_make(33, 48, 56, FP16, device, 4, gated=True), "silu", True,
               which=which)


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,k,n,t", [(1, 64, 64, BF16), (5, 40, 37, FP16),
                                     (64, 96, 128, BF16),
                                     (130, 200, 72, FP16)])
def test_checkpoint_in_8_bits(m, k, n, t, gated, device):
    for act in ("gelu", "relu", "silu") + (() if gated else (None,)):
        _check(*_make(m, k, n, t, device, n, gated=gated), act, gated,
               eight=True)


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("gated", [False, True])
def test_checkpoint_in_8_bits_is_that_of_the_kept_values(gated, device):
    """Small whole numbers make the pre-activations exact, so that nothing but
    the definition decides what is kept; the gradients are those of the kept
    values to the bounds of 16 bits."""
    g = torch.Generator().manual_seed(5)
    m, k, n = 70, 64, 48
    outs = 2 * n if gated else n

    def whole(a, b, *s):
        return torch.randint(a, b, s, generator=g).double()

    X, W = whole(-9, 10, m, k), whole(-1, 2, outs, k) / 8
    D = torch.randn(m, n, generator=g).to(BF16).double()
    x, w, dy = (v.to(BF16).to(device) for v in (X, W, D))
    x.requires_grad_(), w.requires_grad_()
    if gated:
        y = gated_linear(x, w, activation="silu", checkpoint="8bit")
    else:
        y = linear_act(x, w, activation="silu", checkpoint="8bit")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    P, X8 = X @ W.t(), _kept8(X)[0]
    if gated:
        A, U = _kept8(P[:, :n])[0], _kept8(P[:, n:])[0]
        G = torch.cat([D * U * _slope(A, "silu"), D * _act(A, "silu")], 1)
    else:
        G = D * _slope(_kept8(P)[0], "silu")
    eg = _round(G, BF16) * 1.01 + 16 * _H * G.abs() + 16 * _H * D.abs().repeat(
        1, outs // n)
    GM = G.abs() + eg
    _within(dx, G @ W, eg @ W.abs() + (outs + 8) * _H * (GM @ W.abs())
            + _round(G @ W, BF16), "dx")
    _within(dw, G.t() @ X8, eg.t() @ X8.abs()
            + (m + 8) * _H * (GM.t() @ X8.abs()) + _round(G.t() @ X8, BF16),
            "dw")


@pytest.mark.parametrize("device", _devices())
def test_gradients_against_differences(device):
    """A step along random directions changes the output as the gradients
    say.  float64 on the CPU, where that is what is computed; on the GPU the
    16-bit gradients against the float64 layer's differences."""
    t = torch.float64 if device == "cpu" else BF16
    for gated in (False, True):
        x, w, b, r, dy = _make(40, 64, 48, BF16, device, 6, gated=gated,
                               res=not gated)
        live = [v for v in (x, w, b, r) if v is not None]
        leaves = [v.to(t).detach().requires_grad_() for v in live]

        def f(v):
            if gated:
                return gated_linear(*v, activation="silu")
            return linear_act(*v, activation="gelu")

        grads = torch.autograd.grad(f(leaves), leaves, dy.to(t))
        base = [v.detach().cpu().double() for v in live]
        D = dy.cpu().double()
        g = torch.Generator().manual_seed(7)
        for i, grad in enumerate(grads):
            way = torch.randn(base[i].shape, generator=g).double()
            h = 1e-6
            up = [v + h * way if j == i else v for j, v in enumerate(base)]
            dn = [v - h * way if j == i else v for j, v in enumerate(base)]
            want = ((f(up) - f(dn)) * D).sum() / (2 * h)
            got = (grad.cpu().double() * way).sum()
            # differences: 1e-6 of the size; each 16-bit entry: at most three
            # roundings (kept value, g, itself), of random sign
            size = (grad.cpu().double() * way).norm()
            rough = 3 * 4 * torch.finfo(t).eps / 2 * size
            assert abs(got - want) <= rough + 1e-6 * (size + abs(want))


@pytest.mark.parametrize("device", _devices())
def test_strides_and_leading_axes(device):
    x, w, b, r, dy = _make(60, 64, 48, BF16, device, 8, res=True)
    want = linear_act(x, w, b, r, activation="gelu")
    wide = torch.zeros(60, 200, dtype=BF16, device=device)
    for at in (0, 8, 3):  # aligned, aligned further on, not aligned
        wide[:, at:at + 64] = x
        assert torch.equal(linear_act(wide[:, at:at + 64], w, b, r,
                                      activation="gelu"), want)
    assert torch.equal(linear_act(x.t().contiguous().t(), w, b, r,
                                  activation="gelu"), want)
    assert torch.equal(linear_act(x, w.t().contiguous().t(), b, r,
                                  activation="gelu"), want)
    rw = torch.zeros(60, 51, dtype=BF16, device=device)
    rw[:, 1:49] = r
    assert torch.equal(linear_act(x, w, b, rw[:, 1:49], activation="gelu"),
                       want)
    x3, r3 = x.reshape(3, 4, 5, 64), r.reshape(3, 4, 5, 48)
    assert torch.equal(linear_act(x3, w, b, r3, activation="gelu"),
                       want.reshape(3, 4, 5, 48))
    assert torch.equal(linear_act(x[0], w, b, r[0], activation="gelu"),
                       linear_act(x[:1], w, b, r[:1], activation="gelu")[0])
    # a gradient that is one row for all, and one that lies by columns
    for d in (dy[:1].expand(60, 48), dy.t().contiguous().t()):
        _check(x, w, b, r, d, "gelu", False)
        _check(x, w, b, r, d, None, False)
    _check(x[:1].expand(60, 64), w, b, r, dy, "gelu", False)


@pytest.mark.parametrize("device", _devices())
def test_no_rows(device):
    w = torch.ones(6, 8, dtype=BF16, device=device, requires_grad=True)
    b = torch.ones(6, dtype=BF16, device=device, requires_grad=True)
    x = torch.empty(2, 0, 8, dtype=BF16, device=device, requires_grad=True)
    for y in (linear_act(x, w, b, activation="gelu"),
              gated_linear(x, w, b),
              gated_linear(x, w, b, checkpoint="8bit"),
              linear_act(x, w, b, checkpoint="8bit")):
        assert y.shape == (2, 0, y.shape[-1])
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert dx.shape == x.shape and not dw.any() and not db.any()
    e = torch.empty(0, 40, dtype=BF16, device=device)
    assert unpack_activation(pack_activation(e)).shape == (0, 40)
    e = torch.empty(3, 0, dtype=BF16, device=device)
    assert unpack_activation(pack_activation(e)).shape == (3, 0)


@pytest.mark.parametrize("device", _devices())
def test_not_finite_values_stay_in_their_rows(device):
    x, w, b, r, dy = _make(80, 72, 64, BF16, device, 9)
    want = linear_act(x, w, b, activation="gelu")
    x2 = x.clone()
    x2[3, 70] = float("nan")
    x2[77, 0] = float("inf")
    got = linear_act(x2, w, b, activation="gelu")
    rows = [i for i in range(80) if i not in (3, 77)]
    assert torch.equal(got[rows], want[rows])
    assert got[3].isnan().all() and not got[77].isfinite().all()
    w2 = w.clone()
    w2[5, 1] = float("nan")
    got = gated_linear(x, w2, b)
    assert got[:, 5].isnan().all()
    cols = [i for i in range(32) if i != 5]
    assert torch.equal(got[:, cols], gated_linear(x, w, b)[:, cols])


@pytest.mark.parametrize("device", _devices())
def test_large_values_reach_the_limits_of_the_activation(device):
    x = torch.tensor([[1e30], [-1e30], [200.0], [-200.0], [0.0]],
                     dtype=BF16, device=device, requires_grad=True)
    w = torch.ones(8, 1, dtype=BF16, device=device)
    for act in ("relu", "gelu", "silu"):
        y = linear_act(x, w, activation=act)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        x0 = x.detach()[:, :1]
        assert torch.equal(y[:, :1], x0.clamp(min=0)), act
        half = 0 if act == "relu" else 4
        assert dx.flatten().tolist() == [8, 0, 8, 0, half], act


# ---- 8 bits ------------------------------------------------------------------


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("t", [BF16, FP16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33),
                                   (64, 768), (2, 3, 200), (7, 4097), (40,)])
def test_pack_is_its_definition(shape, t, device):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(*shape, generator=g) * torch.exp(
        2 * torch.randn(shape[-1], generator=g))
    x = x.to(t)
    p = pack_activation(x.to(device))
    y = unpack_activation(p)
    assert y.shape == x.shape and y.dtype == t and y.device.type == device
    want = _kept8(x.reshape(-1, shape[-1]))[0].reshape(shape)
    most = torch.finfo(t).max
    assert torch.equal(y.cpu().double(),
                       want.clamp(-most, most).to(t).double())
    assert torch.equal(unpack_activation(p, torch.float32).cpu().double(),
                       want)
    rows = x.numel() // shape[-1]
    assert p.nbytes == rows * (-(-shape[-1] // 32) * 33)


@pytest.mark.parametrize("device", _devices())
def test_pack_every_16_bit_value(device):
    """Each of the 65536 patterns, in groups of one magnitude and mixed."""
    bits = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).short()
    for t in (BF16, FP16):
        v = bits.view(t)
        if t == BF16:  # below 2**-110 the GPU's float32 would be subnormal
            v = torch.where(v.float().abs() < 2.0 ** -110,
                            torch.zeros_like(v), v)
        mixed = v[torch.randperm(65536, generator=torch.Generator()
                                 .manual_seed(1))]
        for x in (v.reshape(-1, 32), mixed.reshape(-1, 64)):
            got = unpack_activation(pack_activation(x.to(device))).cpu()
            fine = x.isfinite()
            want = _kept8(torch.where(fine, x, torch.zeros_like(x)))[0]
            most = torch.finfo(t).max
            want = want.clamp(-most, most).to(t)
            assert torch.equal(got[fine], want[fine])
            assert got[~fine].isnan().all()


@pytest.mark.parametrize("device", _devices())
def test_pack_strided_rows(device):
    x = torch.randn(9, 100, generator=torch.Generator().manual_seed(2)
                    ).to(BF16).to(device)
    want = unpack_activation(pack_activation(x[:, 8:72].contiguous()))
    assert torch.equal(unpack_activation(pack_activation(x[:, 8:72])), want)
    assert torch.equal(
        unpack_activation(pack_activation(x.t()[8:72])),
        unpack_activation(pack_activation(x.t()[8:72].contiguous())))
    assert torch.equal(
        unpack_activation(pack_activation(x[:, 3:40])),
        unpack_activation(pack_activation(x[:, 3:40].contiguous())))


# ---- refusals ----------------------------------------------------------------


def test_refusals():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    b, r = torch.zeros(6), torch.zeros(4, 6)
    for wrong in (
            lambda: linear_act(x, w, activation="tanh"),
            lambda: linear_act(x, w, checkpoint="4bit"),
            lambda: linear_act(x, torch.zeros(6, 9)),
            lambda: linear_act(x, torch.zeros(8)),
            lambda: linear_act(x, torch.zeros(0, 8)),
            lambda: linear_act(torch.zeros(4, 0), torch.zeros(6, 0)),
            lambda: linear_act(torch.tensor(1.0), w),
            lambda: linear_act(x, w, torch.zeros(5)),
            lambda: linear_act(x, w, b[None]),
            lambda: linear_act(x, w, b, r[:1]),
            lambda: linear_act(x, w, b, torch.zeros(4, 5)),
            lambda: gated_linear(x, w, activation=None),
            lambda: gated_linear(x, torch.zeros(7, 8)),
            lambda: gated_linear(x, w, b[:3]),
            lambda: pack_activation(torch.tensor(1.0))):
        with pytest.raises(ValueError):
            wrong()
    for wrong in (
            lambda: linear_act(x, w.double()),
            lambda: linear_act(x, w, b.double()),
            lambda: linear_act(x, w, b, r.half()),
            lambda: linear_act(x.long(), w.long()),
            lambda: linear_act(x.double(), w.double(), checkpoint="8bit"),
            lambda: gated_linear(x.half(), w),
            lambda: pack_activation(x.double()),
            lambda: pack_activation(x.long()),
            lambda: unpack_activation(pack_activation(x), torch.int8)):
        with pytest.raises(TypeError):
            wrong()


@pytest.mark.parametrize("device", _devices())
def test_second_derivatives_are_refused(device):
    t = torch.float32 if device == "cpu" else BF16
    x = torch.randn(3, 8, device=device, dtype=t, requires_grad=True)
    w = torch.randn(6, 8, device=device, dtype=t, requires_grad=True)
    for leaf in (x, w):
        g, = torch.autograd.grad(linear_act(x, w, activation="gelu").sum(),
                                 leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


@pytest.mark.parametrize("device", _devices())
def test_changed_inputs_are_noticed(device):
    """What the backward pass needs must not have changed since."""
    t = torch.float32 if device == "cpu" else BF16
    x = torch.randn(3, 8, device=device, dtype=t)
    w = torch.randn(6, 8, device=device, dtype=t, requires_grad=True)
    y = linear_act(x, w, activation="gelu")
    x.zero_()
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(6, 8, device="cuda")
    with pytest.raises(TypeError):
        linear_act(x, w)
    with pytest.raises(TypeError):
        linear_act(x.half(), w.half().cpu())
    with pytest.raises(TypeError):
        gated_linear(x.double(), w.double())
    with pytest.raises(TypeError):
        linear_act(x.half(), w.half(), residual=torch.zeros(
            4, 6, dtype=FP16))
    x, w = x.half(), w.half()
    b = torch.zeros(6, device="cuda").half()
    for wrong in (
            lambda: linear_act(x, w, activation="tanh"),
            lambda: linear_act(x, w, checkpoint="4bit"),
            lambda: linear_act(x, w[:, :7]),
            lambda: linear_act(x, w[0]),
            lambda: linear_act(x, w[:0]),
            lambda: linear_act(x[0, 0], w),
            lambda: linear_act(x[:, :0], w[:, :0]),
            lambda: linear_act(x, w, b[:5]),
            lambda: linear_act(x, w, b[None]),
            lambda: linear_act(x, w, b, x),
            lambda: linear_act(x, w, b, b),
            lambda: gated_linear(x, w, activation=None),
            lambda: gated_linear(x, w[:5]),
            lambda: gated_linear(x, w, b[:3])):
        with pytest.raises(ValueError):
            wrong()
    with pytest.raises(TypeError):
        linear_act(x, w, b.float())
    with pytest.raises(TypeError):
        linear_act(x, w.bfloat16())


# ---- on the GPU alone ----------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,gated", [
    (4096, 128, 4096, False), (2100, 520, 3000, True), (700, 2048, 768, False),
    (24, 4096, 1024, False), (16, 2048, 1500, True), (3, 8192, 512, False),
    (2048, 256, 2050, True), (5000, 264, 272, False)])
def test_larger_sizes(m, k, n, gated):
    """Every tile size and split that the rules choose."""
    for t in (BF16, FP16):
        _check(*_make(m, k, n, t, "cuda", m, gated=gated, res=not gated),
               "silu", gated)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [
    (1, 2048, 40), (9, 1030, 33), (16, 8200, 40), (17, 64, 80),
    (31, 513, 16), (32, 4104, 72), (33, 200, 4097), (48, 1000, 100),
    (49, 520, 1000), (63, 40, 5000), (64, 3000, 30), (64, 1536, 9000)])
def test_few_rows(m, k, n):
    """Each count of 16 rows, k's that end inside a turn or give a wave none,
    and columns that end inside a block."""
    for t, gated in ((BF16, False), (FP16, True)):
        _check(*_make(m, k, n, t, "cuda", n, gated=gated, res=not gated),
               "gelu", gated)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_the_same_inputs_give_the_same_bits(gated):
    x, w, b, r, dy = _make(513, 777, 650, BF16, "cuda", 11, gated=gated)
    runs = []
    for _ in range(3):
        ls = [v.detach().requires_grad_() for v in (x, w, b)]
        y = (gated_linear(*ls) if gated else linear_act(*ls))
        runs.append([y, *torch.autograd.grad(y, ls, dy)])
    for one in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(one, runs[0]))


@pytest.mark.gpu
def test_neighbours_of_the_operands_are_not_read_or_written():
    """Operands in the middle of NaN: an out-of-range read that counts would
    show in the result, and the surroundings stay."""
    for m, k, n in ((70, 72, 136), (33, 50, 41), (130, 200, 264),
                    (5, 136, 96)):
        for gated in (False, True):
            x, w, b, r, dy = _make(m, k, n, BF16, "cuda", 12, gated=gated)
            held = []

            def inside(v):
                big = torch.full((v.numel() + 4096,), float("nan"),
                                 dtype=BF16, device="cuda")
                big[2048:2048 + v.numel()] = v.flatten()
                held.append((big, v.numel()))
                return big[2048:2048 + v.numel()].view(v.shape)

            _check(inside(x), inside(w), inside(b), None, inside(dy), "gelu",
                   gated)
            for big, count in held:
                assert big[:2048].isnan().all()
                assert big[2048 + count:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("k,n,gated,keep", [
    (32768, 64, False, None), (64, 32768, False, None),
    (64, 32768, False, "8bit"), (64, 32768, True, None)])
def test_more_than_2_to_31_values(k, n, gated, keep):
    """Small whole numbers: every sum is one below 2**24, exact in float32 in
    any order, and is rounded once.  In 8 bits, pre-activations of 64 at most
    keep their sign: one that is not 0 is 2**-6 of its group's largest at
    least."""
    m, part = 70016, 8752
    gen = torch.Generator("cuda").manual_seed(7)

    def whole(*shape):
        t = torch.empty(*shape, device="cuda", dtype=BF16)
        for a in range(0, shape[0], part):  # no larger temporary
            t[a:a + part] = torch.randint(-1, 2, t[a:a + part].shape,
                                          generator=gen, device="cuda")
        return t

    x, w, dy = whole(m, k), whole(n * (1 + gated), k), whole(m, n)
    b = torch.zeros(w.shape[0], device="cuda", dtype=BF16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    if gated:
        y = gated_linear(x, w, b, activation="relu", checkpoint=keep)
    else:
        y = linear_act(x, w, b, activation="relu", checkpoint=keep)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    want_w = torch.zeros(w.shape, device="cuda")
    want_b = torch.zeros(b.shape, device="cuda")
    with torch.no_grad():
        wide = w.float()
        for a in range(0, m, part):
            rows = slice(a, a + part)
            p, d = x[rows].float() @ wide.t(), dy[rows].float()
            if gated:
                g, u = p[:, :n], p[:, n:]
                assert torch.equal(y[rows], (g.clamp(min=0) * u).to(BF16))
                g = torch.cat([d * u * (g > 0), d * g.clamp(min=0)], 1)
            else:
                assert torch.equal(y[rows], p.clamp(min=0).to(BF16))
                g = d * (p > 0)
            assert torch.equal(dx[rows], (g @ wide).to(BF16))
            want_w += g.t() @ x[rows].float()
            want_b += g.sum(0)
        assert torch.equal(dw, want_w.to(BF16))
        assert torch.equal(db, want_b.to(BF16))
    if x.numel() > 2 ** 31:
        del y, dx, dw
        back = unpack_activation(pack_activation(x))
        for a in range(0, m, part):
            assert torch.equal(back[a:a + part], x[a:a + part])


@pytest.mark.gpu
def test_on_another_stream():
    x, w, b, r, dy = _make(600, 512, 768, BF16, "cuda", 13, gated=True)
    want = gated_linear(x, w, b)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = x * 1  # made on this stream: the layer has to wait for it
        got = gated_linear(late, w, b)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that overlap share no workspace: splits of k, copies of odd rows,
    few rows and training, each on its own stream, over and over."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = [_make(m, k, n, BF16, "cuda", m, gated=g)
            for m, k, n, g in ((600, 2049, 300, False), (40, 1111, 500, True),
                               (1500, 512, 264, True), (7, 4096, 96, False))]

    def step(i):
        x, w, b, _, dy = made[i]
        ls = [v.detach().requires_grad_() for v in (x, w, b)]
        y = (gated_linear(*ls) if i in (1, 2)
             else linear_act(*ls, activation="gelu"))
        return [y.detach(), *torch.autograd.grad(y, ls, dy)]

    want = [step(i) for i in range(len(made))]
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        for i in range(len(made)):
            s = streams[(turn + i) % 2]
            with torch.cuda.stream(s):
                got.append((i, step(i)))
    torch.cuda.synchronize()
    for i, out in got:
        for p, q in zip(out, want[i]):
            assert torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 24, 64])
def test_captured_few_rows(m):
    x, w, b, _, _ = _make(m, 1500, 700, BF16, "cuda", m, gated=True)
    v = torch.randn(1500, 700, device="cuda").to(BF16) / 26

    def block(x):
        with torch.no_grad():
            return linear_act(gated_linear(x, w, b), v, None, x)

    block(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = block(x)
    for _ in range(4):
        new = torch.randn(m, 1500, device="cuda").to(BF16)
        x.copy_(new)
        g.replay()
        assert torch.equal(out, block(new))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_captured_training_step():
    """A feed-forward block's step in a graph, replayed on new inputs, against
    the eager step; two graphs share nothing."""
    m, k, f = 96, 128, 192
    x, w1, b1, _, dy = _make(m, k, f, BF16, "cuda", 14, gated=True)
    _, w2, b2, _, dy = _make(m, f, k, BF16, "cuda", 15)
    ws = [v.requires_grad_() for v in (w1, b1, w2, b2)]

    def step(x, dy, keep):
        h = gated_linear(x, ws[0], ws[1], checkpoint=keep)
        y = linear_act(h, ws[2], ws[3], x, checkpoint=keep)
        return [y.detach(), *torch.autograd.grad(y, ws, dy)]

    graphs = []
    for keep in (None, "8bit"):
        sx, sdy = x.clone(), dy.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                step(sx, sdy, keep)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(sx, sdy, keep)
        graphs.append((g, sx, sdy, out, keep))
    for i in range(4):
        nx = torch.randn(m, k, device="cuda").to(BF16)
        nd = torch.randn(m, k, device="cuda").to(BF16)
        for g, sx, sdy, out, keep in graphs:
            sx.copy_(nx), sdy.copy_(nd)
            g.replay()
        for g, sx, sdy, out, keep in graphs:
            for p, q in zip(out, step(nx, nd, keep)):
                assert torch.equal(p, q)
        torch.cuda.synchronize()


# ---- the operators together ------------------------------------------------------


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("m,k,f", [(1, 64, 96), (70, 96, 200), (300, 130, 77)])
def test_block_against_float64(m, k, f, device):
    """A gated block with its residual, forward and backward, the second
    layer's bounds resting on the first's."""
    t = BF16
    x, w1, b1, _, _ = _make(m, k, f, t, device, 20, gated=True)
    _, w2, b2, _, dy = _make(m, f, k, t, device, 21)
    ls = [v.detach().requires_grad_() for v in (x, w1, b1, w2, b2)]
    h = gated_linear(*ls[:3], activation="silu")
    y = linear_act(h, ls[3], ls[4], ls[0])
    got = torch.autograd.grad(y, ls, dy)
    X, W1, B1, W2, B2, D = (v.detach().cpu().double()
                            for v in (x, w1, b1, w2, b2, dy))
    # forward
    P = X @ W1.t() + B1
    ep = (k + 8) * _H * (X.abs() @ W1.abs().t() + B1.abs())
    A, U, ea, eu = P[:, :f], P[:, f:], ep[:, :f], ep[:, f:]
    F = _act(A, "silu")
    Hh = F * U
    eh = 1.13 * ea * (U.abs() + eu) + F.abs() * eu + 8 * _H * Hh.abs()
    eh = 1.01 * (eh + _round(Hh, t))
    Y = Hh @ W2.t() + B2 + X
    HM = Hh.abs() + eh
    ey = eh @ W2.abs().t() + (f + 16) * _H * (HM @ W2.abs().t() + B2.abs()
                                              + X.abs())
    _within(y, Y, 1.01 * (ey + _round(Y, t)), "y")
    # backward
    _within(got[4], D.sum(0), (m + 8) * _H * D.abs().sum(0)
            + _round(D.sum(0), t), "db2")
    dW2 = D.t() @ Hh
    _within(got[3], dW2, 1.01 * (D.abs().t() @ eh + (m + 8) * _H
                                 * (D.abs().t() @ HM) + _round(dW2, t)),
            "dw2")
    dH = D @ W2
    ed = (k + 8) * _H * (D.abs() @ W2.abs())
    ed = 1.01 * (ed + _round(dH, t))
    sa = _slope(A, "silu")
    es = 1.01 * (ea + 2.0 ** -16 * A.abs()) + 8 * _H   # kept in 24 bits
    eu = 1.01 * (eu + 2.0 ** -16 * U.abs())
    G = torch.cat([dH * U * sa, dH * F], 1)
    DM = dH.abs() + ed
    eg = torch.cat([
        ed * (U * sa).abs() + DM * (eu * (sa.abs() + es) + U.abs() * es),
        ed * F.abs() + DM * (1.13 * es + 8 * _H * F.abs())], 1)
    eg = 1.01 * eg + 8 * _H * G.abs()
    er = eg + 1.01 * _round(G, t)
    GM = G.abs() + er
    dW1 = G.t() @ X
    _within(got[1], dW1, 1.01 * (er.t() @ X.abs() + (m + 8) * _H
                                 * (GM.t() @ X.abs()) + _round(dW1, t)),
            "dw1")
    dB1 = G.sum(0)
    _within(got[2], dB1, 1.01 * (eg.sum(0) + (m + 8) * _H * GM.sum(0)
                                 + _round(dB1, t)), "db1")
    # x: through the layers, rounded, plus the residual's dy, rounded
    dX1 = G @ W1
    e1 = er @ W1.abs() + (2 * f + 8) * _H * (GM @ W1.abs()) + _round(dX1, t)
    _within(got[0], dX1 + D, 1.01 * (e1 + _round(dX1.abs() + D.abs(), t)),
            "dx")


def _bert(**kw):
    from rocps.models.bert import bert_base
    torch.manual_seed(3)
    return bert_base(layers=2, hidden=64, heads=4, intermediate=96, vocab=300,
                     max_pos=32, **kw)


def test_bert_with_a_gated_block():
    """The model's gradients against the same model of torch operations."""
    import torch.nn.functional as F

    from rocps.models.bert import BertLayer
    ids = torch.randint(0, 300, (3, 16), generator=torch.Generator()
                        .manual_seed(4))
    for ff, act in (("geglu", lambda v: F.gelu(v, approximate="tanh")),
                    ("swiglu", F.silu)):
        m = _bert(feed_forward=ff)
        assert m.layers[0].fc1.weight.shape == (192, 64)
        m.loss(ids, ids).backward()
        own = [p.grad.clone() for p in m.parameters()]
        m.zero_grad()

        def composed(self, x):
            a, u = self.fc1(x).chunk(2, dim=-1)
            return self.fc2(act(a) * u) + x

        old = BertLayer._feed_forward
        try:
            BertLayer._feed_forward = composed
            m.loss(ids, ids).backward()
        finally:
            BertLayer._feed_forward = old
        for a, p in zip(own, m.parameters()):
            # float32 on both sides: some hundred roundings of 2**-24
            assert (a - p.grad).norm() <= 1e-5 * p.grad.norm() + 1e-9


def test_bert_act_checkpoint_keeps_the_output():
    ids = torch.randint(0, 300, (3, 16), generator=torch.Generator()
                        .manual_seed(5))
    for ff in ("gelu", "geglu"):
        plain, small = _bert(feed_forward=ff), _bert(feed_forward=ff,
                                                     act_checkpoint="8bit")
        assert list(plain.state_dict()) == list(small.state_dict())
        a, b = plain.loss(ids, ids), small.loss(ids, ids)
        assert abs(a - b) <= 1e-5 * abs(a)
        a.backward(), b.backward()
        for p, q in zip(plain.parameters(), small.parameters()):
            # a kept value is off by 2**-4 at most and 2**-4 / sqrt(3) in the
            # mean square; a gradient here meets at most eight of them (two
            # layers, two products each, an input and a slope): sqrt(8) times
            # that is a tenth
            assert (p.grad - q.grad).norm() <= 0.25 * p.grad.norm() + 1e-9
    with pytest.raises(ValueError):
        _bert(feed_forward="relu")
    with pytest.raises(ValueError):
        _bert(act_checkpoint="4bit")


@pytest.mark.gpu
@pytest.mark.parametrize("ff", ["gelu", "geglu", "swiglu"])
@pytest.mark.parametrize("keep", [None, "8bit"])
def test_bert_trains_on_the_gpu(ff, keep):
    from rocps.engine.comm import Comm
    from rocps.engine.sync_engine import SyncEngine
    from rocps.train.optimizer import AdamOptimizer
    m = _bert(feed_forward=ff, act_checkpoint=keep).cuda().bfloat16()
    before = [p.detach().clone() for p in m.layers.parameters()]
    eng = SyncEngine(m, Comm(device=torch.device("cuda:0")))
    opt = AdamOptimizer(1e-2)
    ids = torch.randint(0, 300, (4, 16), device="cuda")
    for _ in range(2):
        eng.zero_grad()
        opt.begin_step()
        loss = m.loss(ids, ids)
        eng.step(loss, opt)
    torch.cuda.synchronize()
    assert torch.isfinite(loss.detach())
    for p, q in zip(before, m.layers.parameters()):
        assert q.isfinite().all() and not torch.equal(p, q)
