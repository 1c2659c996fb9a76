"""The feed-forward operators at the ends of their types and of what they
take: values past the kept type's range, derivatives that they do not have,
lengths at their limits, and every kernel that a choice can lead to."""

import pytest
import torch

from rocps.ops.act8 import pack_activation, unpack_activation
from rocps.ops.gated import gated_linear
from rocps.ops.linear import linear_act
from test_feed_forward import _H, _act, _kept8, _round, _slope

BF16, FP16 = torch.bfloat16, torch.float16


def _devices():
    return ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("keep", [None, "8bit"])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_slopes_past_the_kept_types_range(act, keep, device):
    """Pre-activations of +-80000 are finite in float32 and infinite in
    float16, the type that they are kept in.  There the slope is 1 or 0, and
    the gradients are sums of a few whole numbers: exact in any order."""
    k, n = 8, 16
    s = torch.tensor([1.0, -1.0, 1.0, -1.0])
    x = (100 * s)[:, None].expand(4, k).to(FP16).to(device).contiguous()
    w = torch.full((n, k), 100.0, dtype=FP16, device=device)
    b = torch.zeros(n, dtype=FP16, device=device)
    ls = [v.requires_grad_() for v in (x, w, b)]
    y = linear_act(*ls, activation=act, checkpoint=keep)
    assert torch.equal(y[1::2], torch.zeros_like(y[1::2]))
    assert (y[::2] == float("inf")).all()  # past float16
    dx, dw, db = torch.autograd.grad(y, ls, torch.ones_like(y))
    assert torch.equal(dx[::2], torch.full_like(dx[::2], n * 100.0))
    assert torch.equal(dx[1::2], torch.zeros_like(dx[1::2]))
    # two rows of slope 1
    if keep is None:
        assert torch.equal(dw, torch.full_like(dw, 200.0))
    else:  # 100 * 2**2 lies halfway between 384 and 416 and goes to the even
        assert torch.equal(dw, torch.full_like(dw, 192.0))
    assert torch.equal(db, torch.full_like(db, 2.0))


@pytest.mark.parametrize("device", _devices())
def test_slopes_pass_not_a_number_on(device):
    x = torch.tensor([[float("nan")], [1.0]], dtype=FP16, device=device,
                     requires_grad=True)
    w = torch.ones(8, 1, dtype=FP16, device=device)
    for act in ("gelu", "silu"):
        y = linear_act(x, w, activation=act)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert dx[0].isnan().all() and dx[1].isfinite().all(), act


@pytest.mark.gpu
@pytest.mark.parametrize("k", [2 ** 22 - 7, 2 ** 22 - 1, 2 ** 22])
def test_rows_that_are_too_long_are_refused(k):
    """Filled to whole 16 bytes, these have 2**22 values; a tile's 256 rows of
    them would pass the extent that its loads are checked against."""
    x = torch.zeros(1, k, dtype=BF16, device="cuda")
    for m in (1, 65):
        with pytest.raises(RuntimeError, match="too long"):
            linear_act(x.expand(m, k), x)
    with pytest.raises(RuntimeError, match="too long"):
        linear_act(x.clone().requires_grad_(), x, checkpoint="8bit")


@pytest.mark.gpu
def test_the_longest_rows():
    """Values of -1, 0 and 1: every sum is a whole number below 2**24, exact
    in float32 in any order, and those of the gradients are at most 256."""
    k, m, part = 2 ** 22 - 8, 256, 2 ** 19
    gen = torch.Generator("cuda").manual_seed(1)

    def whole(*shape):
        t = torch.empty(shape, dtype=torch.int8, device="cuda")
        return t.random_(-1, 2, generator=gen).to(BF16)

    x, w, dy = whole(m, k), whole(m, k), whole(m, m)
    few = linear_act(x[:3], w)
    y = linear_act(x.requires_grad_(), w.requires_grad_())
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = torch.zeros(m, m, device="cuda")
    d = dy.float()
    with torch.no_grad():
        for a in range(0, k, part):
            xs, ws = x[:, a:a + part].float(), w[:, a:a + part].float()
            want += xs @ ws.t()
            assert torch.equal(dx[:, a:a + part].float(), d @ ws)
            assert torch.equal(dw[:, a:a + part].float(), d.t() @ xs)
    assert torch.equal(y.float(), want.to(BF16).float())
    assert torch.equal(few, y[:3])


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("grads", [False, True])
def test_forward_mode_is_refused(grads, device):
    """A tangent of any input raises; it is never dropped."""
    import torch.autograd.forward_ad as forward

    def inputs(gated):
        shapes = [(4, 8), (12, 8), (12,), (4, 12)][:3 if gated else 4]
        return [torch.ones(s, dtype=BF16, device=device) for s in shapes]

    for gated in (False, True):
        layer = gated_linear if gated else linear_act
        for i in range(3 if gated else 4):
            v = inputs(gated)
            with forward.dual_level():
                v[i] = forward.make_dual(v[i], torch.ones_like(v[i]))
                if grads:
                    for j, t in enumerate(v):
                        if j != i:
                            t.requires_grad_()
                with pytest.raises(NotImplementedError):
                    layer(*v)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    layer(*v)
        layer(*inputs(gated))


@pytest.mark.gpu
@pytest.mark.parametrize("act,gated", [(None, False), ("relu", False),
                                       ("relu", True)])
def test_features_that_no_backward_pass_takes(act, gated):
    """More than 2**22 - 8 rows of the weight: used without gradients, refused
    before the forward pass with them, and at the limit trained.  Whole
    numbers below 2**24 are exact in float32."""
    def run(x, w):
        if gated:
            return gated_linear(x, w, activation=act)
        return linear_act(x, w, activation=act)

    gen = torch.Generator("cuda").manual_seed(2)
    for outs in (2 ** 22 - 8, 2 ** 22 - 6, 2 ** 22):
        w = torch.randint(-1, 2, (outs, 1), generator=gen, device="cuda")
        w = w.to(BF16)
        x = torch.tensor([[1.0], [-2.0], [0.0]], dtype=BF16, device="cuda")
        p = x.float() @ w.t().float()
        a, u = (p.chunk(2, 1) if gated else (p, None))
        want = a.clamp(min=0) if act else a
        y = run(x, w)
        assert torch.equal(y.float(), want * u if gated else want)
        ls = [x.requires_grad_(), w.requires_grad_()]
        if outs > 2 ** 22 - 8:
            with pytest.raises(RuntimeError, match="too many"):
                run(x, w)
            assert run(x[:0], w).shape == (0, y.shape[1])
            continue
        dx, dw = torch.autograd.grad(run(x, w), ls, torch.ones_like(y))
        s = (a > 0).float() if act else torch.ones_like(a)
        g = torch.cat([u * s, want], 1) if gated else s
        with torch.no_grad():
            assert torch.equal(dx.float(), (g @ w.float()).to(BF16).float())
            assert torch.equal(dw.float(), g.t() @ x.float())


def test_dist_train_refuses_what_the_gpu_does_not_run():
    """A gated block or 8-bit checkpoints in fp32 on a GPU: the script says so
    before it starts a server.  (torch is told that there is a GPU.)"""
    import os
    import subprocess
    import sys
    root = os.path.join(os.path.dirname(__file__), "..")

    def run(code, *args):
        return subprocess.run(
            [sys.executable, "-c", "import runpy, sys, torch\n" + code, *args],
            cwd=root, capture_output=True, text=True, timeout=120)

    r = run("torch.cuda.is_available = lambda: True\n"
            "runpy.run_path('examples/dist_train.py', run_name='__main__')",
            "--model=bert_base", "--dtype=fp32", "--feed_forward=geglu",
            "--job_name=worker", "--worker_hosts=127.0.0.1:1")
    assert r.returncode != 0 and "--dtype=bf16" in r.stderr, r.stderr
    r = run("args = runpy.run_path('examples/dist_train.py')['bert_args']\n"
            "for gpu in (False, True):\n"
            "    for dtype in ('bf16', 'fp32'):\n"
            "        for ff in ('gelu', 'geglu', 'swiglu'):\n"
            "            for keep in ('', '8bit'):\n"
            "                try:\n"
            "                    kw = args(ff, keep, dtype, gpu)\n"
            "                    wide = kw.get('intermediate', 0)\n"
            "                    assert kw['act_checkpoint'] == (keep or None)\n"
            "                    assert wide == (0 if ff == 'gelu' else 2048)\n"
            "                    print('y', end='')\n"
            "                except ValueError:\n"
            "                    print('n', end='')\n")
    assert r.stdout == 18 * "y" + "y" + 5 * "n", r.stderr


def _held(v):
    """What 8 bits give back of v: its finite values by their definition, the
    others as NaN."""
    fine = v.isfinite()
    return torch.where(fine, _kept8(torch.where(fine, v, 0.0))[0],
                       float("nan"))


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("m,k,n,gated", [
    (70, 64, 48, False), (70, 64, 48, True), (300, 72, 136, False),
    (66, 1334, 40, False), (72, 1160, 33, True)])  # the last two: k split
def test_infinite_pre_activations_in_8_bits(m, k, n, gated, device):
    """Products of 2**100 and +-2**100 make two columns of the odd rows
    infinite; their neighbours in the group of 32 are kept as if they were not
    there, and only gradients that use them are NaN.  Everything else is a
    whole number of eighths, exact in float32."""
    gen = torch.Generator().manual_seed(k)
    outs = 2 * n if gated else n

    def whole(a, b, *s):
        return torch.randint(a, b, s, generator=gen).double()

    X, W = whole(-9, 10, m, k), whole(-1, 2, outs, k) / 8
    D = torch.randn(m, n, generator=gen).to(BF16).double()
    W[:, 0], X[:, 0] = 0, 0
    W[5, 0], W[n + 6 if gated else 6, 0] = 2.0 ** 100, -2.0 ** 100
    X[1::2, 0] = 2.0 ** 100
    P = X @ W.t()
    P[P.abs() > 2.0 ** 128] *= float("inf")
    assert (~P.isfinite()).sum() == 2 * (m // 2)
    x, w, dy = (v.to(BF16).to(device) for v in (X, W, D))
    ls = [x.requires_grad_(), w.requires_grad_()]
    if gated:
        y = gated_linear(*ls, activation="silu", checkpoint="8bit")
    else:
        y = linear_act(*ls, activation="silu", checkpoint="8bit")
    got = torch.autograd.grad(y, ls, dy)
    odd = torch.zeros(m, n, dtype=torch.bool)
    odd[1::2, 5] = odd[1::2, 6] = True
    assert torch.equal(~y.detach().cpu().isfinite(), odd)

    X8 = _held(X)
    if gated:
        A, U = _held(P[:, :n]), _held(P[:, n:])
        G = torch.cat([D * U * _slope(A, "silu"), D * _act(A, "silu")], 1)
    else:
        G = D * _slope(_held(P), "silu")
    eg = _round(G, BF16) * 1.01 + 16 * _H * G.abs() + 16 * _H * D.abs().repeat(
        1, outs // n)
    GM = G.abs() + eg
    for what, g, want, bound in (
            ("dx", got[0], G @ W, eg @ W.abs()
             + (outs + 8) * _H * (GM @ W.abs())),
            ("dw", got[1], G.t() @ X8, eg.t() @ X8.abs()
             + (m + 8) * _H * (GM.t() @ X8.abs()))):
        g = g.cpu().double()
        lost = want.isnan()
        assert lost.any() and not lost.all()
        assert torch.equal(g.isnan(), lost), what
        bound = bound + _round(want, BF16)
        worst = ((g - want).abs() / bound)[~lost].max()
        assert worst <= 1, f"{what}: {worst:.3g} times its bound"


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("gated", [False, True])
def test_not_a_number_in_a_row_in_8_bits(gated, device):
    """A row of NaN stays one: the other rows' results and gradients keep
    their bits, and the weight's gradient, a sum over all, is NaN."""
    gen = torch.Generator().manual_seed(3)
    m, k, n = 80, 72, 50
    x = torch.randn(m, k, generator=gen).to(BF16).to(device)
    w = torch.randn(n * (1 + gated), k, generator=gen).to(BF16).to(device)
    runs = []
    for spoil in (False, True):
        v = x.clone()
        if spoil:
            v[3, 70] = float("nan")
        ls = [v.requires_grad_(), w.clone().requires_grad_()]
        if gated:
            y = gated_linear(*ls, checkpoint="8bit")
        else:
            y = linear_act(*ls, activation="gelu", checkpoint="8bit")
        runs.append([y.detach(), *torch.autograd.grad(y, ls,
                                                      torch.ones_like(y))])
    rows = [i for i in range(m) if i != 3]
    for a, b in zip(runs[0][:2], runs[1][:2]):
        assert torch.equal(a[rows], b[rows])
        assert b[3].isnan().all() and not a.isnan().any()
    assert runs[1][2].isnan().all() and not runs[0][2].isnan().any()


@pytest.mark.parametrize("device", _devices())
@pytest.mark.parametrize("t", [BF16, torch.float32])
def test_pack_the_smallest_values(t, device):
    """Down to the type's subnormals, where the scale is at its least, 2**-118:
    off by 2**-4 of the value or 2**-10 of the scale, and on the GPU, where
    float32 below 2**-126 counts as 0, by that (before and after)."""
    e = torch.arange(-150, -100).double()
    v = (2.0 ** e)[:, None] * torch.tensor([1.0, -1.25, 1.5, 1.9375]).double()
    x = v.reshape(-1, 8).float().to(t)
    v = x.double()
    y = unpack_activation(pack_activation(x.to(device))).cpu().double()
    bound = torch.maximum(v.abs() * 2.0 ** -4, torch.tensor(2.0 ** -128))
    if device == "cuda":
        bound = bound + 2 * 2.0 ** -126
    # a group is a row here, and its scale is its own: at most 448 * 2**e
    top = v.abs().amax(1, keepdim=True)
    bound = torch.maximum(bound, top / 224 * 2.0 ** -10)
    assert ((y - v).abs() <= bound).all()
    assert torch.equal(y[v == 0], v[v == 0])
