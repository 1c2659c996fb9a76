"""Every kernel that the rules of the feed-forward products can choose, against
the exact result.

A tile, what it keeps, a split and its join, and the backward pass's pairs are
each a kernel of their own.  SHAPES lead to every one of them, which the first
test holds the list to: it compiles the rules for the host and asks them.

The operands are -1, 0 and 1.  Sums are then whole numbers below 2**24, exact
in float32 in any order; in 8 bits such sums are held as whole numbers of four
binary digits, by their definition.  So a result of relu has one right value,
and so has each gradient of it.  The bounds of the other activations are
derived beside them."""

import ctypes
import math
import os
import shutil
import subprocess

import pytest
import torch

from rocps.ops.gated import gated_linear
from rocps.ops.linear import linear_act
from test_feed_forward import _H, _act, _kept8, _round

BF16, FP16 = torch.bfloat16, torch.float16
TILES = {(256, 256), (256, 128), (128, 192), (128, 128), (64, 128), (64, 64)}

SHAPES = [  # rows, k, n, gated
    (65, 1265, 41, False), (331, 74, 2565, True), (393, 65, 2765, True),
    (6818, 333, 66, False), (7273, 139, 449, False), (398, 258, 8370, False),
    (1431, 196, 3857, False), (781, 2785, 386, True), (1429, 42, 226, True),
    (1193, 529, 4374, False), (387, 1876, 4908, True), (7084, 834, 854, True),
    (16563, 2212, 205, False), (4122, 853, 2972, False),
    (2289, 7397, 909, False), (1025, 5764, 1053, False),
    (1955, 948, 4103, True), (3450, 2957, 1667, False),
    (130, 10619, 5879, True),
]

_HOST = """
#include "tile_choice.h"
extern "C" void tile(int i, long* o) {
  o[0] = ff::tile_cost(i).bm, o[1] = ff::tile_cost(i).bn;
}
extern "C" int tiles() { return ff::kTiles; }
extern "C" void forward(long m, long width, long k, int gated, int keep,
                        long* o) {
  auto c = ff::choose_tile(m, width, k, gated, keep);
  o[0] = c.tile, o[1] = c.splits;
}
extern "C" void backward(long m, long outs, long k, long* o) {
  const long ms[2] = {m, outs}, ns[2] = {k, k}, ks[2] = {outs, m};
  auto c = ff::choose_pair(ms, ns, ks);
  o[0] = c.tile, o[1] = c.splits[0], o[2] = c.splits[1],
  o[3] = c.second_first;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_the_shapes_lead_to_every_kernel(tmp_path):
    src, lib = tmp_path / "host.cc", tmp_path / "host.so"
    src.write_text(_HOST)
    kernels = os.path.join(os.path.dirname(__file__), "..", "csrc", "kernels")
    subprocess.run(["g++", "-shared", "-fPIC", "-I", kernels, str(src), "-o",
                    str(lib)], check=True)
    host = ctypes.CDLL(str(lib))
    out = (ctypes.c_long * 4)()

    def ask(f, *a):
        f(*(ctypes.c_long(v) for v in a), out)
        return list(out)

    sizes = [tuple(ask(host.tile, i)[:2]) for i in range(host.tiles())]
    assert set(sizes) == TILES
    halves = TILES - {(128, 192), (64, 64)}  # no two runs of whole 32 columns
    want = {("forward", s, False, keep) for s in TILES for keep in range(3)}
    want |= {("forward", s, True, keep) for s in halves for keep in range(3)}
    want |= {("split", s) for s in TILES}
    want |= {("join", g, keep) for g in (False, True) for keep in range(3)}
    want |= {("backward", s, swap) for s in TILES for swap in (0, 1)}
    want |= {("pair", a, b, swap) for a in (False, True)
             for b in (False, True) for swap in (0, 1)}
    got = set()
    for m, k, n, gated in SHAPES:
        outs = n * (1 + gated)
        for keep in range(3):
            tile, splits = ask(host.forward, m, outs, k, gated, keep)[:2]
            got |= ({("forward", sizes[tile], gated, keep)} if splits == 1 else
                    {("split", sizes[tile]), ("join", gated, keep)})
        tile, a, b, swap = ask(host.backward, m, outs, k)
        got |= {("backward", sizes[tile], swap), ("pair", a > 1, b > 1, swap)}
    assert got == want, (want - got, got - want)


def _argument(v, act):
    """What the activation's sigmoid is taken of."""
    if act == "gelu":
        return 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("t", [BF16, FP16])
@pytest.mark.parametrize("m,k,n,gated", SHAPES)
def test_each_kernel_exactly(m, k, n, gated, t):
    gen = torch.Generator("cuda").manual_seed(m)

    def whole(*shape):
        return torch.randint(-1, 2, shape, generator=gen, device="cuda").to(t)

    x, w, dy = whole(m, k), whole(n * (1 + gated), k), whole(m, n)
    b = whole(w.shape[0])
    r = None if gated else whole(m, n)
    wide = {"x": x.float(), "w": w.float(), "d": dy.float()}
    p = wide["x"] @ wide["w"].t() + b.float()
    assert p.abs().max() < 2048  # kept in 16 bits, fp16 exactly

    def layer(v, act, keep=None):
        if gated:
            return gated_linear(v[0], v[1], v[2], activation=act,
                                checkpoint=keep)
        return linear_act(*v, activation=act, checkpoint=keep)

    def check_forward(y, act, what):
        P = p.double()
        a, u = P.chunk(2, 1) if gated else (P, None)
        Y = _act(a, act) * (u if gated else 1)
        # the sigmoid's argument has four roundings, each of which moves the
        # sigmoid by 1 less itself of so much; 8 for the rest.  A sigmoid below
        # 2**-126 is flushed to 0 (the kernels are compiled so) before a and u
        # multiply it: silu of -88 is 88 * 6.1e-39, and is lost.
        e = torch.zeros_like(Y)
        if act in ("gelu", "silu"):
            arg = _argument(a, act)
            e = Y.abs() * _H * (8 + 4 * arg.abs() * torch.sigmoid(-arg))
            e = e + 2.0 ** -126 * (a * u if gated else a).abs()
        if r is not None:
            Y = Y + r.double()
        if not e.any():
            assert torch.equal(y, Y.float().to(t)), what
            return
        e = 1.001 * e + _H * Y.abs() + 1.001 * _round(Y, t)
        worst = ((y.double() - Y).abs() / e).max().item()
        assert worst <= 1, f"{what}: {worst:.3g} times its bound"

    v = [x, w, b] + ([] if gated else [r])
    for act in (["relu", "gelu", "silu"] + ([] if gated else [None])):
        check_forward(layer(v, act), act, f"{act}, nothing kept")

    for keep in (None, "8bit"):
        ls = [q.detach().requires_grad_() for q in v]
        for act in ("gelu", "silu"):
            check_forward(layer(ls, act, keep).detach(), act, f"{act}, {keep}")
        y = layer(ls, "relu", keep)
        check_forward(y.detach(), "relu", f"relu, {keep}")
        grads = torch.autograd.grad(y, ls, dy)
        a, u = p.chunk(2, 1) if gated else (p, None)
        if keep == "8bit":  # x, of -1, 0 and 1, is held as it is
            # (on the CPU, whose powers of two are exact; the GPU's are not)
            a = _kept8(a.cpu())[0].float().cuda()
            u = _kept8(u.cpu())[0].float().cuda() if gated else None
        d = wide["d"]
        g = d * (a > 0)
        if gated:
            g = torch.cat([g * u, d * a.clamp(min=0)], 1)
        seen = g.to(t).float()  # by the products
        assert torch.equal(grads[0], (seen @ wide["w"]).to(t)), f"dx, {keep}"
        assert torch.equal(grads[1], (seen.t() @ wide["x"]).to(t)), \
            f"dw, {keep}"
        assert torch.equal(grads[2], g.sum(0, dtype=torch.float64).float()
                           .to(t)), f"db, {keep}"
        if not gated:
            assert torch.equal(grads[3], dy)
