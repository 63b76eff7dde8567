"""Rotary positions on the device (swq_rope_table, swq_rope) against their definitions in 64 bits.

Bars.  Tables: 4 * 2^-24 times the magnitude: the fraction of a turn is exact to 2^-30, sine and cosine to two units in
the last place, and two roundings follow.  Turned heads in f32: an element is x (scale w) c - y (scale w) s, six roundings
and a sum of squares of up to 512 terms (a tree of 9 levels, or a lane's 16 in a row): 16 * 2^-24 of its pair's size.  bf16: 2^-8 of the
value more."""

import math

import pytest
import torch

from swiftlet_amd._lib import SwqError
from swiftlet_amd.rope import RopeGPU, RopeScaling

pytestmark = pytest.mark.gpu


def frequencies(rot, theta, sc):
    """f_j and the magnitude, one pair after another."""
    out = []
    for j in range(rot // 2):
        t = theta * sc.factor ** (rot / (rot - 2)) if sc and sc.kind == "ntk" else theta
        f = t ** (-2 * j / rot)
        if sc and sc.kind == "linear":
            f /= sc.factor
        if sc and sc.kind == "yarn":
            lo, hi = (rot * math.log(sc.original_positions / (2 * math.pi * n)) / (2 * math.log(theta)) for n in (sc.beta_fast, sc.beta_slow))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
            x = min(max((j - lo) / max(hi - lo, 0.001), 0), 1)
            f = f * (1 - x) + f / sc.factor * x
        out.append(f)
    size = 1.0
    if sc and sc.kind == "yarn":
        size = sc.magnitude or (1 + 0.1 * math.log(sc.factor) if sc.factor > 1 else 1.0)
    return torch.tensor(out, dtype=torch.float64), size


SCALINGS = [None, RopeScaling("linear", 4.0), RopeScaling("ntk", 8.0), RopeScaling("yarn", 4.0, 262144), RopeScaling("yarn", 40.0, 4096, 16.0, 2.0),
            RopeScaling("yarn", 2.5, 32768, magnitude=1.25), RopeScaling("yarn", 0.5, 4096), RopeScaling("linear", 1.3)]


@pytest.mark.parametrize("sc", SCALINGS, ids=lambda s: "plain" if s is None else f"{s.kind}{s.factor}")
@pytest.mark.parametrize("rot,theta", [(64, 1e7), (128, 1e4), (6, 5e5), (512, 1e6)])
def test_table(rot, theta, sc):
    r = RopeGPU(rot, theta, scaling=sc)
    freq, size = frequencies(rot, theta, sc)
    given = torch.tensor([0, 1, 2, 77, 4095, 100001, 262143, 1 << 20, 5, 5], dtype=torch.int32, device="cuda")
    for pos, got in ((given.cpu().double(), r.table(given)), (torch.arange(3000, 3007).double(), r.table(first=3000, count=7))):
        ang = pos[:, None] * freq
        want = torch.stack([ang.cos(), ang.sin()], -1) * size
        assert got.shape == want.shape and float((got.cpu().double() - want).abs().max()) < 4 * 2.0 ** -24 * size


def test_no_positions():
    r = RopeGPU(64, 1e7)
    assert r.table(first=9, count=0).shape == (0, 32, 2)
    assert r.table(torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 32, 2)


def test_many_positions():
    """A table of 2 GB, the last rows right."""
    r = RopeGPU(64, 1e7)
    t = r.table(first=0, count=(1 << 23) + 3)
    at = torch.tensor([(1 << 23) + 2], dtype=torch.int32, device="cuda")
    assert torch.equal(t[-1:], r.table(at))


def turned(x, table, rows, layout, rot, w, eps, inverse):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    t = table.double()[rows.long().clamp(0, len(table) - 1)] if rows is not None else table.double()[:len(x)]
    c, s = t[:, None, :, 0], t[:, None, :, 1] * (-1 if inverse else 1)
    a, b = (y[..., :rot // 2], y[..., rot // 2:rot]) if layout == "half" else (y[..., 0:rot:2], y[..., 1:rot:2])
    u, v = a * c - b * s, b * c + a * s
    z = y.clone()
    size = y.abs().clone()
    both = (a.abs() + b.abs()) * (c.abs() + s.abs())
    if layout == "half":
        z[..., :rot // 2], z[..., rot // 2:rot] = u, v
        size[..., :rot // 2], size[..., rot // 2:rot] = both, both
    else:
        z[..., 0:rot:2], z[..., 1:rot:2] = u, v
        size[..., 0:rot:2], size[..., 1:rot:2] = both, both
    return z, size


def check(got, x, table, rows, layout, rot, w=None, eps=1e-6, inverse=False):
    want, size = turned(x, table, rows, layout, rot, w, eps, inverse)
    allowed = 16 * 2.0 ** -24 * size + (want.abs() * 2.0 ** -8 if got.dtype == torch.bfloat16 else 0) + 1e-38
    assert bool(((got.double() - want).abs() <= allowed).all()), float(((got.double() - want).abs() / allowed).max())


def inputs(N, heads, hd, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xs = [torch.randn((N, h, hd), generator=g, device="cuda").to(dtype) for h in heads]
    return g, xs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(256, 64), (128, 128), (64, 32), (16, 6), (5, 2), (2, 2), (96, 96), (512, 512), (511, 510), (80, 24), (320, 64), (257, 100)])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
def test_heads(hd, rot, layout, dtype, norm):
    for N, heads in ((1, [3]), (37, [16, 2]), (5, [1, 7, 2, 1])):
        g, xs = inputs(N, heads, hd, dtype, seed=hd + N)
        r = RopeGPU(rot, 1e6, layout)
        table = r.table(first=100, count=60)
        ws = [1 + 0.1 * torch.randn(hd, generator=g, device="cuda") if norm else None for _ in heads]
        rows = torch.randint(-3, 65, (N,), generator=g, device="cuda", dtype=torch.int32)
        for at in (None, rows):
            for inverse in (False, True):
                outs = r.apply(xs, table, rows=at, norm_weights=ws, inverse=inverse)
                for x, y, w in zip(xs, outs, ws):
                    check(y, x, table, at, layout, rot, w, inverse=inverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot", [(256, 64), (128, 128), (12, 6)])
def test_strides_and_in_place(hd, rot, layout, dtype):
    """Queries between their output gates, heads in front of tokens, rows that start anywhere; results where the
    inputs were, beside what is not the heads' own."""
    g, (proj, wide) = inputs(9, [8, 5], 2 * hd, dtype, seed=2)
    r = RopeGPU(rot, 1e6, layout)
    table = r.table(count=9)
    q, k = proj[..., :hd], wide[..., 3:3 + hd]
    heads_first = torch.randn((6, 9, hd), generator=g, device="cuda").to(dtype).transpose(0, 1)
    for x in (q, k, heads_first):
        check(r.apply([x], table)[0], x, table, None, layout, rot)
    was = proj.clone()
    got = r.apply([q], table, out=[q])[0]
    assert got.data_ptr() == proj.data_ptr()
    check(q, was[..., :hd], table, None, layout, rot)
    assert torch.equal(proj[..., hd:], was[..., hd:])
    was = wide.clone()
    r.apply([k], table, out=[k])
    check(k, was[..., 3:3 + hd], table, None, layout, rot)
    assert torch.equal(wide[..., :3], was[..., :3]) and torch.equal(wide[..., 3 + hd:], was[..., 3 + hd:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("N,heads,hd,rot", [(4100, [16, 2], 256, 64), (2500, [48, 8], 128, 128)])
def test_outputs_beyond_the_caches(N, heads, hd, rot, layout, dtype):
    """More than 32 MB of results, into tensors of their own and in place between what stays."""
    g, xs = inputs(N, heads, hd + 16, dtype, seed=7)
    r = RopeGPU(rot, 1e6, layout)
    table, w = r.table(count=N), 1 + 0.1 * torch.randn(hd, generator=g, device="cuda")
    heads_of = [x[..., :hd] for x in xs]
    want = [x.clone() for x in xs]
    outs = r.apply(heads_of, table, norm_weights=[w, None])
    for x, y, n in zip(heads_of, outs, (w, None)):
        check(y, x, table, None, layout, rot, n)
    r.apply(heads_of, table, norm_weights=[w, None], out=heads_of)
    for x, y, was in zip(heads_of, outs, want):
        assert torch.equal(x, y)
    assert all(torch.equal(x[..., hd:], was[..., hd:]) for x, was in zip(xs, want))


def test_refusals_in_python():
    r = RopeGPU(64, 1e6)
    table, x = r.table(count=5), torch.zeros((5, 4, 128), device="cuda")
    w, y = torch.ones(128, device="cuda"), torch.empty_like(x)
    for kw in (dict(xs=[]), dict(xs=[x] * 5), dict(xs=[x[0]]), dict(xs=[x, x[:4]]), dict(xs=[x, x[..., :64]]), dict(xs=[x, x.bfloat16()]), dict(xs=[x.half()]),
               dict(xs=[x.transpose(1, 2)]), dict(xs=[x.cpu()]), dict(xs=[x, x], out=[y]), dict(out=[y[..., :64]]), dict(out=[y[:, :1].expand(5, 4, 128)]),
               dict(out=[y[:1].expand(5, 4, 128)]), dict(out=[y.bfloat16()]), dict(out=[y.cpu()]), dict(norm_weights=[]), dict(norm_weights=[w[:64]]),
               dict(norm_weights=[w.bfloat16()]), dict(norm_weights=[w.cpu()]), dict(table=table[:4]), dict(table=table[:, :16]), dict(table=table.cpu()),
               dict(table=table.double()), dict(table=table[::2]), dict(table=table[0]), dict(rows=torch.zeros(4, dtype=torch.int32, device="cuda")),
               dict(rows=torch.zeros(5, dtype=torch.int64, device="cuda")), dict(rows=torch.zeros(5, dtype=torch.int32))):
        with pytest.raises(SwqError):
            r.apply(**{**dict(xs=[x], table=table), **kw})
    at = torch.zeros(5, dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(positions=at, count=4), dict(positions=at.long()), dict(positions=at.cpu()), dict(positions=at[::2]), dict(count=-1),
               dict(count=5, out=torch.empty((4, 32, 2), device="cuda")), dict(count=5, out=torch.empty((5, 32, 2))),
               dict(count=5, out=torch.empty((5, 32, 2), device="cuda", dtype=torch.bfloat16)), dict(count=5, out=torch.empty((10, 32, 2), device="cuda")[::2])):
        with pytest.raises(SwqError):
            r.table(**kw)
    torch.cuda.synchronize()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_there_and_back_and_gradient(layout):
    """The inverse is the gradient: <turn(x), y> = <x, inverse(y)>, also with a magnitude; and back is where x was."""
    g, (x, y) = inputs(33, [6, 6], 64, torch.float32, seed=3)
    r = RopeGPU(48, 1e4, layout, RopeScaling("yarn", 8.0, 1024))
    table = r.table(count=33)
    fx, by = r.apply([x], table)[0].double(), r.apply([y], table, inverse=True)[0].double()
    a, b = (fx * y.double()).sum(), (x.double() * by).sum()
    assert abs(float(a - b)) < 1e-6 * float(fx.norm() * y.double().norm())
    plain = RopeGPU(48, 1e4, layout)
    table = plain.table(count=33)
    back = plain.apply(plain.apply([x], table), table, inverse=True)[0]
    assert float((back - x).abs().max()) < 2e-6


def test_zeros_and_what_is_not_finite():
    """A row of zeros is normalised to zeros; a NaN or an infinity stays with its row."""
    g, (x,) = inputs(7, [4], 128, torch.bfloat16, seed=4)
    w = torch.ones(128, device="cuda")
    r = RopeGPU(64, 1e6)
    table = r.table(count=7)
    want = r.apply([x], table, norm_weights=[w])[0]
    x[2, 1] = 0
    x[3, 0, 5], x[4, 3, 100] = float("nan"), float("inf")
    got = r.apply([x], table, norm_weights=[w])[0]
    assert bool((got[2, 1] == 0).all())
    live = torch.ones((7, 4), dtype=torch.bool, device="cuda")
    live[2, 1] = live[3, 0] = live[4, 3] = False
    assert torch.equal(got[live], want[live])


def test_no_tokens():
    r = RopeGPU(64, 1e6)
    assert r.apply([torch.empty((0, 4, 128), device="cuda")], r.table(count=1))[0].shape == (0, 4, 128)


def test_captured_and_replayed():
    """A decode step's table and turned heads follow the positions that the device holds."""
    g, (q, k) = inputs(5, [16, 2], 256, torch.bfloat16, seed=5)
    r = RopeGPU(64, 1e7, scaling=RopeScaling("yarn", 4.0, 262144))
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    table, outs = torch.empty((5, 32, 2), device="cuda"), [torch.empty_like(q), torch.empty_like(k)]
    r.apply([q, k], r.table(pos, out=table), out=outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r.apply([q, k], r.table(pos, out=table), out=outs)
    for _ in range(3):
        pos.mul_(7).add_(1)
        want = r.apply([q, k], r.table(pos))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_on_another_stream():
    g, (q,) = inputs(300, [16], 256, torch.float32, seed=6)
    r = RopeGPU(64, 1e7)
    want = r.apply([q], r.table(count=300))[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = r.apply([q], r.table(count=300, stream=side), stream=side)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_many_rows():
    """Elements past 2^31 of a tensor."""
    N, hd = 70000, 256
    x = torch.zeros((N, 128, hd), dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn((128, hd), device="cuda").to(torch.bfloat16)
    r = RopeGPU(64, 1e7)
    table, rows = r.table(first=500, count=2), torch.ones(N, dtype=torch.int32, device="cuda")
    got = r.apply([x], table, rows=rows)[0]
    check(got[-1:], x[-1:], table, rows[-1:], "half", 64)
    assert not bool(got[:-1].any())
