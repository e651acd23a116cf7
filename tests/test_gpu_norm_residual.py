"""The norms around a block with gate and residual scale, forward and backward, against the definition in 64 bits.

Tolerances, derived before the first run.  Every result is a short chain of 32-bit operations on sums
over a row: a chain of at most 8 columns a thread (and 24 for the tree) and at most a dozen further
roundings, K = 64 half steps of 2^-24 in all, applied to the sum of the absolute values that the formula adds
(so that cancellation is allowed for).  With B(.) for those sums of absolute values:
  u:  B = |gamma| r (|h| + mean|h|) + |beta|   (r itself is off by half the relative error of its sum)
  y:  K 2^-24 (|residual_scale x| + |block_scale a| B(u)) + eps/2 |y|
  n:  the error of y goes through the norm: |gamma| r (dy + mean dy + |yhat| mean(|yhat| dy)), plus K 2^-24 of its own B
  D:  B = |dy| + r (|g dn| + mean|g dn| + H mean(|g dn| H)), H = (|y| + |mean|) r; and dh alike from B(du)
  sums over rows: (K + rows) 2^-24 of the sum of the absolute values (any order of addition).
The result is rounded once, by eps/2 of its type.
"""
import itertools

import pytest
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
K = 64 * 2.0 ** -24
NONE, RMS, LAYER = 0, 1, 2
PLAIN, SIGMOID, TANH = 0, 1, 2


def act(code, g):
    return torch.sigmoid(g) if code == SIGMOID else torch.tanh(g) if code == TANH else g


def slope(code, a):
    return a * (1 - a) if code == SIGMOID else 1 - a * a if code == TANH else torch.ones_like(a)


def stats_of(kind, v, eps):
    if kind == NONE:
        return torch.zeros_like(v[:, :1]), torch.ones_like(v[:, :1])
    mean = v.mean(1, keepdim=True) if kind == LAYER else torch.zeros_like(v[:, :1])
    return mean, 1 / torch.sqrt((v - mean).pow(2).mean(1, keepdim=True) + eps)


def or_(w, none, cols):
    return torch.full((cols,), float(none), dtype=torch.float64) if w is None else w.double().cpu()


class Case:
    def __init__(self, rows, cols, kind, post=RMS, pre=RMS, gates=0, gate_act=PLAIN, affine=True, seed=0, mean=0.3, eps=1e-5):
        g = torch.Generator().manual_seed(seed + rows * 7 + cols)

        def normal(*shape, std=1.0, mean=0.0):
            return (torch.randn(*shape, generator=g) * std + mean)

        t = TYPES[kind]
        self.rows, self.cols, self.type = rows, cols, t
        self.post, self.pre, self.gate_act, self.eps = post, pre, gate_act, eps
        self.x = normal(rows, cols, std=2.0).to(t)
        self.h = normal(rows, cols, std=1.5, mean=mean).to(t)
        self.gate = normal(gates, cols, mean=0.5).to(t) if gates else None
        self.post_gamma = normal(cols, std=0.2, mean=1.0) if affine and post else None
        self.post_beta = normal(cols, std=0.2) if affine and post == LAYER else None
        self.pre_gamma = normal(cols, std=0.2, mean=1.0) if affine and pre else None
        self.pre_beta = normal(cols, std=0.2) if affine and pre == LAYER else None
        self.dy, self.dn = normal(rows, cols).to(t), normal(rows, cols).to(t)
        self.residual_scale, self.block_scale = 0.75, 0.5

    def expand(self, g):
        return g.repeat_interleave(self.rows // g.shape[0], 0)

    def cuda(self):
        for name, v in vars(self).items():
            if isinstance(v, torch.Tensor):
                setattr(self, name, v.cuda())
        return self

    def common(self):
        return dict(post=self.post, pre=self.pre, gate=self.gate, gate_act=self.gate_act, post_gamma=self.post_gamma,
                    post_beta=self.post_beta, pre_gamma=self.pre_gamma, residual_scale=self.residual_scale,
                    block_scale=self.block_scale)

    def forward(self, fdl, **more):
        return fdl.norm_residual(self.x, self.h, pre_beta=self.pre_beta, eps=self.eps, **self.common(), **more)

    def backward(self, fdl, y, stats, dy, dn):
        return fdl.norm_residual_backward(dy, dn, y, self.h, stats, want_post_beta=self.post == LAYER,
                                          want_pre_beta=self.pre == LAYER, **self.common())

    def d(self, t):
        return t.double().cpu()

    def want_forward(self):
        h, x = self.d(self.h), self.d(self.x)
        mean1, r1 = stats_of(self.post, h, self.eps)
        g1, b1 = or_(self.post_gamma, 1, self.cols), or_(self.post_beta, 0, self.cols)
        u = (h - mean1) * r1 * g1 + b1
        size = g1.abs() * r1 * (h.abs() + (h.abs().mean(1, keepdim=True) if self.post else 0)) + b1.abs()
        a = torch.ones_like(h) if self.gate is None else self.expand(act(self.gate_act, self.d(self.gate)))
        y = self.residual_scale * x + self.block_scale * a * u
        dy = K * ((self.residual_scale * x).abs() + self.block_scale * a.abs() * size)
        if self.gate is not None and self.gate_act != PLAIN:
            dy = dy + 8 * 2.0 ** -24 * self.block_scale * u.abs()   # the activation itself, next to 0
        mean2, r2 = stats_of(self.pre, y, self.eps)
        hat = (y - mean2) * r2
        g2, b2 = or_(self.pre_gamma, 1, self.cols), or_(self.pre_beta, 0, self.cols)
        n = hat * g2 + b2
        dn = g2.abs() * r2 * (dy + dy.mean(1, keepdim=True) + hat.abs() * (hat.abs() * dy).mean(1, keepdim=True))
        dn = dn + K * (g2.abs() * r2 * (y.abs() + y.abs().mean(1, keepdim=True)) + b2.abs())
        return y, n, dy, dn, torch.cat([mean1, r1, mean2, r2], 1)

    def want_backward(self, y, stats, dy, dn):
        st, h = self.d(stats), self.d(self.h)
        out, tol = {}, {}
        zero = torch.zeros_like(h)
        dy, dn = zero if dy is None else self.d(dy), zero if dn is None else self.d(dn)
        y = zero if y is None else self.d(y)
        many = K + self.rows * 2.0 ** -24

        def back(kind, v, size, mean, r, hat):
            if kind == NONE:
                return v, size
            big = hat.abs() + 2 * mean.abs() * r
            along = (v * hat).mean(1, keepdim=True)
            level = v.mean(1, keepdim=True) if kind == LAYER else 0.0
            b = r * (size + size.mean(1, keepdim=True) * (kind == LAYER) + big * (size * big).mean(1, keepdim=True))
            return r * (v - level - hat * along), b

        m2, r2 = st[:, 2:3], st[:, 3:4]
        hat = (y - m2) * r2
        big = hat.abs() + 2 * m2.abs() * r2
        g2 = or_(self.pre_gamma, 1, self.cols)
        if self.pre:
            out["pre_gamma"], tol["pre_gamma"] = (dn * hat).sum(0), many * (dn.abs() * big).sum(0)
            out["pre_beta"], tol["pre_beta"] = dn.sum(0), many * dn.abs().sum(0)
            through, size = back(self.pre, dn * g2, (dn * g2).abs(), m2, r2, hat)
        else:
            through, size = zero, zero
        whole, size = dy + through, dy.abs() + size
        out["x"], tol["x"] = self.residual_scale * whole, K * abs(self.residual_scale) * size
        e, size = self.block_scale * whole, abs(self.block_scale) * size
        m1, r1 = st[:, 0:1], st[:, 1:2]
        hat = (h - m1) * r1
        big = hat.abs() + 2 * m1.abs() * r1
        g1, b1 = or_(self.post_gamma, 1, self.cols), or_(self.post_beta, 0, self.cols)
        if self.gate is not None:
            a = act(self.gate_act, self.d(self.gate))
            gates = a.shape[0]
            u, usize = hat * g1 + b1, big * g1.abs() + b1.abs()
            s = slope(self.gate_act, a)
            sums = lambda v: v.view(gates, -1, self.cols).sum(1)  # noqa: E731
            out["gate"] = sums(e * u) * s
            # the slope is 1 - a^2 or a (1 - a) of a rounded a: off by a few half steps of 1
            tol["gate"] = many * sums(size * usize) * s.abs() + sums((e * u).abs() + K * size * usize) * 8 * 2.0 ** -24 * (self.gate_act != PLAIN)
            full = self.expand(a)
            extra = 8 * 2.0 ** -24 / K * (self.gate_act != PLAIN)
            e, size = e * full, size * (full.abs() + extra)
        if self.post:
            out["post_gamma"], tol["post_gamma"] = (e * hat).sum(0), 2 * many * (size * big).sum(0)
            out["post_beta"], tol["post_beta"] = e.sum(0), 2 * many * size.sum(0)
        out["h"], size = back(self.post, e * g1, size * g1.abs(), m1, r1, hat)
        tol["h"] = 2 * K * size
        return out, tol


def close(got, want, tol, what):
    half, tiny = HALF[got.dtype], TINY[got.dtype]
    off = (got.double().cpu() - want).abs()
    tol = tol + half * want.abs() + half * tol + tiny
    assert bool((off <= tol).all()), (what, (off - tol).max().item(), (off / tol).max().item())


def check(fdl, c, which=("both",)):
    y, n, stats = c.forward(fdl)
    want_y, want_n, tol_y, tol_n, want_stats = c.want_forward()
    close(y, want_y, tol_y, "y")
    if c.pre:
        close(n, want_n, tol_n, "n")
    else:
        assert n is None
    close(stats, want_stats, K * (want_stats.abs() + want_stats.abs().amax(0) + 2.0), "stats")
    for w in which:
        dy = None if w == "dn" else c.dy
        dn = None if w == "dy" or not c.pre else c.dn
        got = c.backward(fdl, y, stats, dy, dn)
        want, tol = c.want_backward(y, stats, dy, dn)
        for name, g in got.items():
            if g is not None:
                close(g, want[name], tol[name], (w, name))
        again = c.backward(fdl, y, stats, dy, dn)
        for name, g in got.items():
            assert g is None or torch.equal(g, again[name]), name


def test_formulas_against_differences():
    """The gradient formulas that the GPU tests compare with, against central differences in 64 bits (CPU)."""
    for post, pre, gates, code in itertools.product((NONE, RMS, LAYER), (RMS, LAYER, NONE), (0, 1, 2, 6), (PLAIN, SIGMOID, TANH)):
        c = Case(6, 5, "f32", post, pre, gates, code, seed=3)
        for name, v in vars(c).items():
            if isinstance(v, torch.Tensor):
                setattr(c, name, v.double())
        y, n, _, _, stats = c.want_forward()
        got, _ = c.want_backward(y, stats, c.dy, c.dn if pre else None)

        def value():
            y, n, *_ = c.want_forward()
            return (c.dy * y).sum() + ((c.dn * n).sum() if pre else 0.0)

        for name, leaf in (("x", c.x), ("h", c.h), ("gate", c.gate), ("post_gamma", c.post_gamma), ("post_beta", c.post_beta),
                           ("pre_gamma", c.pre_gamma), ("pre_beta", c.pre_beta)):
            if leaf is None:
                continue
            for i in range(0, leaf.numel(), 3):
                flat, step = leaf.view(-1), 1e-5
                old = flat[i].item()
                flat[i] = old + step
                up = value()
                flat[i] = old - step
                down = value()
                flat[i] = old
                # third derivatives of size up to 100: 1e-10 / 6 of them, and 2^-52 of values below 100, over the step
                assert abs((up - down).item() / (2 * step) - got[name].reshape(-1)[i].item()) < 1e-7, (post, pre, gates, code, name, i)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (5, 64), (37, 256), (9, 257), (4, 264), (300, 100), (2, 1001),
                                       (65, 1024), (7, 4096), (3, 4100), (2, 5000), (2, 8192), (1, 12289), (2, 32768), (1, 32761)])
def test_against_the_definition(fdl, cuda, rows, cols, kind):
    for post, pre in ((RMS, RMS), (LAYER, LAYER)):
        check(fdl, Case(rows, cols, kind, post, pre).cuda())
    check(fdl, Case(rows, cols, kind, RMS, LAYER, gates=1, gate_act=SIGMOID).cuda())
    check(fdl, Case(rows, cols, kind, LAYER, RMS, gates=rows, gate_act=TANH).cuda())
    fdl.take_device_error()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [96, 640, 1001])
def test_every_combination(fdl, cuda, cols):
    for post, pre, gates, code in itertools.product((NONE, RMS, LAYER), (NONE, RMS, LAYER), (0, 1, 4, 12), (PLAIN, SIGMOID, TANH)):
        if gates or code == PLAIN:
            check(fdl, Case(12, cols, "f32", post, pre, gates, code, affine=gates != 4).cuda(), ("both", "dy") + (("dn",) if pre else ()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,gates", [(6000, 1), (6000, 3), (6000, 500), (6000, 3000), (6000, 6000), (4999, 1), (5000, 1000), (3001, 3001)])
@pytest.mark.parametrize("cols", [40, 300])
def test_many_rows_and_their_gates(fdl, cuda, rows, gates, cols):
    """More rows than teams: each takes several, and gates shared by few and by many rows."""
    check(fdl, Case(rows, cols, "bf16", RMS, RMS, gates, SIGMOID).cuda())
    check(fdl, Case(rows, cols, "f32", LAYER, LAYER, gates, PLAIN).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,gates", [(1400, 264, 7), (2500, 512, 1), (601, 1000, 601), (700, 2048, 0), (450, 4096, 450),
                                             (450, 4096, 150), (330, 4104, 3), (400, 8192, 2), (151, 8200, 1), (160, 16384, 160),
                                             (90, 32768, 9), (1500, 257, 3), (1201, 330, 1201), (500, 1001, 0), (600, 2049, 2), (301, 4095, 301),
                                             (170, 5003, 10), (160, 9001, 1), (75, 30001, 75)])
def test_more_rows_than_teams(fdl, cuda, rows, cols, gates, kind):
    """Several rows for each team, from one to eight CTAs wide, rows of whole packs and rows off the 16-byte grid."""
    check(fdl, Case(rows, cols, kind, RMS, RMS, gates, SIGMOID if gates else PLAIN).cuda(), ("both", "dn"))
    check(fdl, Case(rows, cols, kind, LAYER, LAYER, gates, TANH if gates else PLAIN, seed=2).cuda(), ("both", "dy"))
    check(fdl, Case(rows, cols, kind, NONE, NONE, gates, PLAIN).cuda())
    fdl.take_device_error()


@pytest.mark.gpu
def test_shifted_starts_take_the_element_path(fdl, cuda):
    c = Case(5, 512, "bf16", LAYER, LAYER, 5, TANH).cuda()
    y, n, stats = c.forward(fdl)

    def shift(t):
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    for name in ("x", "h", "gate", "dy", "dn", "post_gamma", "post_beta", "pre_gamma", "pre_beta"):
        d = Case(5, 512, "bf16", LAYER, LAYER, 5, TANH).cuda()
        setattr(d, name, shift(getattr(d, name)))
        check(fdl, d)


@pytest.mark.gpu
def test_in_place(fdl, cuda):
    for rows, cols in ((9, 200), (4, 2048), (3, 9000)):
        c = Case(rows, cols, "f32", RMS, LAYER, rows, SIGMOID).cuda()
        y, n, stats = c.forward(fdl)
        x0, h0 = c.x.clone(), c.h.clone()
        y2, n2, stats2 = c.forward(fdl, out=c.x, out_n=c.h)
        assert y2.data_ptr() == c.x.data_ptr() and n2.data_ptr() == c.h.data_ptr()
        assert torch.equal(y, y2) and torch.equal(n, n2) and torch.equal(stats, stats2)
        c.x, c.h = x0, h0
        want = c.backward(fdl, y, stats, c.dy, c.dn)
        # dx over dy, dh over h, dgate over gate through the C entry
        dy, h, gate = c.dy.clone(), c.h.clone(), c.gate.clone()
        size = fdl.lib().fdl_norm_residual_backward_scratch_bytes(rows, cols, rows)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        fdl.check(fdl.lib().fdl_norm_residual_backward(
            dy.data_ptr(), c.dn.data_ptr(), y.data_ptr(), h.data_ptr(), stats.data_ptr(), gate.data_ptr(), rows, SIGMOID, RMS,
            c.post_gamma.data_ptr(), None, LAYER, c.pre_gamma.data_ptr(), dy.data_ptr(), h.data_ptr(), gate.data_ptr(), None, None,
            None, None, rows, cols, c.residual_scale, c.block_scale, 0, scratch.data_ptr(), size,
            torch.cuda.current_stream().cuda_stream), "backward in place")
        assert torch.equal(dy, want["x"]) and torch.equal(h, want["h"]) and torch.equal(gate, want["gate"])


@pytest.mark.gpu
def test_constant_and_huge_rows(fdl, cuda):
    """A row of equal values has variance 0: eps holds.  Values whose squares pass 16 bits stay finite in 32."""
    c = Case(4, 777, "f16", LAYER, RMS, seed=1).cuda()
    c.h[0] = 2.0
    c.h[1] = 0.0
    c.h[2] = 60000.0
    c.x[3] = -60000.0
    check(fdl, c)


@pytest.mark.gpu
def test_no_rows(fdl, cuda):
    c = Case(0, 64, "f32").cuda()
    y, n, stats = c.forward(fdl)
    assert y.shape == (0, 64)
    got = c.backward(fdl, y, stats, c.dy, c.dn)
    assert not got["post_gamma"].any() and not got["pre_gamma"].any()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(fdl, cuda):
    rows, cols = 270000, 8192
    free, _ = cuda.cuda.mem_get_info()
    if free < 6 * rows * cols * 2:
        pytest.skip("not enough free device memory")
    c = Case(4, cols, "bf16").cuda()
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-4:], h[-4:] = c.x, c.h
    yy, nn, ss = fdl.norm_residual(x, h, eps=c.eps, **c.common())
    want_y, want_n, tol_y, tol_n, want_stats = c.want_forward()
    close(yy[-4:], want_y, tol_y, "y")
    close(nn[-4:], want_n, tol_n, "n")
    assert not yy[:-4].any() and not nn[:-4].any()
    dy = torch.zeros_like(x)
    dy[-4:] = c.dy
    del x, nn
    got = fdl.norm_residual_backward(dy, None, yy, h, ss, **c.common())
    want, tol = c.want_backward(yy[-4:], ss[-4:], c.dy, None)
    for name in ("x", "h"):
        close(got[name][-4:], want[name], tol[name], name)
        assert not got[name][:-4].any()
    c.rows = rows  # the sums run over all rows
    want, tol = c.want_backward(yy[-4:], ss[-4:], c.dy, None)
    close(got["post_gamma"], want["post_gamma"], tol["post_gamma"], "post_gamma")


@pytest.mark.gpu
def test_streams_and_graph_capture(fdl, cuda):
    a, b = Case(300, 2048, "bf16", gates=3).cuda(), Case(77, 1001, "f32", LAYER, LAYER).cuda()

    def both(c):
        y, n, stats = c.forward(fdl)
        g = c.backward(fdl, y, stats, c.dy, c.dn)
        return [y, n, stats] + [g[k] for k in sorted(g) if g[k] is not None]

    want_a, want_b = both(a), both(b)
    cuda.cuda.synchronize()
    one, two = cuda.cuda.Stream(), cuda.cuda.Stream()
    for _ in range(5):
        with cuda.cuda.stream(one):
            got_a = both(a)
        with cuda.cuda.stream(two):
            got_b = both(b)
        cuda.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got_a + got_b, want_a + want_b))
    first, second = cuda.cuda.CUDAGraph(), cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(first):
        got_a = both(a)
    with cuda.cuda.graph(second):
        got_b = both(b)
    first.replay(), second.replay(), first.replay()
    cuda.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got_a + got_b, want_a + want_b))
    d = Case(300, 2048, "bf16", gates=3, seed=9).cuda()
    for name in ("x", "h", "gate", "dy", "dn", "post_gamma", "pre_gamma"):
        getattr(a, name).copy_(getattr(d, name))
    first.replay()
    cuda.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got_a, both(d)))
