"""Learned projections on the GPU against their formulas in 64 bits.

Tolerance of a result that is a sum of products: the inputs are exact in 64 bits, the kernels round each of the K additions
of a sum by at most one unit in the last place (2^-23 of the partial sum, which is at most S, the sum of the terms'
magnitudes), a second stage adds its own K, and a 16-bit output is off by half a step more:
  |error| <= (K + 8) 2^-23 S + u |value| + the type's smallest step,   u = 2^-8 (bf16), 2^-11 (fp16), 0 (fp32)
with 8 for the few roundings of scales and of intermediates between the stages.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from vectordb_amd import _lib                                    # noqa: E402
from vectordb_amd._lib import VdbError                           # noqa: E402
from vectordb_amd.projection import Projection                   # noqa: E402

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
SENTINEL = 77.0


def tensor(gen, shape, dtype, scale=1.0, shift=0, ld=None):
    """Values on the GPU, `shift` elements behind an aligned address, rows ld apart."""
    rows = int(np.prod(shape[:-1]))
    ld = ld or shape[-1]
    buf = torch.full((shift + rows * ld + 16,), float("nan"), dtype=dtype, device="cuda")
    view = buf[shift:shift + rows * ld].view(rows, ld)[:, :shape[-1]]
    view.copy_((torch.randn(rows, shape[-1], generator=gen) * scale).to(dtype))
    return view if ld != shape[-1] else buf[shift:shift + rows * ld].view(*shape)


def output(shape, dtype, shift=0, ld=None):
    ld = ld or shape[-1]
    rows = int(np.prod(shape[:-1]))
    buf = torch.full((shift + rows * ld + 16,), SENTINEL, dtype=dtype, device="cuda")
    view = buf[shift:shift + rows * ld].view(rows, ld)[:, :shape[-1]] if ld != shape[-1] else buf[shift:shift + rows * ld].view(*shape)
    return buf, view


def f64(t):
    return t.detach().cpu().double().numpy()


def close(got, want, mag, terms, what):
    """want, mag: value and sum of magnitudes in 64 bits."""
    dt = got.dtype
    g = f64(got).reshape(want.shape)
    tol = (terms + 8) * 2.0 ** -23 * mag + HALF_STEP[dt] * np.abs(want) + TINY[dt]
    bad = ~(np.abs(g - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, first %s: %r, not %r (tolerance %g)" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], g[tuple(np.argwhere(bad)[0])], want[tuple(np.argwhere(bad)[0])],
        np.broadcast_to(tol, want.shape)[tuple(np.argwhere(bad)[0])])


def spans(offsets, n):
    return [(s, min(max(offsets[s], 0), n), min(max(offsets[s + 1], 0), n)) for s in range(len(offsets) - 1)]


class Case:
    def __init__(self, n, din, dout, offsets, dtype, out, adapters=0, rank=0, ids=None, seed=0, shift=0, pad=0, scale=True, groups=None):
        gen = torch.Generator().manual_seed(seed + 1000 * n + din)
        dt = DT[dtype]
        self.n, self.din, self.dout, self.off, self.ids = n, din, dout, list(offsets), ids
        self.dt, self.out, self.shift, self.pad = dt, DT[out], shift, pad
        self.groups = 1 if adapters else len(offsets) - 1
        self.x = tensor(gen, (n, din), dt, 1.0, shift, din + pad)
        self.dy = tensor(gen, (n, dout), dt, 1.0, shift, dout + pad)
        self.w = tensor(gen, (self.groups, dout, din), dt, din ** -0.5, shift)
        self.a = self.b = self.s = None
        if adapters:
            self.a = tensor(gen, (adapters, rank, din), dt, din ** -0.5, shift)
            self.b = tensor(gen, (adapters, dout, rank), dt, rank ** -0.5, shift)
            self.s = tensor(gen, (adapters,), torch.float32, 1.0) if scale else None
        self.proj = Projection(self.w, a=self.a, b=self.b, scale=self.s, out_dtype=self.out)
        self.offsets = torch.tensor(self.off, dtype=torch.int64, device="cuda")
        self.ids_dev = torch.tensor(ids, dtype=torch.int32, device="cuda") if ids is not None else None

    def ws(self, engine, backward):
        size = engine.projection_workspace_bytes(self.proj, self.n, len(self.off) - 1, backward)
        return torch.full((max(size // 4, 4) + 4,), float("nan"), device="cuda"), size

    def forward(self, engine, stream=0, out=None):
        buf, y = out or output((self.n, self.dout), self.out, self.shift, self.dout + self.pad)
        self.buf = buf
        if self.ids is None:
            engine.project_grouped_dev(self.proj, self.n, self.x.data_ptr(), self.din + self.pad, self.offsets.data_ptr(),
                                       y.data_ptr(), self.dout + self.pad, stream=stream)
        else:
            self.keep, size = self.ws(engine, False)
            engine.project_adapted_dev(self.proj, self.n, self.x.data_ptr(), self.din + self.pad, len(self.off) - 1,
                                       self.offsets.data_ptr(), self.ids_dev.data_ptr(), y.data_ptr(), self.dout + self.pad,
                                       self.keep.data_ptr(), size, stream=stream)
        return y

    def backward(self, engine, stream=0):
        self.bufs, (dx, dw, da, db) = zip(*[
            output((self.n, self.din), self.out, self.shift, self.din + self.pad), output(self.w.shape, self.out, self.shift),
            output(self.a.shape if self.a is not None else (1, 1), self.out, self.shift),
            output(self.b.shape if self.b is not None else (1, 1), self.out, self.shift)])
        self.keep, size = self.ws(engine, True)
        if self.ids is None:
            engine.project_grouped_backward_dev(self.proj, self.n, self.dy.data_ptr(), self.dout + self.pad, self.x.data_ptr(),
                                                self.din + self.pad, self.offsets.data_ptr(), dx.data_ptr(), self.din + self.pad,
                                                dw.data_ptr(), self.keep.data_ptr(), size, stream=stream)
            return dx, dw
        engine.project_adapted_backward_dev(self.proj, self.n, self.dy.data_ptr(), self.dout + self.pad, self.x.data_ptr(),
                                            self.din + self.pad, len(self.off) - 1, self.offsets.data_ptr(), self.ids_dev.data_ptr(),
                                            dx.data_ptr(), self.din + self.pad, da.data_ptr(), db.data_ptr(), self.keep.data_ptr(), size,
                                            stream=stream)
        return dx, da, db

    # ---- formulas in 64 bits: value and sum of magnitudes, row by row of segments
    def adapter(self, s):
        k = self.ids[s]
        return k if 0 <= k < self.proj.adapters else -1

    def want_forward(self):
        x, w = f64(self.x), f64(self.w)
        y, m = np.full((self.n, self.dout), SENTINEL), np.zeros((self.n, self.dout))
        for s, b, e in spans(self.off, self.n):
            wg = w[0 if self.ids is not None else s]
            y[b:e], m[b:e] = x[b:e] @ wg.T, np.abs(x[b:e]) @ np.abs(wg).T
            if self.ids is not None and self.adapter(s) >= 0:
                k = self.adapter(s)
                A, B, sc = f64(self.a)[k], f64(self.b)[k], 1.0 if self.s is None else f64(self.s)[k]
                y[b:e] += sc * (x[b:e] @ A.T) @ B.T
                m[b:e] += abs(sc) * (np.abs(x[b:e]) @ np.abs(A).T) @ np.abs(B).T
        return y, m

    def want_backward(self):
        x, dy, w = f64(self.x), f64(self.dy), f64(self.w)
        dx, mx = np.full((self.n, self.din), SENTINEL), np.zeros((self.n, self.din))
        dw, mw = np.zeros_like(w), np.zeros_like(w)
        if self.ids is not None:
            a, b_, sc = f64(self.a), f64(self.b), np.ones(self.proj.adapters) if self.s is None else f64(self.s)
            da, ma, db, mb = np.zeros_like(a), np.zeros_like(a), np.zeros_like(b_), np.zeros_like(b_)
        for s, b, e in spans(self.off, self.n):
            g = 0 if self.ids is not None else s
            dx[b:e], mx[b:e] = dy[b:e] @ w[g], np.abs(dy[b:e]) @ np.abs(w[g])
            dw[g] += dy[b:e].T @ x[b:e]
            mw[g] += np.abs(dy[b:e]).T @ np.abs(x[b:e])
            if self.ids is not None and self.adapter(s) >= 0:
                k = self.adapter(s)
                gg, mg = sc[k] * dy[b:e] @ b_[k], abs(sc[k]) * np.abs(dy[b:e]) @ np.abs(b_[k])
                hh, mh = sc[k] * x[b:e] @ a[k].T, abs(sc[k]) * np.abs(x[b:e]) @ np.abs(a[k]).T
                dx[b:e] += gg @ a[k]
                mx[b:e] += mg @ np.abs(a[k])
                da[k] += gg.T @ x[b:e]
                ma[k] += mg.T @ np.abs(x[b:e])
                db[k] += dy[b:e].T @ hh
                mb[k] += np.abs(dy[b:e]).T @ mh
        return ((dx, mx), (dw, mw)) if self.ids is None else ((dx, mx), (da, ma), (db, mb))

    def check(self, engine, stream=0):
        rank = self.proj.rank
        y = self.forward(engine, stream)
        torch.cuda.synchronize()
        want, mag = self.want_forward()
        close(y, want, mag, self.din + rank, "y")
        self.frame(self.buf, y)
        got = self.backward(engine, stream)
        torch.cuda.synchronize()
        rows = max([e - b for _, b, e in spans(self.off, self.n)] + [0]) if self.ids is None else self.n
        terms = [self.dout + rank, rows + max(self.din, self.dout) * (rank > 0), self.din + self.n]
        for name, g, (v, m), t in zip(("dx", "dw" if self.ids is None else "da", "db"), got, self.want_backward(), terms):
            close(g, v, m, t, name)
        self.frame(self.bufs[0], got[0])

    def frame(self, buf, view):
        """Nothing but the view's elements was written."""
        n = view.numel()
        view.fill_(SENTINEL)
        assert bool((buf == SENTINEL).all()), "written outside the output (%d elements in it)" % n


GROUPED = [
    # n, din, dout, offsets
    (1, 8, 8, [0, 1]),
    (1, 1, 1, [0, 1]),
    (5, 3, 7, [0, 2, 2, 5]),
    (64, 64, 64, [0, 0, 64, 64]),
    (130, 136, 72, [0, 1, 129, 130]),
    (300, 384, 384, [0, 127, 255, 256, 300]),
    (257, 200, 264, [3, 60, 60, 250]),                    # rows before the first group and behind the last
    (128, 515, 387, [0, 128]),
    (97, 33, 130, [0, 10, 96]),
    (40, 768, 128, [0, 0, 0]),                            # no group has rows
    (150, 72, 80, list(range(0, 151, 2)) + [150] * 60),   # more groups than a wave has lanes
]


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("case", GROUPED, ids=lambda c: "%dx%dx%d_%dg" % (c[0], c[1], c[2], len(c[3]) - 1))
def test_grouped(engine, case, dtype, out):
    n, din, dout, off = case
    Case(n, din, dout, off, dtype, out).check(engine)


# rows enough for the gradient of the matrices to be summed in chunks, and for every shape of tile
LARGE = [
    (2000, 136, 72, [0, 1500, 1500, 1501, 2000]),
    (3001, 67, 45, [5, 1000, 2990]),
    (1300, 384, 384, [0, 400, 400, 1300]),
    (9000, 256, 520, [0, 3, 5000, 9000]),
    (40000, 136, 768, [0, 20000, 20000, 39990]),
    (16000, 768, 640, [100, 7000, 7001, 16000]),
    (70000, 128, 272, [0, 12345, 70000]),
]


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: "%dx%dx%d_%dg" % (c[0], c[1], c[2], len(c[3]) - 1))
def test_grouped_large(engine, case, dtype, out):
    n, din, dout, off = case
    Case(n, din, dout, off, dtype, out).check(engine)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,rank", [(3000, 128, 200, 16), (20000, 256, 768, 24), (52000, 128, 264, 8), (9000, 520, 256, 100)])
def test_adapted_large(engine, n, din, dout, rank, dtype, out):
    """Requests of very different length: one row, a few, thousands; many adapters within 16 rows and one over many tiles."""
    lens = [1] * 40 + [3] * 20 + [n // 3, 0, 17, 1, 100] + [n // 5]
    off = [0]
    for v in lens:
        off.append(off[-1] + v)
    off.append(n - 9)
    ids = [(5 * i) % 12 - 1 for i in range(len(off) - 1)]
    Case(n, din, dout, off, dtype, out, 11, rank, ids).check(engine)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift,pad", [(1, 0), (0, 3), (4, 8), (8, 16), (3, 5)])
def test_grouped_strides_and_alignment(engine, dtype, shift, pad):
    Case(140, 96, 160, [0, 50, 140], dtype, "f32", shift=shift, pad=pad).check(engine)
    if dtype != "f32":
        Case(140, 96, 160, [0, 50, 139], dtype, dtype, shift=shift, pad=pad).check(engine)


ADAPTED = [
    # n, din, dout, offsets, adapters, rank, ids
    (1, 8, 8, [0, 1], 1, 1, [0]),
    (1, 768, 768, [0, 1], 3, 16, [2]),
    (1, 64, 64, [0, 1], 3, 16, [-1]),
    (17, 72, 40, [0, 1, 2, 3, 3, 10, 17], 4, 5, [3, -1, 0, 1, 3, 9]),      # an adapter twice, one out of range, one empty request
    (64, 384, 384, list(range(65)), 20, 8, [(7 * i) % 20 - (i % 9 == 0) * 40 for i in range(64)]),
    (200, 136, 264, [2, 90, 91, 180], 3, 33, [1, 2, 1]),                   # rows outside every request
    (260, 256, 128, [0, 200, 260], 2, 128, [1, 0]),
    (150, 130, 77, [0, 7, 60, 150], 3, 17, [0, 1, 2]),
    (90, 515, 66, [0, 40, 41, 90], 5, 64, [4, 4, 0]),
    (48, 64, 64, [0, 48], 2, 16, [7]),
    (300, 64, 96, [0] + [3 * i for i in range(1, 101)], 7, 12, [(i * 3) % 8 - 1 for i in range(100)]),
]


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("case", ADAPTED, ids=lambda c: "%dx%dx%d_%dr_rank%d" % (c[0], c[1], c[2], len(c[3]) - 1, c[5]))
def test_adapted(engine, case, dtype, out):
    n, din, dout, off, adapters, rank, ids = case
    Case(n, din, dout, off, dtype, out, adapters, rank, ids).check(engine)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift,pad", [(1, 0), (0, 3), (4, 8), (8, 16), (3, 5)])
def test_adapted_strides_and_alignment(engine, dtype, shift, pad):
    Case(140, 96, 160, [0, 50, 140], dtype, "f32", 3, 16, [2, 0], shift=shift, pad=pad, scale=False).check(engine)
    if dtype != "f32":
        Case(140, 96, 160, [0, 50, 140], dtype, dtype, 3, 24, [1, 0], shift=shift, pad=pad).check(engine)


@pytest.mark.parametrize("requests", [63, 64, 65, 128, 129, 256, 4096, 4097])
def test_rows_behind_the_last_of_many_requests(engine, requests):
    """The search for a row's request divides the offsets by 64 a step; rows in front of, between and behind all requests."""
    n = requests + 40
    ids = [i % 5 - 1 for i in range(requests)]
    Case(n, 16, 24, list(range(7, 8 + requests)), "bf16", "f32", 4, 4, ids).check(engine)


def test_large_values_of_the_low_rank_intermediate(engine):
    """A x beyond what fp16 holds, with B small enough that the product fits."""
    c = Case(33, 64, 48, [0, 20, 33], "f16", "f32", 2, 16, [1, 0], scale=False)
    c.x.mul_(100.0)
    c.a.mul_(2000.0)
    c.b.mul_(2.0 ** -10)
    assert float((c.x.float() @ c.a[1].float().T).abs().max()) > 65504
    c.check(engine)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_nan_and_infinity_stay_with_their_rows(engine, dtype):
    """A row, a group's matrix or an adapter that is not finite changes no other row and no other gradient."""
    for bad in (float("nan"), float("inf"), torch.finfo(DT[dtype]).min):
        c = Case(40, 72, 80, [0, 9, 20, 40], dtype, "f32")
        y0, (dx0, dw0) = c.forward(engine).clone(), [t.clone() for t in c.backward(engine)]
        c.w[1].fill_(bad)
        c.x[9:20] = bad
        c.dy[9:20] = bad
        y, (dx, dw) = c.forward(engine), c.backward(engine)
        keep = [i for i in range(40) if not 9 <= i < 20]
        assert torch.equal(y[keep], y0[keep]) and torch.equal(dx[keep], dx0[keep]) and torch.equal(dw[[0, 2]], dw0[[0, 2]])
        c = Case(40, 72, 80, [0, 9, 20, 40], dtype, "f32", 3, 20, [0, 1, 2])
        y0, (dx0, da0, db0) = c.forward(engine).clone(), [t.clone() for t in c.backward(engine)]
        for t in (c.a[1], c.b[1], c.s[1:2], c.x[9:20], c.dy[9:20]):
            t.fill_(bad)
        y, (dx, da, db) = c.forward(engine), c.backward(engine)
        assert torch.equal(y[keep], y0[keep]) and torch.equal(dx[keep], dx0[keep])
        assert torch.equal(da[[0, 2]], da0[[0, 2]]) and torch.equal(db[[0, 2]], db0[[0, 2]])
        if bad != bad:
            assert bool(y[9:20].isnan().all()) and bool(da[1].isnan().all())


def test_infinite_row_without_an_adapter_gives_what_the_formula_gives(engine):
    c = Case(3, 16, 16, [0, 1, 3], "bf16", "f32", 2, 4, [-1, 0])
    c.x[0] = 0
    c.x[0, 3] = float("inf")
    y = c.forward(engine)
    w = c.w[0, :, 3].float()
    assert torch.equal(y[0], torch.where(w > 0, float("inf"), -float("inf"))) or bool((w == 0).any())
    assert bool(y[1:].isfinite().all())


@pytest.mark.parametrize("offsets", [[5, 3, 60, 20, 70], [-4, 10, 90, 1000, 1 << 40], [-9, -9, -1, -1, 0], [99, 99, 99, 99, 99],
                                     [1 << 62, -(1 << 62), 1 << 62, 0, 70], [0, 70, 0, 70, 0]])
@pytest.mark.parametrize("adapted", [False, True])
@pytest.mark.parametrize("times", [1, 100, 700])
def test_offsets_that_are_wrong_reach_nothing_outside(engine, offsets, adapted, times):
    """Values of rows in such segments are undefined; the bytes around every output stay, and the call returns."""
    n, offsets = 70 * times, [o * times if abs(o) < 1 << 41 else o for o in offsets]
    ids = [i % 6 for i in range(len(offsets) - 1)]
    c = Case(n, 128, 48 if times < 700 else 520, offsets, "bf16", "f32", *((3, 8, ids) if adapted else ()))
    y = c.forward(engine)
    torch.cuda.synchronize()
    c.frame(c.buf, y)
    outs = c.backward(engine)
    torch.cuda.synchronize()
    for buf, t in zip((c.bufs[0],) + (c.bufs[2:4] if adapted else c.bufs[1:2]), outs):
        c.frame(buf, t)


def test_gradients_against_differences(engine):
    """y is linear in each argument alone, so f(p + e) - f(p - e) = 2 <gradient, e> exactly for f = <dy, y>; what is left is
    the fp32 rounding of the two forward passes, bounded like every result here."""
    c = Case(70, 48, 40, [0, 20, 33, 70], "f32", "f32", 3, 8, [2, 0, 2])
    dx, da, db = (t.clone() for t in c.backward(engine))
    gen = torch.Generator().manual_seed(5)
    dy = f64(c.dy)
    for p, grad in ((c.x, dx), (c.a, da), (c.b, db)):
        # steps of a quarter on a grid, so that p + e and p - e are exact after p is put on a grid too
        p.copy_((p * 64).round() / 64)
    dx, da, db = (t.clone() for t in c.backward(engine))
    for p, grad in ((c.x, dx), (c.a, da), (c.b, db)):
        e = (torch.randint(-1, 2, p.shape, generator=gen).float() / 4).cuda()
        saved = p.clone()
        p.copy_(saved + e)
        up, mup = f64(c.forward(engine)), c.want_forward()[1]
        p.copy_(saved - e)
        down, mdown = f64(c.forward(engine)), c.want_forward()[1]
        p.copy_(saved)
        diff = float((dy * (up - down)).sum()) / 2
        want = float((f64(grad) * f64(e)).sum())
        terms = 48 + 8 + 8
        tol = terms * 2.0 ** -23 * float((np.abs(dy) * (mup + mdown)).sum()) / 2
        mag = c.want_backward()
        m = {id(dx): mag[0][1], id(da): mag[1][1], id(db): mag[2][1]}[id(grad)]
        tol += (70 + 48 + 8) * 2.0 ** -23 * float((m * np.abs(f64(e))).sum())
        assert abs(diff - want) <= tol, (diff, want, tol)


def test_two_calls_give_the_same_bits(engine):
    c = Case(600, 136, 200, [0, 100, 333, 600], "bf16", "f32", 2, 16, [1, 0, 1])
    g = Case(600, 136, 200, [0, 100, 333, 600], "f16", "f32")
    for case in (c, g):
        y, grads = case.forward(engine).clone(), [t.clone() for t in case.backward(engine)]
        for _ in range(3):
            assert torch.equal(case.forward(engine), y)
            assert all(torch.equal(a, b) for a, b in zip(case.backward(engine), grads))


def test_outputs_may_be_left_out(engine):
    c = Case(50, 64, 48, [0, 20, 50], "bf16", "f32")
    dx, dw = (t.clone() for t in c.backward(engine))
    _, dx1 = output((50, 64), torch.float32)
    _, dw1 = output(tuple(c.w.shape), torch.float32)
    args = (c.proj, 50, c.dy.data_ptr(), 48, c.x.data_ptr(), 64, c.offsets.data_ptr())
    engine.project_grouped_backward_dev(*args, dx1.data_ptr(), 64, 0, c.keep.data_ptr(), c.keep.numel() * 4)
    engine.project_grouped_backward_dev(*args, 0, 0, dw1.data_ptr(), c.keep.data_ptr(), c.keep.numel() * 4)
    assert torch.equal(dx, dx1) and torch.equal(dw, dw1)
    c = Case(50, 64, 48, [0, 20, 50], "bf16", "f32", 2, 8, [0, 1])
    dx, da, db = (t.clone() for t in c.backward(engine))
    _, dx1 = output((50, 64), torch.float32)
    _, da1 = output(tuple(c.a.shape), torch.float32)
    _, db1 = output(tuple(c.b.shape), torch.float32)
    args = (c.proj, 50, c.dy.data_ptr(), 48, c.x.data_ptr(), 64, 2, c.offsets.data_ptr(), c.ids_dev.data_ptr())
    ws, size = c.ws(engine, True)
    engine.project_adapted_backward_dev(*args, dx1.data_ptr(), 64, 0, 0, ws.data_ptr(), size)
    engine.project_adapted_backward_dev(*args, 0, 0, da1.data_ptr(), db1.data_ptr(), ws.data_ptr(), size)
    assert torch.equal(dx, dx1) and torch.equal(da, da1) and torch.equal(db, db1)


def test_no_rows_and_no_requests(engine):
    c = Case(30, 64, 48, [0, 20, 30], "bf16", "f32")
    _, dw = output(tuple(c.w.shape), torch.float32)
    zero = torch.zeros(3, dtype=torch.int64, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    engine.project_grouped_dev(c.proj, 0, 0, 0, zero.data_ptr(), 0, 0)
    engine.project_grouped_backward_dev(c.proj, 0, 0, 0, 0, 0, zero.data_ptr(), 0, 0, dw.data_ptr(), ws.data_ptr(), 1 << 20)
    assert bool((dw == 0).all())
    c = Case(30, 64, 48, [0, 30], "bf16", "f32", 2, 8, [1])
    y = output((30, 48), torch.float32)[1]
    da, db = output(tuple(c.a.shape), torch.float32)[1], output(tuple(c.b.shape), torch.float32)[1]
    engine.project_adapted_dev(c.proj, 30, c.x.data_ptr(), 64, 0, c.offsets.data_ptr(), 0, y.data_ptr(), 48, ws.data_ptr(), 1 << 20)
    assert bool((y == SENTINEL).all())
    engine.project_adapted_backward_dev(c.proj, 30, c.dy.data_ptr(), 48, c.x.data_ptr(), 64, 0, c.offsets.data_ptr(), 0, 0, 0,
                                        da.data_ptr(), db.data_ptr(), ws.data_ptr(), 1 << 20)
    assert bool((da == 0).all()) and bool((db == 0).all())


def test_row_addresses_past_32_bits(engine):
    """Rows 65 536 elements apart: the last ones lie more than 2^31 elements behind the first."""
    n, ld, din, dout = 33000, 65536, 64, 32
    gen = torch.Generator().manual_seed(3)
    for adapted in (False, True):
        off = [0, 100, 32900, n]
        c = Case(n, din, dout, off, "bf16", "f32", *((2, 8, [0, 1, 0]) if adapted else ()))
        y, grads = c.forward(engine).clone(), [t.clone() for t in c.backward(engine)]
        big = torch.empty(n * ld, dtype=torch.bfloat16, device="cuda").view(n, ld)
        big[:, 1024:1024 + din] = c.x
        big[:, 2048:2048 + dout] = c.dy
        x, dy = big[:, 1024:1024 + din], big[:, 2048:2048 + dout]
        big_out = torch.empty(n * ld, dtype=torch.float32, device="cuda").view(n, ld)
        ws, size = c.ws(engine, True)
        rest = ([t.clone() for t in grads[1:]])
        o = big_out.data_ptr()
        if adapted:
            seg = (3, c.offsets.data_ptr(), c.ids_dev.data_ptr())
            engine.project_adapted_dev(c.proj, n, x.data_ptr(), ld, *seg, o + 4 * 64, ld, ws.data_ptr(), size)
            engine.project_adapted_backward_dev(c.proj, n, dy.data_ptr(), ld, x.data_ptr(), ld, *seg, o + 4 * 256, ld,
                                                rest[0].data_ptr(), rest[1].data_ptr(), ws.data_ptr(), size)
        else:
            engine.project_grouped_dev(c.proj, n, x.data_ptr(), ld, c.offsets.data_ptr(), o + 4 * 64, ld)
            engine.project_grouped_backward_dev(c.proj, n, dy.data_ptr(), ld, x.data_ptr(), ld, c.offsets.data_ptr(), o + 4 * 256, ld,
                                                rest[0].data_ptr(), ws.data_ptr(), size)
        assert torch.equal(big_out[:, 64:64 + dout], y) and torch.equal(big_out[:, 256:256 + din], grads[0])
        assert all(torch.equal(a, b) for a, b in zip(rest, grads[1:]))
        del big, big_out


def test_other_streams_and_concurrent_calls(engine):
    """Two streams, each with its own workspace, many calls in flight; results as on the default stream."""
    cases = [Case(500, 136, 264, [0, 200, 500], "bf16", "f32", 3, 16, [2, 0]), Case(400, 264, 136, [0, 1, 400], "f16", "f32", 3, 40, [1, 1]),
             Case(500, 136, 264, [0, 200, 500], "bf16", "f32")]
    want = [(c.forward(engine).clone(), [t.clone() for t in c.backward(engine)]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                y = c.forward(engine, s.cuda_stream)
                keep = c.keep if c.ids is not None else None
                got.append((y, c.backward(engine, s.cuda_stream), keep, c.keep, c.buf, c.bufs))
        torch.cuda.synchronize()
        for (y, grads), g in zip(want, got):
            assert torch.equal(g[0], y) and all(torch.equal(a, b) for a, b in zip(g[1], grads))


@pytest.mark.parametrize("adapted", [False, True])
def test_captured_and_replayed(engine, adapted):
    """Forward and backward in one graph; other inputs, other segments and other adapters at each replay, with eager work between."""
    args = (3, 16, [2, 0, 1]) if adapted else ()
    c = Case(300, 136, 200, [0, 100, 180, 300], "bf16", "f32", *args)
    y, grads = c.forward(engine), c.backward(engine)
    torch.cuda.synchronize()
    y = output((300, 200), torch.float32)[1]
    dx = output((300, 136), torch.float32)[1]
    parts = [output(tuple(t.shape), torch.float32)[1] for t in grads[1:]]
    ws, size = c.ws(engine, True)

    def step(stream):
        if adapted:
            seg = (3, c.offsets.data_ptr(), c.ids_dev.data_ptr())
            engine.project_adapted_dev(c.proj, 300, c.x.data_ptr(), 136, *seg, y.data_ptr(), 200, ws.data_ptr(), size, stream=stream)
            engine.project_adapted_backward_dev(c.proj, 300, c.dy.data_ptr(), 200, c.x.data_ptr(), 136, *seg, dx.data_ptr(), 136,
                                                parts[0].data_ptr(), parts[1].data_ptr(), ws.data_ptr(), size, stream=stream)
        else:
            engine.project_grouped_dev(c.proj, 300, c.x.data_ptr(), 136, c.offsets.data_ptr(), y.data_ptr(), 200, stream=stream)
            engine.project_grouped_backward_dev(c.proj, 300, c.dy.data_ptr(), 200, c.x.data_ptr(), 136, c.offsets.data_ptr(),
                                                dx.data_ptr(), 136, parts[0].data_ptr(), ws.data_ptr(), size, stream=stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    gen = torch.Generator().manual_seed(11)
    for turn in range(4):
        c.x.copy_(torch.randn(300, 136, generator=gen))
        c.dy.copy_(torch.randn(300, 200, generator=gen))
        c.offsets.copy_(torch.tensor([0, 10 * turn, 150 + turn, 300]))
        if adapted:
            c.ids_dev.copy_(torch.tensor([turn % 3, -1, (turn + 1) % 3], dtype=torch.int32))
        for t in [y, dx] + parts:
            t.fill_(SENTINEL)
        graph.replay()
        torch.cuda.synchronize()
        want_y, want = c.forward(engine), c.backward(engine)
        torch.cuda.synchronize()
        assert torch.equal(y, want_y), turn
        assert all(torch.equal(a, b) for a, b in zip([dx] + parts, want)), turn


def test_large_gradients_captured_and_replayed(engine):
    """Sizes at which the gradient of the matrices goes through the workspace, captured and replayed beside eager calls."""
    n = 15000
    c = Case(n, 768, 640, [0, 4000, 4001, n], "bf16", "f32")
    dx, dw = (t.clone() for t in c.backward(engine))
    ws, size = c.ws(engine, True)
    assert size > 0
    out = output((n, 768), torch.float32)[1], output(tuple(c.w.shape), torch.float32)[1]

    def step(stream):
        engine.project_grouped_backward_dev(c.proj, n, c.dy.data_ptr(), 640, c.x.data_ptr(), 768, c.offsets.data_ptr(), out[0].data_ptr(),
                                            768, out[1].data_ptr(), ws.data_ptr(), size, stream=stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for t in out:
            t.fill_(SENTINEL)
        graph.replay()
        again = c.backward(engine)
        torch.cuda.synchronize()
        assert torch.equal(out[0], dx) and torch.equal(out[1], dw) and torch.equal(again[1], dw)
    with pytest.raises(VdbError) as err:
        engine.project_grouped_backward_dev(c.proj, n, c.dy.data_ptr(), 640, c.x.data_ptr(), 768, c.offsets.data_ptr(), out[0].data_ptr(),
                                            768, out[1].data_ptr(), ws.data_ptr(), size - 4)
    assert err.value.code == _lib.EINVAL


def test_many_groups(engine):
    """More groups than rows, and as many as a call takes."""
    off = [min(3 * max(0, i - 4000), 40) for i in range(4097)]
    Case(40, 32, 24, off, "bf16", "f32").check(engine)
    off = [i // 2 for i in range(4097)]
    Case(2048, 40, 16, off, "f16", "f16").check(engine)


def test_calls_from_several_threads(engine):
    """Calls side by side from host threads, each with its own stream, outputs and workspace."""
    import threading
    cases = [Case(200 + 50 * i, 72, 136, [0, 90, 200 + 50 * i], "bf16", "f32", *((3, 16, [2, i % 3]) if i % 2 else ())) for i in range(6)]
    want = [(c.forward(engine).clone(), [t.clone() for t in c.backward(engine)]) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * len(cases), []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            for _ in range(10):
                with torch.cuda.stream(stream):
                    y = cases[i].forward(engine, stream.cuda_stream)
                    keep = getattr(cases[i], "keep", None)
                    got[i] = (y, cases[i].backward(engine, stream.cuda_stream), keep)
                    stream.synchronize()
        except Exception as exc:                                  # noqa: BLE001 (reported below)
            errors.append(exc)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (y, grads), g in zip(want, got):
        assert torch.equal(g[0], y) and all(torch.equal(a, b) for a, b in zip(g[1], grads))


@pytest.mark.parametrize("metric", [_lib.METRIC_IP, _lib.METRIC_COSINE, _lib.METRIC_L2])
def test_ingest_and_search_through_projections(engine, table_name, metric):
    """As they are used together: rows of three encoders go through their matrices into one table, queries of several tenants
    through the shared matrix and their adapters, and the answers are the exact ones for the projected values."""
    dim, n, nq, k = 128, 3000, 40, 7
    rows = Case(n, 256, dim, [0, 1000, 1000, n], "bf16", "f32")
    q = Case(nq, 192, dim, [0, 1, 5, 22, 38], "bf16", "f32", 3, 8, [2, -1, 0, 2])
    engine.create_table(table_name, dim, metric, _lib.F32)
    ids = torch.arange(n, dtype=torch.int64, device="cuda") * 3 - 500
    engine.insert_projected_dev(table_name, rows.proj, n, rows.x.data_ptr(), 256, rows.offsets.data_ptr(), ids.data_ptr())
    y = rows.forward(engine)
    want_rows, mag = rows.want_forward()
    close(y, want_rows, mag, 256, "rows")
    if metric != _lib.METRIC_COSINE:
        stored, got_ids = engine.fetch_rows(table_name, 0, n)
        assert np.array_equal(stored, y.cpu().numpy()) and np.array_equal(got_ids, ids.cpu().numpy())

    def outs():
        return (torch.full((nq, k), -5, dtype=torch.int64, device="cuda"), torch.zeros(nq, k, device="cuda"),
                torch.zeros(nq, dtype=torch.int32, device="cuda"))
    a, b = outs(), outs()
    engine.search_projected_dev(table_name, q.proj, nq, q.x.data_ptr(), 192, 4, q.offsets.data_ptr(), q.ids_dev.data_ptr(), k,
                                *(t.data_ptr() for t in a))
    z = torch.zeros(nq, dim, device="cuda")                       # the two queries behind the last request: zero vectors
    q.forward(engine, out=(z, z))
    engine.search_dev(table_name, nq, z.data_ptr(), k, *(t.data_ptr() for t in b))
    torch.cuda.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    # the first request against the formula: best ids in 64 bits, wherever they are further apart than the rounding
    yq = f64(z)[:38]
    wq, mq = q.want_forward()
    close(z[:38], wq[:38], mq[:38], 192 + 8, "queries")
    yr = f64(y)
    if metric == _lib.METRIC_COSINE:
        yr, yq = yr / np.linalg.norm(yr, axis=1, keepdims=True), yq / np.linalg.norm(yq, axis=1, keepdims=True)
    score = yq @ yr.T if metric != _lib.METRIC_L2 else -((yq[:, None, :] - yr[None]) ** 2).sum(-1)
    best = np.argsort(-score, axis=1, kind="stable")[:, 0]
    gap = np.sort(score, axis=1)
    clear = gap[:, -1] - gap[:, -2] > 1e-5 * np.abs(gap[:, -1])   # stored and scored in fp32: relative 2^-24 a step
    assert clear.sum() > 30
    assert np.array_equal(a[0].cpu().numpy()[:38, 0][clear], (best * 3 - 500)[clear])


def test_projected_insert_and_search_refusals(engine, table_name):
    engine.create_table(table_name, 64, _lib.METRIC_IP, _lib.F32)
    rows = Case(20, 48, 64, [0, 5, 20], "f32", "f32")
    ids = torch.arange(20, dtype=torch.int64, device="cuda")

    def insert(offsets, name=table_name, case=rows):
        off = torch.tensor(offsets, dtype=torch.int64, device="cuda")
        engine.insert_projected_dev(name, case.proj, 20, case.x.data_ptr(), case.din, off.data_ptr(), ids.data_ptr())

    for bad in ([0, 5, 19], [1, 5, 20], [0, 21, 20], [0, -1, 20], [0, 5, 21]):
        with pytest.raises(VdbError) as err:
            insert(bad)
        assert err.value.code == _lib.EINVAL
    with pytest.raises(VdbError) as err:
        insert([0, 5, 20], name="nosuch")
    assert err.value.code == _lib.ENOTFOUND
    with pytest.raises(VdbError) as err:
        insert([0, 5, 20], case=Case(20, 48, 63, [0, 5, 20], "f32", "f32"))
    assert err.value.code == _lib.EINVAL and engine.count(table_name) == 0
    rows.w[1, 0, 0] = float("inf")                                # a projected row that is not finite: nothing is inserted
    with pytest.raises(VdbError):
        insert([0, 5, 20])
    assert engine.count(table_name) == 0
    rows.w[1, 0, 0] = 0.5
    insert([0, 5, 20])
    insert([0, 0, 20])
    assert engine.count(table_name) == 40


# middle sizes in fp32: 32 x 32 tiles, aligned and not, one adapter, a few and many in 16 rows
MIDDLE = [
    (1100, 384, 384, 0),
    (700, 515, 515, 0),
    (1090, 384, 372, 8),
    (610, 640, 640, 64),
    (690, 261, 515, 19),
]


@pytest.mark.parametrize("n,din,dout,rank", MIDDLE)
def test_middle_sizes(engine, n, din, dout, rank):
    if not rank:
        Case(n, din, dout, [1, 300, 300, 301, 640, n - 3], "f32", "f32").check(engine)
        return
    off = list(range(0, 40)) + [56, 60, 64, 300, 301, n - 3]
    ids = [(5 * i) % 12 - 1 for i in range(len(off) - 1)]
    Case(n, din, dout, off, "f32", "f32", 11, rank, ids).check(engine)
    Case(n, din, dout, [0, n], "f32", "f32", 2, rank, [1]).check(engine)


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,rank,segments", [(1, 8, 8, 1, 1), (70, 33, 17, 5, 9), (300, 384, 384, 8, 200), (5000, 136, 200, 64, 3),
                                                      (9000, 256, 264, 0, 5), (40, 16, 24, 0, 3)])
def test_workspace_of_the_stated_size_is_not_exceeded(engine, n, din, dout, rank, segments, dtype, out):
    off = [n * s // segments for s in range(segments + 1)]
    ids = [s % 3 - 1 for s in range(segments)] if rank else None
    case = Case(n, din, dout, off, dtype, out, 2 if rank else 0, rank, ids)
    for call, backward in ((case.forward, False), (case.backward, True)):
        case.keep = None
        call(engine)
        torch.cuda.synchronize()
        size = engine.projection_workspace_bytes(case.proj, n, segments, backward)
        if case.keep is not None:
            assert bool(case.keep.view(torch.uint8)[size:].view(torch.float32).isnan().all())


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,adapters,rank", [(2100, 72, 136, 1, 5), (5000, 64, 200, 3, 20), (9000, 136, 72, 2, 70), (12000, 40, 66, 17, 8)])
def test_factor_gradients_of_many_rows_to_an_adapter(engine, n, din, dout, adapters, rank, dtype, out):
    """Rows of an adapter shared by several workgroups, requests that end inside blocks of 16 rows, one adapter without rows."""
    cuts = [0, n // 3 + 1, n // 3 + 1, n // 2, n // 2 + 5, n - 7]
    ids = [0, 1 % adapters, 0, adapters - 1, 0]
    case = Case(n, din, dout, cuts, dtype, out, adapters, rank, ids)
    case.check(engine)
    first = [t.clone() for t in case.backward(engine)[1:]]
    again = case.backward(engine)[1:]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,rank", [(4100, 256, 384, 16), (33000, 256, 520, 9)])
def test_requests_that_meet_in_a_tile(engine, n, din, dout, rank, dtype, out):
    """Requests of 5 to 40 rows and of hundreds: one, a few and many adapters in the rows of a wave, some without one; what an
    adapter of infinities holds stays with its own rows."""
    off, i = [0], 0
    while off[-1] < n - 50:
        off.append(min(off[-1] + (5, 40, 17, 700, 33, 24, 150)[i % 7], n - 50))
        i += 1
    ids = [(3 * s) % 8 - 1 for s in range(len(off) - 1)]
    case = Case(n, din, dout, off, dtype, out, 7, rank, ids)
    case.check(engine)
    clean = case.forward(engine).clone()
    case.b[4].fill_(float("inf"))
    got = case.forward(engine)
    torch.cuda.synchronize()
    other = torch.ones(n, dtype=torch.bool)
    for s, b, e in spans(off, n):
        if ids[s] == 4:
            other[b:e] = False
    assert torch.equal(got.cpu()[other], clean.cpu()[other])
    assert not torch.isfinite(got.cpu()[~other].float()).all(dim=1).any()


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout", [(5000, 3, 70), (9000, 5, 7), (4500, 70, 2), (2500, 131, 257), (4200, 9, 8), (4200, 67, 12), (3000, 193, 450)])
def test_sizes_that_are_no_vectors_in_tiles(engine, n, din, dout, dtype, out):
    """Rows shorter than a vector, and rows that end inside one, where the products are in tiles."""
    Case(n, din, dout, [2, n // 3, n // 3 + 1, n - 1], dtype, out).check(engine)
    Case(n, din, dout, [0, n // 2, n], dtype, out, 2, 5, [1, 0], shift=1, pad=1).check(engine)


def test_shared_factor_gradients_captured_and_replayed(engine):
    """One adapter's rows divided among workgroups, whose sums go through the workspace: replays beside eager calls."""
    n = 6000
    c = Case(n, 136, 200, [0, 2500, 2503, n - 1], "bf16", "f32", 1, 24, [0, 0, 0])
    dx, da, db = (t.clone() for t in c.backward(engine))
    ws, size = c.ws(engine, True)
    out = [output(tuple(t.shape), torch.float32)[1] for t in (dx, da, db)]

    def step(stream, have=size):
        engine.project_adapted_backward_dev(c.proj, n, c.dy.data_ptr(), 200, c.x.data_ptr(), 136, 3, c.offsets.data_ptr(), c.ids_dev.data_ptr(),
                                            out[0].data_ptr(), 136, out[1].data_ptr(), out[2].data_ptr(), ws.data_ptr(), have, stream=stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        for t in out:
            t.fill_(SENTINEL)
        graph.replay()
        again = c.backward(engine)
        torch.cuda.synchronize()
        for got, eager, want in zip(out, again, (dx, da, db)):
            assert torch.equal(got, want) and torch.equal(eager, want)
    with pytest.raises(VdbError) as err:
        step(0, size - 4)
    assert err.value.code == _lib.EINVAL
