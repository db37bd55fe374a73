"""Learned projections on the GPU at the edges of what the header allows, against their formulas in 64 bits (tolerances: see
test_gpu_projection, whose cases and comparison these are)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_projection import Case, close, f64                 # noqa: E402
from vectordb_amd import _lib                                    # noqa: E402
from vectordb_amd._lib import VdbError                           # noqa: E402
from vectordb_amd.projection import Projection                   # noqa: E402


def close_in_range(got, want, mag, terms, what):
    """`close` for results that may lie beyond what fp16 holds: 65 520 is half way between its largest value and the next step, so
    that the kernel's sum, which is within its own error of the wanted one, may round to infinity from there on."""
    if got.dtype == torch.float16:
        g, err = f64(got).reshape(want.shape), (terms + 8) * 2.0 ** -23 * mag
        inf = np.isinf(g)
        assert (np.abs(want[inf]) + err[inf] >= 65520).all() and (np.sign(g[inf]) == np.sign(want[inf])).all(), what
        got, want, mag = got.reshape(want.shape)[torch.from_numpy(~inf).cuda()], want[~inf], mag[~inf]
    close(got, want, mag, terms, what)


def check_in_range(c, engine):
    """Case.check of an adapted case, for results beyond the range of fp16."""
    rank = c.proj.rank
    y, (want, mag) = c.forward(engine), c.want_forward()
    close_in_range(y, want, mag, c.din + rank, "y")
    got = c.backward(engine)
    for name, g, (v, m), t in zip(("dx", "da", "db"), got, c.want_backward(), (c.dout + rank, c.n + max(c.din, c.dout), c.din + c.n)):
        close_in_range(g, v, m, t, name)


def many_adapters(n, adapters):
    """Requests of 1 to 5 rows, then of hundreds: 16 rows meet up to nine adapters."""
    off, i = [1], 0
    while off[-1] < n - 3:
        off.append(min(off[-1] + ((1, 2, 1, 5, 1, 3)[i % 6] if off[-1] < 300 or off[-1] > n - 200 else 130), n - 3))
        i += 1
    return off, [(5 * s) % (adapters + 1) - 1 for s in range(len(off) - 1)]


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("rank", [4, 8, 16])
@pytest.mark.parametrize("n", [90, 4200, 9000])
@pytest.mark.parametrize("din,dout", [(1, 40), (40, 1), (1, 1), (2, 3), (3, 8), (4, 2)])
def test_adapters_of_narrow_rows(engine, din, dout, n, rank, dtype, out):
    """Rows of 1 to 4 elements, where a factor's ranks and columns both lie one element apart, or hold no vector."""
    off, ids = many_adapters(n, 11)
    Case(n, din, dout, off, dtype, out, 11, rank, ids).check(engine)


def spread(c, bits):
    """Ranks of A x (and of dy B) that span `bits` powers of two, with the other factor making up for it."""
    r = c.proj.rank
    e = torch.tensor([float((7 * q) % r) for q in range(r)]).mul_(bits / max(1, r - 1)).sub_(bits / 2).round_()
    c.a.mul_((2.0 ** e).to(c.dt).cuda()[None, :, None])
    c.b.mul_((2.0 ** -e).to(c.dt).cuda()[None, None, :])
    return c


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,rank", [(40, 64, 72, 16), (300, 136, 264, 40), (4300, 128, 264, 16), (17000, 72, 264, 24), (17000, 72, 136, 64)])
def test_ranks_of_very_different_size(engine, n, din, dout, rank, dtype, out):
    """A rank that is small in A x but large through B counts as much as any other: the intermediate has the bits of fp32 in every rank."""
    off, ids = many_adapters(n, 11)
    check_in_range(spread(Case(n, din, dout, off, dtype, out, 11, rank, ids), 20), engine)
    check_in_range(spread(Case(n, din, dout, [0, n // 2, n], dtype, out, 2, rank, [1, 0]), 20), engine)


@pytest.mark.parametrize("n,requests", [(1, 1), (16, 1), (16, 16), (300, 1), (300, 300), (5000, 1)])
def test_small_rank_beside_a_large_one(engine, n, requests):
    """h = (60000, 0.001), B = (2^-20, 30000): the second rank is nearly all of the sum; alone and in a batch."""
    off = [n * s // requests for s in range(requests + 1)]
    c = Case(n, 8, 16, off, "f16", "f32", 8, 2, [s % 8 for s in range(requests)], scale=False)
    c.w.zero_()
    c.x.zero_()
    c.x[:, 0] = 1
    c.a.zero_()
    c.a[:, 0, 0], c.a[:, 1, 0] = 60000, 0.001
    c.b[:, :, 0], c.b[:, :, 1] = 2.0 ** -20, 30000
    c.dy.fill_(0.25)
    c.check(engine)
    assert abs(float(c.forward(engine)[n - 1, 3]) - 30.06) < 0.01


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,requests", [(1, 1), (16, 16), (300, 1), (300, 300), (5000, 1)])
def test_intermediates_next_to_the_limit_of_fp32(engine, n, requests, dtype):
    """A x s = 3.3995e38, which bf16 rounds to infinity and fp32 holds; with a small B the result is finite, and so are the gradients."""
    off = [n * s // requests for s in range(requests + 1)]
    c = Case(n, 16, 24, off, dtype, "f32", 8, 8, [s % 8 for s in range(requests)])
    c.x.fill_(0.25)
    c.a.fill_(0.25)
    c.s.fill_(3.3995e38)
    c.b.fill_(2.0 ** -20)
    c.dy.fill_(2.0 ** -30)
    assert abs(float(c.s[0]) - 3.3995e38) < 1e33
    c.w.zero_()
    y = c.forward(engine)
    want, mag = c.want_forward()
    assert 1e33 < abs(want).max() < 1e35
    close(y, want, mag, 16 + 8, "y")
    dx = c.backward(engine)[0]
    (want, mag) = c.want_backward()[0]
    close(dx, want, mag, 24 + 8, "dx")
    # and with g = dy B s at the limit
    c.dy.fill_(0.25)
    c.b.fill_(0.25)
    c.a.fill_(2.0 ** -20)
    c.x.fill_(2.0 ** -20)
    c.s.fill_(3.3995e38 / float(0.25 * 24 * c.b[0, 0, 0]))
    dx = c.backward(engine)[0]
    (want, mag) = c.want_backward()[0]
    close(dx, want, mag, 24 + 8, "dx")


def same_with_infinities(got, want, mag, terms, what):
    """NaN where the formula gives NaN, infinities of the formula's sign, and the finite rest within rounding."""
    g = f64(got).reshape(want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(g), np.isnan(want)), "%s: %d NaN, not %d" % (what, np.isnan(g).sum(), np.isnan(want).sum())
    assert np.array_equal(g[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), what
    close(got.reshape(want.shape)[torch.from_numpy(fin).cuda()], want[fin], mag[fin], terms, what)


@pytest.mark.filterwarnings("ignore:invalid value:RuntimeWarning")
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,din,dout,rank,long", [(1, 64, 72, 16, True), (40, 64, 72, 16, False), (90, 33, 41, 5, False), (300, 136, 264, 40, True),
                                                  (4300, 128, 264, 16, False), (9000, 128, 264, 16, True), (17000, 72, 136, 64, True)])
def test_infinities_give_what_the_formula_gives(engine, n, din, dout, rank, long, dtype):
    """Infinite entries of a factor, of a row and of a scale, on every way to the low-rank term."""
    if long:
        off, ids = [0, n - n // 2, n], [1, 0]
    else:
        off, ids = many_adapters(n, 11)
    inf = float("inf")

    def check(c, what):
        (want, mag), got = c.want_forward(), c.forward(engine)
        same_with_infinities(got, want, mag, c.din + rank, what + " y")
        (want, mag), got = c.want_backward()[0], c.backward(engine)[0]
        same_with_infinities(got, want, mag, c.dout + rank, what + " dx")

    c = Case(n, din, dout, off, dtype, "f32", 11, rank, ids)
    c.b[:, 3, rank // 2] = inf
    c.b[:, 5, 0] = -inf
    got = c.forward(engine)
    same_with_infinities(got, *c.want_forward(), din + rank, "columns of b")
    c = Case(n, din, dout, off, dtype, "f32", 11, rank, ids)
    c.a[:, rank // 2, 3] = inf
    c.a[:, 0, 5] = -inf
    got = c.backward(engine)[0]
    same_with_infinities(got, *c.want_backward()[0], dout + rank, "columns of a")
    # everything positive, so that infinities of one sign meet
    c = Case(n, din, dout, off, dtype, "f32", 11, rank, ids)
    for t in (c.x, c.dy, c.w, c.a, c.b, c.s):
        t.copy_(t.abs() + 0.125)
    c.x[n // 3, 1] = inf
    c.dy[n // 3, 1] = inf
    check(c, "row")
    c.s[1] = inf
    check(c, "row and scale")


def test_both_gradients_of_a_handle_with_adapters_in_its_workspace(engine):
    """The workspace stated for the handle is enough for the gradient of its shared matrix too."""
    n, din, dout = 16384, 768, 768
    c = Case(n, din, dout, [0, 5000, 5000, n], "bf16", "f32", 3, 16, [2, 0, 1])
    ws, size = c.ws(engine, True)
    dx, dw = torch.empty(n, din, device="cuda"), torch.empty(1, dout, din, device="cuda")
    whole = torch.tensor([0, n], dtype=torch.int64, device="cuda")
    engine.project_grouped_backward_dev(c.proj, n, c.dy.data_ptr(), dout, c.x.data_ptr(), din, whole.data_ptr(), dx.data_ptr(), din,
                                        dw.data_ptr(), ws.data_ptr(), size)
    torch.cuda.synchronize()
    assert bool(ws.view(torch.uint8)[size:].view(torch.float32).isnan().all())
    dy, x, w = f64(c.dy), f64(c.x), f64(c.w)
    close(dw[0], dy.T @ x, np.abs(dy).T @ np.abs(x), n, "dw")
    close(dx, dy @ w[0], np.abs(dy) @ np.abs(w[0]), dout, "dx")
    da, db = torch.empty_like(c.a, dtype=torch.float32), torch.empty_like(c.b, dtype=torch.float32)
    engine.project_adapted_backward_dev(c.proj, n, c.dy.data_ptr(), dout, c.x.data_ptr(), din, 3, c.offsets.data_ptr(), c.ids_dev.data_ptr(),
                                        dx.data_ptr(), din, da.data_ptr(), db.data_ptr(), ws.data_ptr(), size)
    (want, mag), (want_a, mag_a), (want_b, mag_b) = c.want_backward()
    close(dx, want, mag, dout + 16, "dx")
    close(da, want_a, mag_a, n + dout, "da")
    close(db, want_b, mag_b, n + din, "db")


def test_gradients_of_more_adapters_than_one_launch_takes(engine):
    """8192 wide, 40 000 adapters: two launches (32 768 adapters at most in one); adapters on both sides of the border, all others zero."""
    n, din, dout, adapters, off, ids = 90, 8192, 16, 40000, [0, 20, 21, 60, 88, 90], [0, 32767, 32768, 39999, 32767]
    gen = torch.Generator(device="cuda").manual_seed(9)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(torch.bfloat16)
    x, dy, w, a, b = normal(n, din), normal(n, dout), normal(dout, din), normal(adapters, 1, din), normal(adapters, dout, 1)
    proj = Projection(w, a=a, b=b, out_dtype=torch.float32)
    offsets, ids_dev = torch.tensor(off, device="cuda"), torch.tensor(ids, dtype=torch.int32, device="cuda")
    da, db = torch.full_like(a, 7, dtype=torch.float32), torch.full_like(b, 7, dtype=torch.float32)
    size = engine.projection_workspace_bytes(proj, n, 5, True)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    engine.project_adapted_backward_dev(proj, n, dy.data_ptr(), dout, x.data_ptr(), din, 5, offsets.data_ptr(), ids_dev.data_ptr(), 0, 0,
                                        da.data_ptr(), db.data_ptr(), ws.data_ptr(), size)
    used = torch.zeros(adapters, dtype=torch.bool, device="cuda")
    used[torch.tensor(ids, device="cuda").unique()] = True
    assert int(used.sum()) == 4 and float(da[~used].abs().max()) == 0 and float(db[~used].abs().max()) == 0
    for k in sorted(set(ids)):
        rows = [i for s in range(5) if ids[s] == k for i in range(off[s], off[s + 1])]
        xr, dr, ak, bk = f64(x[rows]), f64(dy[rows]), f64(a[k]), f64(b[k])
        close(da[k], (dr @ bk).T @ xr, (np.abs(dr) @ np.abs(bk)).T @ np.abs(xr), len(rows) + dout, "da")
        close(db[k], dr.T @ (xr @ ak.T), np.abs(dr).T @ (np.abs(xr) @ np.abs(ak).T), len(rows) + din, "db")


def test_twelve_million_rows(engine):
    """More 16-row blocks than a launch takes workgroups for 768 columns.  Values of -1, 0 and 1: every sum is exact in fp32."""
    n, din, dout, cut = 12_000_003, 768, 8, 5_592_407
    gen = torch.Generator(device="cuda").manual_seed(12)

    def signs(*shape):
        return torch.randint(-1, 2, shape, generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    x = torch.empty(n, din, dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, 1_000_000):
        x[i:i + 1_000_000] = signs(min(1_000_000, n - i), din)
    dy, w = signs(n, dout), signs(2, dout, din)
    proj = Projection(w, out_dtype=torch.float32)
    offsets = torch.tensor([0, cut, n], device="cuda")
    y = torch.full((n, dout), 0.5, device="cuda")
    engine.project_grouped_dev(proj, n, x.data_ptr(), din, offsets.data_ptr(), y.data_ptr(), dout)
    size = engine.projection_workspace_bytes(proj, n, 2, True)
    ws, dw = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.full((2, dout, din), 0.5, device="cuda")
    engine.project_grouped_backward_dev(proj, n, dy.data_ptr(), dout, x.data_ptr(), din, offsets.data_ptr(), 0, 0, dw.data_ptr(), ws.data_ptr(), size)
    for g, (b, e) in enumerate([(0, cut), (cut, n)]):
        want, wt = torch.zeros(dout, din, dtype=torch.float64, device="cuda"), w[g].double().t().contiguous()
        for i in range(b, e, 500_000):
            r = x[i:min(i + 500_000, e)].double()
            assert torch.equal(y[i:i + r.shape[0]].double(), r @ wt), i
            want += dy[i:i + r.shape[0]].double().t().contiguous() @ r
        assert torch.equal(dw[g].double(), want)


def spin(seconds):
    """Keeps one workgroup of the current stream busy for about that long."""
    spin.rate = getattr(spin, "rate", None)
    if spin.rate is None:
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda._sleep(1000)
        torch.cuda.synchronize()
        a.record()
        torch.cuda._sleep(1_000_000)
        b.record()
        torch.cuda.synchronize()
        spin.rate = 1e9 / a.elapsed_time(b)                       # cycles a second
    torch.cuda._sleep(int(seconds * spin.rate))


def test_a_projected_insert_does_not_wait_for_other_streams(engine, table_name):
    """Warm inserts free and allocate nothing: one returns while another stream is still at work, as a plain insert does."""
    n, dim = 2000, 64
    c = Case(n, 48, dim, [0, 700, n], "bf16", "f32")
    engine.create_table(table_name, dim, _lib.METRIC_IP, _lib.F32)
    ids = torch.arange(n, dtype=torch.int64, device="cuda")
    rows = torch.randn(n, dim, device="cuda")
    mine = torch.cuda.Stream()

    def plain():
        engine.insert_dev(table_name, n, rows.data_ptr(), ids.data_ptr(), stream=mine.cuda_stream)

    def projected():
        engine.insert_projected_dev(table_name, c.proj, n, c.x.data_ptr(), 48, c.offsets.data_ptr(), ids.data_ptr(), stream=mine.cuda_stream)
    engine.reserve(table_name, 1 << 17)
    plain()
    projected()
    for _ in range(8):                                            # streams of one hardware queue wait for each other: another one
        other, done = torch.cuda.Stream(), torch.cuda.Event()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            spin(0.5)
            done.record()
        plain()
        if done.query():
            continue
        projected()
        assert not done.query(), "the projected insert waited for work of another stream"
        done.synchronize()
        assert engine.count(table_name) % n == 0
        return
    pytest.skip("every stream shares its hardware queue with this one")


@pytest.mark.parametrize("rows_of_a_piece", [1, 100, 333, 1200, 2999])
def test_projected_insert_in_pieces(engine, table_name, rows_of_a_piece):
    """An insert larger than the insert buffer: groups that end inside pieces, pieces inside groups; nothing is inserted if the last
    piece holds a row that is not finite."""
    n, dim = 3000, 96
    c = Case(n, 136, dim, [0, 1, 1, 400, 1700, n], "bf16", "f32")
    engine.create_table(table_name, dim, _lib.METRIC_IP, _lib.F32)
    ids = torch.arange(n, dtype=torch.int64, device="cuda") * 7 - 3
    engine.set_option("insert_buffer_size_gb", rows_of_a_piece * dim * 4 / 2.0 ** 30)
    try:
        last = c.x[n - 1].clone()
        c.x[n - 1, 5] = float("inf")
        with pytest.raises(VdbError) as err:
            engine.insert_projected_dev(table_name, c.proj, n, c.x.data_ptr(), 136, c.offsets.data_ptr(), ids.data_ptr())
        assert err.value.code == _lib.EINVAL and engine.count(table_name) == 0
        c.x[n - 1] = last
        engine.insert_projected_dev(table_name, c.proj, n, c.x.data_ptr(), 136, c.offsets.data_ptr(), ids.data_ptr())
    finally:
        engine.set_option("insert_buffer_size_gb", 1.0)
    stored, got_ids = engine.fetch_rows(table_name, 0, n)
    assert np.array_equal(got_ids, ids.cpu().numpy())
    want, mag = c.want_forward()
    close(torch.from_numpy(stored), want, mag, 136, "rows")


def guarded(size, guard):
    """(everything, address of `size` bytes with `guard` bytes of ones on both sides)."""
    guard = (guard + 255) // 256 * 256
    buf = torch.full((guard + (size + 255) // 256 * 256 + guard,), 255, dtype=torch.uint8, device="cuda")
    return buf, buf.data_ptr() + guard, guard


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,off", [
    (20100, 128, 136, list(range(101)) + [20100]),                           # a hundred groups of one row and a long one
    (20100, 128, 136, [0] + [20000 + i for i in range(101)]),
    (193 * 60, 120, 130, [193 * i for i in range(61)]),                      # chunks of one row behind full ones in every group
    (7000, 67, 515, [0, 3500, 3500, 7000]),
    (33000, 256, 136, [0, 1, 32999]),
])
def test_partial_sums_of_the_matrices_stay_in_the_workspace(engine, n, din, dout, off, dtype, out):
    c = Case(n, din, dout, off, dtype, out)
    size = engine.projection_workspace_bytes(c.proj, n, len(off) - 1, True)
    assert size > 0
    buf, ws, guard = guarded(size, max(1 << 20, din * dout * 4))
    dw = torch.empty_like(c.w, dtype=c.out)
    engine.project_grouped_backward_dev(c.proj, n, c.dy.data_ptr(), dout, c.x.data_ptr(), din, c.offsets.data_ptr(), 0, 0, dw.data_ptr(), ws, size)
    torch.cuda.synchronize()
    assert bool((buf[:guard] == 255).all()) and bool((buf[guard + size:] == 255).all())
    want, mag = c.want_backward()[1]
    close(dw, want, mag, n, "dw")


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,adapters,rank", [(1, 8, 8, 1, 1), (5000, 131, 257, 3, 100), (9000, 72, 66, 1, 128), (2100, 515, 33, 7, 65),
                                                      (17000, 64, 136, 2, 70), (300, 65, 63, 40, 128)])
def test_adapted_calls_stay_in_the_workspace(engine, n, din, dout, adapters, rank, dtype, out):
    off = [0, n // 5, n // 5, n // 2, n - n // 9]
    c = Case(n, din, dout, off, dtype, out, adapters, rank, [s % adapters for s in range(4)])
    want, want_back = c.want_forward(), c.want_backward()
    for backward in (False, True):
        size = engine.projection_workspace_bytes(c.proj, n, 4, backward)
        buf, ws, guard = guarded(size, max(1 << 20, 4 * rank * max(din, dout)))
        seg = (4, c.offsets.data_ptr(), c.ids_dev.data_ptr())
        y, dx = torch.full((n, dout), 77.0, dtype=c.out, device="cuda"), torch.full((n, din), 77.0, dtype=c.out, device="cuda")
        da, db = torch.empty_like(c.a, dtype=c.out), torch.empty_like(c.b, dtype=c.out)
        if backward:
            engine.project_adapted_backward_dev(c.proj, n, c.dy.data_ptr(), dout, c.x.data_ptr(), din, *seg, dx.data_ptr(), din,
                                                da.data_ptr(), db.data_ptr(), ws, size)
        else:
            engine.project_adapted_dev(c.proj, n, c.x.data_ptr(), din, *seg, y.data_ptr(), dout, ws, size)
        torch.cuda.synchronize()
        assert bool((buf[:guard] == 255).all()) and bool((buf[guard + size:] == 255).all())
        if backward:
            for name, got, (v, m), terms in zip(("dx", "da", "db"), (dx, da, db), want_back, (dout + rank, n + dout, n + din)):
                close(got, v, m, terms, name)
        else:
            close(y, *want, din + rank, "y")


@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("n,din,dout,rank", [(1, 65536, 3, 128), (5, 3, 65536, 17), (40, 65536, 24, 64), (70, 40, 65535, 8), (300, 65536, 8, 16)])
def test_the_widest_rows(engine, n, din, dout, rank, dtype, out):
    """65 536 elements in or out, alone and with adapters of the largest rank."""
    Case(n, din, dout, [0, n // 2, n], dtype, out).check(engine)
    off = [0, n // 3, n // 2, n]
    c = Case(n, din, dout, off, dtype, out, 4, rank, [3, -1, 1])
    if out == "f16":
        check_in_range(c, engine)
    else:
        c.check(engine)


def test_projected_inserts_and_searches_at_once(engine, table_name):
    """Host threads with streams of their own: three search one table through different projections, two insert into others."""
    import threading
    dim, n, k = 96, 5000, 5
    engine.create_table(table_name, dim, _lib.METRIC_L2, _lib.F32)
    rows = torch.randn(n, dim, generator=torch.Generator().manual_seed(3)).cuda()
    ids = torch.arange(n, dtype=torch.int64, device="cuda")
    engine.insert_dev(table_name, n, rows.data_ptr(), ids.data_ptr())
    queries = [Case(30 + 100 * i, 64 + 8 * i, dim, [0, 10, 11, 30 + 100 * i], d, "f32", 3, 8 + 4 * i, [2, -1, 0], seed=i)
               for i, d in enumerate(("bf16", "f32", "f16"))]
    sources = [Case(2000 + 500 * i, 72, dim, [0, 600, 2000 + 500 * i], "bf16", "f32", seed=9 + i) for i in range(2)]
    others = [table_name + "_a", table_name + "_b"]
    for o in others:
        engine.create_table(o, dim, _lib.METRIC_L2, _lib.F32)

    def search(c, stream):
        out = (torch.full((c.n, k), -5, dtype=torch.int64, device="cuda"), torch.zeros(c.n, k, device="cuda"),
               torch.zeros(c.n, dtype=torch.int32, device="cuda"))
        engine.search_projected_dev(table_name, c.proj, c.n, c.x.data_ptr(), c.din, 3, c.offsets.data_ptr(), c.ids_dev.data_ptr(), k,
                                    *(t.data_ptr() for t in out), stream=stream)
        return out
    try:
        want = [search(c, 0) for c in queries]
        torch.cuda.synchronize()
        errors = []

        def searcher(i):
            try:
                stream = torch.cuda.Stream()
                with torch.cuda.stream(stream):
                    for _ in range(20):
                        got = search(queries[i], stream.cuda_stream)
                        stream.synchronize()
                        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
            except BaseException as exc:                          # noqa: BLE001 (reported below)
                errors.append(exc)

        def inserter(i):
            try:
                stream, c = torch.cuda.Stream(), sources[i]
                for _ in range(10):
                    engine.insert_projected_dev(others[i], c.proj, c.n, c.x.data_ptr(), c.din, c.offsets.data_ptr(), ids.data_ptr(),
                                                stream=stream.cuda_stream)
            except BaseException as exc:                          # noqa: BLE001
                errors.append(exc)
        threads = [threading.Thread(target=searcher, args=(i,)) for i in range(3)] + [threading.Thread(target=inserter, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors, errors[0]
        for o, c in zip(others, sources):
            assert engine.count(o) == 10 * c.n
            stored, _ = engine.fetch_rows(o, 0, 10 * c.n)
            want_rows, mag = c.want_forward()
            for i in range(10):
                close(torch.from_numpy(stored[i * c.n:(i + 1) * c.n]), want_rows, mag, 72, "rows")
    finally:
        for o in others:
            engine.drop_table(o)
