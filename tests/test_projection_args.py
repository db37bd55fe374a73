"""CPU tests of the learned projections' boundary: what the entry points refuse (arguments are checked before the library's
state, so no GPU is needed), and what vectordb_amd.projection.Projection refuses.  The addresses are never read."""
import ctypes as C

import pytest

from vectordb_amd import _lib
from vectordb_amd._lib import ProjectionStruct, VdbError
from vectordb_amd.projection import Projection

X, Y, W, A, B, S, OFF, IDS, DX, DW, DA, DB, WS, DY = (0x100000000 * (i + 1) for i in range(14))
N, DIN, DOUT, RANK = 100, 64, 48, 8


def _gpu():
    try:
        import torch
        return torch.cuda.is_available()
    except Exception:
        return False


def struct(**kw):
    v = dict(dim_in=DIN, dim_out=DOUT, dtype=_lib.BF16, out_dtype=_lib.F32, groups=3, adapters=0, rank=0, reserved=0,
             w=W, a=None, b=None, scale=None)
    v.update(kw)
    return ProjectionStruct(*[v[f] for f, _ in ProjectionStruct._fields_])


def adapter_struct(**kw):
    v = dict(groups=1, adapters=5, rank=RANK, a=A, b=B, scale=S)
    v.update(kw)
    return struct(**v)


def call(fn, p, **kw):
    lib = _lib.load()
    v = dict(n=N, x=X, ldx=DIN, off=OFF, y=Y, ldy=DOUT, dy=DY, lddy=DOUT, dx=DX, lddx=DIN, dw=DW, da=DA, db=DB, req=4, ids=IDS,
             ws=WS, wsb=1 << 30, st=None, name=b"nosuch", k=3)
    v.update(kw)
    g = lambda *names: [v[n] for n in names]                                                       # noqa: E731
    ref = C.byref(p) if p is not None else None
    if fn == "grouped":
        return lib.vdb_project_grouped_dev(ref, *g("n", "x", "ldx", "off", "y", "ldy", "st"))
    if fn == "grouped_backward":
        return lib.vdb_project_grouped_backward_dev(ref, *g("n", "dy", "lddy", "x", "ldx", "off", "dx", "lddx", "dw", "ws", "wsb", "st"))
    if fn == "adapted":
        return lib.vdb_project_adapted_dev(ref, *g("n", "x", "ldx", "req", "off", "ids", "y", "ldy", "ws", "wsb", "st"))
    if fn == "adapted_backward":
        return lib.vdb_project_adapted_backward_dev(ref, *g("n", "dy", "lddy", "x", "ldx", "req", "off", "ids", "dx", "lddx", "da", "db",
                                                            "ws", "wsb", "st"))
    if fn == "insert":
        return lib.vdb_insert_projected_dev(v["name"], ref, *g("n", "x", "ldx", "off", "ids", "st"))
    return lib.vdb_search_projected_dev(v["name"], ref, *g("n", "x", "ldx", "req", "off", "ids", "k", "y", "dx", "dy", "st"))


GROUPED = ["grouped", "grouped_backward", "insert"]
ADAPTED = ["adapted", "adapted_backward", "search"]


@pytest.mark.parametrize("fn", GROUPED + ADAPTED)
@pytest.mark.parametrize("kw", [dict(dim_in=0), dict(dim_in=65537), dict(dim_out=0), dict(dim_out=-1), dict(dtype=3), dict(dtype=-1),
                                dict(out_dtype=_lib.F16), dict(groups=0), dict(groups=4097), dict(reserved=1), dict(w=None), dict(w=W + 1)])
def test_projection_itself_is_checked(fn, kw):
    make = struct if fn in GROUPED else adapter_struct
    assert call(fn, make(**kw)) == _lib.EINVAL
    assert call(fn, None) == _lib.EINVAL and "null projection" in _lib.last_error()


@pytest.mark.parametrize("fn", ADAPTED)
@pytest.mark.parametrize("kw", [dict(groups=2), dict(adapters=0), dict(adapters=65536), dict(rank=0), dict(rank=129), dict(a=None),
                                dict(b=None), dict(a=A + 1), dict(b=B + 1), dict(scale=S + 2)])
def test_adapters_are_checked(fn, kw):
    assert call(fn, adapter_struct(**kw)) == _lib.EINVAL


@pytest.mark.parametrize("fn,kw", [
    ("grouped", dict(n=-1)), ("grouped", dict(x=None)), ("grouped", dict(y=None)), ("grouped", dict(off=None)),
    ("grouped", dict(off=OFF + 4)), ("grouped", dict(ldx=DIN - 1)), ("grouped", dict(ldy=DOUT - 1)), ("grouped", dict(ldy=1 << 40)),
    ("grouped", dict(x=X + 1)), ("grouped", dict(y=Y + 2)), ("grouped", dict(n=1 << 40)),
    ("grouped", dict(y=X)), ("grouped", dict(y=X + 4 * 8)), ("grouped", dict(y=W)), ("grouped", dict(y=OFF)),
    ("grouped_backward", dict(dx=None, dw=None)), ("grouped_backward", dict(dy=None)), ("grouped_backward", dict(x=None)),
    ("grouped_backward", dict(off=None)), ("grouped_backward", dict(lddy=1)), ("grouped_backward", dict(lddx=1)),
    ("grouped_backward", dict(dw=DW + 1)), ("grouped_backward", dict(dx=DY)), ("grouped_backward", dict(dx=X)),
    ("grouped_backward", dict(dw=X)), ("grouped_backward", dict(dw=DY)), ("grouped_backward", dict(dw=W)), ("grouped_backward", dict(dx=DW)),
    ("adapted", dict(req=-1)), ("adapted", dict(req=(1 << 20) + 1)), ("adapted", dict(n=1 << 33)), ("adapted", dict(ids=None)), ("adapted", dict(ids=IDS + 2)), ("adapted", dict(ws=None)),
    ("adapted", dict(wsb=10)), ("adapted", dict(ws=WS + 4)), ("adapted", dict(y=A)), ("adapted", dict(y=B)), ("adapted", dict(y=S)),
    ("adapted", dict(y=IDS)), ("adapted", dict(y=WS)), ("adapted", dict(x=WS)), ("adapted", dict(off=None)), ("adapted", dict(ldx=3)),
    ("adapted_backward", dict(da=None)), ("adapted_backward", dict(db=None)), ("adapted_backward", dict(dx=None, da=None, db=None)),
    ("adapted_backward", dict(wsb=100)), ("adapted_backward", dict(da=DB)), ("adapted_backward", dict(da=A)), ("adapted_backward", dict(db=B)),
    ("adapted_backward", dict(dx=DY)), ("adapted_backward", dict(da=DX)), ("adapted_backward", dict(db=WS)), ("adapted_backward", dict(da=DA + 1)),
    ("insert", dict(name=None)), ("insert", dict(x=None)), ("insert", dict(off=None)), ("insert", dict(ids=None)), ("insert", dict(ldx=1)),
    ("search", dict(name=None)), ("search", dict(k=0)), ("search", dict(k=1025)), ("search", dict(x=None)), ("search", dict(y=None)),
    ("search", dict(ids=None)), ("search", dict(off=None)), ("search", dict(ldx=1)),
])
def test_calls_are_refused(fn, kw):
    p = struct() if fn in GROUPED else adapter_struct()
    assert call(fn, p, **kw) == _lib.EINVAL, _lib.last_error()


@pytest.mark.skipif(_gpu(), reason="the addresses do not exist: only without a GPU")
@pytest.mark.parametrize("fn,kw", [(f, {}) for f in GROUPED + ADAPTED] + [
    ("grouped", dict(ldx=200, y=X + 2 * DIN, ldy=100)),              # columns of one buffer: same distance in bytes, side by side
    ("grouped_backward", dict(dx=None, lddx=0)), ("grouped_backward", dict(dw=None, x=None)),
    ("adapted_backward", dict(dx=None)), ("adapted_backward", dict(da=None, db=None, x=None)),
    ("adapted", dict(n=0, x=None, y=None, ws=None, wsb=0)), ("grouped", dict(n=0, x=None, y=None, off=None)),
])
def test_allowed_calls_reach_the_library_state(fn, kw):
    p = struct() if fn in GROUPED else adapter_struct()
    assert call(fn, p, **kw) == _lib.ESTATE, _lib.last_error()


def test_side_by_side_columns_and_overlapping_ones():
    # rows of 400 bytes: x in bytes 0..127, y (fp32, 48 wide) in 192 bytes from `at`
    at = lambda b: call("grouped", struct(), ldx=200, y=X + b, ldy=100)                            # noqa: E731
    assert at(124) == _lib.EINVAL and at(212) == _lib.EINVAL          # 212: y's row ends in the next row's x
    if not _gpu():
        assert at(128) == _lib.ESTATE and at(208) == _lib.ESTATE


def test_workspace_sizes():
    lib = _lib.load()
    size = lambda p, n, s, b: lib.vdb_projection_workspace_bytes(C.byref(p), n, s, b)              # noqa: E731
    p = adapter_struct()
    assert size(p, 0, 4, 0) >= 0 and size(p, 1000, 4, 0) >= 1000 * RANK * 4
    assert size(p, 1000, 4, 1) > size(p, 1000, 4, 0)
    assert size(struct(), 1000, 3, 0) >= 0 and size(p, -1, 4, 0) == _lib.EINVAL
    assert size(adapter_struct(rank=200), 10, 1, 0) == _lib.EINVAL


@pytest.mark.parametrize("n,din,dout,rank", [(16384, 768, 768, 16), (6000, 136, 200, 24), (100, 8, 8, 1), (0, 64, 48, 8), (200000, 1024, 768, 128)])
def test_one_workspace_serves_both_gradients_of_a_handle_with_adapters(n, din, dout, rank):
    """The shared matrix's gradient is that of the grouped backward call; the size stated for the handle has to do for it too."""
    lib = _lib.load()
    p = adapter_struct(dim_in=din, dim_out=dout, rank=rank)
    size = lib.vdb_projection_workspace_bytes(C.byref(p), n, 4, 1)
    alone = lib.vdb_projection_workspace_bytes(C.byref(struct(dim_in=din, dim_out=dout, groups=1)), n, 1, 1)
    assert size >= alone >= 0
    # every address far from the others, whatever n
    far = dict(x=1 << 44, dy=2 << 44, dx=3 << 44, dw=4 << 44, ws=5 << 44, da=6 << 44, db=7 << 44)
    kw = dict(n=n, ldx=din, lddx=din, lddy=dout, wsb=size, **far)
    if not _gpu():
        for fn in ("grouped_backward", "adapted_backward"):
            assert call(fn, p, **kw) == _lib.ESTATE, (fn, _lib.last_error())
    # more groups than one: the grouped calls alone take the handle, and their size is stated
    q = adapter_struct(dim_in=din, dim_out=dout, rank=rank, groups=3)
    assert lib.vdb_projection_workspace_bytes(C.byref(q), n, 3, 1) == \
        lib.vdb_projection_workspace_bytes(C.byref(struct(dim_in=din, dim_out=dout)), n, 3, 1)


def test_an_insert_buffer_is_a_size():
    """The option divides a projected insert into pieces."""
    lib = _lib.load()
    for bad in (0.0, -1.0, float("nan"), float("-inf")):
        assert lib.vdb_set_option(b"insert_buffer_size_gb", bad) == _lib.EINVAL
    assert lib.vdb_set_option(b"insert_buffer_size_gb", 1.0) == _lib.OK


@pytest.mark.parametrize("fn,n,at", [(fn, 5000, at) for fn in ("adapted", "adapted_backward") for at in (W, A, B, S, OFF, IDS)] +
                         [("grouped_backward", 20000, W), ("grouped_backward", 20000, OFF)])
@pytest.mark.parametrize("part", ["first", "last"])
def test_a_workspace_that_lies_on_an_input_is_refused(fn, n, at, part):
    """Whatever a call reads besides rows; the input in the workspace's first and in its last bytes."""
    p = struct() if fn.startswith("grouped") else adapter_struct()
    size = _lib.load().vdb_projection_workspace_bytes(C.byref(p), n, 4, int(fn.endswith("backward")))
    assert size > 1 << 16
    ws = at if part == "first" else (at - size + 16) // 16 * 16
    kw = dict(n=n, wsb=size)
    assert call(fn, p, ws=ws, **kw) == _lib.EINVAL and "workspace shares memory" in _lib.last_error()
    if not _gpu():
        # right in front of the input, and not on it
        assert call(fn, p, ws=(at - size) // 16 * 16, **kw) == _lib.ESTATE, _lib.last_error()


@pytest.mark.parametrize("fn", ["grouped", "grouped_backward", "adapted", "adapted_backward"])
@pytest.mark.parametrize("din,dout,most", [(768, 768, (((1 << 23) - 8) // 12 - 2) * 64 + 63), (1024, 100, (((1 << 23) - 8) // 16 - 2) * 64 + 63),
                                           (64, 8, 1 << 27), (1, 1, 1 << 27), (65536, 64, (8191 - 2) * 64 + 63)])
def test_rows_up_to_the_stated_limit(fn, din, dout, most):
    """One group: (n / 64 + 2) times the longer dimension / 64 up to 2^23 - 8, and 2^27 rows of adapted calls."""
    p = struct(dim_in=din, dim_out=dout, groups=1) if fn.startswith("grouped") else adapter_struct(dim_in=din, dim_out=dout, adapters=65535, rank=1)
    if fn.startswith("grouped"):
        most = (((1 << 23) - 8) // ((max(din, dout) + 63) // 64) - 2) * 64 + 63
    kw = dict(ldx=din, ldy=dout, lddx=din, lddy=dout, wsb=1 << 43, x=1 << 44, y=8 << 44, dy=2 << 44, dx=3 << 44, dw=4 << 44, ws=5 << 44,
              da=6 << 44, db=7 << 44)
    assert call(fn, p, n=most + 1, **kw) == _lib.EINVAL and "too many rows" in _lib.last_error()
    if not _gpu():
        assert call(fn, p, n=most, **kw) == _lib.ESTATE, _lib.last_error()


class FakeTensor:
    """What Projection looks at of a tensor."""
    def __init__(self, shape, dtype="torch.bfloat16", device="cuda", index=0, contiguous=True):
        self.shape, self.dtype, self._contiguous = shape, dtype, contiguous
        self.device = type("D", (), dict(type=device, index=index, __eq__=lambda s, o: (s.type, s.index) == (o.type, o.index)))()

    def is_contiguous(self):
        return self._contiguous

    def data_ptr(self):
        return 4096

    def reshape(self, shape):
        return FakeTensor(shape, self.dtype, self.device.type, self.device.index, self._contiguous)


def test_projection_object():
    p = Projection(FakeTensor((DOUT, DIN)), a=FakeTensor((5, RANK, DIN)), b=FakeTensor((5, DOUT, RANK)),
                   scale=FakeTensor((5,), "torch.float32"), out_dtype="torch.float32")
    assert (p.groups, p.dim_out, p.dim_in, p.adapters, p.rank) == (1, DOUT, DIN, 5, RANK)
    assert (p.struct.dtype, p.struct.out_dtype, p.struct.w, p.struct.scale) == (_lib.BF16, _lib.F32, 4096, 4096)
    assert Projection(FakeTensor((2, DOUT, DIN))).struct.a is None
    w, a, b = FakeTensor((1, DOUT, DIN)), FakeTensor((5, RANK, DIN)), FakeTensor((5, DOUT, RANK))
    for bad in (dict(w=FakeTensor((DIN,))), dict(w=FakeTensor((1, DOUT, DIN), contiguous=False)), dict(w=FakeTensor((1, DOUT, DIN), device="cpu")),
                dict(w=FakeTensor((1, DOUT, DIN), "torch.float64")), dict(w=w, a=a), dict(w=w, b=b), dict(w=w, scale=FakeTensor((5,), "torch.float32")),
                dict(w=w, a=a, b=FakeTensor((5, DOUT, RANK + 1))), dict(w=w, a=FakeTensor((5, RANK, DIN), "torch.float16"), b=b),
                dict(w=w, a=a, b=b, scale=FakeTensor((5,))), dict(w=w, a=FakeTensor((5, RANK, DIN), index=1), b=b),
                dict(w=w, out_dtype="torch.float16"), dict(w=w, out_dtype=7)):
        with pytest.raises(VdbError) as err:
            Projection(**bad)
        assert err.value.code == _lib.EINVAL
