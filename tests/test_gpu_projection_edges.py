"""Learned projections on the GPU at the edges of what the header allows, against their formulas in 64 bits (tolerances: see
test_gpu_projection, whose cases and comparison these are)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_projection import Case                             # noqa: E402


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
