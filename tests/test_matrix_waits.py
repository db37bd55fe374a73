"""CPU test: no kernel of the built library reads a result of the matrix unit before it is there (see matrix_waits)."""
import os
import shutil
import tempfile
from concurrent.futures import ProcessPoolExecutor

import pytest

import matrix_waits

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vectordb_amd", "libvdb.so")
OBJDUMP = shutil.which("llvm-objdump") or os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")


def found(code):
    """(kernels with products, products, [early uses]) of one code object.  Writes over a result are looked at in the projection
    kernels only: in gemm32s_kernel the way to one is there in the code but never taken (a tile's sums are cleared after its epilogue
    has read them)."""
    kernels = products = 0
    bad = []
    with tempfile.NamedTemporaryFile(suffix=".elf") as f:
        f.write(code)
        f.flush()
        for name, ins in matrix_waits.functions(OBJDUMP, f.name):
            n = sum(op.startswith("v_mfma") for op, _, _ in ins)
            if n:
                kernels += 1
                products += n
                bad += [(name,) + e for e in matrix_waits.early(ins, writes="proj_" in name)]
    return kernels, products, bad


def test_no_result_is_read_before_it_is_there():
    if not os.path.exists(LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no llvm-objdump")
    with ProcessPoolExecutor(4) as pool:
        results = list(pool.map(found, matrix_waits.code_objects(LIB)))
    bad = [b for _, _, more in results for b in more]
    assert not bad, "%d early uses, first: %s" % (len(bad), bad[0])
    assert sum(k for k, _, _ in results) > 200 and sum(n for _, n, _ in results) > 10000


def lines(*ins):
    """Text of instructions of four bytes each, as a disassembler prints them."""
    return "\n".join("\t%s // %012X: 00000000" % (t, 4 * i) for i, t in enumerate(ins))


MFMA32 = "v_mfma_f32_16x16x4_f32 v[0:3], v10, v11, v[0:3]"
MFMA16 = "v_mfma_f32_16x16x32_bf16 a[0:3], v[10:13], v[14:17], a[0:3]"


@pytest.mark.parametrize("ins,early", [
    ((MFMA32, "s_nop 8", "v_add_f32_e32 v9, v3, v3"), 1),                       # 9 states, 10 needed
    ((MFMA32, "s_nop 9", "v_add_f32_e32 v9, v3, v3"), 0),
    ((MFMA32, "s_nop 4", "s_nop 3", "s_mov_b32 s0, 0", "v_add_f32_e32 v9, v3, v3"), 0),
    ((MFMA32, "s_nop 7", "v_mov_b32_e32 v2, 0"), 1),                            # a write over it
    ((MFMA32, MFMA32, "s_nop 9", "v_add_f32_e32 v9, v3, v3"), 0),               # adding on waits by itself
    ((MFMA32, "v_mfma_f32_16x16x4_f32 v[4:7], v2, v11, v[4:7]"), 1),            # as a factor it does not
    ((MFMA32, "s_cbranch_scc1 1", "s_nop 9", "global_store_dword v20, v1, s[0:1]"), 1),     # short by the branch
    ((MFMA32, "s_cbranch_scc1 65534", "s_nop 9", "v_add_f32_e32 v9, v3, v3"), 0),           # a loop that it ends
    ((MFMA16, "s_nop 6", "v_accvgpr_read_b32 v9, a3"), 1),
    ((MFMA16, "s_nop 7", "v_accvgpr_read_b32 v9, a3"), 0),
    ((MFMA16, "v_add_f32_e32 v9, v3, v3", "ds_write_b32 v0, v1"), 0),           # other registers
    ((MFMA16, "s_endpgm", "v_accvgpr_read_b32 v9, a3"), 0),
])
def test_the_check_itself(ins, early):
    assert len(list(matrix_waits.early(matrix_waits.parse(lines(*ins))))) == early
