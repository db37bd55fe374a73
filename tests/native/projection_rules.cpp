// Host rules of the learned projections (vectordb_amd/csrc/project.h), built for the CPU: what a launch may read, worked out
// for every small size.  Prints the number of wrong cases.
#include <cstdio>
#include <cstdint>
#include "../../vectordb_amd/csrc/project.h"

using namespace vdb;

// The low-rank factor of one adapter [rows of it][columns of it] as ProjRows has it, read the way the kernels read it in vectors:
// every vector has to lie in the adapter's elements, at a multiple of its size.
static long long factor_reads(int dim_in, int dim_out, int rank, int dtype, bool backward) {
    const int e = dtype == VDB_F32 ? 4 : 2, V = 16 / e;
    ProjRows p{};
    p.row_adapter = (const int*)0x1000;
    p.dtype = dtype;
    p.rank = rank;
    p.w_by_k = backward;
    p.N = backward ? dim_in : dim_out;
    p.K = backward ? dim_out : dim_in;
    p.f = (const void*)0x100000;
    p.f_adapter = (long long)rank * p.N;
    if (backward) { p.f_col = 1; p.f_rank = dim_in; }
    else { p.f_col = rank; p.f_rank = 1; }
    if (!proj_factor_vectors(p)) return 0;
    const long long elements = (long long)rank * p.N;
    long long bad = 0;
    for (int adapter = 0; adapter < 2; ++adapter)
        for (int col = 0; col < (p.N + 63) / 64 * 64; col += backward ? 4 : 1)
            for (int q = 0; q < rank; q += V)
                for (int k = 0; k < (backward ? V : 1); ++k) {
                    if (q + k >= rank) continue;
                    const long long at = (long long)(unsigned)(col < p.N ? col : backward ? 0 : p.N - 1) * p.f_col + (long long)(q + k) * p.f_rank;
                    const long long wide = backward ? 4 : V;
                    bad += at < 0 || at + wide > elements || (at + adapter * p.f_adapter) % wide != 0;
                    // four columns have to be neighbours in memory, as the ranks of a piece have to be
                    bad += backward ? p.f_col != 1 || p.N < 4 : p.f_rank != 1;
                }
    return bad;
}

int main() {
    long long wrong = 0, cases = 0;
    const int dims[] = {1, 2, 3, 4, 5, 7, 8, 12, 16, 63, 64, 65, 68, 96, 130};
    for (int dtype : {VDB_F32, VDB_BF16, VDB_F16})
        for (int di : dims)
            for (int dn : dims)
                for (int rank = 1; rank <= PROJ_MAX_RANK; ++rank)
                    for (int backward = 0; backward < 2; ++backward) {
                        ++cases;
                        const long long bad = factor_reads(di, dn, rank, dtype, backward);
                        if (bad && wrong < 5) printf("factor of %d -> %d, rank %d, type %d, backward %d: %lld reads outside\n", di, dn, rank, dtype, backward, bad);
                        wrong += bad != 0;
                    }
    printf("cases %lld wrong %lld\n", cases, wrong);
    return wrong != 0;
}
