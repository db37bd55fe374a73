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

// Every launch of the largest calls that are taken: workgroups beyond the limit, or no adapter to a launch.
static long long launches(long long n, int dim_in, int dim_out, int groups, bool adapted) {
    long long bad = 0;
    ProjRows r{};
    r.n = n; r.segments = adapted ? 1 : groups;
    if (adapted) r.row_adapter = (const int*)0x1000;
    for (int back = 0; back < 2; ++back) {
        r.N = back ? dim_in : dim_out;
        for (int R : {64, 128}) bad += proj_rows_grid(r, R) > PROJ_MAX_WORKGROUPS;
    }
    ProjWeights w{};
    w.n = n; w.segments = groups; w.M = dim_out; w.N = dim_in;
    proj_weights_plan(n, groups, dim_out, dim_in, w.tile, w.chunk);
    for (int t : {64, 128}) if (t <= w.tile || w.tile == 64) bad += proj_weights_grid(w, t, t) > PROJ_MAX_WORKGROUPS;
    bad += proj_weights_grid(w, 256, 128) > PROJ_MAX_WORKGROUPS;
    if (!adapted || n < 1) return bad;
    for (int requests : {1, 2, 1000, 1 << 15, 1 << 20}) bad += proj_shrink_grid(n, requests) > PROJ_MAX_WORKGROUPS;
    for (int adapters : {1, 2, 7, 16, 1000, 4096, 4097, 65535}) {
        const long long width = dim_in > dim_out ? dim_in : dim_out;
        const int splits = proj_factor_splits(n, adapters), step = proj_factor_adapters(adapters, splits, width);
        bad += step < 1 || step > adapters || (width + 63) / 64 * step * 2 * splits > PROJ_MAX_WORKGROUPS;
        bad += step < adapters && (width + 63) / 64 * (step + 1) * 2 * splits <= PROJ_MAX_WORKGROUPS;        // no launch more than needed
    }
    return bad;
}

static long long limits(long long& cases) {
    long long wrong = 0;
    for (long long di : {1, 64, 65, 128, 384, 768, 1024, 4096, 65536})
        for (long long dn : {1, 64, 65, 384, 768, 4100, 65536})
            for (long long groups : {1, 2, 8, 500, 2048, 4096})
                for (int adapted = 0; adapted < (groups == 1 ? 2 : 1); ++adapted) {
                    ++cases;
                    long long lo = -1, hi = 1LL << 40;                       // lo is taken, hi is not
                    while (lo + 1 < hi) {
                        const long long mid = (lo + hi) / 2;
                        (proj_sizes_fit(mid, di, dn, groups, adapted) ? lo : hi) = mid;
                    }
                    if (lo < 0) continue;
                    // the limit as it is documented
                    const long long ti = (di + 63) / 64, to = (dn + 63) / 64, longer = ti > to ? ti : to;
                    long long most = ((1LL << 23) - 8) / longer - groups - 1;
                    most = most * 64 + 63;
                    if (adapted && most > 1LL << 27) most = 1LL << 27;
                    const bool stated = groups * ti * to <= 1LL << 23 && lo == most;
                    long long bad = !stated;
                    for (long long n : {lo, lo - 1, lo / 2, lo / 3, lo / 64, lo / 4096, 1000LL})
                        if (n >= 0 && n <= lo) bad += launches(n, (int)di, (int)dn, (int)groups, adapted);
                    if (bad && wrong < 5) printf("limit of %lld -> %lld, %lld groups, adapted %d: %lld rows, %lld wrong\n", di, dn, groups, adapted, lo, bad);
                    wrong += bad != 0;
                }
    return wrong;
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
    printf("factors: cases %lld wrong %lld\n", cases, wrong);
    cases = 0;
    const long long beyond = limits(cases);
    printf("limits: cases %lld wrong %lld\n", cases, beyond);
    return 0;
}
