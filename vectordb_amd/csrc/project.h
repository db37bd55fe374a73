// Parameters of the projection kernels (kernels_project.hip): learned maps of embeddings into a table's space.
// Rows lie in segments: segment s holds rows [offsets[s], offsets[s + 1]).  Offsets come from device memory and are
// clamped to [0, n] by every kernel, so that no value of them reaches memory outside the operands.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/vdb.h"

namespace vdb {

constexpr int PROJ_MAX_RANK = 128;
// No launch needs more workgroups; sizes that would are refused (proj_sizes_fit), or take several launches.
constexpr long long PROJ_MAX_WORKGROUPS = 1LL << 23;
constexpr long long PROJ_MAX_REQUESTS = 1LL << 20, PROJ_MAX_ADAPTED_ROWS = 16 * PROJ_MAX_WORKGROUPS;
// Workgroups that the gradient of the matrices is divided into where its output tiles are fewer (32 768 rows of 8 groups, 1024 x 768
// bf16, whole backward pass: 287 us with 256, 206 with 512, 194 with 768, 204 with 1024).
constexpr int PJ_SPLIT_WGS = 768;
// A low-rank intermediate h [n, rank], fp32, is handed to the kernel that multiplies it as it is beside fp32 rows, and as three bf16
// parts that add up to it beside 16-bit ones (three times 8 bits, and each part with an exponent of its own: parts in fp16 would lose
// the small ranks of a row beside its large ones; only what lies below fp32's smallest normal number, 2^-126, may be lost): rows of proj_parts x proj_rank_pad elements (a step of the matrix unit is 32 ranks
// for 16-bit types, 16 for fp32).
__host__ __device__ constexpr int proj_parts(int dtype) { return dtype == VDB_F32 ? 1 : 3; }
__host__ __device__ constexpr int proj_rank_pad(int rank, int dtype) {
    return dtype == VDB_F32 ? (rank + 15) / 16 * 16 : (rank + 31) / 32 * 32;
}

// y = x M^T with M [dim_y, dim_x] per segment or shared; the same kernel takes dx = dy M (M read down its columns).
struct ProjRows {
    const void* x; long long ldx;        // [n, K] rows, K contiguous
    const void* w; long long w_group;    // matrix of segment 0; elements from one segment's matrix to the next (0: shared)
    long long ldw;                       // elements between rows of the matrix as it is stored
    bool w_by_k;                         // false: element (column, k) at column * ldw + k; true: at k * ldw + column
    void* y; long long ldy;              // [n, N]
    long long n; int N, K;
    int dtype, out_dtype;
    const long long* offsets; int segments;
    // low-rank term: y_i += sum_q h[i][q] f[row_adapter[i]][column][q]; null: none
    const int* row_adapter;              // [n], -1: none
    const void* h;                       // [n][proj_parts][proj_rank_pad]
    const void* f; long long f_adapter, f_col, f_rank;       // strides in elements
    int rank;
};

// Workgroups of the products of the rows by tiles of R x R: each segment that can have rows adds at most one tile to those that the
// rows alone would fill; a multiple of eight, for the eight XCDs.
inline long long proj_rows_grid(const ProjRows& p, int R) {
    const long long tiles = p.row_adapter ? (p.n + R - 1) / R : p.n / R + (p.n < p.segments ? p.n : p.segments);
    return (tiles * ((p.N + R - 1) / R) + 7) / 8 * 8;
}

// Do all launches of a call stay within PROJ_MAX_WORKGROUPS?  The products of the rows and the gradient of the matrices by 64 x 64
// tiles (smaller ones are for small calls), the low-rank intermediate by 16 rows.
inline bool proj_sizes_fit(long long n, long long dim_in, long long dim_out, long long groups, bool adapted) {
    const long long ti = (dim_in + 63) / 64, to = (dim_out + 63) / 64, most = PROJ_MAX_WORKGROUPS;
    return n / 64 + groups + 1 <= (most - 8) / (ti > to ? ti : to) && groups * ti <= most / to && (!adapted || n <= PROJ_MAX_ADAPTED_ROWS);
}

// Can the low-rank factor be read in vectors?  Along a matrix stored column by column (forward) the kernels read 16 bytes of ranks
// (PJ_F_RANKS), along one stored by k (backward) four columns (PJ_F_COLS).  It goes by the way the launch will read: with one input
// column, a backward pass has ranks one element apart too.
inline bool proj_factor_vectors(const ProjRows& p) {
    const int e = p.dtype == VDB_F32 ? 4 : 2;
    if (!p.row_adapter) return false;
    if (p.w_by_k) return p.f_col == 1 && p.N % 4 == 0 && (uintptr_t)p.f % (4 * e) == 0;
    return p.f_rank == 1 && p.rank % (16 / e) == 0 && (uintptr_t)p.f % 16 == 0;
}

// h[i][q] = scale[a] * sum_k x[i][k] f[a][q][k] for rows with an adapter; padding is zero
struct ProjShrink {
    const void* x; long long ldx; long long n; int K;
    const void* f; long long f_adapter, f_rank, f_k;
    const float* scale;
    void* h;                             // parts, see ProjRows; null: not wanted
    int* row_adapter;                    // [n]: the adapter of each row, -1: none; may be null
    float* h32; int rp32;                // [n][rp32] fp32; null: not wanted
    int rank, dtype;
    const long long* offsets; int segments; const int* ids; int adapters;
};

// Workgroups for the adapters of one block of 16 rows: as many as it meets if all requests were of one length, and a workgroup to
// a CU.  More are dispatched in vain (1024 rows of 128 requests: 12.4 us with 256 workgroups in all, 15.1 with 1024), fewer
// leave adapters one after the other (15.8 us with 128).
inline long long proj_shrink_share(long long n, int segments) {
    const long long blocks = (n + 15) / 16;
    long long share = segments / blocks;
    if (share < 256 / blocks) share = 256 / blocks;
    if (share > segments) share = segments;
    return share < 1 ? 1 : share > 16 ? 16 : share;
}
// Workgroups of an intermediate by 16 rows, and by 64 rows with the workgroups for those that meet many adapters.
inline long long proj_shrink_grid(long long n, int segments) { return (n + 15) / 16 * proj_shrink_share(n, segments); }
inline long long proj_shrink_tile_grid(long long n) { return (n + 63) / 64 + (n + 15) / 16; }

// dw[g][m][c] = sum over the rows i of segment g of dy[i][m] x[i][c]
struct ProjWeights {
    const void* dy; long long lddy;
    const void* x; long long ldx;
    void* dw; int M, N;                  // [segments][M][N]
    long long n; int dtype, out_dtype;
    const long long* offsets; int segments;
    int tile;                            // 128 or 64, see proj_weights_plan
    int chunk;                           // rows per workgroup where segments are split, 0: they are not
    float* partial;                      // chunk > 0: [n / chunk + segments][M][N]
};

// How the gradient of the matrices is divided: 128 x 128 output tiles where they fill half the chip by themselves, or would with
// segments of 2048 rows split; 64 x 64 ones otherwise; and chunks of rows that give every CU two workgroups.
inline void proj_weights_plan(long long n, int segments, int M, int N, int& tile, int& chunk) {
    const long long t128 = (long long)((M + 127) / 128) * ((N + 127) / 128), t64 = (long long)((M + 63) / 64) * ((N + 63) / 64);
    tile = segments * t128 >= 256 || n / 2048 * t128 >= 256 ? 128 : 64;
    const long long tiles = tile == 128 ? t128 : t64;
    chunk = 0;
    if (segments * tiles >= PJ_SPLIT_WGS) return;
    long long c = (n * tiles + PJ_SPLIT_WGS - 1) / PJ_SPLIT_WGS;
    c = (c + 63) / 64 * 64;
    if (c < 128) c = 128;
    if (c < n) chunk = (int)c;
}

// Workgroups of the gradient of the matrices by tiles of tm x tn.
inline long long proj_weights_grid(const ProjWeights& p, int tm, int tn) {
    const long long tiles = (long long)((p.M + tm - 1) / tm) * ((p.N + tn - 1) / tn);
    const long long items = p.chunk > 0 ? p.n / p.chunk + (p.n < p.segments ? p.n : p.segments) : p.segments;
    return (items * tiles + 7) / 8 * 8;
}

// Workgroups that share the rows of an adapter, as many as leave 512 rows to each, and 16 over all adapters: with few adapters
// there are too few workgroups, with many the ones that find no rows cost more than the others gain (whole backward pass, 768 x
// 768 bf16, rank 16, alone and shared: 16 384 rows of 1 adapter 174 and 76 us, of 4 adapters 105 and 78, of 24 adapters by two 80
// and 83; 1024 x 768 fp16, rank 64, 4096 rows of 10 adapters by three 74 and 81).
constexpr int PJ_FACTOR_SHARES = 16;
inline int proj_factor_splits(long long n, int adapters) {
    const long long most = n / 512, want = PJ_FACTOR_SHARES / adapters;
    const long long s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s);
}
// Adapters whose gradients one launch takes, of factors with up to `width` columns.
inline int proj_factor_adapters(int adapters, int splits, long long width) {
    const long long most = PROJ_MAX_WORKGROUPS / ((width + 63) / 64 * 2 * splits);
    return (int)(adapters < most ? adapters : most);
}
// floats of the partial sums of one factor's gradient
inline long long proj_factor_partial(int splits, int adapters, int rank, long long N) {
    const int nrb = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
    return splits > 1 ? (long long)splits * adapters * ((N + 63) / 64) * (nrb * 1024) : 0;
}

// out[a][q][c] (or, by_col, out[a][c][q]) = sum over the rows i of adapter a of h[i][q] x[i][c]
struct ProjFactor {
    const float* h; int rp, rank;
    const void* x; long long ldx; int N;
    void* out; bool by_col;
    int splits; float* partial;          // workgroups that share an adapter's rows; splits > 1: proj_factor_partial floats
    long long n; int dtype, out_dtype;
    const long long* offsets; int segments; const int* ids; int adapters;
    int first;                           // adapter of the launch's first workgroups
};

hipError_t launch_proj_rows(const ProjRows& p, hipStream_t st);
hipError_t launch_proj_rows_f32(const ProjRows& p, hipStream_t st);
hipError_t launch_proj_rows_bf16(const ProjRows& p, hipStream_t st);
hipError_t launch_proj_rows_f16(const ProjRows& p, hipStream_t st);
hipError_t launch_proj_weights_f32(const ProjWeights& p, hipStream_t st);
hipError_t launch_proj_weights_bf16(const ProjWeights& p, hipStream_t st);
hipError_t launch_proj_weights_f16(const ProjWeights& p, hipStream_t st);
hipError_t launch_proj_shrink(const ProjShrink& p, hipStream_t st);
hipError_t launch_proj_weights(const ProjWeights& p, hipStream_t st);
hipError_t launch_proj_weights_sum(const ProjWeights& p, hipStream_t st);      // the second step where segments are split
// an adapted forward pass: the intermediate, then the rows, or both in one launch for a few rows
hipError_t launch_proj_adapted(const ProjRows& p, const ProjShrink& s, hipStream_t st);
// both intermediates of a backward pass, of dy and of x; the gradients of both factors
hipError_t launch_proj_shrink_pair(const ProjShrink& g, const ProjShrink& h, hipStream_t st);
hipError_t launch_proj_factors(const ProjFactor& a, const ProjFactor& b, hipStream_t st);
hipError_t launch_proj_zero(float* q, long long count, hipStream_t st);

}  // namespace vdb
