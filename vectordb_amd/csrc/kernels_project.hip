// Learned projections in front of a table: the low-rank intermediates, the gradients of the low-rank factors, and the launches
// (see include/vdb.h for the operators, project.h for the parameters and project_tile.h for the tiled products).
#include "project_tile.h"

namespace vdb {

// ------------------------------------------------------------------------------------------- low-rank intermediates
// Writes four consecutive ranks of one row: as fp32, and as the parts that the low-rank term multiplies.
template <int DT>
__device__ __forceinline__ void pj_store_parts(const ProjShrink& p, long long m, int q, int rp, pj_f32x4 v, float down) {
    if (p.h32 && q < p.rp32) *(pj_f32x4*)(p.h32 + m * p.rp32 + q) = v;
    if (!p.h) return;
    if constexpr (DT == VDB_F32) *(pj_f32x4*)((float*)p.h + m * rp + q) = v;
    else {
        constexpr int NP = proj_parts(DT);
        unsigned short* o = (unsigned short*)p.h + m * (NP * rp) + q;
        if constexpr (DT == VDB_F16) v = v * down;
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            pj_s16x4 s;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] = (short)pj_from_f32<DT>(v[j]);
                const float rest = v[j] - pj_to_f32<DT>((unsigned short)s[j]);
                v[j] = rest == rest ? rest : 0.f;            // an infinity leaves nothing for the later parts
            }
            *(pj_s16x4*)(o + u * rp) = s;
        }
    }
}

// h = s x f^T for 16 rows: the four waves take every fourth step of the contracted axis and add up through LDS in wave
// order.  Each request that meets the 16 rows is multiplied on its own and keeps its own rows; where requests are shorter than
// that, `share` workgroups divide the requests of a block of rows among them.
template <int DT, int NRB, bool XV, bool FV>
__global__ void __launch_bounds__(256)
proj_shrink_kernel(ProjShrink p, int share) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, KS = 4 * V;          // elements per lane and per step
    constexpr int U = NRB <= 2 ? 4 : 2;
    __shared__ pj_f32x4 part[3][NRB][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4, wave = threadIdx.x >> 6;
    const long long r0 = (long long)(blockIdx.x / share) * 16, m = r0 + li;
    const int mine = blockIdx.x % share;
    const int rp = proj_rank_pad(p.rank, DT);
    const T* x = (const T*)p.x + (m < p.n ? m : p.n - 1) * p.ldx;
    int turn = 0;
    pj_each_request(p.offsets, p.ids, p.segments, p.adapters, p.n, r0, r0 + 16, [&](long long b, long long e, int ad) {
        if (turn++ % share != mine) return;
        const T* f = (const T*)p.f + (long long)ad * p.f_adapter;
        pj_f32x4 acc[NRB] = {};
        // U steps at a time, all their loads before the first product
        for (int k0 = wave * KS; k0 < p.K; k0 += U * 4 * KS) {
            union frag { T t[V]; pj_u32x4 v; } xa[U], fa[U][NRB];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * 4 * KS + lh * V;
                if constexpr (XV) xa[u].v = *(const pj_u32x4*)(k < p.K ? x + k : (const T*)pj_zero16);
                else
#pragma unroll
                    for (int j = 0; j < V; ++j) xa[u].t[j] = k + j < p.K ? x[k + j] : (T)0;
#pragma unroll
                for (int i = 0; i < NRB; ++i) {
                    const int q = i * 16 + li;
                    if constexpr (FV) fa[u][i].v = *(const pj_u32x4*)(k < p.K && q < p.rank ? f + (long long)q * p.f_rank + k : (const T*)pj_zero16);
                    else
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            fa[u][i].t[j] = k + j < p.K && q < p.rank ? f[(long long)q * p.f_rank + (long long)(k + j) * p.f_k] : (T)0;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < NRB; ++i) acc[i] = pj_mfma<DT>(fa[u][i].v, xa[u].v, acc[i]);      // lane: row m, ranks 16 i + 4 lh + 0..3
        }
        __syncthreads();
        if (wave)
#pragma unroll
            for (int i = 0; i < NRB; ++i) part[wave - 1][i][lane] = acc[i];
        __syncthreads();
        if (wave == 0) {
            const float sc = p.scale ? p.scale[ad] : 1.f;
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < NRB; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v = acc[i][j];
#pragma unroll
                    for (int w = 0; w < 3; ++w) v += part[w][i][lane][j];
                    acc[i][j] = i * 16 + lh * 4 + j < p.rank ? sc * v : 0.f;
                    const float size = fabsf(acc[i][j]);
                    if (size < __builtin_huge_valf()) most = fmaxf(most, size);
                }
            float down = 1.f;
            if constexpr (DT == VDB_F16) {
                // a power of two that brings the row's largest finite entry to 1/2..1 (1 where that entry is next to the limits of fp32)
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                const int ex = (int)(__float_as_uint(most) >> 23);
                const bool scaled = ex > 2 && ex < 253;
                down = scaled ? __uint_as_float((unsigned)(253 - ex) << 23) : 1.f;      // 2^(126 - ex)
                if (p.h_scale && lh == 0 && m >= b && m < e) p.h_scale[m] = scaled ? __uint_as_float((unsigned)(ex + 1) << 23) : 1.f;
            }
            if (m >= b && m < e) {
#pragma unroll
                for (int i = 0; i < NRB; ++i) if (i * 16 < rp) pj_store_parts<DT>(p, m, i * 16 + lh * 4, rp, acc[i], down);
            }
        }
    });
}

// ------------------------------------------------------------------------------------------- gradient of the factors
// One adapter's [rank] x 64 columns: the four waves take its rows 16 at a time in turn, over every request that names the
// adapter, and add up in wave order.  Products on the fp32 matrix unit: h is fp32, x is widened.
// Lane l loads columns 4 (l % 16) + 0..3 of a row, so that product j of a step holds columns j, 4 + j, 8 + j, ...
template <int DT, int ODT, int NRB, bool XV>
__global__ void __launch_bounds__(256)
proj_factor_kernel(ProjFactor p) {
    typedef typename PJ<DT>::T T;
    typedef typename PJ<ODT>::T O;
    __shared__ pj_f32x4 part[3][4][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4, wave = threadIdx.x >> 6;
    const int n0 = blockIdx.x * 64, ad = blockIdx.y, c0 = n0 + li * 4;
    pj_f32x4 acc[NRB][4] = {};
    int turn = 0;                          // blocks of 16 rows met so far
    for (int s0 = 0; s0 < p.segments; s0 += 64) {
        const bool hit = s0 + lane < p.segments && p.ids[s0 + lane] == ad;
        unsigned long long mask = __ballot(hit);
        while (mask) {
            const int s = s0 + __builtin_ctzll(mask);
            mask &= mask - 1;
            const long long b = pj_clamp(p.offsets[s], p.n), e = pj_clamp(p.offsets[s + 1], p.n);
            for (long long r = b; r < e; r += 16) {
                if ((turn++ & 3) != wave) continue;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const long long i = r + u * 4 + lh;
                    const bool ok = i < e;
                    float xv[4];
                    if constexpr (XV) {
                        typedef T tx4 __attribute__((ext_vector_type(4)));
                        const tx4 v = *(const tx4*)(ok && c0 < p.N ? (const T*)p.x + i * p.ldx + c0 : (const T*)pj_zero16);
#pragma unroll
                        for (int j = 0; j < 4; ++j) xv[j] = pj_to_f32<DT>(v[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) xv[j] = ok && c0 + j < p.N ? pj_to_f32<DT>(((const T*)p.x)[i * p.ldx + c0 + j]) : 0.f;
                    }
#pragma unroll
                    for (int q = 0; q < NRB; ++q) {
                        const float hv = ok && q * 16 < p.rp ? p.h[i * p.rp + q * 16 + li] : 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            acc[q][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[j], hv, acc[q][j], 0, 0, 0);
                    }
                }
            }
        }
    }
    O* out = (O*)p.out + (long long)ad * p.rank * p.N;
#pragma unroll
    for (int q = 0; q < NRB; ++q) {
        __syncthreads();
        if (wave)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[wave - 1][j][lane] = acc[q][j];
        __syncthreads();
        const int k = q * 16 + li;
        if (wave || k >= p.rank) continue;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = n0 + lh * 16 + u * 4 + j;
                if (c >= p.N) continue;
                const float v = acc[q][j][u] + part[0][j][lane][u] + part[1][j][lane][u] + part[2][j][lane][u];
                out[p.by_col ? (long long)c * p.rank + k : (long long)k * p.N + c] = pj_from_f32<ODT>(v);
            }
    }
}

__global__ void __launch_bounds__(256)
proj_zero_outside_kernel(float* q, long long dim, long long n, const long long* offsets, int segments) {
    const long long b = segments > 0 ? pj_clamp(offsets[0], n) : 0, e = segments > 0 ? pj_clamp(offsets[segments], n) : 0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n * dim; i += (long long)gridDim.x * 256) {
        const long long r = i / dim;
        if (r < b || r >= e) q[i] = 0.f;
    }
}

// ------------------------------------------------------------------------------------------- launches
#define PJ_BY_TYPE(FN)                                                              \
    do {                                                                            \
        if (p.dtype == VDB_F32) return FN##_f32(p, st);                             \
        return p.dtype == VDB_BF16 ? FN##_bf16(p, st) : FN##_f16(p, st);            \
    } while (0)

hipError_t launch_proj_rows(const ProjRows& p, hipStream_t st) {
    if (p.n <= 0 || p.segments <= 0) return hipSuccess;
    PJ_BY_TYPE(launch_proj_rows);
}

hipError_t launch_proj_weights(const ProjWeights& p, hipStream_t st) { PJ_BY_TYPE(launch_proj_weights); }

template <int DT, int NRB>
static hipError_t shrink_typed(const ProjShrink& p, hipStream_t st) {
    constexpr int E = PJ<DT>::E, V = 16 / E;
    const bool xv = pj_aligned(p.x, p.ldx, E, 16) && p.K % V == 0;
    const bool fv = p.f_k == 1 && pj_aligned(p.f, p.f_rank, E, 16) && p.K % V == 0;
    const long long blocks = (p.n + 15) / 16;
    long long share = (p.segments + blocks - 1) / blocks;       // requests per block of rows, if they are of one length
    share = share < 1 ? 1 : share > 16 ? 16 : share;
    const dim3 grid((unsigned)(blocks * share));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, (int)share);
        return hipGetLastError();
    };
    if (!xv) return fv ? go(proj_shrink_kernel<DT, NRB, false, true>) : go(proj_shrink_kernel<DT, NRB, false, false>);
    return fv ? go(proj_shrink_kernel<DT, NRB, true, true>) : go(proj_shrink_kernel<DT, NRB, true, false>);
}

template <int DT, int ODT, int NRB>
static hipError_t factor_typed(const ProjFactor& p, hipStream_t st) {
    const dim3 grid((unsigned)((p.N + 63) / 64), (unsigned)p.adapters);
    const bool xv = pj_aligned(p.x, p.ldx, PJ<DT>::E, 4 * PJ<DT>::E) && p.N % 4 == 0;
    return xv ? pj_launch(proj_factor_kernel<DT, ODT, NRB, true>, grid, 0, p, st)
              : pj_launch(proj_factor_kernel<DT, ODT, NRB, false>, grid, 0, p, st);
}

// blocks of 16 of the rank, rounded up to a power of two
#define PJ_BY_RANK(CALL)                                       \
    do {                                                       \
        if (p.rank <= 16) { constexpr int NRB = 1; CALL; }     \
        else if (p.rank <= 32) { constexpr int NRB = 2; CALL; }\
        else if (p.rank <= 64) { constexpr int NRB = 4; CALL; }\
        else { constexpr int NRB = 8; CALL; }                  \
    } while (0)

hipError_t launch_proj_shrink(const ProjShrink& p, hipStream_t st) {
    if (p.n <= 0 || p.segments <= 0) return hipSuccess;
    if (p.dtype == VDB_F32) PJ_BY_RANK(return (shrink_typed<VDB_F32, NRB>(p, st)));
    // 16-bit parts are padded to steps of 32 ranks
    const int nrb = proj_rank_pad(p.rank, p.dtype) / 16;
#define PJ_SHRINK(DT) (nrb <= 2 ? shrink_typed<DT, 2>(p, st) : nrb <= 4 ? shrink_typed<DT, 4>(p, st) : shrink_typed<DT, 8>(p, st))
    return p.dtype == VDB_BF16 ? PJ_SHRINK(VDB_BF16) : PJ_SHRINK(VDB_F16);
#undef PJ_SHRINK
}

hipError_t launch_proj_factor(const ProjFactor& p, hipStream_t st) {
    if (p.dtype == VDB_F32) PJ_BY_RANK(return (factor_typed<VDB_F32, VDB_F32, NRB>(p, st)));
    if (p.dtype == VDB_BF16) {
        if (p.out_dtype == VDB_F32) PJ_BY_RANK(return (factor_typed<VDB_BF16, VDB_F32, NRB>(p, st)));
        PJ_BY_RANK(return (factor_typed<VDB_BF16, VDB_BF16, NRB>(p, st)));
    }
    if (p.out_dtype == VDB_F32) PJ_BY_RANK(return (factor_typed<VDB_F16, VDB_F32, NRB>(p, st)));
    PJ_BY_RANK(return (factor_typed<VDB_F16, VDB_F16, NRB>(p, st)));
}

hipError_t launch_proj_zero_outside(float* q, long long dim, long long n, const long long* offsets, int segments, hipStream_t st) {
    const long long blocks = (n * dim + 255) / 256;
    hipLaunchKernelGGL(proj_zero_outside_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, st, q, dim, n, offsets, segments);
    return hipGetLastError();
}

}  // namespace vdb
