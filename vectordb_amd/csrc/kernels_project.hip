// Learned projections in front of a table: the low-rank intermediates, the gradients of the low-rank factors, and the launches
// (see include/vdb.h for the operators, project.h for the parameters and project_tile.h for the tiled products).
#include "project_tile.h"

namespace vdb {

// ------------------------------------------------------------------------------------------- low-rank intermediates
// Writes four consecutive ranks of one row: as fp32, and as the parts that the low-rank term multiplies.
template <int DT>
__device__ __forceinline__ void pj_store_parts(const ProjShrink& p, long long m, int q, int rp, pj_f32x4 v) {
    if (p.h32 && q < p.rp32) *(pj_f32x4*)(p.h32 + m * p.rp32 + q) = v;
    if (!p.h) return;
    if constexpr (DT == VDB_F32) *(pj_f32x4*)((float*)p.h + m * rp + q) = v;
    else {
        constexpr int NP = proj_parts(DT);
        unsigned short* o = (unsigned short*)p.h + m * (NP * rp) + q;
#pragma unroll
        for (int u = 0; u < NP; ++u) {
            pj_s16x4 s;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // cut, not rounded: three times 8 bits are all of them, and no part of a finite value is infinite
                const unsigned part = __float_as_uint(v[j]) & 0xffff0000u;
                s[j] = (short)(part >> 16);
                const float rest = v[j] - __uint_as_float(part);
                v[j] = rest == rest ? rest : 0.f;            // an infinity leaves nothing for the later parts
            }
            *(pj_s16x4*)(o + u * rp) = s;
        }
    }
}

// How the factor of a shrink lies: FK: contiguous along the contracted axis, 16-byte pieces aligned (A of a forward pass);
// FR: contiguous along the ranks, whole 16-byte pieces (B of a backward pass); else any strides.
enum { PJ_S_ANY = 0, PJ_S_FK = 1, PJ_S_FR = 2 };

// The rows' side of XS steps of the contracted axis at k0, k0 + stride, ...
template <int DT, int XS, bool XV>
__device__ __forceinline__ void pj_shrink_load_x(const ProjShrink& p, const typename PJ<DT>::T* x, int k0, int stride, pj_u32x4 (&xa)[XS]) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E;
    const int lh = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int u = 0; u < XS; ++u) {
        const int k = k0 + u * stride + lh * V;
        if constexpr (XV) xa[u] = pj_load_if<pj_u32x4>(k < p.K, x + k);
        else xa[u] = pj_piece<T>(x + k, p.K - k, p.K >= V);
    }
}

// U steps: acc[i] += (ranks 16 i.. of f) x^T, all loads ahead of the products.
// FR, 16-bit: a step's 32 lines of the factor pass through `lds`, a part of it that belongs to this wave, and come back
// transposed (ds_read_b64_tr_b16: blocks of 4 lines x 16 ranks).
template <int DT, int NRB, int F, int U>
__device__ __forceinline__ void pj_shrink_steps(const ProjShrink& p, const pj_u32x4* xa, const typename PJ<DT>::T* f, int k0, int stride,
                                                char* lds, pj_f32x4 (&acc)[NRB]) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E;
    constexpr bool TR = F == PJ_S_FR && DT != VDB_F32;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    union frag { T t[V]; pj_u32x4 v; } fa[U][NRB];
    const unsigned fr = (unsigned)p.f_rank, fk = (unsigned)p.f_k;            // an adapter's elements number less than 2^32
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = k0 + u * stride + lh * V;
        if constexpr (TR) {
            // pieces of 8 ranks: piece c is line c / (rank / 8) of the step
            const int ppl = p.rank / 8, kb = k0 + u * stride;
#pragma unroll
            for (int i = 0; i < NRB; ++i) {
                const int c = i * 64 + lane;
                const bool in = c < 32 * ppl && kb + c / ppl < p.K;
                fa[u][i].v = pj_load_if<pj_u32x4>(in, f + (unsigned)kb * fk + (unsigned)c * 8u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NRB; ++i) {
                const int q = i * 16 + li;
                const unsigned at = (unsigned)q * fr + (unsigned)k * fk;
                if constexpr (F == PJ_S_FK) fa[u][i].v = pj_load_if<pj_u32x4>(k < p.K && q < p.rank, f + at);
                else
#pragma unroll
                    for (int j = 0; j < V; ++j) fa[u][i].t[j] = k + j < p.K && q < p.rank ? f[at + (unsigned)j * fk] : (T)0;
            }
        }
    }
    if constexpr (TR) {
        const int line = p.rank * 2;                   // bytes; ranks past the last read the next line and are dropped by the caller
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NRB; ++i) *(pj_u32x4*)(lds + (u * NRB + i) * 1024 + lane * 16) = fa[u][i].v;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NRB; ++i) {
                const char* at = lds + u * NRB * 1024 + (lh * 8 + (li >> 2)) * line + i * 32 + (li & 3) * 8;
                union { pj_s16x4 h[2]; pj_u32x4 v; } t;
                t.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PJ_LOCAL pj_s16x4*)at);
                t.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PJ_LOCAL pj_s16x4*)(at + 4 * line));
                fa[u][i].v = t.v;
            }
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NRB; ++i) acc[i] = pj_mfma<DT>(fa[u][i].v, xa[u], acc[i]);      // lane: row, ranks 16 i + 4 lh + 0..3
}

// LDS of a wave for pj_shrink_steps: the lines of U steps, and what the reads of ranks past the last may touch behind them
template <int DT, int NRB, int F, int U> constexpr int pj_shrink_lds() { return F == PJ_S_FR && DT != VDB_F32 ? U * NRB * 1024 + 256 : 16; }

// Scales one row block's sums and stores the rows of adapter `ad` (`mine`: this lane's row is one of them).
template <int DT, int NRB>
__device__ __forceinline__ void pj_shrink_store(const ProjShrink& p, long long m, bool mine, int ad, pj_f32x4 (&acc)[NRB]) {
    const int lh = (threadIdx.x & 63) >> 4, rp = proj_rank_pad(p.rank, DT);
    const float sc = p.scale ? p.scale[ad] : 1.f;
#pragma unroll
    for (int i = 0; i < NRB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = i * 16 + lh * 4 + j < p.rank ? sc * acc[i][j] : 0.f;
    if (mine) {
#pragma unroll
        for (int i = 0; i < NRB; ++i) if (i * 16 < rp) pj_store_parts<DT>(p, m, i * 16 + lh * 4, rp, acc[i]);
    }
}

// Adapter of each of B times 16 rows (lane l: row + 16 i + l % 16); -1: none.
template <int B>
__device__ __forceinline__ void pj_row_adapters(const ProjShrink& p, long long row, int (&am)[B]) {
    const int li = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < B; ++i) am[i] = -1;
    pj_each_request(p.offsets, p.ids, p.segments, p.adapters, p.n, row, row + B * 16, [&](long long b, long long e, int a) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const long long m = row + i * 16 + li;
            am[i] = m >= b && m < e ? a : am[i];
        }
    });
}

// LDS of pj_shrink_block: the waves' sums, and each wave's lines
template <int DT, int NRB, int F> constexpr int pj_shrink_block_lds() {
    return 3 * NRB * 1024 + 4 * pj_shrink_lds<DT, NRB, F, (NRB <= 2 ? 4 : 2)>();
}

// h = s x f^T for 16 rows: the four waves take every fourth step of the contracted axis and add up through LDS in wave
// order.  Each adapter that the 16 rows meet is multiplied on its own and keeps its own rows; `share` workgroups divide
// the adapters of a block of rows among them.  The rows are loaded before the adapters are known.
// What bounds it is latency (offsets, then the factor, then the exchange): a wave to 16 rows without the exchange, and 64 rows
// to a workgroup, which reads the factor a quarter as often, were both slower at small ranks (24 and 26 against 18 us for
// 16 384 x 768 of rank 16; for many rows of ranks above 32 see proj_shrink_tile_kernel).
template <int DT, int NRB, bool XV, int F>
__device__ __forceinline__ void pj_shrink_block(const ProjShrink& p, long long r0, int mine, int share, char* smem) {
    typedef typename PJ<DT>::T T;
    constexpr int KS = 64 / PJ<DT>::E, XS = 8, U = NRB <= 2 ? 4 : 2;
    const int lane = threadIdx.x & 63, li = lane & 15, wave = threadIdx.x >> 6;
    pj_f32x4 (*const part)[NRB][64] = (pj_f32x4 (*)[NRB][64])smem;
    char* const lds = smem + 3 * NRB * 1024 + wave * pj_shrink_lds<DT, NRB, F, U>();
    const long long m = r0 + li;
    const T* x = (const T*)p.x + (m < p.n ? m : p.n - 1) * p.ldx;
    pj_u32x4 xa[XS];
    pj_shrink_load_x<DT, XS, XV>(p, x, wave * KS, 4 * KS, xa);
    int am[1];
    pj_row_adapters<1>(p, r0, am);
    if (p.row_adapter && mine == 0 && wave == 0 && lane < 16 && m < p.n) p.row_adapter[m] = am[0];
    unsigned left = (unsigned)__ballot(am[0] >= 0) & 0xffffu;
    for (int turn = 0; left; turn = turn + 1 == share ? 0 : turn + 1) {
        const int ad = __builtin_amdgcn_readlane(am[0], __builtin_ctz(left));
        left &= ~(unsigned)__ballot(am[0] == ad);
        if (turn != mine) continue;
        const T* f = (const T*)p.f + (long long)ad * p.f_adapter;
        pj_f32x4 acc[NRB] = {};
        for (int kc = wave * KS; kc < p.K; kc += XS * 4 * KS) {
            if (p.K > XS * 4 * KS) pj_shrink_load_x<DT, XS, XV>(p, x, kc, 4 * KS, xa);
#pragma unroll
            for (int u = 0; u < XS; u += U)
                if (kc + u * 4 * KS < p.K) pj_shrink_steps<DT, NRB, F, U>(p, xa + u, f, kc + u * 4 * KS, 4 * KS, lds, acc);
        }
        __syncthreads();
        if (wave)
#pragma unroll
            for (int i = 0; i < NRB; ++i) part[wave - 1][i][lane] = acc[i];
        __syncthreads();
        if (wave) continue;
#pragma unroll
        for (int i = 0; i < NRB; ++i)
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += part[w][i][lane][j];
        pj_shrink_store<DT, NRB>(p, m, am[0] == ad, ad, acc);
    }
}

template <int DT, int NRB, bool XV, int F>
__global__ void __launch_bounds__(256)
proj_shrink_kernel(ProjShrink p, int share) {
    __shared__ __attribute__((aligned(16))) char smem[pj_shrink_block_lds<DT, NRB, F>()];
    pj_shrink_block<DT, NRB, XV, F>(p, (long long)(blockIdx.x / share) * 16, blockIdx.x % share, share, smem);
}

// Both intermediates of a backward pass in one launch: g of dy (its factor contiguous along the ranks), h of x.
template <int DT, int NRB>
__global__ void __launch_bounds__(256)
proj_shrink_pair_kernel(ProjShrink g, ProjShrink h, int share) {
    __shared__ __attribute__((aligned(16))) char smem[pj_shrink_block_lds<DT, NRB, PJ_S_FR>()];
    const long long r0 = (long long)(blockIdx.x / share) * 16;
    if (blockIdx.y == 0) pj_shrink_block<DT, NRB, true, PJ_S_FR>(g, r0, blockIdx.x % share, share, smem);
    else pj_shrink_block<DT, NRB, true, PJ_S_FK>(h, r0, blockIdx.x % share, share, smem);
}

// Many rows of long requests: 64 rows by all ranks through LDS, a ring of four stages of 128 bytes of k as in PJProduct, each
// wave 16 rows.  For every adapter of the 64 rows (up to four) the whole product; 64 rows of more adapters are left to the
// workgroups behind the first `tiles`, which take 16 rows each as above and have nothing to do otherwise.
// (32 768 x 1024 rows, rank 64: 29 us, and 52 by 16 rows, which read the factor four times as often.)
template <int DT, int NRB, int F>
__global__ void __launch_bounds__(256)
proj_shrink_tile_kernel(ProjShrink p, int tiles) {
    extern __shared__ __attribute__((aligned(16))) char pj_lds[];
    typedef typename PJ<DT>::T T;
    constexpr bool FB = F == PJ_S_FR;
    constexpr int RN = NRB <= 4 ? 64 : 128, KT = 128 / PJ<DT>::E, S = 4, STAGE = pj_tile_bytes(64) + pj_tile_bytes(RN), L = 2 + RN / 32;
    const int lane = threadIdx.x & 63, li = lane & 15, wave = threadIdx.x >> 6;
    const bool own = (int)blockIdx.x < tiles;
    const long long block = (long long)blockIdx.x - tiles;                   // of 16 rows
    const long long r0 = own ? (long long)blockIdx.x * 64 : block / 4 * 64;
    int am[4];
    pj_row_adapters<4>(p, r0, am);
    int ads[4], count = 0;                                                  // the adapters in the order of their first rows
    unsigned left[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { left[i] = (unsigned)__ballot(am[i] >= 0) & 0xffffu; ads[i] = -1; }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        int ad = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) if (ad < 0 && left[i]) ad = __builtin_amdgcn_readlane(am[i], __builtin_ctz(left[i]));
        if (ad < 0) continue;
        ads[c] = ad;
        ++count;
#pragma unroll
        for (int i = 0; i < 4; ++i) left[i] &= ~(unsigned)__ballot(am[i] == ad);
    }
    const bool many = (left[0] | left[1] | left[2] | left[3]) != 0;
    if (own == many) return;                                                // (for the other kind of workgroup)
    if (many) {
        static_assert(pj_shrink_block_lds<DT, NRB, F>() <= S * STAGE, "the ring's memory");
        pj_shrink_block<DT, NRB, true, F>(p, block * 16, 0, 1, pj_lds);
        return;
    }
    const int mine = wave == 0 ? am[0] : wave == 1 ? am[1] : wave == 2 ? am[2] : am[3];
    const long long m = r0 + wave * 16 + li;
    if (p.row_adapter && lane < 16 && m < p.n) p.row_adapter[m] = mine;
    for (int c = 0; c < count; ++c) {
        const int ad = c == 0 ? ads[0] : c == 1 ? ads[1] : c == 2 ? ads[2] : ads[3];
        const T* f = (const T*)p.f + (long long)ad * p.f_adapter;
        PJOperand<DT, false, 64> ox;
        PJOperand<DT, FB, RN> of;
        ox.init((const T*)p.x, p.ldx, r0, p.n, p.K);
        of.init(f, FB ? p.f_k : p.f_rank, 0, p.rank, p.K);
        long long k = p.K;
        auto next = [&](int stage) {
            const int l = k < KT ? (k > 0 ? (int)k : 0) : KT;
            ox.stage(pj_lds + stage * STAGE, l);
            of.stage(pj_lds + stage * STAGE + pj_tile_bytes(64), l);
            k -= KT;
        };
        __syncthreads();                                                    // the last adapter's stages have been read
#pragma unroll
        for (int i = 0; i < S - 1; ++i) next(i);
        pj_f32x4 acc[NRB] = {};
        const int steps = (p.K + KT - 1) / KT;
        int cur = 0;
        for (int t = 0; t < steps; ++t) {
            pj_wait_and_meet<(S - 2) * L>();
            next(cur == 0 ? S - 1 : cur - 1);
            const char* lx = pj_lds + cur * STAGE;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                pj_u32x4 fx[1], ff[NRB];
                pj_fragments<DT, false, 64, 1>(lx, wave * 16, kk, fx);
                pj_fragments<DT, FB, RN, NRB>(lx + pj_tile_bytes(64), 0, kk, ff);
#pragma unroll
                for (int i = 0; i < NRB; ++i) acc[i] = pj_mfma<DT>(ff[i], fx[0], acc[i]);
            }
            cur = cur + 1 == S ? 0 : cur + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        pj_shrink_store<DT, NRB>(p, m, mine == ad, ad, acc);
    }
}

// ------------------------------------------------------------------------------------------- a few adapted rows, in one launch
// y = x W^T + s (x A^T) B^T for 16 rows by 16 columns per workgroup, where there are so few rows that a second launch costs more
// than what is done again here: every column tile makes its rows' h = s x A^T by itself (one product for each adapter that the 16
// rows meet), the four waves over a quarter of the contracted axis each.  h stays in fp32, in LDS.
// The rows and the matrix are loaded before the adapters are known; K is at most what that holds.
template <int DT, int ODT, int NRB>
__global__ void __launch_bounds__(256)
proj_adapt_few_kernel(ProjRows p, ProjShrink s, int col_tiles) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, KS = 4 * V, XS = 8;
    __shared__ pj_f32x4 part[4][NRB][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4, wave = threadIdx.x >> 6;
    const int c0 = (int)(blockIdx.x % col_tiles) * 16;
    const long long r0 = (long long)(blockIdx.x / col_tiles) * 16, m = r0 + li;
    const T* x = (const T*)p.x + (m < p.n ? m : p.n - 1) * p.ldx;
    const T* w = (const T*)p.w + (long long)(c0 + li < p.N ? c0 + li : p.N - 1) * p.ldw;
    pj_u32x4 xa[XS], wa[XS];
    pj_shrink_load_x<DT, XS, true>(s, x, wave * KS, 4 * KS, xa);
    pj_shrink_load_x<DT, XS, true>(s, w, wave * KS, 4 * KS, wa);
    const long long first = pj_clamp(p.offsets[0], p.n), end = pj_clamp(p.offsets[p.segments], p.n);
    int am[1];
    pj_row_adapters<1>(s, r0, am);
    // what this wave adds of the low-rank term: ranks wave * V.. of its row's factor, for its lanes' four columns
    const int q = wave * V;
    const bool some = am[0] >= 0 && q < p.rank;
    const T* f = (const T*)p.f + (long long)(some ? am[0] : 0) * p.f_adapter;
    union { T t[V]; pj_u32x4 v; } fv[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int col = c0 + lh * 4 + n;
        fv[n].v = pj_load_if<pj_u32x4>(some, f + (unsigned)(col < p.N ? col : p.N - 1) * (unsigned)p.f_col + (unsigned)q);
    }
    const float sc = some ? (s.scale ? s.scale[am[0]] : 1.f) : 0.f;
    // the adapters of the 16 rows one after the other, the factor of the next one on its way while one is multiplied
    pj_f32x4 h[NRB] = {};
    auto load = [&](int ad, pj_u32x4 (&fa)[XS][NRB]) __attribute__((always_inline)) {
        const T* a = (const T*)s.f + (long long)ad * s.f_adapter;
#pragma unroll
        for (int u = 0; u < XS; ++u) {
            const int k = wave * KS + u * 4 * KS + lh * V;
#pragma unroll
            for (int i = 0; i < NRB; ++i)
                fa[u][i] = pj_load_if<pj_u32x4>(k < s.K && i * 16 + li < s.rank, a + (unsigned)(i * 16 + li) * (unsigned)s.f_rank + (unsigned)k);
        }
    };
    pj_u32x4 fa[XS][NRB], fb[XS][NRB];
    unsigned left = (unsigned)__ballot(am[0] >= 0) & 0xffffu;
    int ad = left ? __builtin_amdgcn_readlane(am[0], __builtin_ctz(left)) : -1;
    if (ad >= 0) load(ad, fa);
    while (ad >= 0) {
        left &= ~(unsigned)__ballot(am[0] == ad);
        const int next = left ? __builtin_amdgcn_readlane(am[0], __builtin_ctz(left)) : -1;
        if (next >= 0) load(next, fb);
        pj_f32x4 t[NRB] = {};
#pragma unroll
        for (int u = 0; u < XS; ++u)
#pragma unroll
            for (int i = 0; i < NRB; ++i) t[i] = pj_mfma<DT>(fa[u][i], xa[u], t[i]);
#pragma unroll
        for (int i = 0; i < NRB; ++i) if (am[0] == ad) h[i] = t[i];
#pragma unroll
        for (int u = 0; u < XS; ++u)
#pragma unroll
            for (int i = 0; i < NRB; ++i) fa[u][i] = fb[u][i];
        ad = next;
    }
    pj_f32x4 acc = {};
#pragma unroll
    for (int u = 0; u < XS; ++u) acc = pj_mfma<DT>(wa[u], xa[u], acc);
#pragma unroll
    for (int i = 0; i < NRB; ++i) part[wave][i][lane] = h[i];
    __syncthreads();
    if (some) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            // ranks q + k.. of the lane's row: block (q + k) / 16, lane group (q + k) / 4 % 4
            pj_f32x4 hv = {};
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                const pj_f32x4 t = part[o][(q + k) >> 4][((q + k) >> 2 & 3) * 16 + li];
#pragma unroll
                for (int j = 0; j < 4; ++j) hv[j] += t[j];
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[n] = __builtin_fmaf(sc * hv[j], pj_to_f32<DT>(fv[n].t[k + j]), acc[n]);
        }
    }
    __syncthreads();
    if (wave) part[wave - 1][0][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += part[o][0][lane][j];
    const int c = c0 + lh * 4;
    if (m >= first && m < end && c < p.N) pj_store4<ODT>(p.y, m * p.ldy + c, acc, p.N - c);
}

// ------------------------------------------------------------------------------------------- gradient of the factors
// One adapter's [rank] x 64 columns: eight waves, of one workgroup or of several, take its rows 16 at a time in turn, over every
// request that names the adapter, and add up in wave order.  Several workgroups leave their sums in `partial`, and
// proj_factor_sum_kernel adds them up in their order.  Products on the fp32 matrix unit: h is fp32, x is widened.
// Lane l loads columns 4 (l % 16) + 0..3 of a row, so that product j of a step holds columns j, 4 + j, 8 + j, ...
// The rows of the next turns are loaded while the current ones are multiplied.
constexpr int PJ_FACTOR_WAVES = 8;

template <int DT, int NRB, bool XV> struct PJFactorRows {
    typedef typename PJ<DT>::T T;
    union { T t[4]; unsigned u[PJ<DT>::E]; } x[4];
    union { float f; unsigned u; } h[4][NRB];
    // Rows behind the request's last are read as that one and masked, so that no load waits for a branch; columns and ranks outside
    // are read as the first ones, and what comes of them is not stored.
    __device__ __forceinline__ void load(const ProjFactor& p, long long r, long long e, int c0) {
        const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long long i = r + u * 4 + lh, k = i < e ? i : e - 1;
            const T* px = (const T*)p.x + k * p.ldx;
            if constexpr (XV) __builtin_memcpy(x[u].t, __builtin_assume_aligned(px + (c0 < p.N ? c0 : 0), 4 * sizeof(T)), 4 * sizeof(T));
            else
#pragma unroll
                for (int j = 0; j < 4; ++j) x[u].t[j] = px[c0 + j < p.N ? c0 + j : 0];
#pragma unroll
            for (int q = 0; q < NRB; ++q) h[u][q].f = p.h[k * p.rp + (q * 16 < p.rp ? q * 16 : 0) + li];
        }
    }
    __device__ __forceinline__ void mask(long long r, long long e) {
        const int lh = (threadIdx.x & 63) >> 4;
        if (r + 16 <= e) return;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            unsigned ok = r + u * 4 + lh < e ? ~0u : 0u;
            asm volatile("" : "+v"(ok));                     // not a branch around the loads
#pragma unroll
            for (int j = 0; j < PJ<DT>::E; ++j) x[u].u[j] &= ok;
#pragma unroll
            for (int q = 0; q < NRB; ++q) h[u][q].u &= ok;
        }
    }
    __device__ __forceinline__ void multiply(pj_f32x4 (&acc)[NRB][4]) const {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < NRB; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[q][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(pj_to_f32<DT>(x[u].t[j]), h[u][q].f, acc[q][j], 0, 0, 0);
    }
};

// Where workgroup `split` of an adapter leaves its sum of 64 columns: NRB blocks of 16 ranks, 4 products, 64 lanes of 4 values.
template <int NRB> __device__ __forceinline__ pj_f32x4* pj_factor_partial(const ProjFactor& p, int split, int adapter, int block) {
    return (pj_f32x4*)p.partial + (((long long)split * p.adapters + adapter) * ((p.N + 63) / 64) + block) * (NRB * 4 * 64);
}

// One block of 16 ranks by columns lh * 16 + 4 u + j of the block at n0, product j, into the gradient.
template <int ODT> __device__ __forceinline__ void pj_factor_store(const ProjFactor& p, int adapter, int k, int n0, int j, const pj_f32x4& v) {
    const int lh = (threadIdx.x & 63) >> 4;
    if (k >= p.rank) return;
    typename PJ<ODT>::T* out = (typename PJ<ODT>::T*)p.out + (long long)adapter * p.rank * p.N;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int c = n0 + lh * 16 + u * 4 + j;
        if (c < p.N) out[p.by_col ? (long long)c * p.rank + k : (long long)k * p.N + c] = pj_from_f32<ODT>(v[u]);
    }
}

// blockIdx.z: the gradient of A, of B, for each of the splits.
template <int DT, int ODT, int NRB, bool XV>
__global__ void __launch_bounds__(PJ_FACTOR_WAVES * 64)
proj_factor_kernel(ProjFactor pa, ProjFactor pb) {
    const ProjFactor& p = blockIdx.z % 2 == 0 ? pa : pb;
    if ((int)blockIdx.x * 64 >= p.N) return;
    constexpr int W = PJ_FACTOR_WAVES, D = NRB <= 2 ? 4 : 2;           // blocks of rows in registers
    __shared__ pj_f32x4 part[W - 1][4][64];
    const int lane = threadIdx.x & 63, li = lane & 15, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.z / 2, all = W * p.splits, mine = split * W + wave;
    const int n0 = blockIdx.x * 64, ad = p.first + blockIdx.y, c0 = n0 + li * 4;
    pj_f32x4 acc[NRB][4] = {};
    // this wave's blocks of 16 rows, one after the other: rows [r, min(r + 16, e))
    int s0 = -64, turn = 0;                // requests looked at; blocks of the adapter met so far, modulo all
    unsigned long long mask = 0;           // requests of the 64 at s0 that are left
    long long r = 0, e = 0;
    auto next = [&]() {
        r += all * 16;
        while (r >= e) {
            while (!mask) {
                s0 += 64;
                if (s0 >= p.segments) return false;
                mask = __ballot(s0 + lane < p.segments && p.ids[s0 + lane] == ad);
            }
            const int s = s0 + __builtin_ctzll(mask);
            mask &= mask - 1;
            const long long b = pj_clamp(p.offsets[s], p.n);
            e = pj_clamp(p.offsets[s + 1], p.n);
            if (e <= b) { r = e; continue; }
            r = b + (long long)((mine - turn + all) % all) * 16;
            turn = (int)((turn + (e - b + 15) / 16) % all);
        }
        return true;
    };
    PJFactorRows<DT, NRB, XV> rows[D];
    long long at[D], end[D];               // the slots' rows; at == end: empty
#pragma unroll
    for (int u = 0; u < D; ++u) at[u] = end[u] = 0;
    bool more = true;
    auto fill = [&](int u) {
        more = more && next();
        at[u] = end[u] = 0;
        if (!more) return;
        at[u] = r; end[u] = e;
        rows[u].load(p, r, e, c0);
    };
#pragma unroll
    for (int u = 0; u < D - 1; ++u) fill(u);
    for (bool any = true; any;) {
#pragma unroll
        for (int u = 0; u < D; ++u) {
            fill((u + D - 1) % D);
            any = at[u] < end[u];
            if (!any) break;
            rows[u].mask(at[u], end[u]);
            rows[u].multiply(acc);
        }
    }
#pragma unroll
    for (int q = 0; q < NRB; ++q) {
        __syncthreads();
        if (wave)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[wave - 1][j][lane] = acc[q][j];
        __syncthreads();
        if (wave) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            pj_f32x4 v = acc[q][j];
#pragma unroll
            for (int w = 0; w < W - 1; ++w) v += part[w][j][lane];
            if (p.splits > 1) pj_factor_partial<NRB>(p, split, ad, blockIdx.x)[(q * 4 + j) * 64 + lane] = v;
            else pj_factor_store<ODT>(p, ad, q * 16 + li, n0, j, v);
        }
    }
}

// The sum of an adapter's partial sums; blockIdx.z as above, one block of 16 ranks for each further z.
template <int ODT, int NRB>
__global__ void __launch_bounds__(256)
proj_factor_sum_kernel(ProjFactor pa, ProjFactor pb) {
    const ProjFactor& p = blockIdx.z % 2 == 0 ? pa : pb;
    if ((int)blockIdx.x * 64 >= p.N) return;
    const int lane = threadIdx.x & 63, j = threadIdx.x >> 6, q = blockIdx.z / 2, ad = blockIdx.y;
    pj_f32x4 v = {};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) v += pj_factor_partial<NRB>(p, s, ad, blockIdx.x)[(q * 4 + j) * 64 + lane];
    pj_factor_store<ODT>(p, ad, q * 16 + (lane & 15), blockIdx.x * 64, j, v);
}

// dw of the segments that were split, and zeros for those without rows: the chunks' partial sums in their order.
template <int ODT>
__global__ void __launch_bounds__(256)
proj_weights_sum_kernel(ProjWeights p) {
    typedef typename PJ<ODT>::T O;
    const int seg = blockIdx.y, lane = threadIdx.x & 63;
    const long long size = (long long)p.M * p.N;
    long long first = 0;                     // number of the segment's first chunk
    for (int s0 = 0; s0 < seg; s0 += 64) {
        long long c = 0;
        if (s0 + lane < seg) {
            const long long b = pj_clamp(p.offsets[s0 + lane], p.n), e = pj_clamp(p.offsets[s0 + lane + 1], p.n);
            c = e > b ? (e - b + p.chunk - 1) / p.chunk : 0;
        }
        for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o);
        first += c;
    }
    const long long b = pj_clamp(p.offsets[seg], p.n), e = pj_clamp(p.offsets[seg + 1], p.n);
    long long chunks = e > b ? (e - b + p.chunk - 1) / p.chunk : 0;
    if (chunks == 1) return;
    const long long room = p.n / p.chunk + p.segments - first;       // offsets that decrease could name more chunks than there are
    if (chunks > room) chunks = room < 0 ? 0 : room;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (long long)gridDim.x * 1024) {
        const float* in = p.partial + first * size + i;
        pj_f32x4 v = {};
        if (size % 4 == 0) {
#pragma unroll 4
            for (long long c = 0; c < chunks; ++c) {
                const pj_f32x4 t = *(const pj_f32x4*)(in + c * size);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += t[j];
            }
        } else {
            for (long long c = 0; c < chunks; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) if (i + j < size) v[j] += in[c * size + j];
        }
        O* out = (O*)p.dw + seg * size + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (i + j < size) out[j] = pj_from_f32<ODT>(v[j]);
    }
}

__global__ void __launch_bounds__(256)
proj_zero_kernel(float* q, long long count) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) q[i] = 0.f;
}

// ------------------------------------------------------------------------------------------- launches
// input type x output type (the input's, or fp32)
#define PJ_TYPES(dt, odt, CALL)                                                                              \
    do {                                                                                                     \
        if ((dt) == VDB_F32) { constexpr int DT = VDB_F32, ODT = VDB_F32; CALL; }                            \
        else if ((dt) == VDB_BF16 && (odt) == VDB_F32) { constexpr int DT = VDB_BF16, ODT = VDB_F32; CALL; } \
        else if ((dt) == VDB_BF16) { constexpr int DT = VDB_BF16, ODT = VDB_BF16; CALL; }                    \
        else if ((odt) == VDB_F32) { constexpr int DT = VDB_F16, ODT = VDB_F32; CALL; }                      \
        else { constexpr int DT = VDB_F16, ODT = VDB_F16; CALL; }                                            \
    } while (0)

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

hipError_t launch_proj_weights_sum(const ProjWeights& p, hipStream_t st) {
    const long long size = (long long)p.M * p.N;
    long long blocks = (size + 1023) / 1024;
    if (blocks > 1024) blocks = 1024;
    const dim3 grid((unsigned)blocks, (unsigned)p.segments);
    if (p.out_dtype == VDB_F32) return pj_launch(proj_weights_sum_kernel<VDB_F32>, grid, 0, p, st);
    if (p.out_dtype == VDB_BF16) return pj_launch(proj_weights_sum_kernel<VDB_BF16>, grid, 0, p, st);
    return pj_launch(proj_weights_sum_kernel<VDB_F16>, grid, 0, p, st);
}

// By 64 rows: from rank 33 and 16 384 rows on, for long requests (rank 64, 1024 wide, 48 requests: 32 768 rows 52 -> 29 us, 8192 rows
// 22 -> 33; rank 16, 768 wide: 16 384 rows 12 -> 17).
template <int DT, int NRB> static bool shrink_tiles(const ProjShrink& p) {
    return NRB >= 4 && p.n >= 16384 && p.n / p.segments >= 128 && proj_shrink_tile_grid(p.n) <= PROJ_MAX_WORKGROUPS;
}

template <int DT, int NRB>
static hipError_t shrink_typed(const ProjShrink& p, hipStream_t st) {
    constexpr int E = PJ<DT>::E, V = 16 / E;
    const bool xv = pj_aligned(p.x, p.ldx, E, 16) && p.K % V == 0;
    const bool fk = p.f_k == 1 && pj_aligned(p.f, p.f_rank, E, 16) && p.K % V == 0;
    const bool ftile = p.f_rank == 1 && p.f_k == p.rank && p.rank % V == 0 && (uintptr_t)p.f % 16 == 0;
    const bool fr = DT == VDB_F32 ? p.f_rank == 1 : p.f_rank == 1 && p.f_k == p.rank && p.rank % 8 == 0 && (uintptr_t)p.f % 16 == 0;
    if constexpr (NRB >= 4) if (shrink_tiles<DT, NRB>(p) && xv && (fk || ftile)) {
        const int tiles = (int)((p.n + 63) / 64);
        const dim3 grid((unsigned)proj_shrink_tile_grid(p.n));
        const size_t lds = 4 * (pj_tile_bytes(64) + pj_tile_bytes(NRB <= 4 ? 64 : 128));
        auto go = [&](auto kernel) {
            if (lds > 65536) {
                const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
                if (e != hipSuccess) return e;
            }
            hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, p, tiles);
            return hipGetLastError();
        };
        if (fk) return go(proj_shrink_tile_kernel<DT, NRB, PJ_S_FK>);
        return go(proj_shrink_tile_kernel<DT, NRB, PJ_S_FR>);
    }
    const long long share = proj_shrink_share(p.n, p.segments);
    const dim3 grid((unsigned)proj_shrink_grid(p.n, p.segments));
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p, (int)share);
        return hipGetLastError();
    };
    if (!xv || !(fk || fr)) return go(proj_shrink_kernel<DT, NRB, false, PJ_S_ANY>);
    if (!fk) return go(proj_shrink_kernel<DT, NRB, true, PJ_S_FR>);
    return go(proj_shrink_kernel<DT, NRB, true, PJ_S_FK>);
}

template <int DT, int ODT, int NRB>
static hipError_t factor_typed(ProjFactor p, ProjFactor b, hipStream_t st) {
    const int most = p.N > b.N ? p.N : b.N, step = proj_factor_adapters(p.adapters, p.splits, most);
    const dim3 threads(PJ_FACTOR_WAVES * 64);
    const bool xv = pj_aligned(p.x, p.ldx, PJ<DT>::E, 4 * PJ<DT>::E) && p.N % 4 == 0 &&
                    pj_aligned(b.x, b.ldx, PJ<DT>::E, 4 * PJ<DT>::E) && b.N % 4 == 0;
    for (int first = 0; first < p.adapters; first += step) {
        p.first = b.first = first;
        const int left = p.adapters - first;
        const dim3 grid((unsigned)((most + 63) / 64), (unsigned)(left < step ? left : step), 2 * p.splits);
        if (xv) hipLaunchKernelGGL((proj_factor_kernel<DT, ODT, NRB, true>), grid, threads, 0, st, p, b);
        else hipLaunchKernelGGL((proj_factor_kernel<DT, ODT, NRB, false>), grid, threads, 0, st, p, b);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.splits > 1) {                                      // (of a few adapters)
        const dim3 grid((unsigned)((most + 63) / 64), (unsigned)p.adapters, 2 * ((p.rank + 15) / 16));
        hipLaunchKernelGGL((proj_factor_sum_kernel<ODT, NRB>), grid, dim3(256), 0, st, p, b);
    }
    return hipGetLastError();
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

template <int DT, int ODT>
static hipError_t adapt_few_typed(const ProjRows& p, const ProjShrink& s, hipStream_t st) {
    const int col_tiles = (p.N + 15) / 16;
    const dim3 grid((unsigned)((p.n + 15) / 16 * col_tiles));
    constexpr int V = 16 / PJ<DT>::E;
    if (p.rank <= 16 && p.rank <= 4 * V) hipLaunchKernelGGL((proj_adapt_few_kernel<DT, ODT, 1>), grid, dim3(256), 0, st, p, s, col_tiles);
    else hipLaunchKernelGGL((proj_adapt_few_kernel<DT, ODT, 2>), grid, dim3(256), 0, st, p, s, col_tiles);
    return hipGetLastError();
}

hipError_t launch_proj_adapted(const ProjRows& p, const ProjShrink& s, hipStream_t st) {
    if (p.n <= 0 || p.segments <= 0) return hipSuccess;
    const int e = p.dtype == VDB_F32 ? 4 : 2, v = 16 / e;
    // One launch: up to 256 rows with no more than two requests to 16 of them, as the adapters of 16 rows are multiplied one after the
    // other (768 x 768 bf16, rank 16, one launch against two: 1 row 5.1 and 8.5 us, 256 rows of one request 9.9 and 12.5, 512 rows
    // 17.2 and 13.1; 64 rows of 8 requests 8.9 and 10.0, 64 rows of 64 requests 16.8 and 11.2).
    const bool few = p.n <= 256 && p.segments <= 2 * ((p.n + 15) / 16) && p.K <= 512 / e * 4 && p.rank <= 4 * v && p.rank % v == 0 && p.K % v == 0 &&
                     pj_aligned(p.x, p.ldx, e, 16) && pj_aligned(p.w, p.ldw, e, 16) && (uintptr_t)s.f % 16 == 0 && (uintptr_t)p.f % 16 == 0;
    if (few) PJ_TYPES(p.dtype, p.out_dtype, return (adapt_few_typed<DT, ODT>(p, s, st)));
    const hipError_t err = launch_proj_shrink(s, st);
    return err == hipSuccess ? launch_proj_rows(p, st) : err;
}

template <int DT, int NRB>
static hipError_t shrink_pair_typed(const ProjShrink& g, const ProjShrink& h, hipStream_t st) {
    constexpr int E = PJ<DT>::E, V = 16 / E;
    const bool vec = pj_aligned(g.x, g.ldx, E, 16) && g.K % V == 0 && pj_aligned(h.x, h.ldx, E, 16) && pj_aligned(h.f, h.f_rank, E, 16) &&
                     h.K % V == 0 && (DT == VDB_F32 || (g.rank % 8 == 0 && (uintptr_t)g.f % 16 == 0));
    if (!vec || shrink_tiles<DT, NRB>(g) || 2 * proj_shrink_grid(g.n, g.segments) > PROJ_MAX_WORKGROUPS) {
        const hipError_t e = shrink_typed<DT, NRB>(g, st);
        return e == hipSuccess ? shrink_typed<DT, NRB>(h, st) : e;
    }
    const long long share = proj_shrink_share(g.n, g.segments);
    const dim3 grid((unsigned)proj_shrink_grid(g.n, g.segments), 2);
    hipLaunchKernelGGL((proj_shrink_pair_kernel<DT, NRB>), grid, dim3(256), 0, st, g, h, (int)share);
    return hipGetLastError();
}

hipError_t launch_proj_shrink_pair(const ProjShrink& g, const ProjShrink& h, hipStream_t st) {
    if (g.n <= 0 || g.segments <= 0) return hipSuccess;
    if (g.dtype == VDB_F32) { const ProjShrink& p = g; PJ_BY_RANK(return (shrink_pair_typed<VDB_F32, NRB>(g, h, st))); }
    const int nrb = proj_rank_pad(g.rank, g.dtype) / 16;
#define PJ_PAIR(DT) (nrb <= 2 ? shrink_pair_typed<DT, 2>(g, h, st) : nrb <= 4 ? shrink_pair_typed<DT, 4>(g, h, st) : shrink_pair_typed<DT, 8>(g, h, st))
    return g.dtype == VDB_BF16 ? PJ_PAIR(VDB_BF16) : PJ_PAIR(VDB_F16);
#undef PJ_PAIR
}

hipError_t launch_proj_factors(const ProjFactor& p, const ProjFactor& b, hipStream_t st) {
    PJ_TYPES(p.dtype, p.out_dtype, PJ_BY_RANK(return (factor_typed<DT, ODT, NRB>(p, b, st))));
}

hipError_t launch_proj_zero(float* q, long long count, hipStream_t st) {
    const long long blocks = (count + 255) / 256;
    hipLaunchKernelGGL(proj_zero_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, st, q, count);
    return hipGetLastError();
}

}  // namespace vdb
