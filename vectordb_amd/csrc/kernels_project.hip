// Learned projections in front of a table: products grouped by source, low-rank adapters of many requests beside a
// shared matrix, and their gradients (see include/vdb.h for the operators and project.h for the parameters).
#include "vdb_internal.h"
#include "project.h"

namespace vdb {

typedef float pj_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pj_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pj_f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int pj_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short pj_u16x8 __attribute__((ext_vector_type(8)));
typedef short pj_s16x4 __attribute__((ext_vector_type(4)));

#define PJ_GLOBAL __attribute__((address_space(1)))
#define PJ_LOCAL __attribute__((address_space(3)))

// Sixteen zero bytes: the source of every 16-byte piece of a tile that lies outside its operand.
static __device__ __align__(16) const unsigned int pj_zero16[4] = {0, 0, 0, 0};

template <int DT> struct PJ {            // 16-bit types
    static constexpr int E = 2;
    typedef unsigned short T;
};
template <> struct PJ<VDB_F32> {
    static constexpr int E = 4;
    typedef float T;
};

__device__ __forceinline__ float pj_load(const float* p) { return *p; }
template <int DT> __device__ __forceinline__ float pj_to_f32(typename PJ<DT>::T v) {
    if constexpr (DT == VDB_F32) return v;
    else if constexpr (DT == VDB_BF16) return __uint_as_float((unsigned)v << 16);
    else return (float)__builtin_bit_cast(_Float16, v);
}
// rounded once, to nearest even
template <int DT> __device__ __forceinline__ typename PJ<DT>::T pj_from_f32(float v) {
    if constexpr (DT == VDB_F32) return v;
    else if constexpr (DT == VDB_BF16) return __builtin_bit_cast(unsigned short, (__bf16)v);
    else return __builtin_bit_cast(unsigned short, (_Float16)v);
}

// ------------------------------------------------------------------------------------------- segments
__device__ __forceinline__ long long pj_clamp(long long v, long long n) { return v < 0 ? 0 : v > n ? n : v; }

// Which tile of TM rows workgroup `bid` of a grouped product works on: tiles are numbered segment by segment
// (ceil(size / TM) each), column tiles run fastest, and the numbers are dealt to the eight XCDs in contiguous runs
// (workgroup b runs on XCD b % 8), so that the column tiles that share rows share an L2.
// Every wave does this by itself, 64 segments at a time.  Returns false for workgroups past the last tile.
__device__ __forceinline__ bool pj_find_tile(const long long* offsets, int segments, long long n, int tm, int col_tiles,
                                             unsigned bid, int& seg, long long& row0, long long& row1, int& col) {
    const int lane = threadIdx.x & 63;
    long long total = 0;
    for (int s0 = 0; s0 < segments; s0 += 64) {
        const int s = s0 + lane;
        long long t = 0;
        if (s < segments) {
            const long long b = pj_clamp(offsets[s], n), e = pj_clamp(offsets[s + 1], n);
            t = e > b ? (e - b + tm - 1) / tm : 0;
        }
        for (int o = 32; o >= 1; o >>= 1) t += __shfl_xor(t, o);
        total += t;
    }
    const long long all = total * col_tiles, run = (all + 7) / 8;
    const long long idx = (long long)(bid >> 3);
    if (idx >= run) return false;
    const long long id = (long long)(bid & 7) * run + idx;
    if (id >= all) return false;
    col = (int)(id % col_tiles);
    const long long want = id / col_tiles;
    long long before = 0;
    for (int s0 = 0; s0 < segments; s0 += 64) {
        const int s = s0 + lane;
        long long b = 0, e = 0, t = 0;
        if (s < segments) {
            b = pj_clamp(offsets[s], n); e = pj_clamp(offsets[s + 1], n);
            t = e > b ? (e - b + tm - 1) / tm : 0;
        }
        long long inc = t;
        for (int o = 1; o < 64; o <<= 1) { const long long u = __shfl_up(inc, o); if (lane >= o) inc += u; }
        const bool mine = before + inc - t <= want && want < before + inc;
        const unsigned long long m = __ballot(mine);
        if (m) {
            const int src = __builtin_ctzll(m);
            seg = s0 + src;
            row0 = __shfl(b + (want - (before + inc - t)) * tm, src);
            row1 = __shfl(e, src);
            return true;
        }
        before += __shfl(inc, 63);
    }
    return false;
}

// First segment whose end lies behind `row` (offsets do not decrease); `segments` if there is none.
__device__ __forceinline__ int pj_first_segment(const long long* offsets, int segments, long long row) {
    int lo = 0, hi = segments;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    return lo;
}

// ------------------------------------------------------------------------------------------- tiles in LDS
// One operand tile: 128 rows (or columns) of the product by 128 bytes of the contracted axis, 16 KiB, kept as it lies in
// memory in 16-byte pieces whose place is swizzled so that the fragment reads below touch every bank once:
//   contiguous along k (BYK = false): row r is 128 bytes, piece c sits in slot c ^ ((r >> 1) & 7)
//   contiguous along the rows (BYK = true): one line per k; 16-bit: 256 bytes, piece c in slot c ^ 2 f(k) with
//     f(k) = (k & 3) | (k >> 3 & 1) << 2; fp32: 512 bytes, piece c in slot c ^ 4 (k >> 2 & 3)
constexpr int PJ_TILE = 128, PJ_TILE_BYTES = 16384, PJ_THREADS = 256;

template <int DT, bool BYK> struct PJOperand {
    typedef typename PJ<DT>::T T;
    static constexpr int E = PJ<DT>::E, V = 16 / E, KT = 128 / E;
    const T* src[4];
    long long step[4];
    int kpos[4];                 // k of the piece within a tile
    bool in[4];                  // the piece's rows lie in the operand (VEC); per element otherwise
    int rem[4];                  // BYK: elements of the piece that lie in the operand; else unused
    const T* zero;

    // rows r0 .. r0 + 127 of [0, rows), k from 0
    __device__ __forceinline__ void init(const T* base, long long ld, long long r0, long long rows) {
        zero = (const T*)pj_zero16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = i * PJ_THREADS + (int)threadIdx.x;
            if constexpr (!BYK) {
                const int r = p >> 3, c = (p & 7) ^ ((r >> 1) & 7);
                kpos[i] = c * V;
                in[i] = r0 + r < rows;
                rem[i] = V;
                src[i] = in[i] ? base + (r0 + r) * ld + c * V : zero;
                step[i] = in[i] ? KT : 0;
            } else {
                constexpr int PL = PJ_TILE * E / 16;             // pieces per line
                const int k = p / PL, slot = p % PL;
                const int c = E == 2 ? slot ^ (((k & 3) | ((k >> 3 & 1) << 2)) << 1) : slot ^ ((k >> 2 & 3) << 2);
                kpos[i] = k;
                const long long left = rows - (r0 + c * V);
                rem[i] = left >= V ? V : left > 0 ? (int)left : 0;
                in[i] = rem[i] > 0;
                src[i] = in[i] ? base + (long long)k * ld + r0 + c * V : zero;
                step[i] = in[i] ? KT * ld : 0;
            }
        }
    }
    // pieces of the next KT elements of the contracted axis, of which `kleft` lie in the operand
    template <bool VEC> __device__ __forceinline__ void stage(char* lds, int kleft) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            char* const wave_dst = lds + (i * PJ_THREADS + ((int)threadIdx.x & ~63)) * 16;
            if constexpr (VEC) {
                const T* s = in[i] && kpos[i] < kleft ? src[i] : zero;
                __builtin_amdgcn_global_load_lds((const PJ_GLOBAL void*)s, (PJ_LOCAL void*)wave_dst, 16, 0, 0);
            } else {
                T v[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const bool ok = BYK ? (j < rem[i] && kpos[i] < kleft) : (in[i] && kpos[i] + j < kleft);
                    v[j] = ok ? src[i][j] : (T)0;
                }
                T* d = (T*)(wave_dst + ((int)threadIdx.x & 63) * 16);
#pragma unroll
                for (int j = 0; j < V; ++j) d[j] = v[j];
            }
            src[i] += step[i];
        }
    }
};

// Fragment of 16 rows from `row` (a multiple of 16): lane l holds row + l % 16 and, of the step's 64 bytes of k, the 16 bytes
// number l / 16 (16-bit: k = 8 (l / 16) + 0..7; fp32: k = 4 (l / 16) + 0..3, one element for each of four products).
template <int DT, bool BYK> __device__ __forceinline__ pj_u32x4 pj_fragment(const char* lds, int row, int kk) {
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    if constexpr (!BYK) {
        const int r = row + li;
        return *(const pj_u32x4*)(lds + r * 128 + (((kk * 4 + lh) ^ ((r >> 1) & 7)) << 4));
    } else if constexpr (DT == VDB_F32) {
        pj_u32x4 v;
        const int c = (row + li) >> 2;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = *(const unsigned*)(lds + (kk * 16 + lh * 4 + j) * 512 + ((c ^ (lh << 2)) << 4) + (li & 3) * 4);
        return v;
    } else {
        // ds_read_b64_tr_b16: sixteen lanes read a block of 4 k x 16 rows, lane i its piece of line i / 4 and gets column i
        const int c = (row >> 3) + ((li & 3) >> 1);
        const int f = (li >> 2) | ((lh & 1) << 2);
        const char* a = lds + (kk * 32 + lh * 8 + (li >> 2)) * 256 + ((c ^ (f << 1)) << 4) + (li & 1) * 8;
        union { pj_s16x4 h[2]; pj_u32x4 v; } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PJ_LOCAL pj_s16x4*)a);
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((PJ_LOCAL pj_s16x4*)(a + 4 * 256));
        return u.v;
    }
}

// D[n][m] += sum_k a[n][k] b[m][k] over the step's 64 bytes of k; lane l of D holds m = l % 16, n = 4 (l / 16) + 0..3
template <int DT> __device__ __forceinline__ pj_f32x4 pj_mfma(const pj_u32x4& a, const pj_u32x4& b, pj_f32x4 c) {
    if constexpr (DT == VDB_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pj_bf16x8, a), __builtin_bit_cast(pj_bf16x8, b), c, 0, 0, 0);
    else if constexpr (DT == VDB_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pj_f16x8, a), __builtin_bit_cast(pj_f16x8, b), c, 0, 0, 0);
    else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
}

// Stores the four consecutive columns that a lane holds of one row; `left` of them lie in the output.
template <int DT> __device__ __forceinline__ void pj_store4(void* out, long long at, const pj_f32x4& v, long long left, bool vec) {
    typedef typename PJ<DT>::T T;
    T* p = (T*)out + at;
    T t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = pj_from_f32<DT>(v[j]);
    if (vec && left >= 4) {
        if constexpr (DT == VDB_F32) *(pj_f32x4*)p = v;
        else { pj_s16x4 s = {(short)t[0], (short)t[1], (short)t[2], (short)t[3]}; *(pj_s16x4*)p = s; }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < left) p[j] = t[j];
    }
}

// ------------------------------------------------------------------------------------------- rows x matrix
struct PJRowsArgs {
    ProjRows p;
    int col_tiles;
    bool vec_out;
};

// Sum over the k tiles of one 128 x 128 output tile: two LDS buffers, the loads of the next tile in flight while the
// current one is multiplied.
template <int DT, bool MK, bool NK, bool VEC>
__device__ __forceinline__ void pj_mainloop(PJOperand<DT, MK>& om, PJOperand<DT, NK>& on, long long K, char* lds,
                                            int wm, int wn, pj_f32x4 (&acc)[4][4]) {
    constexpr int KT = 128 / PJ<DT>::E;
    const long long tiles = (K + KT - 1) / KT;
    auto left = [&](long long t) { const long long l = K - t * KT; return l < KT ? (int)l : KT; };
    if (tiles > 0) { om.template stage<VEC>(lds, left(0)); on.template stage<VEC>(lds + PJ_TILE_BYTES, left(0)); }
    for (long long t = 0; t < tiles; ++t) {
        const int cur = (int)(t & 1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (t + 1 < tiles) {
            char* nxt = lds + (cur ^ 1) * 2 * PJ_TILE_BYTES;
            om.template stage<VEC>(nxt, left(t + 1));
            on.template stage<VEC>(nxt + PJ_TILE_BYTES, left(t + 1));
        }
        const char* lm = lds + cur * 2 * PJ_TILE_BYTES;
        const char* ln = lm + PJ_TILE_BYTES;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            pj_u32x4 fm[4], fn[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fm[i] = pj_fragment<DT, MK>(lm, wm * 64 + i * 16, kk);
                fn[i] = pj_fragment<DT, NK>(ln, wn * 64 + i * 16, kk);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = pj_mfma<DT>(fn[j], fm[i], acc[i][j]);
        }
    }
}

// Low-rank term of one wave's 64 x 64 block, before the main product: for every request that meets a block of 16 rows,
// h f^T on the fp32 matrix unit (exact products of the fp32 intermediate), taken over only by the rows of that request,
// so that what one adapter holds never reaches another request's rows.
template <int DT>
__device__ __forceinline__ void pj_low_rank(const ProjRows& p, long long row, int colb, pj_f32x4 (&acc)[4][4]) {
    typedef typename PJ<DT>::T T;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long r0 = row + i * 16, m = r0 + li;
        if (r0 >= p.n) break;
        const long long mc = m < p.n ? m : p.n - 1;
        for (int s = pj_first_segment(p.offsets, p.segments, r0); s < p.segments; ++s) {
            const long long b = pj_clamp(p.offsets[s], p.n), e = pj_clamp(p.offsets[s + 1], p.n);
            if (b >= r0 + 16) break;
            const int a = p.ids[s];
            if (e <= b || a < 0 || a >= p.adapters) continue;
            const bool mine = m >= b && m < e;
            const T* f = (const T*)p.f + (long long)a * p.f_adapter;
            pj_f32x4 t[4] = {};
            for (int q = 0; q < p.rp; q += 16) {
                const pj_f32x4 hv = *(const pj_f32x4*)(p.h + mc * p.rp + q + lh * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = colb + j * 16 + li;
                    const T* fc = f + (long long)(col < p.N ? col : p.N - 1) * p.f_col;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int r = q + lh * 4 + u;
                        const float fv = r < p.rank ? pj_to_f32<DT>(fc[r * p.f_rank]) : 0.f;
                        t[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fv, mine ? hv[u] : 0.f, t[j], 0, 0, 0);
                    }
                }
            }
            if (mine)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = t[j];
        }
    }
}

template <int DT, int ODT, bool NK, bool VEC, bool ADAPT>
__global__ void __launch_bounds__(PJ_THREADS)
proj_rows_kernel(PJRowsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char pj_lds[];
    typedef typename PJ<DT>::T T;
    const ProjRows& p = a.p;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    long long row0, row1, first = 0;         // rows of this tile: [max(row0, first), row1)
    int seg = 0, col;
    if constexpr (ADAPT) {
        // one matrix for all rows: tiles over the rows from the first segment's start to the last one's end
        const long long span[2] = {pj_clamp(p.offsets[0], p.n), pj_clamp(p.offsets[p.segments], p.n)};
        if (span[1] <= span[0]) return;
        const long long t0 = span[0] / PJ_TILE, tiles = (span[1] + PJ_TILE - 1) / PJ_TILE - t0;
        const long long all = tiles * a.col_tiles, run = (all + 7) / 8, idx = blockIdx.x >> 3;
        const long long id = (long long)(blockIdx.x & 7) * run + idx;
        if (idx >= run || id >= all) return;
        col = (int)(id % a.col_tiles);
        row0 = (t0 + id / a.col_tiles) * PJ_TILE;
        first = span[0]; row1 = span[1];
    } else {
        if (!pj_find_tile(p.offsets, p.segments, p.n, PJ_TILE, a.col_tiles, blockIdx.x, seg, row0, row1, col)) return;
    }
    const int col0 = col * PJ_TILE;
    pj_f32x4 acc[4][4] = {};
    if constexpr (ADAPT) pj_low_rank<DT>(p, row0 + wm * 64, col0 + wn * 64, acc);
    PJOperand<DT, false> om;
    PJOperand<DT, NK> on;
    om.init((const T*)p.x, p.ldx, row0, row1);
    on.init((const T*)p.w + (long long)seg * p.w_group, p.ldw, col0, p.N);
    pj_mainloop<DT, false, NK, VEC>(om, on, p.K, pj_lds, wm, wn, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long m = row0 + wm * 64 + i * 16 + li;
        if (m >= row1 || m < first) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = col0 + wn * 64 + j * 16 + lh * 4;
            if (c < p.N) pj_store4<ODT>(p.y, m * p.ldy + c, acc[i][j], p.N - c, a.vec_out);
        }
    }
}

// ------------------------------------------------------------------------------------------- gradient of the matrices
struct PJWeightsArgs {
    ProjWeights p;
    int m_tiles, n_tiles;
    bool vec_out;
};

template <int DT, int ODT, bool VEC>
__global__ void __launch_bounds__(PJ_THREADS)
proj_weights_kernel(PJWeightsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char pj_lds[];
    typedef typename PJ<DT>::T T;
    const ProjWeights& p = a.p;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int seg = blockIdx.x / (a.m_tiles * a.n_tiles), rest = blockIdx.x % (a.m_tiles * a.n_tiles);
    const int m0 = rest / a.n_tiles * PJ_TILE, n0 = rest % a.n_tiles * PJ_TILE;
    const long long b = pj_clamp(p.offsets[seg], p.n), e = pj_clamp(p.offsets[seg + 1], p.n);
    pj_f32x4 acc[4][4] = {};
    PJOperand<DT, true> om, on;
    om.init((const T*)p.dy + b * p.lddy, p.lddy, m0, p.M);
    on.init((const T*)p.x + b * p.ldx, p.ldx, n0, p.N);
    pj_mainloop<DT, true, true, VEC>(om, on, e > b ? e - b : 0, pj_lds, wm, wn, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + wm * 64 + i * 16 + li;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = n0 + wn * 64 + j * 16 + lh * 4;
            if (c < p.N) pj_store4<ODT>(p.dw, ((long long)seg * p.M + m) * p.N + c, acc[i][j], p.N - c, a.vec_out);
        }
    }
}

// ------------------------------------------------------------------------------------------- low-rank intermediates
// h = s x f^T for 16 rows by 16 of the rank: the four waves take every fourth step of the contracted axis and add up
// through LDS in wave order.  Every request that meets the 16 rows is multiplied, and keeps its own rows.
template <int DT>
__global__ void __launch_bounds__(256)
proj_shrink_kernel(ProjShrink p) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, KS = 4 * V;          // elements per lane and per step
    __shared__ pj_f32x4 part[3][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4, wave = threadIdx.x >> 6;
    const long long r0 = (long long)blockIdx.x * 16, m = r0 + li;
    const int q0 = blockIdx.y * 16;
    const long long mc = m < p.n ? m : p.n - 1;
    const T* x = (const T*)p.x + mc * p.ldx;
    for (int s = pj_first_segment(p.offsets, p.segments, r0); s < p.segments; ++s) {
        const long long b = pj_clamp(p.offsets[s], p.n), e = pj_clamp(p.offsets[s + 1], p.n);
        if (b >= r0 + 16) break;
        const int ad = p.ids[s];
        if (e <= b || ad < 0 || ad >= p.adapters) continue;
        const T* f = (const T*)p.f + (long long)ad * p.f_adapter;
        const int q = q0 + li;
        pj_f32x4 acc = {};
        for (int k0 = wave * KS; k0 < p.K; k0 += 4 * KS) {
            union { T t[V]; pj_u32x4 v; } xa, fa;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int k = k0 + lh * V + j;
                xa.t[j] = k < p.K ? x[k] : (T)0;
                fa.t[j] = k < p.K && q < p.rank ? f[(long long)q * p.f_rank + (long long)k * p.f_k] : (T)0;
            }
            acc = pj_mfma<DT>(fa.v, xa.v, acc);            // lane: row m, ranks q0 + 4 lh + 0..3
        }
        __syncthreads();
        if (wave) part[wave - 1][lane] = acc;
        __syncthreads();
        if (wave == 0 && m >= b && m < e) {
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] += part[w][lane][j];
            const float sc = p.scale ? p.scale[ad] : 1.f;
            pj_f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = q0 + lh * 4 + j < p.rank ? sc * acc[j] : 0.f;
            *(pj_f32x4*)(p.h + m * p.rp + q0 + lh * 4) = o;
        }
    }
}

// ------------------------------------------------------------------------------------------- gradient of the factors
// 16 of the rank by 64 columns of one adapter: the four waves take the adapter's rows 16 at a time in turn, over every
// request that names the adapter, and add up in wave order.  Products on the fp32 matrix unit.
template <int DT, int ODT>
__global__ void __launch_bounds__(256)
proj_factor_kernel(ProjFactor p) {
    typedef typename PJ<DT>::T T;
    typedef typename PJ<ODT>::T O;
    __shared__ pj_f32x4 part[3][4][64];
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4, wave = threadIdx.x >> 6;
    const int n0 = blockIdx.x * 64, q0 = blockIdx.y * 16, ad = blockIdx.z;
    pj_f32x4 acc[4] = {};
    long long turn = 0;                    // blocks of 16 rows met so far
    for (int s0 = 0; s0 < p.segments; s0 += 64) {
        const bool hit = s0 + lane < p.segments && p.ids[s0 + lane] == ad;
        unsigned long long mask = __ballot(hit);
        while (mask) {
            const int s = s0 + __builtin_ctzll(mask);
            mask &= mask - 1;
            const long long b = pj_clamp(p.offsets[s], p.n), e = pj_clamp(p.offsets[s + 1], p.n);
            for (long long r = b; r < e; r += 16, ++turn) {
                if ((turn & 3) != wave) continue;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const long long i = r + u * 4 + lh;
                    const bool ok = i < e;
                    const float hv = ok ? p.h[i * p.rp + q0 + li] : 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int c = n0 + j * 16 + li;
                        const float xv = ok && c < p.N ? pj_to_f32<DT>(((const T*)p.x)[i * p.ldx + c]) : 0.f;
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv, hv, acc[j], 0, 0, 0);   // lane: rank q0 + li, columns 4 lh + 0..3
                    }
                }
            }
        }
    }
    if (wave)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[wave - 1][j][lane] = acc[j];
    __syncthreads();
    if (wave) return;
    const int q = q0 + li;
    if (q >= p.rank) return;
    O* out = (O*)p.out + (long long)ad * p.rank * p.N;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = n0 + j * 16 + lh * 4 + u;
            if (c >= p.N) continue;
            const float v = acc[j][u] + part[0][j][lane][u] + part[1][j][lane][u] + part[2][j][lane][u];
            out[p.by_col ? (long long)c * p.rank + q : (long long)q * p.N + c] = pj_from_f32<ODT>(v);
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
static bool pj_aligned(const void* ptr, long long ld, int dtype, int bytes) {
    const long long e = dtype == VDB_F32 ? 4 : 2;
    return (uintptr_t)ptr % bytes == 0 && ld * e % bytes == 0;
}

template <typename K, typename A>
static hipError_t pj_launch(K kernel, dim3 grid, size_t lds, const A& args, hipStream_t st) {
    hipLaunchKernelGGL(kernel, grid, dim3(PJ_THREADS), lds, st, args);
    return hipGetLastError();
}

// input type x output type (the input's, or fp32)
#define PJ_TYPES(dt, odt, CALL)                                                                        \
    do {                                                                                               \
        if ((dt) == VDB_F32) { constexpr int DT = VDB_F32, ODT = VDB_F32; CALL; }                      \
        else if ((dt) == VDB_BF16 && (odt) == VDB_F32) { constexpr int DT = VDB_BF16, ODT = VDB_F32; CALL; } \
        else if ((dt) == VDB_BF16) { constexpr int DT = VDB_BF16, ODT = VDB_BF16; CALL; }              \
        else if ((odt) == VDB_F32) { constexpr int DT = VDB_F16, ODT = VDB_F32; CALL; }                \
        else { constexpr int DT = VDB_F16, ODT = VDB_F16; CALL; }                                      \
    } while (0)

template <int DT, int ODT>
static hipError_t rows_typed(const ProjRows& p, hipStream_t st) {
    PJRowsArgs a;
    a.p = p;
    a.col_tiles = (p.N + PJ_TILE - 1) / PJ_TILE;
    a.vec_out = pj_aligned(p.y, p.ldy, ODT, 4 * PJ<ODT>::E);
    constexpr int V = 16 / PJ<DT>::E;
    const bool vec = pj_aligned(p.x, p.ldx, DT, 16) && pj_aligned(p.w, p.ldw, DT, 16) && p.w_group % V == 0 &&
                     p.K % V == 0 && (!p.w_by_k || p.N % V == 0);
    const long long row_tiles = p.ids ? (p.n + PJ_TILE - 1) / PJ_TILE : p.n / PJ_TILE + p.segments;
    const long long blocks = (row_tiles * a.col_tiles + 7) / 8 * 8;
    const dim3 grid((unsigned)blocks);
    const size_t lds = 4 * PJ_TILE_BYTES;
#define PJ_ROWS(NK, VEC) \
    (p.ids ? pj_launch(proj_rows_kernel<DT, ODT, NK, VEC, true>, grid, lds, a, st) \
           : pj_launch(proj_rows_kernel<DT, ODT, NK, VEC, false>, grid, lds, a, st))
    if (p.w_by_k) return vec ? PJ_ROWS(true, true) : PJ_ROWS(true, false);
    return vec ? PJ_ROWS(false, true) : PJ_ROWS(false, false);
#undef PJ_ROWS
}

hipError_t launch_proj_rows(const ProjRows& p, hipStream_t st) {
    if (p.n <= 0 || p.segments <= 0) return hipSuccess;
    hipError_t e = hipSuccess;
    PJ_TYPES(p.dtype, p.out_dtype, e = (rows_typed<DT, ODT>(p, st)));
    return e;
}

template <int DT, int ODT>
static hipError_t weights_typed(const ProjWeights& p, hipStream_t st) {
    PJWeightsArgs a;
    a.p = p;
    a.m_tiles = (p.M + PJ_TILE - 1) / PJ_TILE;
    a.n_tiles = (p.N + PJ_TILE - 1) / PJ_TILE;
    a.vec_out = pj_aligned(p.dw, p.N, ODT, 4 * PJ<ODT>::E);
    constexpr int V = 16 / PJ<DT>::E;
    const bool vec = pj_aligned(p.dy, p.lddy, DT, 16) && pj_aligned(p.x, p.ldx, DT, 16) && p.M % V == 0 && p.N % V == 0;
    const dim3 grid((unsigned)((long long)p.segments * a.m_tiles * a.n_tiles));
    return vec ? pj_launch(proj_weights_kernel<DT, ODT, true>, grid, 4 * PJ_TILE_BYTES, a, st)
               : pj_launch(proj_weights_kernel<DT, ODT, false>, grid, 4 * PJ_TILE_BYTES, a, st);
}

hipError_t launch_proj_weights(const ProjWeights& p, hipStream_t st) {
    hipError_t e = hipSuccess;
    PJ_TYPES(p.dtype, p.out_dtype, e = (weights_typed<DT, ODT>(p, st)));
    return e;
}

hipError_t launch_proj_shrink(const ProjShrink& p, hipStream_t st) {
    if (p.n <= 0 || p.segments <= 0) return hipSuccess;
    const dim3 grid((unsigned)((p.n + 15) / 16), (unsigned)(p.rp / 16));
    if (p.dtype == VDB_F32) return pj_launch(proj_shrink_kernel<VDB_F32>, grid, 0, p, st);
    if (p.dtype == VDB_BF16) return pj_launch(proj_shrink_kernel<VDB_BF16>, grid, 0, p, st);
    return pj_launch(proj_shrink_kernel<VDB_F16>, grid, 0, p, st);
}

hipError_t launch_proj_zero_outside(float* q, long long dim, long long n, const long long* offsets, int segments, hipStream_t st) {
    const long long blocks = (n * dim + 255) / 256;
    hipLaunchKernelGGL(proj_zero_outside_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, st, q, dim, n, offsets, segments);
    return hipGetLastError();
}

hipError_t launch_proj_factor(const ProjFactor& p, hipStream_t st) {
    const dim3 grid((unsigned)((p.N + 63) / 64), (unsigned)(p.rp / 16), (unsigned)p.adapters);
    hipError_t e = hipSuccess;
    PJ_TYPES(p.dtype, p.out_dtype, e = (pj_launch(proj_factor_kernel<DT, ODT>, grid, 0, p, st)));
    return e;
}

}  // namespace vdb
