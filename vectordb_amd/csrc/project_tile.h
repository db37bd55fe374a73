// Device side of the learned projections: segments, operand tiles in LDS, the tiled products and the low-rank term.
// Included by one source file for each type (kernels_project_*.hip) and by kernels_project.hip.
#pragma once
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

// A value from global memory, or zeros.  The address space is named: of a choice between an argument's memory and a constant the
// compiler makes a flat load, whose wait is for every load in flight.
template <typename V> __device__ __forceinline__ V pj_load_if(bool ok, const void* p) {
    return *(const __attribute__((address_space(1))) V*)(ok ? p : (const void*)pj_zero16);
}

template <int DT> struct PJ {            // 16-bit types
    static constexpr int E = 2;
    typedef unsigned short T;
};
template <> struct PJ<VDB_F32> {
    static constexpr int E = 4;
    typedef float T;
};

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

// Vectors at any address that is aligned to an element of 16 bits.
typedef pj_u32x4 pj_u32x4_any __attribute__((aligned(2)));
typedef pj_f32x4 pj_f32x4_any __attribute__((aligned(4)));
typedef pj_s16x4 pj_s16x4_any __attribute__((aligned(2)));

// The 16 bytes at p of which `left` elements lie in the operand (none: 0 or less), the others zero.  Where the operand's rows hold
// 16 bytes (`whole`), a part is read as the 16 bytes that end where the row does and moved down, so that every piece is one load
// without a branch.
template <typename T> __device__ __forceinline__ int pj_behind(int left) { return left > 0 && left < (int)(16 / sizeof(T)) ? 16 / sizeof(T) - left : 0; }
template <typename T> __device__ __forceinline__ pj_u32x4 pj_moved(const pj_u32x4& v, int behind) {
    return __builtin_bit_cast(pj_u32x4, __builtin_bit_cast(unsigned __int128, v) >> (behind * (int)sizeof(T) * 8));
}
template <typename T> __device__ __forceinline__ pj_u32x4 pj_piece_unmoved(const T* p, int left) {
    return pj_load_if<pj_u32x4_any>(left > 0, p - pj_behind<T>(left));
}
template <typename T> __device__ __forceinline__ pj_u32x4 pj_piece_by_element(const T* p, int left) {
    constexpr int V = 16 / sizeof(T);
    union { T t[V]; pj_u32x4 v; } r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.t[j] = j < left ? p[j] : (T)0;
    return r.v;
}
template <typename T> __device__ __forceinline__ pj_u32x4 pj_piece(const T* p, int left, bool whole) {
    if (whole) return pj_moved<T>(pj_piece_unmoved(p, left), pj_behind<T>(left));
    return pj_piece_by_element(p, left);
}

// ------------------------------------------------------------------------------------------- segments
__device__ __forceinline__ long long pj_clamp(long long v, long long n) { return v < 0 ? 0 : v > n ? n : v; }

// Which tile of TM rows workgroup `bid` of a grouped product works on: tiles are numbered segment by segment
// (ceil(size / TM) each), column tiles run fastest, and the numbers are dealt to the eight XCDs in contiguous runs
// (workgroup b runs on XCD b % 8), so that the column tiles that share rows share an L2.
// Every wave does this by itself, 64 segments at a time.  Returns false for workgroups past the last tile.
__device__ __forceinline__ bool pj_find_tile(const long long* offsets, int segments, long long n, int tm, int col_tiles,
                                             unsigned bid, int& seg, long long& row0, long long& row1, int& col, long long& number) {
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
    number = want;
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

__device__ __forceinline__ bool pj_find_tile(const long long* offsets, int segments, long long n, int tm, int col_tiles,
                                             unsigned bid, int& seg, long long& row0, long long& row1, int& col) {
    long long number;
    return pj_find_tile(offsets, segments, n, tm, col_tiles, bid, seg, row0, row1, col, number);
}

// First segment whose end lies behind `row` (offsets do not decrease); `segments` if there is none.  Called by whole
// waves: 64 ends are compared at a time, so that a search costs one load for each factor of 64.
__device__ __forceinline__ int pj_first_segment(const long long* offsets, int segments, long long row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = segments;                       // the answer lies in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const int at = lo + (lane + 1) * step - 1;   // last segment of this lane's share
        const bool behind = at >= hi || offsets[at + 1] > row;
        const unsigned long long m = __ballot(behind);
        const int k = m ? __builtin_ctzll(m) : 64;   // none: the 64 shares end at hi, and every segment lies before the row
        const int nlo = lo + k * step, nhi = lo + (k + 1) * step - 1;
        lo = nlo < hi ? nlo : hi;
        hi = nhi < hi ? nhi : hi;
    }
    return lo;
}

// (a shuffle of a lane that is the same for all goes through LDS: 0.1 us for each request)
__device__ __forceinline__ long long pj_readlane64(long long v, int lane) {
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)v, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (long long)((unsigned long long)hi << 32 | lo);
}

// Requests with an adapter that meet rows [r0, r1): visited one by one by the whole wave, 64 loaded at a time.
template <typename F>
__device__ __forceinline__ void pj_each_request(const long long* offsets, const int* ids, int segments, int adapters, long long n,
                                                long long r0, long long r1, F&& visit) {
    const int lane = threadIdx.x & 63;
    for (int s0 = segments <= 64 ? 0 : pj_first_segment(offsets, segments, r0); s0 < segments; s0 += 64) {
        const int s = s0 + lane;
        long long b = n, e = 0;
        int a = -1;
        if (s < segments) { b = pj_clamp(offsets[s], n); e = pj_clamp(offsets[s + 1], n); a = ids[s]; }
        unsigned long long m = __ballot(e > b && b < r1 && e > r0 && a >= 0 && a < adapters);
        const bool last = __ballot(s < segments && b >= r1) != 0;
        while (m) {
            const int src = __builtin_ctzll(m);
            m &= m - 1;
            visit(pj_readlane64(b, src), pj_readlane64(e, src), __builtin_amdgcn_readlane(a, src));
        }
        if (last) break;
    }
}

// ------------------------------------------------------------------------------------------- tiles in LDS
// One operand tile: R = 32, 64 or 128 rows (or columns) of the product by 128 bytes of the contracted axis, kept as it lies in
// memory in 16-byte pieces whose place is swizzled so that the fragment reads below touch every bank once:
//   contiguous along k (BYK = false): row r is 128 bytes, piece c sits in slot c ^ ((r >> 1) & 7)
//   contiguous along the rows (BYK = true): one line per k, piece c of line k in slot c ^ pj_line_swizzle(k)
constexpr int PJ_THREADS = 256;
constexpr int pj_tile_bytes(int R) { return R * 128; }

template <int DT, int R> __device__ __forceinline__ int pj_line_swizzle(int k) {
    if constexpr (DT == VDB_F32) return (k >> 2 & (R == 32 ? 1 : 3)) << 2;       // 64-byte spans: the four lane groups read lines k, k + 4, ...
    else if constexpr (R >= 128) return ((k & 3) | (k >> 3 & 1) << 2) << 1;      // 32-byte spans of a line of 256 or 512 bytes
    else return ((k >> 1 & 1) | (k >> 3 & 1) << 1) << 1;                         // 32-byte spans of a 128-byte line, two lines cover the banks
}

template <int DT, bool BYK, int R> struct PJOperand {
    typedef typename PJ<DT>::T T;
    static constexpr int E = PJ<DT>::E, V = 16 / E, KT = 128 / E, P = R / 32;    // P: pieces per thread
    static constexpr int PL = R * E / 16;                                        // BYK: pieces per line
    const T* src[P];
    long long step[P];
    int kpos[P];                 // k of the piece within a tile
    int rem[P];                  // elements of the piece that lie in the operand's rows (V or 0 if !BYK)
    bool whole, ragged;          // (through registers) what is contiguous holds 16 bytes; it ends inside one of this tile's pieces

    // rows r0 .. r0 + R - 1 of [0, rows), k from 0
    __device__ __forceinline__ void init(const T* base, long long ld, long long r0, long long rows, long long K) {
        whole = (BYK ? rows : K) >= V;
        ragged = BYK && r0 + R > rows && rows % V != 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int p = i * PJ_THREADS + (int)threadIdx.x;
            if constexpr (!BYK) {
                const int r = p >> 3, c = (p & 7) ^ ((r >> 1) & 7);
                kpos[i] = c * V;
                rem[i] = r0 + r < rows ? V : 0;
                src[i] = base + (rem[i] ? (r0 + r) * ld + c * V : 0);
                step[i] = rem[i] ? KT : 0;
            } else {
                const int k = p / PL, c = p % PL ^ pj_line_swizzle<DT, R>(k);
                kpos[i] = k;
                const long long left = rows - (r0 + c * V);
                rem[i] = left >= V ? V : left > 0 ? (int)left : 0;
                src[i] = base + (rem[i] ? (long long)k * ld + r0 + c * V : 0);
                step[i] = rem[i] ? KT * ld : 0;
            }
        }
    }
    // the next KT elements of the contracted axis, of which `kleft` lie in the operand: one load per piece whatever kleft is
    __device__ __forceinline__ void stage(char* lds, int kleft) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            char* const wave_dst = lds + (i * PJ_THREADS + ((int)threadIdx.x & ~63)) * 16;
            const T* s = rem[i] && kpos[i] < kleft ? src[i] : (const T*)pj_zero16;
            __builtin_amdgcn_global_load_lds((const PJ_GLOBAL void*)s, (PJ_LOCAL void*)wave_dst, 16, 0, 0);
            src[i] += step[i];
        }
    }
    // the same for operands of any alignment and size, through registers; W: whole
    template <bool W> __device__ __forceinline__ void load(pj_u32x4 (&r)[P], int kleft) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if constexpr (W) r[i] = pj_piece_unmoved(src[i], inside(i, kleft));
            else r[i] = pj_piece_by_element(src[i], inside(i, kleft));
            src[i] += step[i];
        }
    }
    // the same kleft as when they were loaded
    template <bool W> __device__ __forceinline__ void put(char* lds, const pj_u32x4 (&r)[P], int kleft) const {
        const bool parts = W && (BYK ? ragged : kleft < KT);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const pj_u32x4 v = parts ? pj_moved<T>(r[i], pj_behind<T>(inside(i, kleft))) : r[i];
            *(pj_u32x4*)(lds + (i * PJ_THREADS + (int)threadIdx.x) * 16) = v;
        }
    }
    __device__ __forceinline__ int inside(int i, int kleft) const {
        return BYK ? (kpos[i] < kleft ? rem[i] : 0) : (rem[i] ? kleft - kpos[i] : 0);
    }
};

// Fragments of B times 16 rows from `row` (a multiple of 16): lane l holds row + l % 16 and, of the step's 64 bytes of k, the 16
// bytes number l / 16 (16-bit: k = 8 (l / 16) + 0..7; fp32: k = 4 (l / 16) + 0..3, one element for each of four products).
template <int DT, bool BYK, int R, int B>
__device__ __forceinline__ void pj_fragments(const char* lds, int row, int kk, pj_u32x4 (&f)[B]) {
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    constexpr int LINE = R * PJ<DT>::E;
    if constexpr (!BYK) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int r = row + i * 16 + li;
            f[i] = *(const pj_u32x4*)(lds + r * 128 + (((kk * 4 + lh) ^ ((r >> 1) & 7)) << 4));
        }
    } else if constexpr (DT == VDB_F32) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int c = ((row + i * 16 + li) >> 2) ^ pj_line_swizzle<DT, R>(lh * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                f[i][j] = *(const unsigned*)(lds + (kk * 16 + lh * 4 + j) * LINE + (c << 4) + (li & 3) * 4);
        }
    } else if constexpr (B == 8) {
        pj_u32x4 lo[4], hi[4];
        pj_fragments<DT, BYK, R, 4>(lds, row, kk, lo);
        pj_fragments<DT, BYK, R, 4>(lds, row + 64, kk, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[i] = lo[i]; f[4 + i] = hi[i]; }
    } else {
        static_assert(B == 2 || B == 4, "fragments of one asm block");
        // ds_read_b64_tr_b16: sixteen lanes read a block of 4 k x 16 rows, lane i the 8 bytes number i % 4 of line i / 4, and get
        // column i of the block; lines k and k + 4 have the same swizzle.  The reads and their wait are one asm block: through
        // the builtin the compiler waits for every load into LDS in flight first.
        const int k = lh * 8 + (li >> 2), swz = pj_line_swizzle<DT, R>(k);
        const unsigned line = (unsigned)(uintptr_t)(PJ_LOCAL const char*)lds + (unsigned)((kk * 32 + k) * LINE + (li & 1) * 8);
        unsigned at[B];
#pragma unroll
        for (int i = 0; i < B; ++i) at[i] = line + (unsigned)(((((row + i * 16) >> 3) + ((li & 3) >> 1)) ^ swz) << 4);
        unsigned long long v[B][2];
        if constexpr (B == 4)
            asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
                         "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
                         "s_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1]), "=&v"(v[2][0]), "=&v"(v[2][1]), "=&v"(v[3][0]), "=&v"(v[3][1])
                         : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(4 * LINE) : "memory");
        else
            asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                         "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
                         "s_waitcnt lgkmcnt(0)"
                         : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1])
                         : "v"(at[0]), "v"(at[1]), "n"(4 * LINE) : "memory");
#pragma unroll
        for (int i = 0; i < B; ++i) {
            struct two { unsigned long long a, b; } t = {v[i][0], v[i][1]};
            f[i] = __builtin_bit_cast(pj_u32x4, t);
        }
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
template <int DT> __device__ __forceinline__ void pj_store4(void* out, long long at, const pj_f32x4& v, long long left) {
    typedef typename PJ<DT>::T T;
    T* p = (T*)out + at;
    T t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = pj_from_f32<DT>(v[j]);
    if (left >= 4) {
        if constexpr (DT == VDB_F32) *(pj_f32x4_any*)p = v;
        else { pj_s16x4 s = {(short)t[0], (short)t[1], (short)t[2], (short)t[3]}; *(pj_s16x4_any*)p = s; }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < left) p[j] = t[j];
    }
}

// ------------------------------------------------------------------------------------------- tiled products
// Waits until at most N of this wave's loads are in flight and all its LDS reads have returned, then meets the other waves.
template <int N> __device__ __forceinline__ void pj_wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Tiles of a launch: 64 x 64 with four stages of k in flight where there are few of them, 128 x 128 with two stages and
// two workgroups on a CU where there are many (see pj_small_tiles); fp32, whose products take eight times as long, 32 x 32
// with eight stages where 64 x 64 leave CUs without work.
template <int R> struct PJRing {
    static constexpr int STAGES = R == 32 ? 8 : R == 64 ? 4 : 2;
    static constexpr int BYTES = STAGES * 2 * pj_tile_bytes(R);
    static constexpr int HALVES = 2 * 2 * pj_tile_bytes(R);          // through registers: two stages
};

// One R x R output tile: a ring of LDS stages, each the next 128 bytes of k of both operands.  The loads of a stage are
// issued STAGES - 1 steps ahead; every step issues the same number of them (zeros past the end), so that the wait can count.
template <int DT, bool MK, bool NK, bool VEC, int R>
struct PJProduct {
    static constexpr int KT = 128 / PJ<DT>::E, B = R / 32, S = PJRing<R>::STAGES, TB = pj_tile_bytes(R);
    PJOperand<DT, MK, R> om;
    PJOperand<DT, NK, R> on;
    long long left;              // of k, not yet staged
    int tiles;

    // VEC: loads straight into LDS.  Otherwise through D sets of registers, loaded D steps ahead and put into the other half of
    // the ring while the current step is multiplied.
    static constexpr int D = R == 128 ? 2 : 3;
    int kl[D];                   // of k in each
    pj_u32x4 rm[VEC ? 1 : D][VEC ? 1 : PJOperand<DT, MK, R>::P], rn[VEC ? 1 : D][VEC ? 1 : PJOperand<DT, NK, R>::P];

    __device__ __forceinline__ int take() {
        const int l = left < KT ? (left > 0 ? (int)left : 0) : KT;
        left -= KT;
        return l;
    }
    __device__ __forceinline__ void next(char* lds, int stage) {
        const int l = take();
        om.stage(lds + stage * 2 * TB, l);
        on.stage(lds + stage * 2 * TB + TB, l);
    }
    __device__ __forceinline__ void begin(long long K, char* lds) {
        left = K;
        tiles = (int)((K + KT - 1) / KT);
        if (tiles <= 0) return;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < S - 1; ++i) next(lds, i);
        } else if (om.whole && on.whole) {
#pragma unroll
            for (int i = 0; i < D; ++i) load(i);
        }
    }
    __device__ __forceinline__ void load(int d) {
        kl[d] = take();
        om.template load<true>(rm[d], kl[d]);
        on.template load<true>(rn[d], kl[d]);
        asm volatile("" ::: "memory");                              // in this order, for the waits
    }
    __device__ __forceinline__ void multiply(const char* lm, int wm, int wn, pj_f32x4 (&acc)[B][B]) {
        const char* ln = lm + TB;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            pj_u32x4 fm[B], fn[B];
            pj_fragments<DT, MK, R, B>(lm, wm * (R / 2), kk, fm);
            pj_fragments<DT, NK, R, B>(ln, wn * (R / 2), kk, fn);
#pragma unroll
            for (int i = 0; i < B; ++i)
#pragma unroll
                for (int j = 0; j < B; ++j) acc[i][j] = pj_mfma<DT>(fn[j], fm[i], acc[i][j]);
        }
    }
    // acc += om on^T; the wave's block is rows wm * R/2.., columns wn * R/2..
    __device__ __forceinline__ void run(char* lds, int wm, int wn, pj_f32x4 (&acc)[B][B]) {
        if constexpr (VEC) {
            constexpr int L = 2 * PJOperand<DT, MK, R>::P;          // loads per stage and thread
            int cur = 0;
            for (int t = 0; t < tiles; ++t) {
                pj_wait_and_meet<(S - 2) * L>();
                next(lds, cur == 0 ? S - 1 : cur - 1);
                multiply(lds + cur * 2 * TB, wm, wn, acc);
                cur = cur + 1 == S ? 0 : cur + 1;
            }
            // nothing may still be on its way into LDS when the workgroup's memory goes to another one
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else if (om.whole && on.whole) {
            for (int t = 0; t < tiles; t += D)
#pragma unroll
                for (int d = 0; d < D; ++d) {                       // (steps past the end multiply zeros)
                    char* const buf = lds + ((t + d) & 1) * 2 * TB;
                    om.template put<true>(buf, rm[d], kl[d]);
                    on.template put<true>(buf + TB, rn[d], kl[d]);
                    load(d);
                    __syncthreads();                                // (the other half was read a step ago, before the last meeting)
                    multiply(buf, wm, wn, acc);
                }
        } else {
            // rows of less than 16 bytes, element by element
            for (int t = 0; t < tiles; ++t) {
                char* const buf = lds + (t & 1) * 2 * TB;
                const int l = take();
                om.template load<false>(rm[0], l);
                om.template put<false>(buf, rm[0], l);
                on.template load<false>(rn[0], l);
                on.template put<false>(buf + TB, rn[0], l);
                __syncthreads();
                multiply(buf, wm, wn, acc);
            }
        }
    }
};

// ------------------------------------------------------------------------------------------- wide products, 16-bit
// For the gradient of the matrices, which contracts over rows (both operands lie by k): 256 x 128 per workgroup of four waves,
// 128 x 64 each, which read three quarters of the LDS bytes per product that 64 x 64 do; 32 rows per stage, a ring of three
// 24 KiB stages, two workgroups on a CU.  Addresses are 32-bit offsets from bases that move along the rows.
// (dw of 32 768 rows, 1024 x 768: 88 -> 76 us.  For the rows themselves, whose 64 bytes of k per row are half a cache line, such
// tiles gained 6 % at 65 536 rows of fp32 output and nothing elsewhere; 256 x 256 tiles of eight waves, half a step apart, 15 % there.)
constexpr int PJ_WIDE_M = 256, PJ_WIDE_N = 128, PJ_WIDE_S = 3, PJ_WIDE_STAGE = (PJ_WIDE_M + PJ_WIDE_N) * 64;
constexpr int PJ_WIDE_BYTES = PJ_WIDE_S * PJ_WIDE_STAGE;

// Can the offsets within a stage be 32 bits wide?
static inline bool pj_offsets_fit(long long rows, long long ld, int esize) { return rows * ld * esize < ((long long)1 << 31); }

// One operand's part of a stage: 32 lines of R columns, piece c of line k in slot c ^ pj_line_swizzle(k).  Columns past the end repeat
// the last piece of 8: their results are not stored.
template <int DT, int R> struct PJWideOperand {
    typedef typename PJ<DT>::T T;
    static constexpr int P = R / 64, PL = R / 8;
    const char* base;
    long long step;
    unsigned off[P];
    __device__ __forceinline__ void init(const T* first, long long ld, int cols) {
        const int last = (cols < R ? cols : R) / 8 - 1;
        base = (const char*)first;
        step = 64 * ld;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int p = i * PJ_THREADS + (int)threadIdx.x, k = p / PL, c = p % PL ^ pj_line_swizzle<DT, R>(k);
            off[i] = (unsigned)k * (unsigned)(ld * 2) + (unsigned)(c < last ? c : last) * 16u;
        }
    }
    // `left` of the 32 lines lie in the operand, the others are zero
    __device__ __forceinline__ void stage(char* lds, int left) {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const char* src = (i * PJ_THREADS + (int)threadIdx.x) / PL < left ? base + off[i] : (const char*)pj_zero16;
            __builtin_amdgcn_global_load_lds((const PJ_GLOBAL void*)src, (PJ_LOCAL void*)(lds + (i * PJ_THREADS + wave * 64) * 16), 16, 0, 0);
        }
        base += step;
    }
};

template <int DT> struct PJWide {
    static constexpr int BM = 8, BN = 4;
    PJWideOperand<DT, PJ_WIDE_M> om;
    PJWideOperand<DT, PJ_WIDE_N> on;
    long long left;
    // one load per piece also past the end, so that the waits can count
    __device__ __forceinline__ void next(char* lds) {
        const int l = left < 32 ? (left > 0 ? (int)left : 0) : 32;
        om.stage(lds, l);
        on.stage(lds + PJ_WIDE_M * 64, l);
        left -= 32;
    }
    __device__ __forceinline__ void run(long long rows, char* lds, int wm, int wn, pj_f32x4 (&acc)[BM][BN]) {
        left = rows;
        const int steps = (int)((rows + 31) / 32);
        if (steps <= 0) return;
        next(lds);
        next(lds + PJ_WIDE_STAGE);
        int cur = 0;
        for (int t = 0; t < steps; ++t) {
            pj_wait_and_meet<(PJ_WIDE_S - 2) * 6>();
            next(lds + (cur == 0 ? 2 : cur - 1) * PJ_WIDE_STAGE);
            const char* at = lds + cur * PJ_WIDE_STAGE;
            pj_u32x4 fm[BM], fn[BN];
            pj_fragments<DT, true, PJ_WIDE_N, BN>(at + PJ_WIDE_M * 64, wn * 64, 0, fn);
            pj_fragments<DT, true, PJ_WIDE_M, BM>(at, wm * 128, 0, fm);
#pragma unroll
            for (int i = 0; i < BM; ++i)
#pragma unroll
                for (int j = 0; j < BN; ++j) acc[i][j] = pj_mfma<DT>(fn[j], fm[i], acc[i][j]);
            cur = cur == 2 ? 0 : cur + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
};

// ------------------------------------------------------------------------------------------- low-rank term
// The term h f^T of a wave's block, before the main product.  Beside 16-bit rows the fp32 intermediate h comes in three bf16 parts
// that add up to it, so that no way below rounds h; a factor in fp16 is taken apart into two bf16 parts, which hold its 11 bits, as
// it is multiplied.  (Six products instead of two of fp16 parts, whose range is too small: a rank 2^-20 of its row's largest kept 5
// bits.  1024 x 768 fp16, 32 768 rows of 48 requests, rank 64: 110 us against 102, 108 without the product of the smallest parts.)
//   one adapter for all of the wave's rows, or a few and ranks of one step: the matrix unit, all rows by each of them, taken over
//     as below;
//   few adapters in 16 rows (two, or one for each 12 ranks): the matrix unit, all 16 rows by one adapter, taken over by the
//     rows of that adapter only, so that what one adapter holds never reaches another request's rows;
//   more: every lane for itself, its row by its four columns, which waits once for all adapters instead of once for each, in a time
//     that grows with the rank.

// How the factor f lies: entry (column, rank) of an adapter at column * f_col + rank * f_rank elements (32 bits hold it).
//   PJ_F_RANKS   ranks contiguous, 16-byte pieces of them aligned (B of a forward pass)
//   PJ_F_COLS    columns contiguous, groups of four aligned and whole (A of a backward pass)
//   PJ_F_ANY     neither
enum { PJ_F_ANY = 0, PJ_F_RANKS = 1, PJ_F_COLS = 2 };

// Waits until the matrix unit has written t: the compiler's own wait for an fp32 product (10 states) was seen to fall away where the
// products end a loop whose exit reads them at once (columns 3 mod 4 of a 32 x 32 tile held the sum without its last step).
__device__ __forceinline__ void pj_settle(pj_f32x4& t) { asm volatile("s_nop 15" : "+v"(t)); }

// Entry of one adapter's factor, the same adapter for all lanes: 32 bits hold the byte too, which leaves the address to a scalar.
template <typename T> __device__ __forceinline__ T pj_entry(const T* f, unsigned at) {
    return *(const T*)((const char*)f + at * (unsigned)sizeof(T));
}

// t += f h^T over one step of ranks, the products of the smallest parts first.
template <int DT> struct PJFactorParts {
    pj_u32x4 hi;
    __device__ __forceinline__ explicit PJFactorParts(const pj_u32x4& f) : hi(f) {}
    __device__ __forceinline__ void multiply(const pj_u32x4 (&h)[proj_parts(DT)], pj_f32x4& t) const {
#pragma unroll
        for (int u = proj_parts(DT) - 1; u >= 0; --u) t = pj_mfma<DT>(hi, h[u], t);
    }
};
template <> struct PJFactorParts<VDB_F16> {
    pj_u32x4 hi, lo;
    // the first 8 bits, cut, and the other 3
    __device__ __forceinline__ explicit PJFactorParts(const pj_u32x4& f) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float a = pj_to_f32<VDB_F16>((unsigned short)f[w]), b = pj_to_f32<VDB_F16>((unsigned short)(f[w] >> 16));
            const unsigned ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
            hi[w] = __builtin_amdgcn_perm(ub, ua, 0x07060302);               // the upper halves of both
            lo[w] = __builtin_amdgcn_perm(__float_as_uint(b - __uint_as_float(ub)), __float_as_uint(a - __uint_as_float(ua)), 0x07060302);
        }
    }
    __device__ __forceinline__ void multiply(const pj_u32x4 (&h)[3], pj_f32x4& t) const {
#pragma unroll
        for (int u = 2; u >= 0; --u) {
            t = pj_mfma<VDB_BF16>(lo, h[u], t);
            t = pj_mfma<VDB_BF16>(hi, h[u], t);
        }
    }
};

// 16 rows by one adapter on the matrix unit; t: lane's row by columns colb + 16 j + 4 (l / 16) + 0..3
template <int DT, int F, int C>
__device__ __forceinline__ void pj_low_rank_block(const ProjRows& p, long long mc, int colb, int a, pj_f32x4 (&t)[C]) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, QS = 4 * V, NP = proj_parts(DT);
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int rp = proj_rank_pad(p.rank, DT);
    const unsigned fr = (unsigned)p.f_rank, fcol = (unsigned)p.f_col;
    const T* f = (const T*)p.f + (long long)a * p.f_adapter;
    const T* h = (const T*)p.h + mc * (NP * rp);
#pragma unroll F == PJ_F_RANKS ? 2 : 1
    for (int q = 0; q < p.rank; q += QS) {
        pj_u32x4 hv[NP];
#pragma unroll
        for (int u = 0; u < NP; ++u) hv[u] = *(const pj_u32x4*)(h + u * rp + q + lh * V);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int col = colb + j * 16 + li, r = q + lh * V;
            const unsigned at = (unsigned)(col < p.N ? col : p.N - 1) * fcol + (unsigned)r * fr;
            union { T t[V]; pj_u32x4 v; } fv;
            if constexpr (F == PJ_F_RANKS) fv.v = pj_load_if<pj_u32x4>(r < p.rank, f + at);
            else
#pragma unroll
                for (int u = 0; u < V; ++u) { const T e = pj_entry(f, r + u < p.rank ? at + (unsigned)u * fr : 0u); fv.t[u] = r + u < p.rank ? e : (T)0; }
            PJFactorParts<DT>(fv.v).multiply(hv, t[j]);
            if constexpr (F != PJ_F_RANKS) asm volatile("" ::: "memory");       // one block's loads at a time: registers
        }
    }
    if constexpr (DT == VDB_F32)
#pragma unroll
        for (int j = 0; j < C; ++j) pj_settle(t[j]);
}

// All B blocks of 16 rows by one adapter.
template <int DT, int F, int B, int C>
__device__ __forceinline__ void pj_low_rank_all(const ProjRows& p, long long row, int colb, int a, pj_f32x4 (&acc)[B][C]) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, QS = 4 * V, NP = proj_parts(DT);
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int rp = proj_rank_pad(p.rank, DT);
    const unsigned fr = (unsigned)p.f_rank, fcol = (unsigned)p.f_col;
    const T* f = (const T*)p.f + (long long)a * p.f_adapter;
    const T* h = (const T*)p.h + (row + li) * (NP * rp);
#pragma unroll 1
    for (int q = 0; q < p.rank; q += QS) {
        const int r = q + lh * V;
        constexpr int BG = DT == VDB_F16 && B > 2 ? 2 : B;     // blocks of rows at a time: the parts of an fp16 factor take registers
        union { T t[V]; pj_u32x4 v; } fv[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int col = colb + j * 16 + li;
            const unsigned at = (unsigned)(col < p.N ? col : p.N - 1) * fcol + (unsigned)r * fr;
            if constexpr (F == PJ_F_RANKS) fv[j].v = pj_load_if<pj_u32x4>(r < p.rank, f + at);
            else
#pragma unroll
                for (int u = 0; u < V; ++u) { const T e = pj_entry(f, r + u < p.rank ? at + (unsigned)u * fr : 0u); fv[j].t[u] = r + u < p.rank ? e : (T)0; }
        }
#pragma unroll
        for (int g = 0; g < B; g += BG) {
            pj_u32x4 hv[BG][NP];
#pragma unroll
            for (int i = 0; i < BG; ++i)
#pragma unroll
                for (int u = 0; u < NP; ++u) hv[i][u] = *(const pj_u32x4*)(h + (long long)(g + i) * 16 * (NP * rp) + u * rp + q + lh * V);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const PJFactorParts<DT> fp(fv[j].v);
#pragma unroll
                for (int i = 0; i < BG; ++i) fp.multiply(hv[i], acc[g + i][j]);
            }
            if constexpr (BG < B) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Every lane its own row's adapter: t += h[m] f[a]^T for its four columns of each block, ranks q0, q0 + qs, ... in steps of V
template <int DT, int F, int C>
__device__ __forceinline__ void pj_low_rank_lanes(const ProjRows& p, long long mc, int colb, int a, int q0, int qs, pj_f32x4 (&t)[C]) {
    typedef typename PJ<DT>::T T;
    typedef T tx4 __attribute__((ext_vector_type(4)));
    constexpr int V = 16 / PJ<DT>::E, NP = proj_parts(DT);
    const int lh = (threadIdx.x & 63) >> 4;
    const int rp = proj_rank_pad(p.rank, DT);
    const unsigned fr = (unsigned)p.f_rank, fcol = (unsigned)p.f_col;
    const T* f = (const T*)p.f + (long long)(a < 0 ? 0 : a) * p.f_adapter;
    const T* h = (const T*)p.h + mc * (NP * rp);
#pragma unroll F == PJ_F_RANKS ? 2 : 1
    for (int q = q0; q < p.rank; q += qs) {
        float hq[V] = {};
#pragma unroll
        for (int u = NP - 1; u >= 0; --u) {
            union { T t[V]; pj_u32x4 v; } hv;
            hv.v = *(const pj_u32x4*)(h + u * rp + q);
#pragma unroll
            for (int k = 0; k < V; ++k) hq[k] += pj_to_f32<DT == VDB_F32 ? VDB_F32 : VDB_BF16>(hv.t[k]);
        }
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int col = colb + j * 16 + lh * 4;
            if constexpr (F == PJ_F_COLS) {
                const unsigned at = (unsigned)(col < p.N ? col : 0) * fcol + (unsigned)q * fr;
                tx4 fv[V];
#pragma unroll
                for (int k = 0; k < V; ++k) fv[k] = pj_load_if<tx4>(q + k < p.rank, f + at + (unsigned)k * fr);
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int n = 0; n < 4; ++n) t[j][n] = __builtin_fmaf(hq[k], pj_to_f32<DT>(fv[k][n]), t[j][n]);
            } else {
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const unsigned at = (unsigned)(col + n < p.N ? col + n : p.N - 1) * fcol + (unsigned)q * fr;
                    union { T t[V]; pj_u32x4 v; } fv;
                    if constexpr (F == PJ_F_RANKS) fv.v = *(const pj_u32x4*)(f + at);
                    else
#pragma unroll
                        for (int k = 0; k < V; ++k) fv.t[k] = q + k < p.rank ? f[at + (unsigned)k * fr] : (T)0;
#pragma unroll
                    for (int k = 0; k < V; ++k) t[j][n] = __builtin_fmaf(hq[k], pj_to_f32<DT>(fv.t[k]), t[j][n]);
                }
            }
            if constexpr (F != PJ_F_RANKS) asm volatile("" ::: "memory");
        }
    }
}

// Adapters of a wave's rows up to which all of its rows are multiplied by each of them: where two requests meet in a wave's 64 rows
// that waits twice, and 16 rows at a time five times (768 x 768 bf16, rank 16, 16 384 rows of 64 requests: forward pass
// 51.6 -> 47.5 us, the backward pass's kernel 43.6 -> 36.5; up to 8 adapters the same).
constexpr int PJ_EACH_ADAPTER = 4;

// All B blocks of 16 rows by each of their adapters in turn (ranks of one step); `v`: the adapter of row lane, -1: none.
template <int DT, int F, int B, int C>
__device__ __forceinline__ void pj_low_rank_each(const ProjRows& p, long long row, int colb, const int (&am)[B], int v, pj_f32x4 (&acc)[B][C]) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, NP = proj_parts(DT);
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4, r = lh * V;
    const int rp = proj_rank_pad(p.rank, DT);
    const unsigned fcol = (unsigned)p.f_col;
    pj_u32x4 hv[B][NP];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const long long m = row + i * 16 + li;
        const T* h = (const T*)p.h + (m < p.n ? m : p.n - 1) * (NP * rp) + r;
#pragma unroll
        for (int u = 0; u < NP; ++u) hv[i][u] = *(const pj_u32x4*)(h + u * rp);
    }
    for (unsigned long long left = __ballot(v >= 0); left;) {
        const int ad = __builtin_amdgcn_readlane(v, __builtin_ctzll(left));
        left &= ~__ballot(v == ad);
        const T* f = (const T*)p.f + (long long)ad * p.f_adapter;
        unsigned fr = (unsigned)p.f_rank;
        asm volatile("" : "+s"(fr));                           // addresses are not kept over the loop: registers
        union { T t[V]; pj_u32x4 v; } fv[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const int col = colb + j * 16 + li;
            const unsigned at = (unsigned)(col < p.N ? col : p.N - 1) * fcol + (unsigned)r * fr;
            if constexpr (F == PJ_F_RANKS) fv[j].v = pj_load_if<pj_u32x4>(r < p.rank, f + at);
            else
#pragma unroll
                for (int u = 0; u < V; ++u) { const T e = pj_entry(f, r + u < p.rank ? at + (unsigned)u * fr : 0u); fv[j].t[u] = r + u < p.rank ? e : (T)0; }
        }
        constexpr int CG = DT == VDB_F16 && C > 2 ? 2 : C;     // blocks of columns at a time: the parts of an fp16 factor take registers
#pragma unroll
        for (int c = 0; c < C; c += CG) {
#pragma unroll
            for (int i = 0; i < B; ++i) {
                if (__ballot(am[i] == ad) == 0) continue;
                pj_f32x4 t[CG] = {};
#pragma unroll
                for (int j = 0; j < CG; ++j) {
                    PJFactorParts<DT>(fv[c + j].v).multiply(hv[i], t[j]);
                    if constexpr (DT == VDB_F32) pj_settle(t[j]);
                }
#pragma unroll
                for (int j = 0; j < CG; ++j) if (am[i] == ad) acc[i][c + j] = t[j];
            }
            if constexpr (CG < C) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Adapters of B blocks of 16 rows (lane l: row + 16 i + l % 16); -1: none.
template <int B> __device__ __forceinline__ void pj_load_adapters(const ProjRows& p, long long row, int (&am)[B]) {
    const int li = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const long long m = row + i * 16 + li;
        am[i] = m < p.n ? p.row_adapter[m] : -1;
    }
}

// Is a value infinite or NaN in any lane?
template <int C> __device__ __forceinline__ float pj_largest(const pj_f32x4 (&t)[C], float z) {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
        for (int n = 0; n < 4; n += 2)                       // (a maximum that a NaN goes through)
            z = __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(t[j][n]), fabsf(t[j][n + 1])), z);
    return z;
}
template <int C> __device__ __forceinline__ bool pj_any_not_finite(const pj_f32x4 (&t)[C]) {
    return __ballot(!(pj_largest<C>(t, 0.f) < __builtin_huge_valf())) != 0;
}

// B blocks of 16 rows from `row`, C of 16 columns from `colb`; am: the rows' adapters.  `waves` > 1: that many waves share the block, and the sum of
// their accumulators is the term.
// Where parts are multiplied an infinity times the zero that another part holds is NaN, and infinite parts of both signs are too: what
// is not finite is worked out again lane by lane, from h put together, and is then what the formula gives.
template <int DT, int F, int B, int C>
__device__ __forceinline__ void pj_low_rank(const ProjRows& p, long long row, int colb, const int (&am)[B], pj_f32x4 (&acc)[B][C],
                                            int waves = 1, int wave = 0) {
    constexpr int V = 16 / PJ<DT>::E;
    const int li = threadIdx.x & 15;
    bool done = false;
    if constexpr (B > 1 && F != PJ_F_ANY) {
        // one adapter for all rows, as long requests have it: its factor is loaded once for all of them
        const int a0 = __builtin_amdgcn_readlane(am[0], 0);
        bool same = a0 >= 0;
#pragma unroll
        for (int i = 0; i < B; ++i) same = same && am[i] == a0;
        if (__ballot(!same) == 0) {
            pj_low_rank_all<DT, F, B, C>(p, row, colb, a0, acc);
            done = true;
        } else if (p.rank <= 4 * V) {
            // a few adapters, as where requests meet
            int v = -1, met = 0;
#pragma unroll
            for (int i = 0; i < B; ++i) if ((threadIdx.x & 63) >> 4 == i) v = am[i];
            for (unsigned long long left = __ballot(v >= 0); left; ++met) left &= ~__ballot(v == __builtin_amdgcn_readlane(v, __builtin_ctzll(left)));
            if (met <= PJ_EACH_ADAPTER) {
                pj_low_rank_each<DT, F, B, C>(p, row, colb, am, v, acc);
                done = true;
            }
        }
        if (done) {
            float z = 0.f;
            if constexpr (DT != VDB_F32)
#pragma unroll
                for (int i = 0; i < B; ++i) z = pj_largest<C>(acc[i], z);
            if (__ballot(!(z < __builtin_huge_valf())) == 0) return;
        }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const long long m = row + i * 16 + li, mc = m < p.n ? m : p.n - 1;
        const unsigned rows = (unsigned)__ballot(am[i] >= 0) & 0xffffu;
        if (!rows) continue;
        pj_f32x4 t[C] = {};
        bool lanes = false;                                  // (of a value that is not finite: alone)
        if (!done) {
            int met = 0;                                     // adapters in these 16 rows
            for (unsigned left = rows; left; ++met) left &= ~(unsigned)__ballot(am[i] == __builtin_amdgcn_readlane(am[i], __builtin_ctz(left)));
            if (met <= (p.rank < 32 ? 2 : p.rank / 12)) {
                int turn = 0;
                for (unsigned left = rows; left;) {
                    const int ad = __builtin_amdgcn_readlane(am[i], __builtin_ctz(left));
                    left &= ~(unsigned)__ballot(am[i] == ad);
                    const bool mine = turn == wave;
                    turn = turn + 1 == waves ? 0 : turn + 1;
                    if (!mine) continue;
                    pj_f32x4 u[C] = {};
                    pj_low_rank_block<DT, F, C>(p, mc, colb, ad, u);
#pragma unroll
                    for (int j = 0; j < C; ++j) if (am[i] == ad) t[j] = u[j];
                }
            } else lanes = true;
        } else {
#pragma unroll
            for (int j = 0; j < C; ++j) t[j] = acc[i][j];
        }
        if (lanes || (DT != VDB_F32 && pj_any_not_finite<C>(t))) {
            pj_f32x4 u[C] = {};
            pj_low_rank_lanes<DT, F, C>(p, mc, colb, am[i], lanes ? wave * V : 0, lanes ? waves * V : V, u);
#pragma unroll
            for (int j = 0; j < C; ++j)
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (lanes || !(fabsf(t[j][n]) < __builtin_huge_valf())) t[j][n] = u[j][n];
        }
        if (am[i] >= 0) {
#pragma unroll
            for (int j = 0; j < C; ++j) acc[i][j] = t[j];
        }
    }
}

struct PJRowsArgs {
    ProjRows p;
    int col_tiles;
    bool vec_out;                // y can be written in aligned pieces of 16 bytes
};

// Stores a wave's block of 16 B rows by 16 C columns at y as whole cache lines.  A lane holds four columns of a row: stored as they
// are, a wave's store would be sixteen pieces of 32 or 64 bytes.  Turned in `lds` (BYTES of it, this wave's own) it is four or
// eight rows of 64 outputs (65 536 x 768 rows out: 112 -> 99 us bf16, 167 -> 157 us fp32), which need not stay in the L2 that the
// operands of other tiles live in (fp32: 157 -> 142 us).
template <int ODT, int B, int C, int BYTES>
__device__ __forceinline__ void pj_store_turned(typename PJ<ODT>::T* y, long long ldy, char* lds, const pj_f32x4 (&acc)[B][C]) {
    constexpr int LINE = C * 16 * PJ<ODT>::E + 16, LPR = (LINE - 16) / 16, RPI = 64 / LPR;      // lanes to a row, rows to a store
    constexpr int BI = B * 16 * LINE <= BYTES ? B : B * 8 * LINE <= BYTES ? B / 2 : B / 4;      // blocks of 16 rows that fit
    static_assert(BI * 16 * LINE <= BYTES, "a wave's part of the ring");
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
#pragma unroll
    for (int h = 0; h < B; h += BI) {
#pragma unroll
        for (int i = 0; i < BI; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) pj_store4<ODT>(lds + (i * 16 + li) * LINE + (j * 16 + lh * 4) * PJ<ODT>::E, 0, acc[h + i][j], 4);
#pragma unroll
        for (int r = 0; r < BI * 16; r += RPI) {
            const pj_u32x4 v = *(const pj_u32x4*)(lds + (r + lane / LPR) * LINE + lane % LPR * 16);
            __builtin_nontemporal_store(v, (pj_u32x4*)((char*)(y + (h * 16 + r + lane / LPR) * ldy) + lane % LPR * 16));
        }
    }
}

// The tile of `tm` rows that this workgroup works on: rows [max(row0, first), min(row0 + tm, row1)); false: none.
template <bool ADAPT>
__device__ __forceinline__ bool pj_place(const ProjRows& p, int tm, int col_tiles, int& seg, long long& row0, long long& first,
                                         long long& row1, int& col) {
    if constexpr (!ADAPT) return pj_find_tile(p.offsets, p.segments, p.n, tm, col_tiles, blockIdx.x, seg, row0, row1, col);
    else {
        // one matrix for all rows: tiles over the rows from the first segment's start to the last one's end
        first = pj_clamp(p.offsets[0], p.n);
        row1 = pj_clamp(p.offsets[p.segments], p.n);
        if (row1 <= first) return false;
        const long long t0 = first / tm, tiles = (row1 + tm - 1) / tm - t0;
        const long long all = tiles * col_tiles, run = (all + 7) / 8, idx = blockIdx.x >> 3;
        const long long id = (long long)(blockIdx.x & 7) * run + idx;
        if (idx >= run || id >= all) return false;
        col = (int)(id % col_tiles);
        row0 = (t0 + id / col_tiles) * tm;
        return true;
    }
}

template <int DT, int ODT, bool NK, bool VEC, bool ADAPT, int F, int R>
__global__ void __launch_bounds__(PJ_THREADS, 2)
proj_rows_kernel(PJRowsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char pj_lds[];
    typedef typename PJ<DT>::T T;
    constexpr int B = R / 32;
    const ProjRows& p = a.p;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    long long row0, row1, first = 0;         // rows of this tile: [max(row0, first), row1)
    int seg = 0, col;
    if (!pj_place<ADAPT>(p, R, a.col_tiles, seg, row0, first, row1, col)) return;
    const int col0 = col * R;
    pj_f32x4 acc[B][B] = {};
    PJProduct<DT, false, NK, VEC, R> prod;
    prod.om.init((const T*)p.x, p.ldx, row0, row1, p.K);
    prod.on.init((const T*)p.w + (long long)seg * p.w_group, p.ldw, col0, p.N, p.K);
    int am[B] = {};
    if constexpr (ADAPT) pj_load_adapters<B>(p, row0 + wm * (R / 2), am);        // before the stages' loads, which return in order
    prod.begin(p.K, pj_lds);
    if constexpr (ADAPT) pj_low_rank<DT, F, B, B>(p, row0 + wm * (R / 2), col0 + wn * (R / 2), am, acc);
    prod.run(pj_lds, wm, wn, acc);
    if (R == 128 && a.vec_out && row0 >= first && row0 + R <= row1 && col0 + R <= p.N) {
        __syncthreads();                                     // the ring is free: each wave has a quarter of it
        pj_store_turned<ODT, B, B, PJRing<R>::BYTES / 4>((typename PJ<ODT>::T*)p.y + (row0 + wm * (R / 2)) * p.ldy + col0 + wn * (R / 2), p.ldy,
                                                         pj_lds + wave * (PJRing<R>::BYTES / 4), acc);
        return;
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const long long m = row0 + wm * (R / 2) + i * 16 + li;
        if (m >= row1 || m < first) continue;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int c = col0 + wn * (R / 2) + j * 16 + lh * 4;
            if (c < p.N) pj_store4<ODT>(p.y, m * p.ldy + c, acc[i][j], p.N - c);
        }
    }
}

// A few rows: 16 rows x 16 columns per workgroup, so that the matrix is read by many CUs; the four waves take every fourth step
// of the contracted axis, straight from memory into fragments with all loads of U steps ahead of the products, and add up
// through LDS in wave order.  The requests of the low-rank term are divided among the waves as well.
template <int DT, int ODT, bool NK, bool VEC, bool ADAPT, int F>
__global__ void __launch_bounds__(PJ_THREADS)
proj_few_kernel(PJRowsArgs a) {
    typedef typename PJ<DT>::T T;
    constexpr int V = 16 / PJ<DT>::E, KS = 4 * V, U = 4;
    __shared__ pj_f32x4 part[3][64];
    const ProjRows& p = a.p;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    long long row0, row1, first = 0;
    int seg = 0, col;
    if constexpr (ADAPT) {
        col = blockIdx.x % a.col_tiles;
        row0 = (long long)(blockIdx.x / a.col_tiles) * 16;
        first = pj_clamp(p.offsets[0], p.n); row1 = pj_clamp(p.offsets[p.segments], p.n);
        if (row0 >= row1 || row0 + 16 <= first) return;
    } else {
        if (!pj_find_tile(p.offsets, p.segments, p.n, 16, a.col_tiles, blockIdx.x, seg, row0, row1, col)) return;
    }
    const long long m = row0 + li;
    const int c = col * 16 + li;
    const T* x = (const T*)p.x + (m < row1 ? m : row1 - 1) * p.ldx;
    const T* w = (const T*)p.w + (long long)seg * p.w_group + (NK ? (c < p.N ? c : p.N - 1) : (long long)(c < p.N ? c : p.N - 1) * p.ldw);
    pj_f32x4 acc[1][1] = {};
    if constexpr (ADAPT) {
        int am[1];
        pj_load_adapters<1>(p, row0, am);
        pj_low_rank<DT, F, 1, 1>(p, row0, col * 16, am, acc, 4, wave);
    }
    for (int k0 = wave * KS; k0 < p.K; k0 += U * 4 * KS) {
        union frag { T t[V]; pj_u32x4 v; } xa[U], wa[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * 4 * KS + lh * V;
            if constexpr (VEC) xa[u].v = pj_load_if<pj_u32x4>(k < p.K, x + k);
            else xa[u].v = pj_piece<T>(x + k, p.K - k, p.K >= V);
            if constexpr (VEC && !NK) wa[u].v = pj_load_if<pj_u32x4>(k < p.K, w + k);
            else if constexpr (!NK) wa[u].v = pj_piece<T>(w + k, p.K - k, p.K >= V);
            else
#pragma unroll
                for (int j = 0; j < V; ++j) wa[u].t[j] = k + j < p.K ? w[(k + j) * p.ldw] : (T)0;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) acc[0][0] = pj_mfma<DT>(wa[u].v, xa[u].v, acc[0][0]);
    }
    if (wave) part[wave - 1][lane] = acc[0][0];
    __syncthreads();
    if (wave) return;
    pj_f32x4 v = acc[0][0];
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += part[i][lane][j];
    const int cs = col * 16 + lh * 4;
    if (m < row1 && m >= first && cs < p.N) pj_store4<ODT>(p.y, m * p.ldy + cs, v, p.N - cs);
}

struct PJWeightsArgs {
    ProjWeights p;
    int m_tiles, n_tiles;
};

// Segment, output tile and rows [b, e) of this workgroup; item: number of the chunk whose partial sums it leaves, -1: the segment is
// not split.
template <bool SPLIT>
__device__ __forceinline__ bool pj_weights_place(const PJWeightsArgs& a, int& seg, int& tile, long long& b, long long& e, long long& item) {
    const ProjWeights& p = a.p;
    item = -1;
    if constexpr (SPLIT) {
        if (!pj_find_tile(p.offsets, p.segments, p.n, p.chunk, a.m_tiles * a.n_tiles, blockIdx.x, seg, b, e, tile, item)) return false;
        if (item >= p.n / p.chunk + p.segments) return false;       // offsets that decrease: more chunks than the workspace holds
        if (b == pj_clamp(p.offsets[seg], p.n) && e - b <= p.chunk) item = -1;
        e = e - b < p.chunk ? e : b + p.chunk;
    } else {
        seg = blockIdx.x / (a.m_tiles * a.n_tiles);
        tile = blockIdx.x % (a.m_tiles * a.n_tiles);
        if (seg >= p.segments) return false;
        b = pj_clamp(p.offsets[seg], p.n);
        e = pj_clamp(p.offsets[seg + 1], p.n);
    }
    return true;
}

// dw of one segment, or of one chunk of its rows (SPLIT: a segment of more than one chunk leaves fp32 partial sums, which
// proj_weights_sum_kernel adds up in the order of the chunks).
template <int DT, int ODT, bool VEC, bool SPLIT, int R>
__global__ void __launch_bounds__(PJ_THREADS, 2)
proj_weights_kernel(PJWeightsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char pj_lds[];
    typedef typename PJ<DT>::T T;
    constexpr int B = R / 32;
    const ProjWeights& p = a.p;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    int seg, tile;
    long long b, e, item;
    if (!pj_weights_place<SPLIT>(a, seg, tile, b, e, item)) return;
    const int m0 = tile / a.n_tiles * R, n0 = tile % a.n_tiles * R;
    pj_f32x4 acc[B][B] = {};
    PJProduct<DT, true, true, VEC, R> prod;
    prod.om.init((const T*)p.dy + b * p.lddy, p.lddy, m0, p.M, e - b);
    prod.on.init((const T*)p.x + b * p.ldx, p.ldx, n0, p.N, e - b);
    prod.begin(e > b ? e - b : 0, pj_lds);
    prod.run(pj_lds, wm, wn, acc);
#pragma unroll
    for (int i = 0; i < B; ++i) {
        const int m = m0 + wm * (R / 2) + i * 16 + li;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int c = n0 + wn * (R / 2) + j * 16 + lh * 4;
            if (c >= p.N) continue;
            if (SPLIT && item >= 0) pj_store4<VDB_F32>(p.partial, (item * p.M + m) * p.N + c, acc[i][j], p.N - c);
            else pj_store4<ODT>(p.dw, ((long long)seg * p.M + m) * p.N + c, acc[i][j], p.N - c);
        }
    }
}

// The same by wide tiles; M and N are multiples of 8.
template <int DT, int ODT, bool SPLIT>
__global__ void __launch_bounds__(PJ_THREADS, 2)
proj_wide_weights_kernel(PJWeightsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char pj_lds[];
    typedef typename PJ<DT>::T T;
    constexpr int BM = 8, BN = 4;
    const ProjWeights& p = a.p;
    const int lane = threadIdx.x & 63, li = lane & 15, lh = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    int seg, tile;
    long long b, e, item;
    if (!pj_weights_place<SPLIT>(a, seg, tile, b, e, item)) return;
    const int m0 = tile / a.n_tiles * PJ_WIDE_M, n0 = tile % a.n_tiles * PJ_WIDE_N;
    pj_f32x4 acc[BM][BN] = {};
    PJWide<DT> prod;
    prod.om.init((const T*)p.dy + b * p.lddy + m0, p.lddy, p.M - m0);
    prod.on.init((const T*)p.x + b * p.ldx + n0, p.ldx, p.N - n0);
    prod.run(e > b ? e - b : 0, pj_lds, wm, wn, acc);
#pragma unroll
    for (int i = 0; i < BM; ++i) {
        const int m = m0 + wm * 128 + i * 16 + li;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < BN; ++j) {
            const int c = n0 + wn * 64 + j * 16 + lh * 4;
            if (c >= p.N) continue;
            if (SPLIT && item >= 0) pj_store4<VDB_F32>(p.partial, (item * p.M + m) * p.N + c, acc[i][j], p.N - c);
            else pj_store4<ODT>(p.dw, ((long long)seg * p.M + m) * p.N + c, acc[i][j], p.N - c);
        }
    }
}

// ------------------------------------------------------------------------------------------- launches of one type
static inline bool pj_aligned(const void* ptr, long long ld, int esize, int bytes) {
    return (uintptr_t)ptr % bytes == 0 && ld * esize % bytes == 0;
}

template <typename K, typename A>
static hipError_t pj_launch(K kernel, dim3 grid, size_t lds, const A& args, hipStream_t st) {
    hipLaunchKernelGGL(kernel, grid, dim3(PJ_THREADS), lds, st, args);
    return hipGetLastError();
}

// 64 x 64 tiles where 128 x 128 ones would leave CUs without work (bf16, 768 x 768, 8 groups: 8192 rows, 408 tiles of 128 x 128, 18 us
// and 30 by 64 x 64).
static inline bool pj_small_tiles(long long tiles128) { return tiles128 < 256; }

template <int DT, int ODT, int R>
static hipError_t pj_rows_sized(const ProjRows& p, bool vec, hipStream_t st) {
    PJRowsArgs a;
    a.p = p;
    a.col_tiles = (p.N + R - 1) / R;
    a.vec_out = pj_aligned(p.y, p.ldy, PJ<ODT>::E, 16);
    const dim3 grid((unsigned)proj_rows_grid(p, R));
    const size_t lds = vec ? PJRing<R>::BYTES : PJRing<R>::HALVES;
    const bool fv = proj_factor_vectors(p);
#define PJ_ROWS(NK, VEC)                                                                              \
    (!p.row_adapter ? pj_launch(proj_rows_kernel<DT, ODT, NK, VEC, false, PJ_F_ANY, R>, grid, lds, a, st)     \
     : fv   ? pj_launch(proj_rows_kernel<DT, ODT, NK, VEC, true, NK ? PJ_F_COLS : PJ_F_RANKS, R>, grid, lds, a, st) \
            : pj_launch(proj_rows_kernel<DT, ODT, NK, VEC, true, PJ_F_ANY, R>, grid, lds, a, st))
    if constexpr (R == 128) {
        // (a factor that cannot be read in vectors would spill here)
        if constexpr (DT != VDB_F32) if (!vec) return pj_launch(proj_rows_kernel<DT, ODT, false, false, false, PJ_F_ANY, R>, grid, lds, a, st);
#define PJ_BIG(NK)                                                                                                        \
    (p.row_adapter ? pj_launch(proj_rows_kernel<DT, ODT, NK, true, true, NK ? PJ_F_COLS : PJ_F_RANKS, R>, grid, lds, a, st)       \
           : pj_launch(proj_rows_kernel<DT, ODT, NK, true, false, PJ_F_ANY, R>, grid, lds, a, st))
        return p.w_by_k ? PJ_BIG(true) : PJ_BIG(false);
#undef PJ_BIG
    } else {
        if (p.w_by_k) return vec ? PJ_ROWS(true, true) : PJ_ROWS(true, false);
        return vec ? PJ_ROWS(false, true) : PJ_ROWS(false, false);
    }
#undef PJ_ROWS
}

template <int DT, int ODT>
static hipError_t pj_few(const ProjRows& p, bool vec, hipStream_t st) {
    PJRowsArgs a;
    a.p = p;
    a.col_tiles = (p.N + 15) / 16;
    a.vec_out = false;
    const dim3 grid((unsigned)proj_rows_grid(p, 16));
    const bool fv = proj_factor_vectors(p);
#define PJ_FEW(NK, VEC)                                                                          \
    (!p.row_adapter ? pj_launch(proj_few_kernel<DT, ODT, NK, VEC, false, PJ_F_ANY>, grid, 0, a, st)      \
     : fv   ? pj_launch(proj_few_kernel<DT, ODT, NK, VEC, true, NK ? PJ_F_COLS : PJ_F_RANKS>, grid, 0, a, st) \
            : pj_launch(proj_few_kernel<DT, ODT, NK, VEC, true, PJ_F_ANY>, grid, 0, a, st))
    if (p.w_by_k) return vec ? PJ_FEW(true, true) : PJ_FEW(true, false);
    return vec ? PJ_FEW(false, true) : PJ_FEW(false, false);
#undef PJ_FEW
}

// Largest number of 64 x 64 tiles that is left to the kernel for a few rows (one launch, 768 x 768 bf16: 256 rows, 48 tiles, 7.9 us
// by 16 x 16 and 8.2 by 64 x 64; 512 rows 12.4 and 8.4; 384 x 384 fp32: 512 rows, 48 tiles, 9.7 and 12.9; 1024 rows, 96 tiles, 14.3
// and 13.1).
constexpr long long PJ_FEW_TILES = 64;

// fp32 takes 32 x 32 tiles where 64 x 64 would leave half of the CUs without one (384 x 384, in a graph: 1024 rows, 99 tiles, 10.0 us
// by 32 x 32 and 13.1 by 64 x 64; 1000 rows of 515 x 387, 126 tiles, 13.4 and 19.7; 2048 rows, 195 tiles, 18.3 and 13.5; 1024 x 768,
// 192 tiles, 30.4 and 28.2).
constexpr long long PJ_F32_TILES = 128;

template <int DT, int ODT>
static hipError_t pj_rows(const ProjRows& p, hipStream_t st) {
    constexpr int E = PJ<DT>::E, V = 16 / E;
    const bool vec = pj_aligned(p.x, p.ldx, E, 16) && pj_aligned(p.w, p.ldw, E, 16) && p.w_group % V == 0 &&
                     p.K % V == 0 && (!p.w_by_k || p.N % V == 0);
    const long long tiles = ((p.n + 127) / 128 + (p.row_adapter ? 0 : p.segments / 2)) * ((p.N + 127) / 128);
    const long long tiles64 = ((p.n + 63) / 64) * ((p.N + 63) / 64);
    if (tiles64 <= PJ_FEW_TILES) return pj_few<DT, ODT>(p, vec, st);
    if constexpr (DT == VDB_F32)
        if (((p.n + 63) / 64 + (p.row_adapter ? 0 : p.segments / 2)) * ((p.N + 63) / 64) < PJ_F32_TILES) return pj_rows_sized<DT, ODT, 32>(p, vec, st);
    // Through registers 128 x 128 tiles pay later, and not in fp32 (1025 x 769 bf16, 20 000 rows: 106 us by 64 x 64 and 81 by 128 x 128;
    // 515 x 387 fp16, 8000 rows, 264 tiles, 21.6 and 23.5, 12 000 rows, 388 tiles, 28.0 and 25.2, 60 000 rows 105 and 85; fp32, 20 000
    // rows 110 and 129); down the columns of the matrix they would spill.
    const bool big = vec ? !pj_small_tiles(tiles) && (!p.row_adapter || proj_factor_vectors(p))
                         : DT != VDB_F32 && !p.row_adapter && !p.w_by_k && tiles >= 384;
    return big ? pj_rows_sized<DT, ODT, 128>(p, vec, st) : pj_rows_sized<DT, ODT, 64>(p, vec, st);
}

template <int DT, int ODT, int R>
static hipError_t pj_weights_sized(const ProjWeights& p, bool vec, hipStream_t st) {
    PJWeightsArgs a;
    a.p = p;
    a.m_tiles = (p.M + R - 1) / R;
    a.n_tiles = (p.N + R - 1) / R;
    const dim3 grid((unsigned)proj_weights_grid(p, R, R));
    const size_t lds = vec ? PJRing<R>::BYTES : PJRing<R>::HALVES;
    if (p.chunk > 0) {
        if constexpr (R == 128) return pj_launch(proj_weights_kernel<DT, ODT, true, true, R>, grid, lds, a, st);
        else return vec ? pj_launch(proj_weights_kernel<DT, ODT, true, true, R>, grid, lds, a, st)
                        : pj_launch(proj_weights_kernel<DT, ODT, false, true, R>, grid, lds, a, st);
    }
    if constexpr (R == 128) return pj_launch(proj_weights_kernel<DT, ODT, true, false, R>, grid, lds, a, st);
    else return vec ? pj_launch(proj_weights_kernel<DT, ODT, true, false, R>, grid, lds, a, st)
                    : pj_launch(proj_weights_kernel<DT, ODT, false, false, R>, grid, lds, a, st);
}

template <int DT, int ODT>
static hipError_t pj_weights(const ProjWeights& p, hipStream_t st) {
    constexpr int E = PJ<DT>::E, V = 16 / E;
    const bool vec = pj_aligned(p.dy, p.lddy, E, 16) && pj_aligned(p.x, p.ldx, E, 16) && p.M % V == 0 && p.N % V == 0;
    if constexpr (DT != VDB_F32)
        if (vec && p.tile == 128 && pj_offsets_fit(32, p.lddy, 2) && pj_offsets_fit(32, p.ldx, 2)) {
            PJWeightsArgs a;
            a.p = p;
            a.m_tiles = (p.M + PJ_WIDE_M - 1) / PJ_WIDE_M;
            a.n_tiles = (p.N + PJ_WIDE_N - 1) / PJ_WIDE_N;
            const dim3 grid((unsigned)proj_weights_grid(p, PJ_WIDE_M, PJ_WIDE_N));
            auto go = [&](auto kernel) {
                const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, PJ_WIDE_BYTES);
                return e == hipSuccess ? pj_launch(kernel, grid, PJ_WIDE_BYTES, a, st) : e;
            };
            return p.chunk > 0 ? go(proj_wide_weights_kernel<DT, ODT, true>) : go(proj_wide_weights_kernel<DT, ODT, false>);
        }
    return vec && p.tile == 128 ? pj_weights_sized<DT, ODT, 128>(p, vec, st) : pj_weights_sized<DT, ODT, 64>(p, vec, st);
}

// A type's rows and weights products; defined in kernels_project_{f32,bf16,f16}.hip.
#define PJ_DEFINE(NAME, DT)                                                                            \
    hipError_t launch_proj_rows_##NAME(const ProjRows& p, hipStream_t st) {                            \
        return p.out_dtype == VDB_F32 ? pj_rows<DT, VDB_F32>(p, st) : pj_rows<DT, DT>(p, st);          \
    }                                                                                                  \
    hipError_t launch_proj_weights_##NAME(const ProjWeights& p, hipStream_t st) {                      \
        return p.out_dtype == VDB_F32 ? pj_weights<DT, VDB_F32>(p, st) : pj_weights<DT, DT>(p, st);    \
    }

}  // namespace vdb
