// Newton-Schulz orthogonalisation of a list of matrices, and the Muon update built on it (gfx950).
//
//   X = U / max(|U|_F, eps);  steps times:  A = X X^T,  X <- (a I + b A + c A^2) X      (U with more rows than columns: of U^T)
//
// MATHEMATICS.  With Q = a I + b A + c A^2 (symmetric, a polynomial of A) the next step's Gram matrix is A' = Q A Q: it need not be formed
// from X again.  So a HOP of h steps runs on the small side only (m <= n):
//     A = X X^T;   Q_i = a I + b A_i + c A_i^2,   A_{i+1} = (A_i Q_i) Q_i,   R_i = Q_i R_{i-1};   X <- R_h X
// at 3 m^2 n + (4 h - 3) m^3 operations (symmetric products: the lower half only, mirrored) instead of h (3 m^2 n + m^3).  An extra step in
// a hop multiplies the relative error of the smallest eigenvalues by a^2 ~ 12 (they grow by that, the rounding error of A does not shrink):
// hop_cap() says how many a type allows, plan_hops() takes the cheapest schedule.
//
// ARITHMETIC.  fp32 accuracy from the fp16 matrix cores: an operand is kept as two fp16 planes, x 2^k = h + l (h = fp16(x 2^k), l the rest:
// 22 to 24 bits), a product is h h + h l + l h accumulated in fp32 -- three products at the fp16 rate (2.5 PFLOP/s) against one at the
// fp32 rate (0.16).  The power of two puts the largest entry below 2^15, so l keeps its bits down to entries of 2^-24 of that.
// What the small singular values suffer from is an error of Q that is not one of A (they grow by up to a^5 = 485 meanwhile): b A and c A^2 are
// formed of the same planes, and in fp32 below m = 128, where sums of so few terms hide nothing, A^2 takes l l too (400 shapes up to 300 x 1000
// in emulation, largest error: 2.8e-6 of the exact result with b A from the accumulators, 2.1e-6 from the planes, 1.3e-6 with l l).  150 shapes
// of m < 128 measured: rms 0.76e-6, listed with a 2048 x 2048 one 1.07e-6 (larger tiles: a sum is one chain, not four), fp32 products 1.49e-6.
//
// All matrices of a call (up to 12 at a time) go through each stage in ONE launch (problem list in the kernel arguments): five steps are 17 to
// 19 launches whatever their number.  Operand image: row r = chunks of 32 k, each [h: 32 fp16][l: 32 fp16] (128 bytes); columns up to the
// chunk's end are zero, rows end where the matrix does (loads clamp the row).  X is kept in both orientations (X for the Gram product, X^T for
// the product with R: both contract over the last axis).
#include "common.h"

#include <math.h>

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int MAX_MAT = 12;            // matrices of one pass through the stages
constexpr int MAX_PROB = 2 * MAX_MAT;  // products of one launch (a hop's step has two independent ones per matrix)
constexpr int MAX_NORM_BLOCKS = 2048;   // partial sums of squares per matrix

struct Prob {                // out = (alpha acc + cb C + ca I), acc = L R^T over kc chunks of 32
    const _Float16* L;
    const _Float16* R;
    const _Float16* C;       // planes [M][oc] or NULL (symmetric)
    _Float16* out;           // planes [M][oc] or NULL
    _Float16* outT;          // planes [N][otc] or NULL
    void* fin;               // [M, N] of the result type, or [N, M] (fin_t), or NULL
    const float* rdev;       // alpha is multiplied by rdev^rpow
    int M, N, kc, oc, otc, rpow, sym, tiles_n, fin_t;
    float alpha, cb, ca, so, fmul, fdecay;
    int tiles, seg;          // tiles of the result; chunks of a segment of K (kc: not cut)
    int ll;                  // the product of the l planes too
};
// A launch's work items, one a workgroup: the first `whole` tiles uncut, then the rest in segments of K.  Items are ordered by segment, then by
// tile: neighbours share operand rows, not just the tile.  equal: all problems have one K, the rest is `rest` tiles x segments; else every
// problem has segments of its own.
struct Probs {
    int tile0[MAX_PROB], item0[MAX_PROB];      // first tile and first item of every problem; behind the last: INT_MAX
    int tiles, items, whole, rest, equal;
    int fin_dtype, fin_update;    // fin_update: fin = fdecay * fin - fmul * value
    float* part;
    int count;
    Prob p[MAX_PROB];
};

// The entry of `starts` (ascending, INT_MAX behind the last) that `at` belongs to: one load by all lanes and a ballot.  The arguments come
// from host memory, ~1 us a dependent read: a scalar search would pay that per entry.
template <int N> __device__ __forceinline__ int which(const int (&starts)[N], int at)
{
    static_assert(N <= 64, "one entry a lane");
    const int lane = threadIdx.x & 63;
    const int v = lane < N ? starts[lane] : 0x7fffffff;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(v <= at)) - 1);
}
static_assert(sizeof(Probs) <= 3584, "travels in the kernel arguments");

__host__ __device__ inline int chunks(int64_t k) { return (int)((k + 31) / 32); }

// 16 bytes a lane straight into LDS: from base + off (base the same for the wave) to the LDS address dst + 16 * lane; waited for by
// wait_vm in front of a barrier
__device__ __forceinline__ void to_lds16(const char* base, unsigned off, unsigned dst)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(dst) : "memory");
}
template <int N> __device__ __forceinline__ void wait_vm()
{
    static_assert(N >= 0 && N < 64, "vmcnt is a six-bit counter");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ void store_fin(void* p, int dtype, size_t i, float v)
{
    if (dtype == MP_DTYPE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == MP_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
    else static_cast<__bf16*>(p)[i] = (__bf16)v;
}
__device__ __forceinline__ float load_any(const void* p, int dtype, size_t i)
{
    if (dtype == MP_DTYPE_F32) return static_cast<const float*>(p)[i];
    if (dtype == MP_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
    return (float)static_cast<const __bf16*>(p)[i];
}

// four consecutive elements at any element address, zeros from `left` on
__device__ __forceinline__ void load4(const void* p, int dtype, size_t i, int64_t left, float (&v)[4])
{
    if (left >= 4) {
        if (dtype == MP_DTYPE_F32) __builtin_memcpy(v, static_cast<const float*>(p) + i, 16);
        else if (dtype == MP_DTYPE_F16) {
            _Float16 t[4];
            __builtin_memcpy(t, static_cast<const _Float16*>(p) + i, 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
        } else {
            __bf16 t[4];
            __builtin_memcpy(t, static_cast<const __bf16*>(p) + i, 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
        }
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < left ? load_any(p, dtype, i + e) : 0.0f;
}

// Tiles of a symmetric product: row ti of tiles holds the tj with any element on or below the diagonal, tj < (ti + 1) TM / TN (the last row:
// as many as there are columns).  Row-major order.
__host__ __device__ inline int tiles_of(int M, int N, int sym, int TM, int TN)
{
    const int tm = (M + TM - 1) / TM, tn = (N + TN - 1) / TN, q = TM / TN;
    if (!sym) return tm * tn;
    const int last = q * tm < tn ? q * tm : tn;
    return q * (tm * (tm - 1) / 2) + last;
}

__device__ __forceinline__ void tile_at(const Prob& p, int tile, int TM, int TN, int& m0, int& n0)
{
    int ti, tj;
    if (p.sym) {
        const int q = TM / TN;
        const int f = tile / q;                        // q (ti + 1) ti / 2 + tj = tile
        ti = (int)((sqrtf(8.0f * (float)f + 1.0f) - 1.0f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= f) ++ti;
        while (ti * (ti + 1) / 2 > f) --ti;
        tj = tile - q * (ti * (ti + 1) / 2);
    } else {
        ti = tile / p.tiles_n;
        tj = tile % p.tiles_n;
    }
    m0 = ti * TM;
    n0 = tj * TN;
}

__device__ __forceinline__ void put_planes(_Float16* img, int row, int nchunk, int col, const float (&v)[4])
{
    half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = (_Float16)v[e];
        l[e] = (_Float16)(v[e] - (float)h[e]);
    }
    _Float16* q = img + ((size_t)row * nchunk + (col >> 5)) * 64 + (col & 31);
    *reinterpret_cast<half4*>(q) = h;
    *reinterpret_cast<half4*>(q + 32) = l;
}

__device__ __forceinline__ float alpha_of(const Prob& p)
{
    if (!p.rpow) return p.alpha;
    const float r = *p.rdev;
    return p.alpha * (p.rpow == 2 ? r * r : r);
}

// up to eight consecutive elements of the result, at any element address
__device__ __forceinline__ void put_fin(const Probs& a, const Prob& p, size_t at, int left, float (&v)[8])
{
    if (a.fin_update) {
        float w[8];
        load4(p.fin, a.fin_dtype, at, left, reinterpret_cast<float(&)[4]>(w[0]));
        load4(p.fin, a.fin_dtype, at + 4, left - 4, reinterpret_cast<float(&)[4]>(w[4]));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = p.fdecay * w[e] - p.fmul * v[e];
    }
    if (left >= 8) {
        if (a.fin_dtype == MP_DTYPE_F32) __builtin_memcpy(static_cast<float*>(p.fin) + at, v, 32);
        else if (a.fin_dtype == MP_DTYPE_F16) {
            _Float16 h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
            __builtin_memcpy(static_cast<_Float16*>(p.fin) + at, h, 16);
        } else {
            __bf16 h[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = (__bf16)v[e];
            __builtin_memcpy(static_cast<__bf16*>(p.fin) + at, h, 16);
        }
    } else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < left) store_fin(p.fin, a.fin_dtype, at + e, v[e]);
}

typedef unsigned uint4v __attribute__((ext_vector_type(4)));

// fp16 planes of x packed into 32 bits: h below, l above
__device__ __forceinline__ unsigned planes_of(float x)
{
    const _Float16 h = (_Float16)x, l = (_Float16)(x - (float)h);
    unsigned short hb, lb;
    __builtin_memcpy(&hb, &h, 2);
    __builtin_memcpy(&lb, &l, 2);
    return (unsigned)hb | ((unsigned)lb << 16);
}
// eight packed elements to the h and l runs of an image (16 bytes each)
__device__ __forceinline__ void put_packed(_Float16* img, int row, int nchunk, int col, const unsigned (&w)[8])
{
    _Float16* o = img + ((size_t)row * nchunk + (col >> 5)) * 64 + (col & 31);
    uint4v h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x05040100);
        l[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302);
    }
    *reinterpret_cast<uint4v*>(o) = h;
    *reinterpret_cast<uint4v*>(o + 32) = l;
}
constexpr int TPAD = 4;      // a tile's rows in LDS are TN + 4 floats apart: 16-byte pieces, columns spread over the banks

// `rows` (a multiple of 32) x TN accumulators at (r0, c0) of the product, in LDS (COPIES of them, to be added in order), to wherever the
// problem wants them.  Through LDS because a result goes out in two orientations: eight consecutive elements a lane (16 bytes of each
// plane, 64-byte runs) either way.  The first pass forms the values, writes the row orientation and leaves them packed for the second.
// (With one wave a SIMD this is instruction time: 64 x 64 took 5.6 us with values formed and rounded in both passes.)
template <int TN, int COPIES>
__device__ __forceinline__ void epilogue(const Probs& a, const Prob& p, float* t, int rows, int r0, int c0)
{
    constexpr int S = TN + TPAD;
    const float so = p.fin ? 1.0f : p.so, alpha = alpha_of(p) * so, cb = p.cb * so, ca = p.ca * so;
    const int padN = p.oc * 32, padM = p.otc * 32, copy = rows * S;
    const bool diagonal = p.ca != 0.0f && r0 < c0 + TN && c0 < r0 + rows, edge = c0 + TN > p.N;
#pragma unroll 2
    for (int q = threadIdx.x; q < rows * (TN / 8); q += 256) {
        const int rl = q / (TN / 8), cl = q % (TN / 8) * 8, row = r0 + rl, col = c0 + cl;
        float* tt = t + rl * S + cl;
        float v[8];
#pragma unroll
        for (int k = 0; k < COPIES; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(tt + k * copy), y = *reinterpret_cast<const float4*>(tt + k * copy + 4);
            const float w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k == 0 ? w[e] : v[e] + w[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= alpha;
        if (p.C && row < p.M && col < padN) {
            const half8* c = reinterpret_cast<const half8*>(p.C + ((size_t)row * p.oc + (col >> 5)) * 64 + (col & 31));
            const half8 h = c[0], l = c[4];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += cb * ((float)h[e] + (float)l[e]);
        }
        if (diagonal)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += row == col + e ? ca : 0.0f;
        if (p.fin) {
            if (!p.fin_t) {
                if (row < p.M) put_fin(a, p, (size_t)row * p.N + col, p.N - col, v);
            } else {
                *reinterpret_cast<float4*>(tt) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4*>(tt + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
            continue;
        }
        // columns N .. padN - 1 and rows M .. padM - 1 are zeros
        if (edge)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = col + e < p.N ? v[e] : 0.0f;
        unsigned w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = row < p.M ? planes_of(v[e]) : 0u;
        uint4v* wt = reinterpret_cast<uint4v*>(tt);
        wt[0] = uint4v{w[0], w[1], w[2], w[3]};
        wt[1] = uint4v{w[4], w[5], w[6], w[7]};
        // a symmetric result takes its lower half in pieces of 8 x 8: those below the diagonal here and, mirrored, in the second pass
        if (row < p.M && col < padN && (!p.sym || row >> 3 > col >> 3)) put_packed(p.out, row, p.oc, col, w);
    }
    if (p.fin && !p.fin_t) return;
    lds_barrier();          // (not __syncthreads: it would wait for the stores above)
#pragma unroll 2
    for (int q = threadIdx.x; q < rows / 8 * TN; q += 256) {
        const int cl = (q >> 2) % TN, rl = (q / (4 * TN)) * 32 + (q & 3) * 8, row = r0 + rl, col = c0 + cl;
        if (col >= p.N) continue;
        const float* tt = t + rl * S + cl;
        if (p.fin) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = tt[e * S];
            if (row < p.M) put_fin(a, p, (size_t)col * p.M + row, p.M - row, v);
            continue;
        }
        if (row >= padM || (p.sym && row >> 3 < col >> 3)) continue;
        unsigned w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = reinterpret_cast<const unsigned*>(tt)[e * S];
        if (p.sym && row >> 3 == col >> 3) {        // on the diagonal: row `col` of the piece, left of the diagonal from itself
            const unsigned* d = reinterpret_cast<const unsigned*>(t) + (col - r0) * S + (row - c0);
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = row + e < col ? d[e] : w[e];
        }
        put_packed(p.outT, col, p.otc, row, w);
    }
}

// The same for a tile whose results go out as planes and whose accumulators are still in registers: formed and rounded there (a block of
// 32 x 32: register r of lane q is row (r & 3) + 8 (r >> 2) + 4 (q >> 5), column q & 31), one packed word each through LDS, then both
// orientations without another rounding (128 x 128: 5.9 us by way of epilogue(), 5.5 this way).
template <int WM, int WN, int TM, int TN>
__device__ __forceinline__ void epilogue_planes(const Prob& p, unsigned* t, const float16v (&acc)[WM][WN], int m0, int n0, int wm, int wn)
{
    constexpr int S = TN + TPAD;
    const int fr = threadIdx.x & 31, fh = (threadIdx.x & 63) >> 5;
    const float alpha = alpha_of(p) * p.so, cb = p.cb * p.so, ca = p.ca * p.so;
    const int padN = p.oc * 32, padM = p.otc * 32;
    const bool diagonal = p.ca != 0.0f && m0 < n0 + TN && n0 < m0 + TM, edge = m0 + TM > p.M || n0 + TN > p.N;
#pragma unroll
    for (int x = 0; x < WM; ++x)
#pragma unroll
        for (int y = 0; y < WN; ++y) {
            const int cl = wn + 32 * y + fr, col = n0 + cl;
            half4 ch[4], cl4[4];
            if (p.C)            // symmetric: row `col` of it has this lane's rows side by side
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int row = m0 + wm + 32 * x + 8 * g + 4 * fh;
                    ch[g] = cl4[g] = half4{0, 0, 0, 0};
                    if (col < p.N && row < padM) {
                        const _Float16* c = p.C + ((size_t)col * p.oc + (row >> 5)) * 64 + (row & 31);
                        ch[g] = *reinterpret_cast<const half4*>(c);
                        cl4[g] = *reinterpret_cast<const half4*>(c + 32);
                    }
                }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int rl = wm + 32 * x + (r & 3) + 8 * (r >> 2) + 4 * fh, row = m0 + rl;
                float v = alpha * acc[x][y][r];
                if (p.C) v += cb * ((float)ch[r >> 2][r & 3] + (float)cl4[r >> 2][r & 3]);
                if (diagonal) v += row == col ? ca : 0.0f;
                if (edge) v = row < p.M && col < p.N ? v : 0.0f;
                t[rl * S + cl] = planes_of(v);
            }
        }
    lds_barrier();
    // (tiles wholly inside, off the diagonal: no conditions)
#pragma unroll 4
    for (int q = threadIdx.x; q < TM * (TN / 8); q += 256) {
        const int rl = q / (TN / 8), cl = q % (TN / 8) * 8, row = m0 + rl, col = n0 + cl;
        if (row < p.M && col < padN && (!p.sym || row >> 3 > col >> 3)) {
            const uint4v lo = *reinterpret_cast<const uint4v*>(t + rl * S + cl), hi = *reinterpret_cast<const uint4v*>(t + rl * S + cl + 4);
            const unsigned w[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            put_packed(p.out, row, p.oc, col, w);
        }
    }
#pragma unroll 4
    for (int q = threadIdx.x; q < TM / 8 * TN; q += 256) {
        const int cl = (q >> 2) % TN, rl = (q / (4 * TN)) * 32 + (q & 3) * 8, row = m0 + rl, col = n0 + cl;
        if (col < p.N && row < padM && !(p.sym && row >> 3 < col >> 3)) {
            unsigned w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = t[(rl + e) * S + cl];
            if (p.sym && row >> 3 == col >> 3) {        // on the diagonal: row `col` of the piece, left of the diagonal from itself
                const unsigned* d = t + (col - m0) * S + (row - n0);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = row + e < col ? d[e] : w[e];
            }
            put_packed(p.outT, col, p.otc, row, w);
        }
    }
}

// A tile of (64 WM) x (64 WN), four waves (2 x 2), NS LDS buffers of one 32-k chunk.  Halfway through chunk c (its second 16 k are in
// registers by then) the workgroup meets: chunk c + 1 has arrived for everybody, buffer c is free and takes chunk c + NS; the first fragments
// of c + 1 are read while the second half of c is multiplied.  One barrier a chunk, NS - 1 chunks of latency covered.
// An operand row of a buffer is 64 bytes per plane (PL, PR planes); its 16-byte unit u lies at u ^ swz(row), the swizzle applied to the
// source address of the load, so that the 32 rows of a fragment read meet each bank group equally often.
template <int PL> __device__ __forceinline__ int swz(int row) { return PL == 2 ? row & 7 : (row >> 1) & 3; }

// KW: the four waves share a (32 WM) x (32 WN) tile by K instead, wave v taking chunks v, v + 4, ..: each with a ring of its own and no
// meeting at all; their sums meet in LDS at the end, added in the order of the waves.  For 64 x 64 tiles, where a wave of the shared form has
// three products between two meetings (136 tiles of K = 1024: 15.2 us shared, 12.7 this way).
// LL: products of the l planes too, for the problems that ask for them, and the small products in sums of their own: beside h h they would lose
// their last bits.
template <int WM, int WN, int PL, int PR, int NS, bool KW, bool LL>
__global__ __launch_bounds__(256, 1) void ns_gemm_kernel(Probs a)
{
    constexpr int WAVES = KW ? 1 : 4;                              // waves that load a stage together
    constexpr int TM = KW ? 32 * WM : 64 * WM, TN = KW ? 32 * WN : 64 * WN, BL = TM * 64 * PL, BR = TN * 64 * PR, STAGE = BL + BR;
    constexpr int NL = BL / (1024 * WAVES), NR = BR / (1024 * WAVES);      // load instructions a wave and stage
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int fr = lane & 31, fh = lane >> 5;                      // fragment row, k half
    const int wm = KW ? 0 : (wave >> 1) * WM * 32, wn = KW ? 0 : (wave & 1) * WN * 32;
    char* const ring = KW ? lds + wave * (NS * STAGE) : lds;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) char*)lds + wave * (KW ? NS * STAGE : 1024));
    const int lt = KW ? lane : (int)threadIdx.x;                   // this lane among those that load a stage
    auto meet = [&] {       // everybody who reads a stage has it, and has finished with the one before
        if constexpr (KW) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else lds_barrier();
    };

    // the workgroups of one XCD (every eighth) take consecutive items: they share operand rows through its L2
    const int bid = blockIdx.x;
    int w;
    {
        const int base = bid < a.whole ? 0 : a.whole, n = bid < a.whole ? a.whole : a.items - a.whole, b = bid - base;
        const int per = n >> 3, rest = n & 7, x = b & 7, y = b >> 3;
        w = base + x * per + (x < rest ? x : rest) + y;
    }
    {
        const int i = a.count == 1 ? 0 : w < a.whole ? which(a.tile0, w) : a.equal ? which(a.tile0, a.whole + (w - a.whole) % a.rest) : which(a.item0, w);
        const Prob p = a.p[i];
        int tile = w - a.tile0[i], c0 = 0;        // chunks [c0, c0 + n) of the tile
        if (w >= a.whole) {
            const int local = a.equal ? w - a.whole : w - a.item0[i], tiles = a.equal ? a.rest : p.tiles, sgm = local / tiles;
            tile = local - sgm * tiles + (a.equal ? a.whole - a.tile0[i] : 0);
            c0 = sgm * p.seg;
        }
        const int left = p.kc - c0, n = w < a.whole || left < p.seg ? left : p.seg;
        int m0, n0;
        tile_at(p, tile, TM, TN, m0, n0);

        // source offsets of this lane from the tile's first row (below 2^32: rows <= 256, K <= 2^21)
        unsigned offL[NL], offR[NR];
        constexpr int UL = 4 * PL, UR = 4 * PR;        // 16-byte units a row
#pragma unroll
        for (int k = 0; k < NL; ++k) {
            const int lr = (k * 64 * WAVES + lt) / UL, row = m0 + lr < p.M ? lr : p.M - 1 - m0;
            offL[k] = (unsigned)row * (unsigned)(p.kc * 64 * PL) + ((lane % UL) ^ swz<PL>(lr)) * 16;
        }
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int lr = (k * 64 * WAVES + lt) / UR, row = n0 + lr < p.N ? lr : p.N - 1 - n0;
            offR[k] = (unsigned)row * (unsigned)(p.kc * 64 * PR) + ((lane % UR) ^ swz<PR>(lr)) * 16;
        }
        const int v = KW ? __builtin_amdgcn_readfirstlane(wave) : 0, step = KW ? 4 : 1;
        const int nw = KW ? (n - v + 3) / 4 : n;       // chunks of this wave: c0 + v, c0 + v + step, ..
        const char* srcL = reinterpret_cast<const char*>(p.L) + ((size_t)m0 * p.kc + c0 + v) * (64 * PL);
        const char* srcR = reinterpret_cast<const char*>(p.R) + ((size_t)n0 * p.kc + c0 + v) * (64 * PR);
        auto fetch_one = [&](int buf, int k) {         // instruction k of NL + NR; the last one moves on to the next chunk
            const unsigned d = lds0 + buf * STAGE;
            if (k < NL) to_lds16(srcL, offL[k < NL ? k : 0], d + k * (1024 * WAVES));
            else to_lds16(srcR, offR[k >= NL ? k - NL : 0], d + BL + (k - NL) * (1024 * WAVES));
            if (k == NL + NR - 1) {
                srcL += step * 64 * PL;
                srcR += step * 64 * PR;
            }
        };
        float16v acc[WM][WN], low[LL ? WM : 1][LL ? WN : 1];
#pragma unroll
        for (int x = 0; x < WM; ++x)
#pragma unroll
            for (int y = 0; y < WN; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    acc[x][y][r] = 0.0f;
                    if constexpr (LL) low[x][y][r] = 0.0f;
                }

        const int rowL = wm + fr, rowR = wn + fr;        // (32 rows on: the same swizzle)
        half8 fl[2][WM][PL], fq[2][WN][PR];
        constexpr int READS = WM * PL + WN * PR, PRODS = (PL + PR - 1) * WM * WN, FETCHES = NL + NR;
        auto read_one = [&](int buf, int ks, int k) {
            const char* s = ring + buf * STAGE;
            if (k < WM * PL) {
                const int x = k % WM, pl = k / WM % PL;
                fl[ks][x][pl] = *reinterpret_cast<const half8*>(s + (rowL + 32 * x) * (64 * PL) + (((pl * 4 + ks * 2 + fh) ^ swz<PL>(rowL)) * 16));
            } else {
                const int y = (k - WM * PL) % WN, pl = (k - WM * PL) / WN % PR;
                fq[ks][y][pl] = *reinterpret_cast<const half8*>(s + BL + (rowR + 32 * y) * (64 * PR) + (((pl * 4 + ks * 2 + fh) ^ swz<PR>(rowR)) * 16));
            }
        };
        // The PRODS matrix instructions of 16 k, the small products first, a block's WM * WN apart; in the shadow of each (32 cycles) go its
        // share of the reads of the other half's fragments and of the loads of a chunk to come: with one wave a SIMD nothing else fills it.
        auto multiply = [&](int ks, bool reads, int rbuf, bool fetches, int fbuf) {
            if constexpr (LL)        // (a question of its own kernel: asked in all of them it costs 1 % of a small launch)
                if (p.ll)
#pragma unroll
                    for (int g = 0; g < WM * WN; ++g)
                        low[g / WN][g % WN] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[ks][g / WN][1], fq[ks][g % WN][1], low[g / WN][g % WN], 0, 0, 0);
#pragma unroll
            for (int g = 0; g < PRODS; ++g) {
                const int k = g / (WM * WN), x = g / WN % WM, y = g % WN;
                const int pl = PL == 2 && k == 0 ? 1 : 0, pr = PR == 2 && k == PL - 1 ? 1 : 0;
                float16v* to = &acc[x][y];
                if constexpr (LL)
                    if (pl + pr) to = &low[x][y];
                *to = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[ks][x][pl], fq[ks][y][pr], *to, 0, 0, 0);
                if (reads)
#pragma unroll
                    for (int r = g * READS * 2 / PRODS; r < (g + 1) * READS * 2 / PRODS; ++r)        // (in the first half: in time for the next)
                        if (r < READS) read_one(rbuf, ks ^ 1, r);
                if (fetches)
#pragma unroll
                    for (int r = g * FETCHES / PRODS; r < (g + 1) * FETCHES / PRODS; ++r) fetch_one(fbuf, r);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const int ahead = nw < NS ? nw : NS;
        for (int k = 0; k < ahead; ++k)
#pragma unroll
            for (int r = 0; r < FETCHES; ++r) fetch_one(k, r);
        if (nw >= NS) wait_vm<(NS - 1) * FETCHES>();
        else wait_vm<0>();
        meet();
        if (nw > 0)
#pragma unroll
            for (int r = 0; r < READS; ++r) read_one(0, 0, r);
        int buf = 0, c = 0;
        for (; c + NS < nw; ++c) {       // chunks up to c + NS - 1 are on their way
            multiply(0, true, buf, false, 0);
            wait_vm<(NS - 2) * FETCHES>();
            meet();
            const int next = buf + 1 < NS ? buf + 1 : 0;
            multiply(1, true, next, true, buf);
            buf = next;
        }
        for (; c < nw; ++c) {            // the last NS: nothing more to load
            multiply(0, true, buf, false, 0);
            wait_vm<0>();
            meet();
            const int next = buf + 1 < NS ? buf + 1 : 0;
            multiply(1, c + 1 < nw, next, false, 0);
            buf = next;
        }
        // (nobody reads the buffers any more: the last meeting was behind the last fragment reads)
        if constexpr (LL)
#pragma unroll
            for (int x = 0; x < WM; ++x)
#pragma unroll
                for (int y = 0; y < WN; ++y) acc[x][y] += low[x][y];
        if constexpr (KW) lds_barrier();
        if constexpr (!KW)
            if (n == p.kc && !p.fin) {
                epilogue_planes<WM, WN, TM, TN>(p, reinterpret_cast<unsigned*>(lds), acc, m0, n0, wm, wn);
                return;
            }
        float* const t = reinterpret_cast<float*>(lds);
        float* const mine = KW ? t + wave * (TM * (TN + TPAD)) : t;
#pragma unroll
        for (int x = 0; x < WM; ++x)
#pragma unroll
            for (int y = 0; y < WN; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r)      // register r of lane q: row (r & 3) + 8 (r >> 2) + 4 (q >> 5), column q & 31
                    mine[(wm + 32 * x + (r & 3) + 8 * (r >> 2) + 4 * fh) * (TN + TPAD) + wn + 32 * y + fr] = acc[x][y][r];
        lds_barrier();
        if (n == p.kc) epilogue<TN, KW ? 4 : 1>(a, p, t, TM, m0, n0);
        else {
            float4* o = reinterpret_cast<float4*>(a.part + (size_t)(w - a.whole) * (TM * TN));
#pragma unroll 4
            for (int q = threadIdx.x; q < TM * TN / 4; q += 256) {
                const float* tt = t + q / (TN / 4) * (TN + TPAD) + q % (TN / 4) * 4;
                float4 x = *reinterpret_cast<const float4*>(tt);
                if constexpr (KW)
#pragma unroll
                    for (int k = 1; k < 4; ++k) {
                        const float4 y = *reinterpret_cast<const float4*>(tt + k * TM * (TN + TPAD));
                        x.x += y.x;
                        x.y += y.y;
                        x.z += y.z;
                        x.w += y.w;
                    }
                o[q] = x;
            }
        }
    }
}

// Tiles cut along K: the segments' accumulators added in their order, then the same epilogue.  A workgroup takes 32 rows.
template <int TM, int TN>
__global__ __launch_bounds__(256) void ns_join_kernel(Probs a)
{
    constexpr int STRIPS = TM / 32, PER = 32 * TN / 1024;
    __shared__ __align__(16) float t[32 * (TN + TPAD)];
    const int strip = blockIdx.x % STRIPS, tile = a.whole + blockIdx.x / STRIPS;
    const int i = which(a.tile0, tile);
    const Prob p = a.p[i];
    const int segs = (p.kc + p.seg - 1) / p.seg;
    if (segs == 1) return;
    const int first = a.equal ? tile - a.whole : a.item0[i] - a.whole + tile - a.tile0[i], step = a.equal ? a.rest : p.tiles;
    float4 acc[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) acc[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
    for (int sgm = 0; sgm < segs; ++sgm) {
        const float4* o = reinterpret_cast<const float4*>(a.part + ((size_t)first + (size_t)sgm * step) * (TM * TN) + strip * 32 * TN) + threadIdx.x;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const float4 v = o[k * 256];
            acc[k].x += v.x;
            acc[k].y += v.y;
            acc[k].z += v.z;
            acc[k].w += v.w;
        }
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int at = (k * 256 + threadIdx.x) * 4;
        *reinterpret_cast<float4*>(t + at / TN * (TN + TPAD) + at % TN) = acc[k];
    }
    lds_barrier();
    int m0, n0;
    tile_at(p, tile - a.tile0[i], TM, TN, m0, n0);
    epilogue<TN, 1>(a, p, t, 32, m0 + strip * 32, n0);
}

// ---- momentum, norm, planes -------------------------------------------------------------------------------------------------------
struct Mat {
    const void* g;       // gradient / input [rows, cols]
    float* mom;          // momentum or NULL
    double* sums;        // partial sums of squares
    float* r;            // X = (U 2^e) * r[0];  r[1] = r[0] t, r[2] = 1 / t (x_shift)
    _Float16* P;         // planes of U 2^e, [rows][chunks(cols)]
    _Float16* PT;        // of its transpose, [cols][chunks(rows)]
    int rows, cols, blocks;
};
struct Mats {
    int blk0[MAX_MAT], tile0[MAX_MAT];       // first workgroup of every matrix in ns_norm_kernel / ns_planes_kernel; behind the last: INT_MAX
    Mat m[MAX_MAT];
    int count, dtype, nesterov, planes;
    float mu, x_room;
    double eps;
};
static_assert(sizeof(Mats) <= 3584, "travels in the kernel arguments");

// momentum (if any) updated and the sums of squares of the update's direction, one partial sum per workgroup (fp64: the squares of fp32
// numbers neither overflow nor vanish there)
template <int DT, bool MOM>
__global__ __launch_bounds__(256) void ns_norm_kernel(Mats a)
{
    __shared__ double s_acc[4];
    const int i = which(a.blk0, blockIdx.x);
    const Mat m = a.m[i];
    const size_t n = (size_t)m.rows * m.cols;
    const int b = blockIdx.x - a.blk0[i];
    double s = 0.0;
    for (size_t e0 = (size_t)b * 4096 + threadIdx.x * 4; e0 < n; e0 += (size_t)m.blocks * 4096) {
        float u[4][4], v[4][4];        // four loads on their way before the first is used
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t left = (int64_t)n - (int64_t)(e0 + q * 1024);
            load4(m.g, DT, e0 + q * 1024, left, u[q]);
            if constexpr (MOM) load4(m.mom, MP_DTYPE_F32, e0 + q * 1024, left, v[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const size_t e = e0 + q * 1024;
            if (e >= n) break;
            if constexpr (MOM) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[q][k] = v[q][k] + (1.0f - a.mu) * (u[q][k] - v[q][k]);
                    u[q][k] = a.nesterov ? u[q][k] + a.mu * (v[q][k] - u[q][k]) : v[q][k];
                }
                if (n - e >= 4) __builtin_memcpy(m.mom + e, v[q], 16);
                else
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        if (e + k < n) m.mom[e + k] = v[q][k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) s += (double)u[q][k] * (double)u[q][k];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) s_acc[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) m.sums[b] = (s_acc[0] + s_acc[1]) + (s_acc[2] + s_acc[3]);
}

__device__ __forceinline__ void put_plane(_Float16* img, int row, int nchunk, int col, const float (&v)[4])
{
    half4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (_Float16)v[e];
    *reinterpret_cast<half4*>(img + ((size_t)row * nchunk + (col >> 5)) * 32 + (col & 31)) = h;
}

// A norm far below eps: X stays small through all steps, and planes scaled for |X| ~ 1 would lose it in fp16's subnormals (a norm of 5e-8 eps:
// 3e-4 of the result, 5e-12 eps: all of it).  Behind the first hop the planes hold X t, t the largest power of two (one at least) that keeps
// |X| t within the planes' bound in every step: x_room = that bound / the largest product of |Q|, which is what |X| grows by.
__device__ __forceinline__ double x_shift(double norm, double denom, float x_room)
{
    const double v = (double)x_room * denom / norm;
    int e = 0;
    if (norm > 0.0 && v >= 2.0) {
        (void)frexp(v < 1e36 ? v : 1e36, &e);         // v in [2^(e-1), 2^e)
        --e;
    }
    return ldexp(1.0, e);
}

// 64 x 64 elements of a matrix into both plane images.  The power of two 2^e takes the norm into [2^13, 2^14): exact, and every entry
// below 2^14; the division by the norm itself waits for the products' epilogues (r).  A 16-bit matrix without momentum is one plane: fp16
// holds the 8 or 11 bits of an entry exactly (down to 2^-38 of the norm, where the polynomial's slope of 485 is still far below half a step).
__global__ __launch_bounds__(256) void ns_planes_kernel(Mats a)
{
    __shared__ double s_acc[4];
    __shared__ float tile[64][65];
    const int i = which(a.tile0, blockIdx.x);
    const Mat m = a.m[i];
    double s = 0.0;
    for (int k = threadIdx.x; k < m.blocks; k += 256) s += m.sums[k];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) s_acc[threadIdx.x >> 6] = s;
    __syncthreads();
    const double norm = sqrt((s_acc[0] + s_acc[1]) + (s_acc[2] + s_acc[3]));
    int e = 0;
    if (norm > 0.0 && norm < 1e300) {
        (void)frexp(norm, &e);        // norm in [2^(e-1), 2^e)
        e = 14 - e;
    }
    const int local = blockIdx.x - a.tile0[i], tn = (m.cols + 63) / 64;
    const int r0 = (local / tn) * 64, c0 = (local % tn) * 64;
    if (local == 0 && threadIdx.x == 0) {
        const double denom = norm > a.eps || norm != norm ? norm : a.eps, r = 1.0 / ldexp(denom, e), t = x_shift(norm, denom, a.x_room);
        m.r[0] = (float)r;
        m.r[1] = (float)(r * t);
        m.r[2] = (float)(1.0 / t);
    }
    const int tc = (threadIdx.x & 15) * 4, tr = threadIdx.x >> 4;
#pragma unroll
    for (int k = 0; k < 64; k += 16) {
        const int r = r0 + k + tr, c = c0 + tc;
        float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < m.rows) {
            const size_t at = (size_t)r * m.cols + c;
            load4(m.g, a.dtype, at, (int64_t)m.cols - c, u);
            if (m.mom) {
                float v[4];
                load4(m.mom, MP_DTYPE_F32, at, (int64_t)m.cols - c, v);
#pragma unroll
                for (int q = 0; q < 4; ++q) u[q] = a.nesterov ? u[q] + a.mu * (v[q] - u[q]) : v[q];
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) tile[k + tr][tc + q] = ldexpf(u[q], e);
    }
    __syncthreads();
    const int pc = chunks(m.cols), ptc = chunks(m.rows);
    for (int q = threadIdx.x; q < 64 * 16; q += 256) {
        const int a4 = (q & 15) * 4, b = q >> 4;
        float v[4];
        if (r0 + b < m.rows && c0 + a4 < pc * 32) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = tile[b][a4 + k];
            if (a.planes == 1) put_plane(m.P, r0 + b, pc, c0 + a4, v);
            else put_planes(m.P, r0 + b, pc, c0 + a4, v);
        }
        if (c0 + b < m.cols && r0 + a4 < ptc * 32) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = tile[a4 + k][b];
            if (a.planes == 1) put_plane(m.PT, c0 + b, ptc, r0 + a4, v);
            else put_planes(m.PT, c0 + b, ptc, r0 + a4, v);
        }
    }
}

// ---- small matrices: everything in one launch ------------------------------------------------------------------------------------
// m <= 64 and planes that fit a CU's LDS: a workgroup of eight waves has a matrix from gradient to result.  17 launches of a few
// microseconds would be all there is to it (64 x 64 fp32: 100 us, 27 here; from m = 96 on the launches win: 128 x 131 took 118 us this
// way).  Wave v holds the columns of blocks v, v + 8, .. of 32 of X in registers (packed planes, in the accumulator layout of the product
// that made them: that layout is the right operand's of the next product Q X if Q's columns are read in the same order, two runs of four).
// LDS holds X's planes for the Gram product and one m x m matrix, A and then Q.
struct Small {
    const void* g;
    float* mom;
    void* out;
    int rows, cols;
    float fmul, fdecay;
};
constexpr int MAX_SMALL = 64;
struct Smalls {
    int count, nesterov, update, steps;
    float mu, a, b, c, sX, sA, sQ, x_room;
    double eps;
    Small m[MAX_SMALL];
};
static_assert(sizeof(Smalls) <= 3584, "travels in the kernel arguments");

constexpr int SMALL_LDS = 147456 + 256;        // (256: the padding of the fp32 tile that lies over X's planes on the way in and out)
constexpr int small_nb(int mb) { return mb == 1 ? 4 : 2; }      // column blocks a wave
// Waves that share a block of the Gram product by K, from 256 columns on: one wave alone is what 16 x 900 waits for (57 us, with four 45), short
// ones lose two meetings a step (32 x 32: 16 us, 18); with 64 rows four waves have a block each (64 x 500: 65, with two 64).
constexpr int small_ks(int mb) { return mb == 1 ? 4 : 1; }
constexpr int SMALL_KS_CHUNKS = 8;
constexpr int small_s(int mb) { return mb == 1 ? 12288 : 16384; }      // bytes in front of X: the m x m image, before it the sums of those waves

template <int MB, int DT>
__global__ __launch_bounds__(512) void ns_small_kernel(Smalls a)
{
    constexpr int NB = small_nb(MB);
    extern __shared__ __align__(16) char lds[];
    __shared__ double s_sum[8];
    const Small m = a.m[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 31, fh = lane >> 5, odd = lane & 1;
    const bool tall = m.rows > m.cols;
    const int M = tall ? m.cols : m.rows, N = tall ? m.rows : m.cols, npc = chunks(N);
    char* S = lds;
    char* X = lds + small_s(MB);
    auto unit = [&](char* img, int row, int nch, int chunk, int u) { return img + ((size_t)row * nch + chunk) * 128 + ((u ^ (row & 7)) * 16); };

    // In and out by way of LDS (over X's planes): a wave reads rows of the matrix as it lies in memory.
    float* const t = reinterpret_cast<float*>(X);
    const int stride = npc * 32 + 1, sr = tall ? 1 : stride, sc = tall ? stride : 1;       // element (r, c) of the matrix at t[r sr + c sc]
    double sum = 0.0;
    if (M < 32 * MB || N < npc * 32) {         // rows and columns that fill up the blocks: zeros
        for (int q = threadIdx.x; q < 32 * MB * stride; q += 512) t[q] = 0.0f;
        __syncthreads();
    }
    for (int r0 = wave; r0 < m.rows; r0 += 32)
        for (int c = lane; c < m.cols; c += 64) {
            float x[4], v[4];           // four rows on their way at once
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const size_t at = (size_t)(r0 + 8 * q) * m.cols + c;
                if (r0 + 8 * q < m.rows) {
                    x[q] = load_any(m.g, DT, at);
                    v[q] = m.mom ? m.mom[at] : 0.0f;
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int rr = r0 + 8 * q;
                if (rr >= m.rows) continue;
                if (m.mom) {
                    v[q] = v[q] + (1.0f - a.mu) * (x[q] - v[q]);
                    m.mom[(size_t)rr * m.cols + c] = v[q];
                    x[q] = a.nesterov ? x[q] + a.mu * (v[q] - x[q]) : v[q];
                }
                sum += (double)x[q] * (double)x[q];
                t[rr * sr + c * sc] = x[q];
            }
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += s_sum[k];
    const double norm = sqrt(sum);
    int e2 = 0;
    if (norm > 0.0 && norm < 1e300) {       // the norm to [2^13, 2^14), as in ns_planes_kernel
        (void)frexp(norm, &e2);
        e2 = 14 - e2;
    }
    const double denom = norm > a.eps || norm != norm ? norm : a.eps, r = 1.0 / ldexp(denom, e2), shift = x_shift(norm, denom, a.x_room);
    unsigned xp[NB][MB][16];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int row = 32 * i + (k & 3) + 8 * (k >> 2) + 4 * fh, col = (wave + 8 * b) * 32 + fr;
                xp[b][i][k] = wave + 8 * b < npc ? planes_of(ldexpf(t[row * stride + col], e2)) : 0u;
                __builtin_amdgcn_sched_barrier(0);
            }
    __syncthreads();

    float sx = (float)r, so = (float)(r * shift) * a.sX / a.sQ;           // X = planes * sx; so: from a product Q X to the next planes
    for (int step = 0; step < a.steps; ++step) {
        // (a zero the compiler does not know: it would keep the addresses of every access below in registers across the steps, and spill)
        int zero = 0;
        asm volatile("" : "+v"(zero));
        S = lds + zero;
        X = lds + small_s(MB) + zero;
        // X's planes to LDS.  A lane has a column: neighbours swap so that each writes two columns of one row.
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int nb = wave + 8 * b;
            if (nb < npc)
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int k = 0; k < 16; k += 2) {
                    const unsigned p0 = xp[b][i][k], p1 = xp[b][i][k + 1];
                    const unsigned mine = odd ? p1 : p0, got = mp::dpp_u32<mp::DPP_QUAD_XOR1>(odd ? p0 : p1);
                    const unsigned lo = odd ? got : mine, hi = odd ? mine : got;
                    const int row = 32 * i + (k & 3) + 8 * (k >> 2) + 4 * fh + odd;
                    *reinterpret_cast<unsigned*>(unit(X, row, npc, nb, fr >> 3) + (fr & 6) * 2) = __builtin_amdgcn_perm(hi, lo, 0x05040100);
                    *reinterpret_cast<unsigned*>(unit(X, row, npc, nb, 4 + (fr >> 3)) + (fr & 6) * 2) = __builtin_amdgcn_perm(hi, lo, 0x07060302);
                    __builtin_amdgcn_sched_barrier(0);       // (here and below: addresses and fragments of all of it at once do not fit the registers)
                }
        }
        __syncthreads();
        auto product = [&](char* img, int c0, int step, int nch, int i, int j, bool full) {        // rows 32 i .. of the image times rows 32 j ..
            // (h h by itself: a third of the roundings at the size of the sum, and two chains of matrix instructions)
            float16v acc, big;
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k] = big[k] = 0.0f;
            const int ri = 32 * i + fr, rj = 32 * j + fr;
            for (int c = c0; c < nch; c += step)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const half8 lh = *reinterpret_cast<const half8*>(unit(img, ri, nch, c, ks * 2 + fh)), ll = *reinterpret_cast<const half8*>(unit(img, ri, nch, c, 4 + ks * 2 + fh));
                    const half8 rh = *reinterpret_cast<const half8*>(unit(img, rj, nch, c, ks * 2 + fh)), rl = *reinterpret_cast<const half8*>(unit(img, rj, nch, c, 4 + ks * 2 + fh));
                    if (full) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll, rl, acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll, rh, acc, 0, 0, 0);
                    big = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh, rh, big, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh, rl, acc, 0, 0, 0);
                }
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k] += big[k];
            return acc;
        };
        auto keep = [&](float16v& v, float scale, int i, int j) {      // block (i, j) of a symmetric matrix as block (j, i), runs of four; v: what the planes hold
#pragma unroll
            for (int rg = 0; rg < 4; ++rg) {
                half4 h, l;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = v[rg * 4 + e] * scale;
                    h[e] = (_Float16)x;
                    l[e] = (_Float16)(x - (float)h[e]);
                    v[rg * 4 + e] = (float)h[e] + (float)l[e];
                }
                *reinterpret_cast<half4*>(unit(S, 32 * j + fr, MB, i, rg) + fh * 8) = h;
                *reinterpret_cast<half4*>(unit(S, 32 * j + fr, MB, i, 4 + rg) + fh * 8) = l;
            }
        };
        // A, then Q, block (i, j) by wave i MB + j; the Gram product by KS waves
        float16v A;
        constexpr int KS = small_ks(MB), BLOCKS = MB * MB;
        const int block = wave % BLOCKS, part = wave / BLOCKS, i0 = block / MB, j0 = block % MB;
        const bool mine = part == 0;
        const int share = KS > 1 && npc >= SMALL_KS_CHUNKS ? KS : 1;
        if (part < share) A = product(X, part, share, npc, i0, j0, false);
        if (share > 1) {
            float* const sums = reinterpret_cast<float*>(S) + lane;
            if (!mine && part < share)
#pragma unroll
                for (int k = 0; k < 16; ++k) sums[((part - 1) * BLOCKS + block) * 1024 + k * 64] = A[k];
            __syncthreads();
            if (mine)
#pragma unroll
                for (int p = 0; p < KS - 1; ++p)
#pragma unroll
                    for (int k = 0; k < 16; ++k) A[k] += sums[(p * BLOCKS + block) * 1024 + k * 64];
            __syncthreads();
        }
        if (mine) {
#pragma unroll
            for (int k = 0; k < 16; ++k) A[k] *= sx * sx;
            keep(A, a.sA, i0, j0);
        }
        __syncthreads();
        if (mine) {
            const float16v sq = product(S, 0, 1, MB, i0, j0, DT == MP_DTYPE_F32);
            const float cc = a.c / (a.sA * a.sA), bb = a.b / a.sA;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int row = 32 * i0 + (k & 3) + 8 * (k >> 2) + 4 * fh;
                A[k] = cc * sq[k] + bb * A[k] + (row == 32 * j0 + fr && row < M ? a.a : 0.0f);
            }
        }
        __syncthreads();
        if (mine) keep(A, a.sQ, i0, j0);
        __syncthreads();
        const bool last = step + 1 == a.steps;
        const float alpha = sx / a.sQ;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int nb = wave + 8 * b;
            if (nb < npc) {
            float16v acc[MB];
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[i][k] = 0.0f;
#pragma unroll
            for (int c = 0; c < MB; ++c)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    // k slot j of half fh is row 16 ks + 8 (j >> 2) + 4 fh + (j & 3) of the chunk, on both sides
                    uint4v wh, wl;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        wh[e] = __builtin_amdgcn_perm(xp[b][c][8 * ks + 2 * e + 1], xp[b][c][8 * ks + 2 * e], 0x05040100);
                        wl[e] = __builtin_amdgcn_perm(xp[b][c][8 * ks + 2 * e + 1], xp[b][c][8 * ks + 2 * e], 0x07060302);
                    }
                    const half8 rh = __builtin_bit_cast(half8, wh), rl = __builtin_bit_cast(half8, wl);
#pragma unroll
                    for (int i = 0; i < MB; ++i) {
                        const int row = 32 * i + fr;
                        const half4 h0 = *reinterpret_cast<const half4*>(unit(S, row, MB, c, 2 * ks) + fh * 8);
                        const half4 h1 = *reinterpret_cast<const half4*>(unit(S, row, MB, c, 2 * ks + 1) + fh * 8);
                        const half4 l0 = *reinterpret_cast<const half4*>(unit(S, row, MB, c, 4 + 2 * ks) + fh * 8);
                        const half4 l1 = *reinterpret_cast<const half4*>(unit(S, row, MB, c, 4 + 2 * ks + 1) + fh * 8);
                        const half8 lh = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7), ll = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
                        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ll, rh, acc[i], 0, 0, 0);
                        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh, rl, acc[i], 0, 0, 0);
                        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lh, rh, acc[i], 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (!last) {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int k = 0; k < 16; ++k) xp[b][i][k] = planes_of(acc[i][k] * so);
            } else {        // (the planes are not read any more)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const int row = 32 * i + (k & 3) + 8 * (k >> 2) + 4 * fh;
                        t[row * stride + nb * 32 + fr] = acc[i][k] * alpha;
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
            }
        }
        sx = (float)(1.0 / shift) / a.sX;
        so = 1.0f / a.sQ;
    }
    __syncthreads();
    for (int rr = wave; rr < m.rows; rr += 8)
#pragma unroll 2
        for (int c = lane; c < m.cols; c += 64) {
            const size_t at = (size_t)rr * m.cols + c;
            float x = t[rr * sr + c * sc];
            if (a.update) x = m.fdecay * load_any(m.out, DT, at) - m.fmul * x;
            store_fin(m.out, DT, at, x);
        }
}

// ---- up to eight rows (or columns) ---------------------------------------------------------------------------------------------------
// A thread has NC columns of X in fp32 registers: 36 dot products, an 8 x 8 polynomial and 64 multiply-adds a column are little for the vector
// units (blocks of 32 rows of the matrix cores would be three quarters zeros), and fp32 throughout: sums of so few terms leave the planes' 22
// bits bare (165 matrices up to 64 x 512: at most 3.7 times as far from the exact result as fp32 products, 2.3 with this kernel).  fp32, 5 x 100:
// 19 us by ns_small_kernel, 11 this way; 8 x 1000: 45, 12; 8 x 4000: 97 by products' launches, 28.  (Summed value by value over a wave, six
// dependent steps each, it took 43 us whatever the size.)
constexpr int TINY_M = 8, TINY_THREADS = 512;

template <int NC, int DT>
__global__ __launch_bounds__(TINY_THREADS) void ns_tiny_kernel(Smalls a)
{
    __shared__ double s_sum[8];
    __shared__ float part[8][36];
    __shared__ __align__(16) float A[8][8], Q[8][8];
    const Small m = a.m[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool tall = m.rows > m.cols;
    const int M = tall ? m.cols : m.rows, N = tall ? m.rows : m.cols;
    float x[NC][8];
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = c * TINY_THREADS + threadIdx.x;
        float v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool in = col < N && r < M;
            const size_t at = tall ? (size_t)col * M + r : (size_t)r * N + col;
            x[c][r] = in ? load_any(m.g, DT, at) : 0.0f;
            v[r] = in && m.mom ? m.mom[at] : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (m.mom && col < N && r < M) {
                v[r] = v[r] + (1.0f - a.mu) * (x[c][r] - v[r]);
                m.mom[tall ? (size_t)col * M + r : (size_t)r * N + col] = v[r];
                x[c][r] = a.nesterov ? x[c][r] + a.mu * (v[r] - x[c][r]) : v[r];
            }
            sum += (double)x[c][r] * (double)x[c][r];
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += s_sum[k];
    const double norm = sqrt(sum), scale = 1.0 / (norm > a.eps || norm != norm ? norm : a.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int r = 0; r < 8; ++r) x[c][r] = (float)((double)x[c][r] * scale);
    for (int step = 0; step < a.steps; ++step) {
        // A: entry (i, j), j <= i, is number i (i + 1) / 2 + j.  A wave's sums of 36 numbers: halves of the wave keep 18 each, rows of 16 lanes 9 each
        float g[36];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                float v = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; ++c) v = fmaf(x[c][i], x[c][j], v);
                g[i * (i + 1) / 2 + j] = v;
            }
#pragma unroll
        for (int k = 0; k < 18; ++k) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(g[k]), __float_as_uint(g[k + 18]), false, false);
            g[k] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
#pragma unroll
        for (int k = 0; k < 9; ++k) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(g[k]), __float_as_uint(g[k + 9]), false, false);
            float v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
            v += __uint_as_float(mp::dpp_u32<mp::DPP_QUAD_XOR1>(__float_as_uint(v)));
            v += __uint_as_float(mp::dpp_u32<mp::DPP_QUAD_XOR2>(__float_as_uint(v)));
            v += __uint_as_float(mp::dpp_u32<mp::DPP_ROW_HALF_MIRROR>(__float_as_uint(v)));
            v += __uint_as_float(mp::dpp_u32<mp::DPP_ROW_MIRROR>(__float_as_uint(v)));
            if ((lane & 15) == 0) part[wave][k + 9 * (lane >> 4 & 1) + 18 * (lane >> 5)] = v;
        }
        __syncthreads();
        const int i = lane >> 3, j = lane & 7, hi = i > j ? i : j, lo = i > j ? j : i;
        if (wave == 0) {
            float g = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) g += part[w][hi * (hi + 1) / 2 + lo];
            A[i][j] = g;
        }
        __syncthreads();
        if (wave == 0) {
            float q = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) q = fmaf(A[i][k], A[k][j], q);
            Q[i][j] = fmaf(a.c, q, a.b * A[i][j]) + (i == j ? a.a : 0.0f);
        }
        __syncthreads();
        float y[NC][8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            float q[8];
            *reinterpret_cast<float4*>(q) = *reinterpret_cast<const float4*>(Q[r]);
            *reinterpret_cast<float4*>(q + 4) = *reinterpret_cast<const float4*>(Q[r] + 4);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float acc = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) acc = fmaf(q[k], x[c][k], acc);
                y[c][r] = acc;
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 8; ++r) x[c][r] = y[c][r];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int col = c * TINY_THREADS + threadIdx.x;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (col >= N || r >= M) continue;
            const size_t at = tall ? (size_t)col * M + r : (size_t)r * N + col;
            const float v = x[c][r];
            store_fin(m.out, DT, at, a.update ? m.fdecay * load_any(m.out, DT, at) - m.fmul * v : v);
        }
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
struct Shape { int64_t rows, cols, m, n; };

Shape shape_of(int64_t rows, int64_t cols)
{
    Shape s{rows, cols, rows < cols ? rows : cols, rows < cols ? cols : rows};
    return s;
}

constexpr int MAX_STEPS = 16;

struct Bounds { double x, q, r[MAX_STEPS + 1]; bool ok; };    // of |X|, |Q| and |Q^h| (products of up to h successive Q) in spectral norm

// The scalar recursion of a singular value, on a grid of starting values in [0, 1]: what the matrices can grow to.  30 us of host time, the
// same for all steps of a training run: a thread keeps the last one, a property of the coefficients alone (64 x 64 fp32 takes 5 us longer with
// it formed every time).
Bounds bounds_of(int steps, const double* c)
{
    thread_local Bounds b;
    thread_local int of_steps = 0;
    thread_local double of[3];
    if (of_steps == steps && of[0] == c[0] && of[1] == c[1] && of[2] == c[2]) return b;
    of_steps = steps;
    for (int k = 0; k < 3; ++k) of[k] = c[k];
    b.x = 1.0; b.q = 0.0; b.ok = true;
    for (double& v : b.r) v = 0.0;
    for (int g = 0; g < 768; ++g) {
        double s = g < 512 ? g / 511.0 : pow(10.0, -(g - 511) * 8.0 / 256.0), q[MAX_STEPS];
        for (int i = 0; i < steps; ++i) {
            const double l = s * s;
            q[i] = c[0] + c[1] * l + c[2] * l * l;
            s = fabs(q[i] * s);
            if (!(s <= 1e6)) { b.ok = false; return b; }
            if (s > b.x) b.x = s;
            if (fabs(q[i]) > b.q) b.q = fabs(q[i]);
            double p = 1.0;
            for (int k = i; k >= 0; --k) {
                p *= fabs(q[k]);
                if (p > b.r[i - k + 1]) b.r[i - k + 1] = p;
            }
        }
    }
    // beyond 16 the fp16 planes of X, A (256) and A Q would lose the bits the smaller values need
    if (!(b.x <= 16.0) || !(b.q <= 1e4)) b.ok = false;
    return b;
}

float pow2_scale(double bound)      // largest power of two that keeps bound below 2^15 (fp16 ends at 2^16: a factor two of slack)
{
    int e;
    (void)frexp(bound > 0.0 ? bound : 1.0, &e);
    return ldexpf(1.0f, 15 - e);
}

float x_room(const Bounds& b, int steps)        // (x_shift)
{
    double grow = 1.0;
    for (int h = 1; h <= steps; ++h) grow = b.r[h] > grow ? b.r[h] : grow;
    return (float)(b.x / grow);
}

// Steps a hop of every matrix of a chunk.  Allowed, with g = max |Q|^2 (a^2 = 11.9 for the usual coefficients) the growth of the smallest
// eigenvalues' relative error a further step:
//   fp32: two from n = 2 m and m = 256 on (it saves a fifth there; nearer to square less than 15 %, in small matrices nothing, and the error
//         grows: 128 x 131: 2.6e-6 of the exact result against 1.4e-6 step by step, 70 x 600: 2.5e-6 against 1.6e-6);
//   bf16: 2^-22 g^(h-1) <= 5e-3, five steps (worst case measured 6e-4, a matrix dominated by one direction; the result's rounding: 1.7e-3);
//   fp16: 2^-22 g^(h-1) <= 5e-5, three steps (worst case measured 1e-4, rank one; the rounding: 2e-4).
// Of one limit for the whole chunk the cheapest is taken: the work, and 6.5 us for each launch of the matrix that has most of them.
bool hops_in_f32(const Shape& s) { return s.m >= 256 && s.n >= 2 * s.m; }

int hop_cap(const Shape& s, int steps, int dtype, double g)
{
    const double most = dtype == MP_DTYPE_F32 ? (hops_in_f32(s) ? 16.0 : 1.0) : dtype == MP_DTYPE_F16 ? 200.0 : 20000.0;
    int h = 1;
    for (double e = g > 1.5 ? g : 1.5; h < steps && e <= most && (dtype != MP_DTYPE_F32 || h < 2); e *= g > 1.5 ? g : 1.5) ++h;
    return h;
}

// work: operations of plane products, at 0.4 PFLOP/s (1024 x 1024 x 1024 reach 0.25, large ones 1.0)
void plan_hops(const Shape* s, int k, int steps, int dtype, int planes, const Bounds& bd, int* hop)
{
    const double g = bd.q * bd.q;
    double best = 1e300;
    for (int h = 1; h <= steps; ++h) {
        int use[MAX_MAT];
        bool more = h == 1;
        double work = 0.0;
        int launches = 0;
        for (int q = 0; q < k; ++q) {
            int mine = 2;
            const int cap = hop_cap(s[q], steps, dtype, g);
            use[q] = h < cap ? h : cap;
            more = more || use[q] == h;
            const double m = (double)s[q].m, n = (double)s[q].n;
            for (int left = steps; left > 0; left -= use[q]) {
                const int len = left < use[q] ? left : use[q];
                // (the first hop of a one-plane matrix: one product for the Gram matrix, two for the last one)
                work += m * m * ((left == steps && planes == 1 ? 1.0 + 2.0 * 2.0 : 3.0 * 3.0) * n + 3.0 * (4.0 * len - 3.0) * m);
                mine += len == 1 ? 3 : 3 * len + 1;       // Gram, apply; Q a step; T (and R), A between steps; R behind the last
            }
            launches = mine > launches ? mine : launches;
        }
        if (!more) break;        // (no matrix may take that many)
        const double cost = work / 0.4e15 + launches * 6.5e-6;
        if (cost < best * 0.999) {
            best = cost;
            for (int q = 0; q < k; ++q) hop[q] = use[q];
        }
    }
}

size_t up(size_t v) { return (v + 255) & ~(size_t)255; }
size_t image(int64_t rows, int64_t k) { return up((size_t)rows * chunks(k) * 128); }

struct Buffers { char *X, *XT, *XT2, *A, *T, *P[3]; double* sums; float* r; };

int norm_blocks(const Shape& s)
{
    const int64_t b = (s.rows * s.cols + 4095) / 4096;
    return (int)(b < MAX_NORM_BLOCKS ? (b > 0 ? b : 1) : MAX_NORM_BLOCKS);
}

// (what any schedule may use: the size does not depend on the coefficients)
size_t layout(const Shape& s, int steps, int dtype, char* base, Buffers* b)
{
    const bool chain = steps > 1 && (dtype != MP_DTYPE_F32 || hops_in_f32(s));
    size_t at = 0;
    auto take = [&](size_t n) {
        char* p = base ? base + at : nullptr;
        at += n;
        return p;
    };
    Buffers d;
    d.sums = reinterpret_cast<double*>(take(up(norm_blocks(s) * sizeof(double))));
    d.r = reinterpret_cast<float*>(take(256));
    d.X = take(image(s.m, s.n));
    d.XT = take(image(s.n, s.m));
    d.XT2 = steps > 1 ? take(image(s.n, s.m)) : nullptr;
    d.A = take(image(s.m, s.m));
    d.T = chain ? take(image(s.m, s.m)) : nullptr;
    d.P[0] = take(image(s.m, s.m));
    d.P[1] = chain ? take(image(s.m, s.m)) : nullptr;
    d.P[2] = chain ? take(image(s.m, s.m)) : nullptr;
    if (b) *b = d;
    return at;
}

constexpr int CUS = 256;

// What a launch does: tile shape, leading tiles taken whole, and the length of K's segments for the others (kmax: not cut).
struct Plan { int shape, whole, seg; };
// Tile shapes.  cyc: cycles of a chunk on one CU (three plane products) with all CUs at work, as measured; epi: of the epilogue.
struct TileShape { int tm, tn; double cyc, epi; };
constexpr int NSHAPES = 4;
constexpr TileShape SHAPES[NSHAPES] = {{256, 128, 1900.0, 12000.0}, {128, 128, 1150.0, 6500.0}, {64, 64, 450.0, 4500.0}, {32, 32, 210.0, 1500.0}};
// accumulators of the cut tiles
constexpr size_t PART_BYTES = (size_t)96 << 20;
constexpr int MAX_CUT = 32;

// Estimated cycles of the launch for every shape and cut; the cheapest is taken.  A cut sends the accumulators through memory (there and back
// at ~2000 bytes a cycle of the chip) and takes another launch (~10 000 cycles).
Plan plan_of(const Prob* p, int count, int products)
{
    Plan best{-1, 0, 0};
    double best_cost = 1e300;
    for (int s = 0; s < NSHAPES; ++s) {
        int64_t tiles = 0, units = 0;
        int kmin = 1 << 30, kmax = 0;
        for (int i = 0; i < count; ++i) {
            const int t = tiles_of(p[i].M, p[i].N, p[i].sym, SHAPES[s].tm, SHAPES[s].tn);
            tiles += t;
            units += (int64_t)t * p[i].kc;
            kmin = p[i].kc < kmin ? p[i].kc : kmin;
            kmax = p[i].kc > kmax ? p[i].kc : kmax;
        }
        if (tiles > (1 << 28)) continue;
        const double cyc = SHAPES[s].cyc * products / 3.0, epi = SHAPES[s].epi, slot = (double)SHAPES[s].tm * SHAPES[s].tn * 4.0;
        const bool equal = kmin == kmax;
        for (int cut = 1; cut <= MAX_CUT && (cut == 1 || kmax / cut >= 4); ++cut) {
            const int seg = (kmax + cut - 1) / cut;
            for (int keep = 0; keep < 2; ++keep) {       // equal lengths: whole rounds uncut, only what is left cut
                if (keep && (!equal || cut == 1 || tiles < CUS)) continue;
                const int64_t whole = cut == 1 ? tiles : keep ? tiles / CUS * CUS : 0, rest = tiles - whole;
                double c;
                int64_t items = 0;
                if (equal) {
                    items = rest * ((kmax + seg - 1) / seg);
                    c = (double)((whole + CUS - 1) / CUS) * (kmax * cyc + epi) + (double)((items + CUS - 1) / CUS) * (seg * cyc + epi);
                } else {        // rounds of mixed lengths: the mean load and a part of the longest item
                    for (int i = 0; i < count; ++i)
                        items += (int64_t)tiles_of(p[i].M, p[i].N, p[i].sym, SHAPES[s].tm, SHAPES[s].tn) * ((p[i].kc + seg - 1) / seg);
                    const double mean = ((double)units * cyc + (double)items * epi) / CUS, one = seg * cyc + epi;
                    c = items <= CUS ? one : mean + 0.6 * one;
                }
                if (cut > 1) {
                    if (rest == 0 || (double)items * slot > (double)PART_BYTES) continue;
                    c += 2.0 * (double)items * slot / 2000.0 + 10000.0;
                }
                if (c < best_cost) {
                    best_cost = c;
                    best = Plan{s, (int)whole, seg};
                }
            }
        }
    }
    return best;
}

template <int WM, int WN, int PL, int PR, int NS, bool KW, bool LL>
int launch_ring(const Probs& a, double flops, hipStream_t stream)
{
    static mp::DynLds dyn;
    constexpr int TM = KW ? 32 * WM : 64 * WM, TN = KW ? 32 * WN : 64 * WN, RINGS = KW ? 4 : 1;
    constexpr size_t ring = (size_t)RINGS * NS * 64 * (TM * PL + TN * PR), tile = (size_t)RINGS * TM * (TN + TPAD) * sizeof(float);
    constexpr size_t smem = ring > tile ? ring : tile;
    if (!dyn.ensure(reinterpret_cast<const void*>(&ns_gemm_kernel<WM, WN, PL, PR, NS, KW, LL>), smem)) return MP_ELAUNCH;
    MP_LAUNCH("ns_gemm_kernel", flops, 0.0, (ns_gemm_kernel<WM, WN, PL, PR, NS, KW, LL>), dim3((unsigned)a.items), dim3(256), smem, stream, a);
    MP_CHECK_LAUNCH();
    if (a.whole < a.tiles) {
        MP_LAUNCH("ns_join_kernel", 0.0, 0.0, (ns_join_kernel<TM, TN>), dim3((unsigned)(a.tiles - a.whole) * (TM / 32)), dim3(256), 0, stream, a);
        MP_CHECK_LAUNCH();
    }
    return MP_OK;
}

// Depth of the ring: what 144 KB hold (at most 8 chunks) where the launch has one workgroup a CU at most, else half of that so that two
// share a CU (256 x 128 and the K-sharing 64 x 64: always one).
template <int WM, int WN, int PL, int PR, bool KW>
int launch_as(const Probs& a, double flops, hipStream_t stream)
{
    constexpr int lds = 147456, stage = KW ? 4 * 64 * 32 * (WM * PL + WN * PR) : 64 * 64 * (WM * PL + WN * PR);
    constexpr int deep = lds / stage < 8 ? lds / stage : 8, half = KW || WM * WN >= 8 ? deep : (lds / 2 / stage < 8 ? lds / 2 / stage : 8);
    if constexpr (PL == 2 && PR == 2) {
        bool ll = false;
        for (int i = 0; i < a.count; ++i) ll = ll || a.p[i].ll;
        // (in every tile shape: a small matrix keeps its product whatever else is in the list)
        if (ll && a.items <= CUS) return launch_ring<WM, WN, PL, PR, deep, KW, true>(a, flops, stream);
        if (ll) return launch_ring<WM, WN, PL, PR, half, KW, true>(a, flops, stream);
    }
    if (a.items <= CUS) return launch_ring<WM, WN, PL, PR, deep, KW, false>(a, flops, stream);
    return launch_ring<WM, WN, PL, PR, half, KW, false>(a, flops, stream);
}

// planes of the left and the right operands: (2, 2), (2, 1) or (1, 1)
int launch(Probs& a, int left, int right, hipStream_t stream)
{
    if (a.count == 0) return MP_OK;
    const int products = left + right - 1;
    const Plan pl = plan_of(a.p, a.count, products);
    if (pl.shape < 0) return MP_EUNSUPPORTED;
    const TileShape ts = SHAPES[pl.shape];
    int64_t tiles = 0, items = pl.whole;
    double flops = 0.0;
    a.equal = 1;
    for (int i = 0; i < a.count; ++i) {
        Prob& p = a.p[i];
        p.tiles_n = (p.N + ts.tn - 1) / ts.tn;
        p.tiles = tiles_of(p.M, p.N, p.sym, ts.tm, ts.tn);
        const int segs = (p.kc + pl.seg - 1) / pl.seg;
        p.seg = (p.kc + segs - 1) / segs;
        a.tile0[i] = (int)tiles;
        a.item0[i] = (int)items;
        tiles += p.tiles;
        items += (int64_t)p.tiles * segs;
        a.equal &= p.kc == a.p[0].kc;
        flops += 2.0 * products * p.M * p.N * 32.0 * p.kc * (p.sym ? 0.5 : 1.0);
    }
    for (int i = a.count; i < MAX_PROB; ++i) a.tile0[i] = a.item0[i] = 0x7fffffff;
    a.tiles = (int)tiles;
    a.whole = pl.whole;
    a.rest = a.tiles - a.whole;
    if (a.whole == a.tiles) items = tiles;
    else if (a.equal) items = a.whole + (int64_t)a.rest * ((a.p[0].kc + a.p[0].seg - 1) / a.p[0].seg);
    a.items = (int)items;
#define NS_SHAPES(PL, PR)                                                     \
    return pl.shape == 0   ? launch_as<4, 2, PL, PR, false>(a, flops, stream) \
           : pl.shape == 1 ? launch_as<2, 2, PL, PR, false>(a, flops, stream) \
           : pl.shape == 2 ? launch_as<2, 2, PL, PR, true>(a, flops, stream)  \
                           : launch_as<1, 1, PL, PR, true>(a, flops, stream)
    if (left == 2 && right == 2) NS_SHAPES(2, 2);
    if (left == 2) NS_SHAPES(2, 1);
    NS_SHAPES(1, 1);
#undef NS_SHAPES
}

struct Update { int on; double lr, mu, decay; int nesterov, scale; };

double update_scale(const Update& u, int64_t rows, int64_t cols)
{
    const double r = (double)rows, c = (double)cols;
    return u.scale == MP_MUON_SCALE_MATCH_RMS ? 0.2 * sqrt(r > c ? r : c) : u.scale == MP_MUON_SCALE_ORIGINAL ? sqrt(r > c ? r / c : 1.0) : 1.0;
}

// Which of the one-launch kernels a matrix is for: TINY_2 / TINY_8 (ns_tiny_kernel with that many columns a thread), SMALL_1 / SMALL_2 (blocks of
// 32 rows in ns_small_kernel; lds: what it needs), or none
enum Kind { NOT_SMALL, TINY_2, TINY_8, SMALL_1, SMALL_2 };
Kind kind_of(int64_t rows, int64_t cols, size_t* lds = nullptr)
{
    const Shape s = shape_of(rows, cols);
    if (s.m <= TINY_M && s.n <= 8 * TINY_THREADS) return s.n <= 2 * TINY_THREADS ? TINY_2 : TINY_8;
    if (s.m > 64 || s.n > 1024) return NOT_SMALL;
    const int mb = chunks(s.m), npc = chunks(s.n);
    const size_t need = (size_t)32 * mb * 128 * npc + small_s(mb) + 256;
    if (npc > 8 * small_nb(mb) || need > SMALL_LDS) return NOT_SMALL;
    if (lds) *lds = need;
    return mb == 1 ? SMALL_1 : SMALL_2;
}

bool all_small(int64_t count, const int64_t* rows, const int64_t* cols)
{
    for (int64_t i = 0; i < count; ++i)
        if (rows[i] > 0 && cols[i] > 0 && kind_of(rows[i], cols[i]) == NOT_SMALL) return false;
    return true;
}

template <int NC>
int launch_tiny(const Smalls& a, int dtype, double flops, double bytes, hipStream_t stream)
{
#define NS_TINY(DT) MP_LAUNCH("ns_tiny_kernel", flops, bytes, (ns_tiny_kernel<NC, DT>), dim3((unsigned)a.count), dim3(TINY_THREADS), 0, stream, a)
    if (dtype == MP_DTYPE_F32) NS_TINY(MP_DTYPE_F32);
    else if (dtype == MP_DTYPE_F16) NS_TINY(MP_DTYPE_F16);
    else NS_TINY(MP_DTYPE_BF16);
#undef NS_TINY
    MP_CHECK_LAUNCH();
    return MP_OK;
}

template <int MB, int DT>
int launch_small(const Smalls& a, double flops, double bytes, size_t lds, hipStream_t stream)
{
    static mp::DynLds dyn;
    if (!dyn.ensure(reinterpret_cast<const void*>(&ns_small_kernel<MB, DT>), SMALL_LDS)) return MP_ELAUNCH;
    MP_LAUNCH("ns_small_kernel", flops, bytes, (ns_small_kernel<MB, DT>), dim3((unsigned)a.count), dim3(512), lds, stream, a);
    MP_CHECK_LAUNCH();
    return MP_OK;
}
template <int MB>
int launch_small_of(const Smalls& a, int dtype, double flops, double bytes, size_t lds, hipStream_t stream)
{
    if (dtype == MP_DTYPE_F32) return launch_small<MB, MP_DTYPE_F32>(a, flops, bytes, lds, stream);
    if (dtype == MP_DTYPE_F16) return launch_small<MB, MP_DTYPE_F16>(a, flops, bytes, lds, stream);
    return launch_small<MB, MP_DTYPE_BF16>(a, flops, bytes, lds, stream);
}

// one launch for the matrices of each kind
int run_small(int64_t count, const void* const* in, void* const* out, float* const* mom, const int64_t* rows, const int64_t* cols, int dtype, int steps,
              const double* coef, double eps, const Bounds& bd, const Update& u, hipStream_t stream)
{
    Smalls a;
    a.nesterov = u.nesterov; a.update = u.on; a.steps = steps;
    a.mu = (float)u.mu; a.a = (float)coef[0]; a.b = (float)coef[1]; a.c = (float)coef[2]; a.eps = eps;
    a.sX = pow2_scale(bd.x); a.sA = pow2_scale(bd.x * bd.x); a.sQ = pow2_scale(bd.q); a.x_room = x_room(bd, steps);
    for (int kind = TINY_2; kind <= SMALL_2; ++kind)
        for (int64_t i = 0; i < count;) {
            size_t lds = 0;
            double elems = 0.0, flops = 0.0;
            for (a.count = 0; i < count && a.count < MAX_SMALL; ++i) {
                const Shape s = shape_of(rows[i], cols[i]);
                size_t need = 0;
                if (s.m <= 0 || kind_of(rows[i], cols[i], &need) != kind) continue;
                lds = need > lds ? need : lds;
                a.m[a.count++] = Small{in[i], mom ? mom[i] : nullptr, out[i], (int)rows[i], (int)cols[i], (float)(u.lr * update_scale(u, rows[i], cols[i])),
                                       (float)(1.0 - u.lr * u.decay)};
                elems += (double)s.m * s.n;
                flops += 6.0 * steps * s.m * s.m * (2.0 * s.n + s.m);
            }
            if (a.count == 0) break;
            const int rc = kind == TINY_2    ? launch_tiny<2>(a, dtype, flops, elems * 8.0, stream)
                           : kind == TINY_8  ? launch_tiny<8>(a, dtype, flops, elems * 8.0, stream)
                           : kind == SMALL_1 ? launch_small_of<1>(a, dtype, flops, elems * 8.0, lds, stream)
                                             : launch_small_of<2>(a, dtype, flops, elems * 8.0, lds, stream);
            if (rc) return rc;
        }
    return MP_OK;
}

// next chunk of matrices that have elements, from index i on: their indices (<= MAX_MAT)
int next_chunk(int64_t count, const int64_t* rows, const int64_t* cols, int64_t& i, int64_t* idx)
{
    int k = 0;
    for (; i < count && k < MAX_MAT; ++i)
        if (rows[i] > 0 && cols[i] > 0) idx[k++] = i;
    return k;
}

size_t chunk_bytes(const int64_t* rows, const int64_t* cols, const int64_t* idx, int k, int steps, int dtype)
{
    size_t bytes = 0, part = 0;
    for (int q = 0; q < k; ++q) {
        const Shape s = shape_of(rows[idx[q]], cols[idx[q]]);
        bytes += layout(s, steps, dtype, nullptr, nullptr);
        // cut tiles of any of its products (two m x m ones may share a launch): at most MAX_CUT segments of every tile
        part += (size_t)MAX_CUT * 2 * ((s.m + 255) / 256 * 256) * ((s.n + 255) / 256 * 256) * sizeof(float);
    }
    return bytes + up(part < PART_BYTES ? part : PART_BYTES);
}

int check_args(int64_t count, const int64_t* rows, const int64_t* cols, int dtype, int steps)
{
    if (count < 0 || (count > 0 && (!rows || !cols)) || steps < 1) return MP_EINVAL;
    if (dtype != MP_DTYPE_F32 && dtype != MP_DTYPE_F16 && dtype != MP_DTYPE_BF16) return MP_EUNSUPPORTED;
    if (steps > MAX_STEPS) return MP_EUNSUPPORTED;
    for (int64_t i = 0; i < count; ++i) {
        if (rows[i] < 0 || cols[i] < 0) return MP_EINVAL;
        const int64_t m = rows[i] < cols[i] ? rows[i] : cols[i], n = rows[i] < cols[i] ? cols[i] : rows[i];
        // (the last: units of a product are counted in 31 bits; such a matrix and its planes do not fit the card)
        if (m > 65536 || n > ((int64_t)1 << 21) || (double)m * (double)m * (double)n > 1125899906842624.0) return MP_EUNSUPPORTED;
    }
    return MP_OK;
}

int run_chunk(const void* const* in, void* const* out, float* const* mom, const int64_t* rows, const int64_t* cols, const int64_t* idx, int k,
              int dtype, int steps, const double* coef, double eps, const Bounds& bd, const Update& up_, char* ws, hipStream_t stream)
{
    Shape sh[MAX_MAT];
    Buffers bf[MAX_MAT];
    int hop[MAX_MAT];
    Mats a;
    a.count = k; a.dtype = dtype; a.nesterov = up_.nesterov; a.mu = (float)up_.mu; a.eps = eps;
    a.planes = dtype != MP_DTYPE_F32 && !mom ? 1 : 2;
    a.x_room = x_room(bd, steps);
    int64_t blocks = 0, tiles = 0;
    double elems = 0.0;
    for (int q = 0; q < k; ++q) sh[q] = shape_of(rows[idx[q]], cols[idx[q]]);
    plan_hops(sh, k, steps, dtype, a.planes, bd, hop);
    for (int q = 0; q < k; ++q) {
        ws += layout(sh[q], steps, dtype, ws, &bf[q]);
        Mat& m = a.m[q];
        const bool tall = sh[q].rows > sh[q].cols;
        m.g = in[idx[q]];
        m.mom = mom ? mom[idx[q]] : nullptr;
        m.sums = bf[q].sums;
        m.r = bf[q].r;
        m.P = reinterpret_cast<_Float16*>(tall ? bf[q].XT : bf[q].X);
        m.PT = reinterpret_cast<_Float16*>(tall ? bf[q].X : bf[q].XT);
        m.rows = (int)sh[q].rows; m.cols = (int)sh[q].cols;
        m.blocks = norm_blocks(sh[q]);
        a.blk0[q] = (int)blocks;
        a.tile0[q] = (int)tiles;
        blocks += m.blocks;
        tiles += ((sh[q].rows + 63) / 64) * ((sh[q].cols + 63) / 64);
        elems += (double)sh[q].rows * (double)sh[q].cols;
    }
    for (int q = k; q < MAX_MAT; ++q) a.blk0[q] = a.tile0[q] = 0x7fffffff;
    const double esz = dtype == MP_DTYPE_F32 ? 4.0 : 2.0;
#define NS_NORM(DT, MOM) \
    MP_LAUNCH("ns_norm_kernel", 2.0 * elems, elems * (esz + (mom ? 8.0 : 0.0)), (ns_norm_kernel<DT, MOM>), dim3((unsigned)blocks), dim3(256), 0, stream, a)
    if (dtype == MP_DTYPE_F32) {
        if (mom) NS_NORM(MP_DTYPE_F32, true);
        else NS_NORM(MP_DTYPE_F32, false);
    } else if (dtype == MP_DTYPE_F16) {
        if (mom) NS_NORM(MP_DTYPE_F16, true);
        else NS_NORM(MP_DTYPE_F16, false);
    } else {
        if (mom) NS_NORM(MP_DTYPE_BF16, true);
        else NS_NORM(MP_DTYPE_BF16, false);
    }
#undef NS_NORM
    MP_CHECK_LAUNCH();
    MP_LAUNCH("ns_planes_kernel", 2.0 * elems, elems * (esz + (mom ? 4.0 : 0.0) + 8.0), ns_planes_kernel, dim3((unsigned)tiles), dim3(256), 0, stream, a);
    MP_CHECK_LAUNCH();

    const float sX = pow2_scale(bd.x), sA = pow2_scale(bd.x * bd.x), sT = pow2_scale(bd.x * bd.x * bd.q), sQ = pow2_scale(bd.q);
    // Every matrix walks through its hops by itself; a launch takes the present stage of each, whatever it is, so that hops of different lengths
    // fill each other's launches (seven matrices up to 11988 x 1024, hops of two steps and of one: 23 products' launches in turns, 17 this way).
    enum Stage { GRAM, SQUARE, STEP, NEXT, APPLY, END };
    struct Walk {
        Stage at;
        int done, len, s, r, q;      // steps behind it, steps of this hop, step inside it, which P holds R / Q
        float sR;
        bool first;                  // X is still the input's planes (to be multiplied by r)
    } w[MAX_MAT];
    Probs g;
    g.fin_dtype = dtype;
    g.fin_update = up_.on;
    g.part = reinterpret_cast<float*>(ws);
    auto sym_prob = [&](int q, const void* L, const void* R, float sl, float sr, void* o, float so) {
        Prob p{};
        p.L = static_cast<const _Float16*>(L);
        p.R = static_cast<const _Float16*>(R);
        p.out = p.outT = static_cast<_Float16*>(o);
        p.M = p.N = (int)sh[q].m;
        p.kc = p.oc = p.otc = chunks(sh[q].m);
        p.sym = 1;
        p.alpha = 1.0f / (sl * sr);
        p.so = so;
        return p;
    };
    for (int q = 0; q < k; ++q) w[q] = Walk{GRAM, 0, steps < hop[q] ? steps : hop[q], 0, 0, 0, sQ, true};
    for (;;) {
        bool more = false;
        int planes[MAX_MAT];        // of the operands: 0 (2, 2), 1 (1, 1), 2 (2, 1); one plane: the input's
        for (int q = 0; q < k; ++q) planes[q] = w[q].first && a.planes == 1 ? (w[q].at == GRAM ? 1 : w[q].at == APPLY ? 2 : 0) : 0;
        for (int kind = 0; kind < 3; ++kind) {
            g.count = 0;
            for (int q = 0; q < k; ++q) {
                Walk& v = w[q];
                if (v.at == END || kind != planes[q]) continue;
                more = true;
                if (v.at == GRAM) {                   // A = X X^T
                    Prob p = sym_prob(q, bf[q].X, bf[q].X, v.first ? 1.0f : sX, v.first ? 1.0f : sX, bf[q].A, sA);
                    p.kc = chunks(sh[q].n);
                    p.rdev = bf[q].r + (v.first ? 0 : 2);
                    p.rpow = 2;
                    g.p[g.count++] = p;
                } else if (v.at == SQUARE) {          // Q = a I + b A + c A^2
                    v.q = v.s == 0 ? 0 : (v.r + 1) % 3;
                    Prob p = sym_prob(q, bf[q].A, bf[q].A, sA, sA, bf[q].P[v.q], sQ);
                    p.alpha *= (float)coef[2];
                    p.C = reinterpret_cast<const _Float16*>(bf[q].A);
                    p.cb = (float)(coef[1] / sA);
                    p.ca = (float)coef[0];
                    p.ll = dtype == MP_DTYPE_F32 && sh[q].m < 128;
                    g.p[g.count++] = p;
                    if (v.s == 0) { v.r = v.q; v.sR = sQ; }
                } else if (v.at == STEP) {            // T = A Q (another step follows), R = Q R: independent
                    if (v.s + 1 < v.len) g.p[g.count++] = sym_prob(q, bf[q].A, bf[q].P[v.q], sA, sQ, bf[q].T, sT);
                    if (v.s > 0) {
                        const int to = 3 - v.r - v.q;
                        const float so = pow2_scale(bd.r[v.s + 1]);
                        g.p[g.count++] = sym_prob(q, bf[q].P[v.q], bf[q].P[v.r], sQ, v.sR, bf[q].P[to], so);
                        v.r = to;
                        v.sR = so;
                    }
                } else if (v.at == NEXT) {            // A = T Q
                    g.p[g.count++] = sym_prob(q, bf[q].T, bf[q].P[v.q], sT, sQ, bf[q].A, sA);
                } else {                              // X <- R X
                    Prob p{};
                    p.L = reinterpret_cast<const _Float16*>(bf[q].P[v.r]);
                    p.R = reinterpret_cast<const _Float16*>(bf[q].XT);
                    p.M = (int)sh[q].m;
                    p.N = (int)sh[q].n;
                    p.kc = chunks(sh[q].m);
                    p.alpha = 1.0f / (v.sR * (v.first ? 1.0f : sX));
                    const bool last = v.done + v.len == steps;
                    if (v.first || last) { p.rdev = bf[q].r + (!v.first ? 2 : last ? 0 : 1); p.rpow = 1; }       // (between hops: planes to planes)
                    if (last) {
                        p.fin = out[idx[q]];
                        p.fin_t = sh[q].rows > sh[q].cols;
                        if (up_.on) {
                            p.fmul = (float)(up_.lr * update_scale(up_, sh[q].rows, sh[q].cols));
                            p.fdecay = (float)(1.0 - up_.lr * up_.decay);
                        }
                    } else {
                        p.out = reinterpret_cast<_Float16*>(bf[q].X);
                        p.outT = reinterpret_cast<_Float16*>(bf[q].XT2);
                        p.oc = chunks(sh[q].n);
                        p.otc = chunks(sh[q].m);
                        p.so = sX;
                        char* t = bf[q].XT;
                        bf[q].XT = bf[q].XT2;
                        bf[q].XT2 = t;
                    }
                    g.p[g.count++] = p;
                }
            }
            const int rc = kind == 0 ? launch(g, 2, 2, stream) : kind == 1 ? launch(g, 1, 1, stream) : launch(g, 2, 1, stream);
            if (rc) return rc;
        }
        if (!more) return MP_OK;
        for (int q = 0; q < k; ++q) {
            Walk& v = w[q];
            if (v.at == GRAM || v.at == STEP) v.at = v.at == GRAM ? SQUARE : v.s + 1 < v.len ? NEXT : APPLY;
            else if (v.at == SQUARE) v.at = v.len == 1 ? APPLY : STEP;
            else if (v.at == NEXT) { ++v.s; v.at = SQUARE; }
            else if (v.at == APPLY) {
                v.done += v.len;
                v.len = steps - v.done < hop[q] ? steps - v.done : hop[q];
                v.s = 0;
                v.first = false;
                v.at = v.len ? GRAM : END;
            }
        }
    }
}

int run_all(int64_t count, const void* const* in, void* const* out, float* const* mom, const int64_t* rows, const int64_t* cols, int dtype, int steps,
            const double* coef, double eps, const Update& u, void* workspace, size_t workspace_bytes, hipStream_t stream)
{
    int rc = check_args(count, rows, cols, dtype, steps);
    if (rc) return rc;
    if (count == 0) return MP_OK;
    if (!in || !out || !coef || !(eps >= 0.0) || (u.on && !mom)) return MP_EINVAL;
    if (!isfinite(coef[0]) || !isfinite(coef[1]) || !isfinite(coef[2])) return MP_EINVAL;
    const Bounds bd = bounds_of(steps, coef);
    if (!bd.ok) return MP_EUNSUPPORTED;
    int64_t idx[MAX_MAT];
    const bool small = all_small(count, rows, cols);
    for (int64_t i = 0; i < count;) {       // everything is checked before anything is launched
        const int k = next_chunk(count, rows, cols, i, idx);
        if (k == 0) continue;
        for (int q = 0; q < k; ++q)
            if (!in[idx[q]] || !out[idx[q]] || (u.on && !mom[idx[q]])) return MP_EINVAL;
        if (small) continue;
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)) return MP_EWORKSPACE;
        if (chunk_bytes(rows, cols, idx, k, steps, dtype) > workspace_bytes) return MP_EWORKSPACE;
    }
    if (small) return run_small(count, in, out, mom, rows, cols, dtype, steps, coef, eps, bd, u, stream);
    for (int64_t i = 0; i < count;) {
        const int k = next_chunk(count, rows, cols, i, idx);
        if (k == 0) continue;
        rc = run_chunk(in, out, mom, rows, cols, idx, k, dtype, steps, coef, eps, bd, u, static_cast<char*>(workspace), stream);
        if (rc) return rc;
    }
    return MP_OK;
}

}  // namespace

extern "C" size_t mp_orthogonalize_workspace_bytes(int64_t count, const int64_t* rows, const int64_t* cols, int dtype, int steps)
{
    if (check_args(count, rows, cols, dtype, steps)) return 0;
    size_t most = 0;
    int64_t idx[MAX_MAT];
    if (all_small(count, rows, cols)) return 0;
    for (int64_t i = 0; i < count;) {
        const int k = next_chunk(count, rows, cols, i, idx);
        const size_t b = k ? chunk_bytes(rows, cols, idx, k, steps, dtype) : 0;
        most = b > most ? b : most;
    }
    return most;
}

extern "C" int mp_orthogonalize(int64_t count, const void* const* in, void* const* out, const int64_t* rows, const int64_t* cols, int dtype, int steps,
                                const double* coefficients, double eps, void* workspace, size_t workspace_bytes, mp_stream_t stream)
{
    const Update none{};
    return run_all(count, in, out, nullptr, rows, cols, dtype, steps, coefficients, eps, none, workspace, workspace_bytes, mp_stream(stream));
}

extern "C" int mp_muon_step(int64_t count, void* const* params, const void* const* grads, float* const* momentum, const int64_t* rows,
                            const int64_t* cols, int dtype, double lr, double mu, int nesterov, double weight_decay, int scale, int steps,
                            const double* coefficients, double eps, void* workspace, size_t workspace_bytes, mp_stream_t stream)
{
    if (count > 0 && !momentum) return MP_EINVAL;
    if (scale != MP_MUON_SCALE_NONE && scale != MP_MUON_SCALE_ORIGINAL && scale != MP_MUON_SCALE_MATCH_RMS) return MP_EINVAL;
    Update u{};
    u.on = 1; u.lr = lr; u.mu = mu; u.decay = weight_decay; u.nesterov = nesterov ? 1 : 0; u.scale = scale;
    return run_all(count, grads, params, momentum, rows, cols, dtype, steps, coefficients, eps, u, workspace, workspace_bytes, mp_stream(stream));
}
