// Newton-Schulz orthogonalisation of a list of matrices, and the Muon update built on it (gfx950).
//
//   X = U / max(|U|_F, eps);  steps times:  A = X X^T,  X <- (a I + b A + c A^2) X      (U with more rows than columns: of U^T)
//
// MATHEMATICS.  With Q = a I + b A + c A^2 (symmetric, a polynomial of A) the next step's Gram matrix is A' = Q A Q: it need not be formed
// from X again.  So a HOP of h steps runs on the small side only (m <= n):
//     A = X X^T;   Q_i = a I + b A_i + c A_i^2,   A_{i+1} = (A_i Q_i) Q_i,   R_i = Q_i R_{i-1};   X <- R_h X
// at 3 m^2 n + (4 h - 3) m^3 multiply-adds (symmetric products: the lower half only, mirrored) instead of h (3 m^2 n + m^3).  An extra step in
// a hop multiplies the relative error of the smallest eigenvalues by a^2 ~ 12 (they grow by that, the rounding error of A does not shrink):
// fp32 results take hops of at most two steps (error within 2x of the step-by-step form in fp32), 16-bit results of up to all five
// (measured worst case 6e-4 relative for a matrix dominated by one direction, half a step of bf16 is 4e-3); hop_plan() takes the
// cheapest schedule.
//
// ARITHMETIC.  fp32 accuracy from the fp16 matrix cores: an operand is kept as two fp16 planes, x 2^k = h + l (h = fp16(x 2^k), l the rest:
// 22 to 24 bits), a product is h h + h l + l h accumulated in fp32 -- three products at the fp16 rate (2.5 PFLOP/s) against one at the
// fp32 rate (0.16).  The power of two puts the largest entry below 2^15, so l keeps its bits down to entries of 2^-24 of that.
//
// All matrices of a call go through each stage in ONE launch (problem list in the kernel arguments): a call is 2 + 3..17 launches
// whatever the number of matrices.  Operand image: row r = chunks of 32 k, each [h: 32 fp16][l: 32 fp16] (128 bytes); columns up to the
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
constexpr int MAX_NORM_BLOCKS = 512;   // partial sums of squares per matrix

struct Prob {                // out = (alpha acc + cb C + ca I), acc = L R^T over kc chunks of 32
    const _Float16* L;
    const _Float16* R;
    const _Float16* C;       // planes [M][oc] or NULL
    _Float16* out;           // planes [M][oc] or NULL
    _Float16* outT;          // planes [N][otc] or NULL
    void* fin;               // [M, N] of the result type or NULL
    const float* rdev;       // alpha is multiplied by rdev^rpow
    int M, N, kc, oc, otc, rpow, sym, tiles_n;
    float alpha, cb, ca, so, fmul, fdecay;
    int tile0;               // first workgroup
};
struct Probs {
    Prob p[MAX_PROB];
    int count, splits, kper;      // splits > 1: chunks of kper, partial accumulators to memory
    int fin_dtype, fin_update;    // fin_update: fin = fdecay * fin - fmul * value
    float* part;
};
static_assert(sizeof(Probs) <= 3584, "travels in the kernel arguments");

__host__ __device__ inline int chunks(int64_t k) { return (int)((k + 31) / 32); }

// 16 bytes a lane straight into LDS (lane i at dst + 16 i); waited for by wait_vm0 in front of a barrier
__device__ __forceinline__ void to_lds16(const void* src, void* dst)
{
    const unsigned l = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) void*)dst);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(l) : "memory");
}
__device__ __forceinline__ void wait_vm0() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
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

struct TileAt { int prob, m0, n0, split, index; };

__device__ __forceinline__ TileAt find_tile(const Probs& a, int block, int TM, int TN)
{
    TileAt t;
    int i = 0;
    while (i + 1 < a.count && block >= a.p[i + 1].tile0) ++i;       // uniform: scalar loop over <= 24 entries
    t.prob = i;
    const int local = block - a.p[i].tile0;
    t.split = local % a.splits;
    const int tile = local / a.splits;
    int ti, tj;
    if (a.p[i].sym) {        // lower triangle: tile = ti (ti + 1) / 2 + tj
        ti = (int)((sqrtf(8.0f * (float)tile + 1.0f) - 1.0f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        while (ti * (ti + 1) / 2 > tile) --ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        ti = tile / a.p[i].tiles_n;
        tj = tile % a.p[i].tiles_n;
    }
    t.m0 = ti * TM;
    t.n0 = tj * TN;
    t.index = block / a.splits;       // (tile0 is a multiple of splits)
    return t;
}

__device__ __forceinline__ void put_planes(_Float16* img, int row, int nchunk, int col, const float (&v)[4], int n)
{
    half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = (_Float16)v[e];
        l[e] = (_Float16)(v[e] - (float)h[e]);
    }
    _Float16* q = img + ((size_t)row * nchunk + (col >> 5)) * 64 + (col & 31);
    if (n == 4) {
        *reinterpret_cast<half4*>(q) = h;
        *reinterpret_cast<half4*>(q + 32) = l;
    } else
        for (int e = 0; e < n; ++e) {
            q[e] = h[e];
            q[32 + e] = l[e];
        }
}

// Wave (wm, wn) of 2 x 2 holds WM x WN blocks of 32 x 32; block register r of lane q: row (r & 3) + 8 (r >> 2) + 4 (q >> 5), column q & 31.
template <int WM, int WN>
__device__ __forceinline__ void epilogue(const Probs& a, const Prob& p, const TileAt& t, float16v (&acc)[WM][WN])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * WM * 32, wn = (wave & 1) * WN * 32;
    float alpha = p.alpha;
    if (p.rpow) {
        const float r = *p.rdev;
        alpha *= p.rpow == 2 ? r * r : r;
    }
    const int padN = p.oc * 32, padM = p.otc * 32;
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j) {
            const int col = t.n0 + wn + j * 32 + (lane & 31);
#pragma unroll
            for (int rg = 0; rg < 4; ++rg) {
                const int row0 = t.m0 + wm + i * 32 + rg * 8 + (lane >> 5) * 4;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = row0 + e;
                    float x = alpha * acc[i][j][rg * 4 + e];
                    if (p.C && row < p.M && col < p.N) {
                        const _Float16* c = p.C + ((size_t)row * p.oc + (col >> 5)) * 64 + (col & 31);
                        x += p.cb * ((float)c[0] + (float)c[32]);
                    }
                    if (row == col) x += p.ca;
                    v[e] = x;
                }
                if (p.fin) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = row0 + e;
                        if (row < p.M && col < p.N) {
                            const size_t at = (size_t)row * p.N + col;
                            float x = v[e];
                            if (a.fin_update) x = p.fdecay * load_any(p.fin, a.fin_dtype, at) - p.fmul * x;
                            store_fin(p.fin, a.fin_dtype, at, x);
                        }
                    }
                }
                if (p.out) {
                    // columns N .. padN - 1 are written as zeros.  A symmetric result takes its lower half: row >= column here, mirrored below.
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = row0 + e;
                        if (row < p.M && col < padN && (!p.sym || row >= col)) {
                            const float x = col < p.N ? v[e] * p.so : 0.0f;
                            const _Float16 h = (_Float16)x;
                            _Float16* q = p.out + ((size_t)row * p.oc + (col >> 5)) * 64 + (col & 31);
                            q[0] = h;
                            q[32] = (_Float16)(x - (float)h);
                        }
                    }
                }
                if (p.outT && col < p.N) {
                    float y[4];
                    bool all = row0 + 3 < padM;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[e] = row0 + e < p.M ? v[e] * p.so : 0.0f;
                        if (p.sym && row0 + e <= col) all = false;        // (row == col was written above)
                    }
                    if (all) put_planes(p.outT, col, p.otc, row0, y, 4);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (row0 + e < padM && (!p.sym || row0 + e > col)) {
                                const _Float16 h = (_Float16)y[e];
                                _Float16* q = p.outT + ((size_t)col * p.otc + ((row0 + e) >> 5)) * 64 + ((row0 + e) & 31);
                                q[0] = h;
                                q[32] = (_Float16)(y[e] - (float)h);
                            }
                }
            }
        }
}

// One tile of (64 WM) x (64 WN), four waves, two LDS buffers of one 32-k chunk: chunk c + 1 is on its way into one while c is multiplied
// out of the other (one barrier a chunk: whoever passed it has finished with the buffer that is filled next).  A row of a buffer is 128
// bytes; its 16-byte unit u lies at u ^ (row & 7), so that the 32 rows a fragment read touches meet each bank group equally often.
template <int WM, int WN>
__global__ __launch_bounds__(256) void ns_gemm_kernel(Probs a)
{
    constexpr int TM = 64 * WM, TN = 64 * WN, STAGE = (TM + TN) * 128;
    __shared__ __align__(16) char lds[2 * STAGE];
    const TileAt t = find_tile(a, blockIdx.x, TM, TN);
    const Prob& p = a.p[t.prob];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c0 = t.split * a.kper, c1 = a.splits == 1 ? p.kc : (c0 + a.kper < p.kc ? c0 + a.kper : p.kc);

    // load unit of this lane: rows (8 a wave and instruction), 16-byte unit of the row's chunk (swizzled at the source)
    const int lr = wave * 8 + (lane >> 3), lu = (lane & 7) ^ (lr & 7);
    const char* srcL[2 * WM];
    const char* srcR[2 * WN];
#pragma unroll
    for (int i = 0; i < 2 * WM; ++i) {
        int row = t.m0 + lr + 32 * i;
        row = row < p.M ? row : p.M - 1;
        srcL[i] = reinterpret_cast<const char*>(p.L) + ((size_t)row * p.kc + c0) * 128 + lu * 16;
    }
#pragma unroll
    for (int i = 0; i < 2 * WN; ++i) {
        int row = t.n0 + lr + 32 * i;
        row = row < p.N ? row : p.N - 1;
        srcR[i] = reinterpret_cast<const char*>(p.R) + ((size_t)row * p.kc + c0) * 128 + lu * 16;
    }
    auto fetch = [&](int buf) {
        char* d = lds + buf * STAGE + wave * 1024;
#pragma unroll
        for (int i = 0; i < 2 * WM; ++i) {
            to_lds16(srcL[i], d + i * 4096);
            srcL[i] += 128;
        }
#pragma unroll
        for (int i = 0; i < 2 * WN; ++i) {
            to_lds16(srcR[i], d + TM * 128 + i * 4096);
            srcR[i] += 128;
        }
    };
    float16v acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    const int fr = lane & 31, fh = lane >> 5;                  // fragment row, k half
    const int rowL = (wave >> 1) * WM * 32 + fr, rowR = (wave & 1) * WN * 32 + fr;      // (32 i more: same row & 7)
    if (c0 < c1) fetch(0);
    for (int c = c0; c < c1; ++c) {
        wait_vm0();
        lds_barrier();
        const char* s = lds + ((c - c0) & 1) * STAGE;
        if (c + 1 < c1) fetch((c - c0 + 1) & 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            half8 fl[WM][2], fq[WN][2];
#pragma unroll
            for (int pl = 0; pl < 2; ++pl) {
                const int u = pl * 4 + ks * 2 + fh;
#pragma unroll
                for (int i = 0; i < WM; ++i) fl[i][pl] = *reinterpret_cast<const half8*>(s + (rowL + 32 * i) * 128 + ((u ^ (rowL & 7)) * 16));
#pragma unroll
                for (int j = 0; j < WN; ++j) fq[j][pl] = *reinterpret_cast<const half8*>(s + TM * 128 + (rowR + 32 * j) * 128 + ((u ^ (rowR & 7)) * 16));
            }
            // the small products first; a block's three stay WM * WN apart (independent accumulators between them)
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int i = 0; i < WM; ++i)
#pragma unroll
                    for (int j = 0; j < WN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl[i][k == 0], fq[j][k == 1], acc[i][j], 0, 0, 0);
        }
    }
    if (a.splits > 1) {
        float4* o = reinterpret_cast<float4*>(a.part) + (size_t)blockIdx.x * (WM * WN * 4 * 256) + threadIdx.x;
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    o[((i * WN + j) * 4 + r) * 256] = make_float4(acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]);
        return;
    }
    epilogue<WM, WN>(a, p, t, acc);
}

// the split tiles' accumulators added in the order of the splits, then the same epilogue
template <int WM, int WN>
__global__ __launch_bounds__(256) void ns_join_kernel(Probs a)
{
    const TileAt t = find_tile(a, blockIdx.x * a.splits, 64 * WM, 64 * WN);
    float16v acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    const float4* o = reinterpret_cast<const float4*>(a.part) + (size_t)blockIdx.x * a.splits * (WM * WN * 4 * 256) + threadIdx.x;
    for (int s = 0; s < a.splits; ++s, o += WM * WN * 4 * 256)
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float4 v = o[((i * WN + j) * 4 + r) * 256];
                    acc[i][j][4 * r] += v.x;
                    acc[i][j][4 * r + 1] += v.y;
                    acc[i][j][4 * r + 2] += v.z;
                    acc[i][j][4 * r + 3] += v.w;
                }
    epilogue<WM, WN>(a, a.p[t.prob], t, acc);
}

// ---- momentum, norm, planes -------------------------------------------------------------------------------------------------------
struct Mat {
    const void* g;       // gradient / input [rows, cols]
    float* mom;          // momentum or NULL
    double* sums;        // partial sums of squares
    float* r;            // X = (U 2^e) * r
    _Float16* P;         // planes of U 2^e, [rows][chunks(cols)]
    _Float16* PT;        // of its transpose, [cols][chunks(rows)]
    int rows, cols, blocks, blk0, tile0;
};
struct Mats {
    Mat m[MAX_MAT];
    int count, dtype, nesterov;
    float mu;
    double eps;
};
static_assert(sizeof(Mats) <= 3584, "travels in the kernel arguments");

// momentum (if any) updated and the sums of squares of the update's direction, one partial sum per workgroup (fp64: the squares of fp32
// numbers neither overflow nor vanish there)
__global__ __launch_bounds__(256) void ns_norm_kernel(Mats a)
{
    __shared__ double s_acc[4];
    int i = 0;
    while (i + 1 < a.count && (int)blockIdx.x >= a.m[i + 1].blk0) ++i;
    const Mat& m = a.m[i];
    const size_t n = (size_t)m.rows * m.cols;
    const int b = blockIdx.x - m.blk0;
    double s = 0.0;
    for (size_t e = (size_t)b * 256 + threadIdx.x; e < n; e += (size_t)m.blocks * 256) {
        float u = load_any(m.g, a.dtype, e);
        if (m.mom) {
            float v = m.mom[e];
            v = v + (1.0f - a.mu) * (u - v);
            m.mom[e] = v;
            u = a.nesterov ? u + a.mu * (v - u) : v;
        }
        s += (double)u * (double)u;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) s_acc[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) m.sums[b] = (s_acc[0] + s_acc[1]) + (s_acc[2] + s_acc[3]);
}

// 64 x 64 elements of a matrix into both plane images.  The power of two 2^e takes the norm into [2^13, 2^14): exact, and every entry
// below 2^14; the division by the norm itself waits for the products' epilogues (r).
__global__ __launch_bounds__(256) void ns_planes_kernel(Mats a)
{
    __shared__ double s_acc[4];
    __shared__ float tile[64][65];
    int i = 0;
    while (i + 1 < a.count && (int)blockIdx.x >= a.m[i + 1].tile0) ++i;
    const Mat& m = a.m[i];
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
    const int local = blockIdx.x - m.tile0, tn = (m.cols + 63) / 64;
    const int r0 = (local / tn) * 64, c0 = (local % tn) * 64;
    if (local == 0 && threadIdx.x == 0) *m.r = (float)(1.0 / ldexp(norm > a.eps || norm != norm ? norm : a.eps, e));
    const int tc = threadIdx.x & 63, tr = threadIdx.x >> 6;
    for (int k = 0; k < 64; k += 4) {
        const int r = r0 + k + tr, c = c0 + tc;
        float u = 0.0f;
        if (r < m.rows && c < m.cols) {
            const size_t at = (size_t)r * m.cols + c;
            u = load_any(m.g, a.dtype, at);
            if (m.mom) {
                const float v = m.mom[at];
                u = a.nesterov ? u + a.mu * (v - u) : v;
            }
            u = ldexpf(u, e);
        }
        tile[k + tr][tc] = u;
    }
    __syncthreads();
    const int pc = chunks(m.cols), ptc = chunks(m.rows);
    for (int q = threadIdx.x; q < 64 * 16; q += 256) {
        const int a4 = (q & 15) * 4, b = q >> 4;
        float v[4];
        if (r0 + b < m.rows && c0 + a4 < pc * 32) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = tile[b][a4 + k];
            put_planes(m.P, r0 + b, pc, c0 + a4, v, 4);
        }
        if (c0 + b < m.cols && r0 + a4 < ptc * 32) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = tile[a4 + k][b];
            put_planes(m.PT, c0 + b, ptc, r0 + a4, v, 4);
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

// The scalar recursion of a singular value, on a grid of starting values in [0, 1]: what the matrices can grow to.
Bounds bounds_of(int steps, const double* c)
{
    Bounds b;
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

int hop_plan(const Shape& s, int steps, int dtype)
{
    // steps of a hop: cheapest of the allowed lengths (a hop of h: 3 m^2 n + (4 h - 3) m^3 against h (3 m^2 n + m^3)); ties to the short one
    const int most = dtype == MP_DTYPE_F32 ? 2 : steps;
    int best = 1;
    double cost = 1e300;
    for (int h = 1; h <= most; ++h) {
        double c = 0.0;
        for (int left = steps; left > 0;) {
            const int k = left < h ? left : h;
            c += 3.0 * (double)s.n + (4.0 * k - 3.0) * (double)s.m;
            left -= k;
        }
        if (c < cost * 0.999) {
            cost = c;
            best = h;
        }
    }
    return best;
}

size_t up(size_t v) { return (v + 255) & ~(size_t)255; }
size_t image(int64_t rows, int64_t k) { return up((size_t)rows * chunks(k) * 128); }

struct Buffers { char *X, *XT, *XT2, *A, *T, *P[3]; double* sums; float* r; };

int norm_blocks(const Shape& s)
{
    const int64_t b = (s.rows * s.cols + 4095) / 4096;
    return (int)(b < MAX_NORM_BLOCKS ? (b > 0 ? b : 1) : MAX_NORM_BLOCKS);
}

size_t layout(const Shape& s, int steps, int dtype, char* base, Buffers* b)
{
    const int hop = hop_plan(s, steps, dtype);
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
    d.XT2 = steps > hop ? take(image(s.n, s.m)) : nullptr;
    d.A = take(image(s.m, s.m));
    d.T = hop > 1 ? take(image(s.m, s.m)) : nullptr;
    d.P[0] = take(image(s.m, s.m));
    d.P[1] = hop > 1 ? take(image(s.m, s.m)) : nullptr;
    d.P[2] = hop > 1 ? take(image(s.m, s.m)) : nullptr;
    if (b) *b = d;
    return at;
}

constexpr int CUS = 256;
constexpr int SPLIT_FROM = 32;       // chunks of K from which a split pays for its trip through memory

// tiles of a product in TM x TM pieces
int64_t tiles_of(const Prob& p, int T)
{
    const int64_t tm = (p.M + T - 1) / T, tn = (p.N + T - 1) / T;
    return p.sym ? tm * (tm + 1) / 2 : tm * tn;
}

// The launch's tile size and split.  128 x 128 tiles read each operand half as often as 64 x 64 ones but are a quarter as many: they are
// taken when the launch has at least 3/4 of a tile per CU.  Fewer tiles than CUs and a long K: the K axis is split so that the launch has
// about one workgroup per CU, at least 8 chunks each (a split's accumulators pass through memory once).
struct Plan { int T, splits, kper; };
Plan plan_of(const Prob* p, int count, bool may_split)
{
    int64_t t128 = 0, t64 = 0;
    int kc = 0;
    for (int i = 0; i < count; ++i) {
        t128 += tiles_of(p[i], 128);
        t64 += tiles_of(p[i], 64);
        kc = p[i].kc > kc ? p[i].kc : kc;
    }
    Plan r{128, 1, kc};
    int64_t tiles = t128;
    if (may_split && t128 < CUS * 3 / 4 && kc >= 64) {       // long K: keep the large tiles and split
        r.T = t128 * 8 >= CUS / 4 ? 128 : 64;
    } else if (t128 < CUS * 3 / 4)
        r.T = 64;
    if (r.T == 64) tiles = t64;
    if (may_split && tiles < CUS && kc >= SPLIT_FROM) {
        int64_t s = (CUS + tiles / 2) / tiles;
        if (s > kc / 8) s = kc / 8;
        if (s > 32) s = 32;
        if (s > 1) {
            r.kper = (int)((kc + s - 1) / s);
            r.splits = (kc + r.kper - 1) / r.kper;
        }
    }
    return r;
}

// Accumulators of a split launch: tiles * splits <= CUS + tiles / 2 < 1.5 CUS whatever set of matrices the launch has.
constexpr size_t PART_BYTES = (size_t)(CUS + CUS / 2) * 128 * 128 * sizeof(float);

int launch(Probs& a, bool may_split, const char* tag, hipStream_t stream)
{
    if (a.count == 0) return MP_OK;
    const Plan pl = plan_of(a.p, a.count, may_split);
    a.splits = pl.splits;
    a.kper = pl.kper;
    int64_t blocks = 0;
    double flops = 0.0;
    for (int i = 0; i < a.count; ++i) {
        Prob& p = a.p[i];
        p.tiles_n = (p.N + pl.T - 1) / pl.T;
        p.tile0 = (int)blocks;
        blocks += tiles_of(p, pl.T) * pl.splits;
        flops += 6.0 * p.M * p.N * 32.0 * p.kc * (p.sym ? 0.5 : 1.0);
        if (blocks > 0x7fffffff) return MP_EUNSUPPORTED;
    }
    if (pl.T == 128) {
        MP_LAUNCH(tag, flops, 0.0, (ns_gemm_kernel<2, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
        MP_CHECK_LAUNCH();
        if (pl.splits > 1) MP_LAUNCH("ns_join_kernel", 0.0, 0.0, (ns_join_kernel<2, 2>), dim3((unsigned)(blocks / pl.splits)), dim3(256), 0, stream, a);
    } else {
        MP_LAUNCH(tag, flops, 0.0, (ns_gemm_kernel<1, 1>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
        MP_CHECK_LAUNCH();
        if (pl.splits > 1) MP_LAUNCH("ns_join_kernel", 0.0, 0.0, (ns_join_kernel<1, 1>), dim3((unsigned)(blocks / pl.splits)), dim3(256), 0, stream, a);
    }
    MP_CHECK_LAUNCH();
    return MP_OK;
}

struct Update { int on; double lr, mu, decay; int nesterov, scale; };

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
    size_t bytes = 0;
    bool split = false;
    for (int q = 0; q < k; ++q) {
        const Shape s = shape_of(rows[idx[q]], cols[idx[q]]);
        bytes += layout(s, steps, dtype, nullptr, nullptr);
        split = split || chunks(s.n) >= SPLIT_FROM;
    }
    return bytes + (split ? PART_BYTES : 0);
}

int check_args(int64_t count, const int64_t* rows, const int64_t* cols, int dtype, int steps)
{
    if (count < 0 || (count > 0 && (!rows || !cols)) || steps < 1) return MP_EINVAL;
    if (dtype != MP_DTYPE_F32 && dtype != MP_DTYPE_F16 && dtype != MP_DTYPE_BF16) return MP_EUNSUPPORTED;
    if (steps > MAX_STEPS) return MP_EUNSUPPORTED;
    for (int64_t i = 0; i < count; ++i) {
        if (rows[i] < 0 || cols[i] < 0) return MP_EINVAL;
        const int64_t m = rows[i] < cols[i] ? rows[i] : cols[i], n = rows[i] < cols[i] ? cols[i] : rows[i];
        if (m > 65536 || n > ((int64_t)1 << 30)) return MP_EUNSUPPORTED;
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
    int64_t blocks = 0, tiles = 0;
    double elems = 0.0;
    for (int q = 0; q < k; ++q) {
        sh[q] = shape_of(rows[idx[q]], cols[idx[q]]);
        hop[q] = hop_plan(sh[q], steps, dtype);
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
        m.blk0 = (int)blocks;
        m.tile0 = (int)tiles;
        blocks += m.blocks;
        tiles += ((sh[q].rows + 63) / 64) * ((sh[q].cols + 63) / 64);
        elems += (double)sh[q].rows * (double)sh[q].cols;
    }
    if (tiles > 0x7fffffff) return MP_EUNSUPPORTED;
    const double esz = dtype == MP_DTYPE_F32 ? 4.0 : 2.0;
    MP_LAUNCH("ns_norm_kernel", 2.0 * elems, elems * (esz + (mom ? 8.0 : 0.0)), ns_norm_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    MP_CHECK_LAUNCH();
    MP_LAUNCH("ns_planes_kernel", 2.0 * elems, elems * (esz + (mom ? 4.0 : 0.0) + 8.0), ns_planes_kernel, dim3((unsigned)tiles), dim3(256), 0, stream, a);
    MP_CHECK_LAUNCH();

    const float sX = pow2_scale(bd.x), sA = pow2_scale(bd.x * bd.x), sT = pow2_scale(bd.x * bd.x * bd.q), sQ = pow2_scale(bd.q);
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
    int done[MAX_MAT], at[MAX_MAT], rbuf[MAX_MAT], qbuf[MAX_MAT];       // steps finished, step inside the hop, which P holds R / Q
    bool first[MAX_MAT];
    for (int q = 0; q < k; ++q) { done[q] = at[q] = 0; first[q] = true; rbuf[q] = qbuf[q] = 0; }
    int left = k;
    while (left > 0) {        // every matrix is at the start of a hop (or finished); hops of one chunk may differ in length
        int len[MAX_MAT], longest = 0;
        float sR[MAX_MAT];
        g.count = 0;
        for (int q = 0; q < k; ++q) {       // A = X X^T
            len[q] = done[q] < steps ? (steps - done[q] < hop[q] ? steps - done[q] : hop[q]) : 0;
            longest = len[q] > longest ? len[q] : longest;
            if (!len[q]) continue;
            Prob p = sym_prob(q, bf[q].X, bf[q].X, first[q] ? 1.0f : sX, first[q] ? 1.0f : sX, bf[q].A, sA);
            p.kc = chunks(sh[q].n);
            if (first[q]) { p.rdev = bf[q].r; p.rpow = 2; }
            g.p[g.count++] = p;
        }
        int rc = launch(g, true, "ns_gemm_kernel (gram)", stream);
        if (rc) return rc;
        for (int s = 0; s < longest; ++s) {
            g.count = 0;
            for (int q = 0; q < k; ++q) {      // Q = a I + b A + c A^2
                if (s >= len[q]) continue;
                qbuf[q] = s == 0 ? 0 : (rbuf[q] + 1) % 3;
                Prob p = sym_prob(q, bf[q].A, bf[q].A, sA, sA, bf[q].P[qbuf[q]], sQ);
                p.alpha *= (float)coef[2];
                p.C = reinterpret_cast<const _Float16*>(bf[q].A);
                p.cb = (float)(coef[1] / sA);
                p.ca = (float)coef[0];
                g.p[g.count++] = p;
            }
            rc = launch(g, false, "ns_gemm_kernel (square)", stream);
            if (rc) return rc;
            g.count = 0;
            for (int q = 0; q < k; ++q) {      // T = A Q (another step follows), R = Q R: independent, one launch
                if (s >= len[q]) continue;
                if (s + 1 < len[q]) g.p[g.count++] = sym_prob(q, bf[q].A, bf[q].P[qbuf[q]], sA, sQ, bf[q].T, sT);
                if (s == 0) {
                    rbuf[q] = qbuf[q];
                    sR[q] = sQ;
                } else {
                    const int to = 3 - rbuf[q] - qbuf[q];
                    const float so = pow2_scale(bd.r[s + 1]);
                    g.p[g.count++] = sym_prob(q, bf[q].P[qbuf[q]], bf[q].P[rbuf[q]], sQ, sR[q], bf[q].P[to], so);
                    rbuf[q] = to;
                    sR[q] = so;
                }
            }
            rc = launch(g, false, "ns_gemm_kernel (step)", stream);
            if (rc) return rc;
            g.count = 0;
            for (int q = 0; q < k; ++q)        // A = T Q
                if (s + 1 < len[q]) g.p[g.count++] = sym_prob(q, bf[q].T, bf[q].P[qbuf[q]], sT, sQ, bf[q].A, sA);
            rc = launch(g, false, "ns_gemm_kernel (step)", stream);
            if (rc) return rc;
        }
        g.count = 0;
        for (int q = 0; q < k; ++q) {          // X <- R X
            if (!len[q]) continue;
            done[q] += len[q];
            const bool last = done[q] == steps, tall = sh[q].rows > sh[q].cols;
            Prob p{};
            const _Float16* R = reinterpret_cast<const _Float16*>(bf[q].P[rbuf[q]]);
            const _Float16* XT = reinterpret_cast<const _Float16*>(bf[q].XT);
            const bool flip = last && tall;        // the result in the matrix's own orientation: X^T R
            p.L = flip ? XT : R;
            p.R = flip ? R : XT;
            p.M = (int)(flip ? sh[q].n : sh[q].m);
            p.N = (int)(flip ? sh[q].m : sh[q].n);
            p.kc = chunks(sh[q].m);
            p.alpha = 1.0f / (sR[q] * (first[q] ? 1.0f : sX));
            if (first[q]) { p.rdev = bf[q].r; p.rpow = 1; }
            if (last) {
                p.fin = out[idx[q]];
                if (up_.on) {
                    const double rr = (double)sh[q].rows, cc = (double)sh[q].cols;
                    const double sc = up_.scale == MP_MUON_SCALE_MATCH_RMS ? 0.2 * sqrt(rr > cc ? rr : cc) : up_.scale == MP_MUON_SCALE_ORIGINAL ? sqrt(rr > cc ? rr / cc : 1.0) : 1.0;
                    p.fmul = (float)(up_.lr * sc);
                    p.fdecay = (float)(1.0 - up_.lr * up_.decay);
                }
                --left;
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
            first[q] = false;
            g.p[g.count++] = p;
        }
        rc = launch(g, false, "ns_gemm_kernel (apply)", stream);
        if (rc) return rc;
    }
    return MP_OK;
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
    for (int64_t i = 0; i < count;) {       // everything is checked before anything is launched
        const int k = next_chunk(count, rows, cols, i, idx);
        if (k == 0) continue;
        for (int q = 0; q < k; ++q)
            if (!in[idx[q]] || !out[idx[q]] || (u.on && !mom[idx[q]])) return MP_EINVAL;
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)) return MP_EWORKSPACE;
        if (chunk_bytes(rows, cols, idx, k, steps, dtype) > workspace_bytes) return MP_EWORKSPACE;
    }
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
