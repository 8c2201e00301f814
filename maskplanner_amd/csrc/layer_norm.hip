// Layer normalisation over the last axis, forward and backward (gfx950).
//
//   mean_r = sum_j x_rj / D,  rstd_r = 1 / sqrt(sum_j (x_rj - mean_r)^2 / D + eps),  z = (x - mean) rstd,  y = w z + b
//   g = w dy:  dx = rstd (g - mean_j(g) - z mean_j(g z)),   dw_j = sum_r dy z,   db_j = sum_r dy
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx (~1 flop per byte).  So every value is loaded
// once: a row is held in the registers of TPR threads (NV vectors of 16 bytes each), the mean is taken before the squares (two passes
// over registers, no cancellation of E[x^2] - mean^2), and the backward kernel sums dw and db on the same pass: a thread owns the same
// columns of every row its workgroup walks, its sums stay in registers, and one row of partial sums per workgroup goes through memory to
// a second small kernel that adds them in a fixed order (no atomics: two calls give the same bits).  All sums in fp32 (partial rows: fp64).
//
// Rows wider than the register form (2048 vectors) loop over the row in memory: the second and third reading come from the caches, and dw / db
// take a kernel of their own over column strips.
#include "common.h"

namespace {

// N values in whole registers, two of 16 bits to one (as an array of them the compiler gives each a register of its own)
template <typename T, int N_> struct LnPack {
    static constexpr int N = N_, WORDS = N * (int)sizeof(T) / 4;
    unsigned w[WORDS];
    __device__ __forceinline__ float at(int e) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else {
            const unsigned short h = (unsigned short)(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
            T t;
            __builtin_memcpy(&t, &h, 2);
            return (float)t;
        }
    }
    __device__ __forceinline__ void set(int e, T v)        // of a zero value, once
    {
        unsigned short h;
        if constexpr (sizeof(T) == 4) __builtin_memcpy(&w[e], &v, 4);
        else {
            __builtin_memcpy(&h, &v, 2);
            w[e / 2] |= (unsigned)h << (e & 1 ? 16 : 0);
        }
    }
};
// 16 bytes that may lie at any element address: rows of odd width are not aligned
template <typename T> using LnVec = LnPack<T, 16 / (int)sizeof(T)>;

// `left` > 0 elements from p on (16 bytes where that many are left), zeros behind
template <typename T>
__device__ __forceinline__ LnVec<T> ln_raw(const T* __restrict__ p, int left)
{
    constexpr int V = LnVec<T>::N;
    LnVec<T> t{};
    if (left >= V) __builtin_memcpy(t.w, p, 16);
    else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < left) t.set(e, p[e]);
    }
    return t;
}

template <typename T>
__device__ __forceinline__ void ln_store(T* __restrict__ p, int left, const float (&in)[LnVec<T>::N])
{
    constexpr int V = LnVec<T>::N;
    if (left >= V) {
        T t[V];
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = (T)in[e];       // the one rounding of the result: to nearest, ties to even
        __builtin_memcpy(p, t, 16);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < left) p[e] = (T)in[e];
    }
}

// V parameters (16 or, fp32 parameters of 16-bit rows, 32 bytes), kept as they are for all rows of a workgroup
template <typename W, int V>
__device__ __forceinline__ LnPack<W, V> ln_param(const W* __restrict__ p, int c, int D, float def)
{
    LnPack<W, V> t{};
    if (p && c + V <= D) __builtin_memcpy(t.w, p + c, sizeof(t));
    else {
#pragma unroll
        for (int e = 0; e < V; ++e) t.set(e, p && c + e < D ? p[c + e] : (W)def);
    }
    return t;
}

// 16-bit values that are to stay as they came: the compiler would keep them converted from one use to the next, in twice the registers
template <typename T, int N>
__device__ __forceinline__ void ln_packed(LnPack<T, N>& t)
{
    if constexpr (sizeof(T) == 2)
#pragma unroll
        for (unsigned& x : t.w) asm volatile("" : "+v"(x));
}

// Sums of A values over the TPR threads of a row, left in all of them.  TPR <= 64: lanes of one wave, in registers (DPP inside rows of 16
// lanes, row and half swaps above), every lane adding the same pairs; wider: the waves' sums through LDS (buf: TPR / 64 x A floats that the
// previous call did not use: one barrier).
template <int CTRL> __device__ __forceinline__ float dpp_f32(float v) { return __uint_as_float(mp::dpp_u32<CTRL>(__float_as_uint(v))); }
template <int TPR, int A>
__device__ __forceinline__ void row_sum(float (&v)[A], float* buf)
{
#pragma unroll
    for (int a = 0; a < A; ++a) {
        v[a] += dpp_f32<mp::DPP_QUAD_XOR1>(v[a]);
        v[a] += dpp_f32<mp::DPP_QUAD_XOR2>(v[a]);
        v[a] += dpp_f32<mp::DPP_ROW_HALF_MIRROR>(v[a]);
        if constexpr (TPR >= 16) v[a] += dpp_f32<mp::DPP_ROW_MIRROR>(v[a]);
        if constexpr (TPR >= 32) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[a]), __float_as_uint(v[a]), false, false);
            v[a] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        if constexpr (TPR >= 64) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[a]), __float_as_uint(v[a]), false, false);
            v[a] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
    }
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int a = 0; a < A; ++a) buf[w * A + a] = v[a];
        __syncthreads();
#pragma unroll
        for (int a = 0; a < A; ++a) {
            float p[TPR / 64];
#pragma unroll
            for (int k = 0; k < TPR / 64; ++k) p[k] = buf[k * A + a];
#pragma unroll
            for (int o = TPR / 128; o > 0; o >>= 1)
#pragma unroll
                for (int k = 0; k < o; ++k) p[k] += p[k + o];
            v[a] = p[0];
        }
    }
}

// A workgroup walks rows gridDim.x apart; the next row's values are on their way while one is reduced.
constexpr int ln_block(int tpr) { return tpr > 256 ? tpr : 256; }

// row of the workgroup that this thread is on: the same for a wave from 64 threads a row on, and then its addresses are scalar
template <int TPR> __device__ __forceinline__ int ln_slot()
{
    if constexpr (TPR >= 256) return 0;
    else if constexpr (TPR == 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    else return threadIdx.x / TPR;
}

template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__(ln_block(TPR)) void ln_fwd_kernel(const T* __restrict__ x, int64_t rows, int D, int64_t xs, const W* __restrict__ w,
                                                     const W* __restrict__ b, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                                                     float* __restrict__ rstd_out)
{
    constexpr int V = LnVec<T>::N, RPB = ln_block(TPR) / TPR;
    __shared__ float buf[2][8];
    const int t = threadIdx.x % TPR, slot = ln_slot<TPR>();
    const int64_t stride = (int64_t)gridDim.x * RPB;
    LnPack<W, V> ww[NV], bb[NV];
    LnVec<T> next[NV];
    auto fetch = [&](int64_t r) {
        const T* xr = x + (r < rows ? r : 0) * xs;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
            next[i] = c < D ? ln_raw(xr + c, D - c) : LnVec<T>{};
        }
    };
    const bool full = D == NV * TPR * V;        // no columns behind D in any thread
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    fetch(r0 + slot);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ww[i] = ln_param<W, V>(w, (i * TPR + t) * V, D, 1.0f);
        bb[i] = ln_param<W, V>(b, (i * TPR + t) * V, D, 0.0f);
    }
    for (; r0 < rows; r0 += stride) {       // (uniform: row_sum has barriers)
        const int64_t r = r0 + slot;
        float v[NV][V];
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] = next[i].at(e);       // (0 behind D)
                s[0] += v[i][e];
            }
        if (r0 + stride < rows) fetch(r + stride);
        row_sum<TPR>(s, buf[0]);
        const float mean = s[0] / (float)D;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= mean;
                s[0] += full || (i * TPR + t) * V + e < D ? v[i][e] * v[i][e] : 0.0f;
            }
        row_sum<TPR>(s, buf[1]);
        const float rstd = 1.0f / sqrtf(s[0] / (float)D + eps);
        if (r < rows) {
            if (t == 0 && mean_out) {
                mean_out[r] = mean;
                rstd_out[r] = rstd;
            }
            T* yr = y + r * D;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + t) * V;
                if (c < D) {
#pragma unroll
                    for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] * rstd, ww[i].at(e), bb[i].at(e));
                    ln_store(yr + c, D - c, v[i]);
                }
            }
        }
    }
}

// part: [gridDim.x][2][D] fp32 (dw row, db row), or NULL when neither is wanted
template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__(ln_block(TPR)) void ln_bwd_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, int64_t rows,
                                                     int D, const W* __restrict__ w, const float* __restrict__ mean_in,
                                                     const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part)
{
    constexpr int V = LnVec<T>::N, RPB = ln_block(TPR) / TPR;
    __shared__ float buf[2][16];
    __shared__ float fold[TPR < 256 ? 256 * V : 1];
    const int t = threadIdx.x % TPR, slot = ln_slot<TPR>();
    const int64_t stride = (int64_t)gridDim.x * RPB;
    LnPack<W, V> ww[NV];
    float aw[NV][V], ab[NV][V];
    LnVec<T> nx[NV], ng[NV];
    float nmean = 0.0f, nrstd = 0.0f;
    auto fetch = [&](int64_t r) {
        // zeros behind D and behind the last row (mean and rstd too): they add exact zeros to every sum
        const T* xr = x + r * xs;
        const T* gr = dy + r * dys;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
            nx[i] = ng[i] = LnVec<T>{};
            if (c < D && r < rows) {
                nx[i] = ln_raw(xr + c, D - c);
                ng[i] = ln_raw(gr + c, D - c);
            }
        }
        nmean = r < rows ? mean_in[r] : 0.0f;
        nrstd = r < rows ? rstd_in[r] : 0.0f;
    };
    int64_t r0 = (int64_t)blockIdx.x * RPB;
    fetch(r0 + slot);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ww[i] = ln_param<W, V>(w, (i * TPR + t) * V, D, 1.0f);
#pragma unroll
        for (int e = 0; e < V; ++e) aw[i][e] = ab[i][e] = 0.0f;
    }
    const float inv = 1.0f / (float)D;
    int flip = 0;
    for (; r0 < rows; r0 += stride) {     // (uniform: row_sum has barriers)
        const int64_t r = r0 + slot;
        const bool live = r < rows;
        const float mean = nmean, rstd = nrstd;
        // the row stays as it came (half the registers of 16-bit values converted); z and g are formed again for dx
        LnVec<T> cx[NV], cg[NV];
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            cx[i] = nx[i];
            cg[i] = ng[i];
            ln_packed(ww[i]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float z = (cx[i].at(e) - mean) * rstd, g = cg[i].at(e), gw = g * ww[i].at(e);
                aw[i][e] += g * z;
                ab[i][e] += g;
                s[0] += gw;
                s[1] += gw * z;
            }
            if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);        // (one vector converted at a time)
        }
        if (r0 + stride < rows) fetch(r + stride);
        if (!dx) continue;
        row_sum<TPR>(s, buf[flip]);
        flip ^= 1;
        if (live) {
            const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + t) * V;
                ln_packed(cx[i]);
                ln_packed(cg[i]);
                ln_packed(ww[i]);
                if (c < D) {
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float z = (cx[i].at(e) - mean) * rstd;
                        o[e] = rstd * (cg[i].at(e) * ww[i].at(e) - c1 - z * c2);
                    }
                    ln_store(dx + r * D + c, D - c, o);
                }
                if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    if (!part) return;
    float* pw = part + (size_t)blockIdx.x * 2 * D;
    if constexpr (TPR >= 256) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (c + e < D) {
                    pw[c + e] = aw[i][e];
                    pw[D + c + e] = ab[i][e];
                }
        }
    } else {      // the RPB row slots of the workgroup meet in LDS, one vector of columns at a time, in the order of the slots
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < V; ++e) fold[e * 256 + threadIdx.x] = k ? ab[i][e] : aw[i][e];
                __syncthreads();
                for (int q = threadIdx.x; q < TPR * V; q += 256) {     // q = thread of the row * V + e
                    const int e = q % V, tt = q / V, c = (i * TPR + tt) * V + e;
                    float sum = 0.0f;
#pragma unroll
                    for (int sl = 0; sl < RPB; ++sl) sum += fold[e * 256 + sl * TPR + tt];
                    if (c < D) pw[(size_t)k * D + c] = sum;
                }
            }
    }
}

// Few rows (a head's batch): one launch and no workspace.  Workgroups 0 .. rows - 1 take dx of a row, the others 256 columns of dw / db each
// over all rows, in their order.
template <typename T, typename W, int NV>
__global__ __launch_bounds__(256) void ln_bwd_few_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, int rows, int D,
                                                         const W* __restrict__ w, const float* __restrict__ mean_in,
                                                         const float* __restrict__ rstd_in, T* __restrict__ dx, W* __restrict__ dw, W* __restrict__ db)
{
    constexpr int V = LnVec<T>::N;
    __shared__ float buf[8];
    const int r = blockIdx.x;
    if (r >= rows) {
        const int c = (r - rows) * 256 + threadIdx.x;
        if (c >= D) return;
        float aw = 0.0f, ab = 0.0f;
#pragma unroll 8
        for (int k = 0; k < rows; ++k) {
            const float g = (float)dy[k * dys + c];
            aw += g * (((float)x[k * xs + c] - mean_in[k]) * rstd_in[k]);
            ab += g;
        }
        if (dw) dw[c] = (W)aw;
        if (db) db[c] = (W)ab;
        return;
    }
    if (!dx) return;
    const float mean = mean_in[r], rstd = rstd_in[r], inv = 1.0f / (float)D;
    float z[NV][V], g[NV][V];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 256 + (int)threadIdx.x) * V;
        if (c >= D) {
#pragma unroll
            for (int e = 0; e < V; ++e) z[i][e] = g[i][e] = 0.0f;
            continue;
        }
        const LnVec<T> nx = ln_raw(x + r * xs + c, D - c), ng = ln_raw(dy + r * dys + c, D - c);
        const LnPack<W, V> ww = ln_param<W, V>(w, c, D, 1.0f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const bool in = c + e < D;
            z[i][e] = in ? (nx.at(e) - mean) * rstd : 0.0f;
            g[i][e] = in ? ng.at(e) * ww.at(e) : 0.0f;
            s[0] += g[i][e];
            s[1] += g[i][e] * z[i][e];
        }
    }
    row_sum<256>(s, buf);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 256 + (int)threadIdx.x) * V;
        if (c < D) {
#pragma unroll
            for (int e = 0; e < V; ++e) g[i][e] = rstd * (g[i][e] - c1 - z[i][e] * c2);
            ln_store(dx + (int64_t)r * D + c, D - c, g[i]);
        }
    }
}

// ---- rows wider than the register form: one workgroup walks a row three times (twice from the caches) -------------------------------
// A thread adds cols / 256 (or rows / 64) terms one after the other: in fp64, fp32 sums of 2^26 columns left y off by 1.7e-4.
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_fwd_wide_kernel(const T* __restrict__ x, int64_t rows, int64_t D, int64_t xs, const W* __restrict__ w,
                                                          const W* __restrict__ b, float eps, T* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out)
{
    __shared__ float buf[8];
    const int64_t r = blockIdx.x;
    const T* xr = x + r * xs;
    double sum = 0.0;
    for (int64_t c = threadIdx.x; c < D; c += 256) sum += (double)(float)xr[c];
    float s[1] = {(float)sum};
    row_sum<256>(s, buf);
    const float mean = s[0] / (float)D;
    sum = 0.0;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
        const float d = (float)xr[c] - mean;
        sum += (double)(d * d);
    }
    s[0] = (float)sum;
    row_sum<256>(s, buf + 4);
    const float rstd = 1.0f / sqrtf(s[0] / (float)D + eps);
    if (threadIdx.x == 0 && mean_out) {
        mean_out[r] = mean;
        rstd_out[r] = rstd;
    }
    for (int64_t c = threadIdx.x; c < D; c += 256)
        y[r * D + c] = (T)fmaf(((float)xr[c] - mean) * rstd, w ? (float)w[c] : 1.0f, b ? (float)b[c] : 0.0f);
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_bwd_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, int64_t rows,
                                                          int64_t D, const W* __restrict__ w, const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, T* __restrict__ dx)
{
    __shared__ float buf[8];
    const int64_t r = blockIdx.x;
    const T* xr = x + r * xs;
    const T* gr = dy + r * dys;
    const float mean = mean_in[r], rstd = rstd_in[r];
    double sg = 0.0, sgz = 0.0;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
        const float g = (float)gr[c] * (w ? (float)w[c] : 1.0f);
        sg += (double)g;
        sgz += (double)(g * (((float)xr[c] - mean) * rstd));
    }
    float s[2] = {(float)sg, (float)sgz};
    row_sum<256>(s, buf);
    const float inv = 1.0f / (float)D, c1 = s[0] * inv, c2 = s[1] * inv;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
        const float g = (float)gr[c] * (w ? (float)w[c] : 1.0f);
        dx[r * D + c] = (T)(rstd * (g - c1 - (((float)xr[c] - mean) * rstd) * c2));
    }
}

// partial dw / db of one slab of rows over a strip of 256 columns: part [gridDim.y][2][D]
template <typename T>
__global__ __launch_bounds__(256) void ln_param_grad_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                                                                 int64_t rows, int64_t D, const float* __restrict__ mean_in,
                                                                 const float* __restrict__ rstd_in, float* __restrict__ part)
{
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= D) return;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    double aw = 0.0, ab = 0.0;
    for (int64_t r = r0; r < r1; ++r) {
        const float g = (float)dy[r * dys + c];
        aw += (double)(g * (((float)x[r * xs + c] - mean_in[r]) * rstd_in[r]));
        ab += (double)g;
    }
    part[(size_t)blockIdx.y * 2 * D + c] = (float)aw;
    part[(size_t)blockIdx.y * 2 * D + D + c] = (float)ab;
}

// dw, db = sums of the n partial rows, fp64, in a fixed order: 16 columns x 64 row groups a workgroup, then the next 16 that are nobody else's
// (a grid has fewer than 2^32 threads: 2^26 columns at once were left unwritten); y: dw or db
template <typename W>
__global__ __launch_bounds__(1024) void ln_param_reduce_kernel(const float* __restrict__ part, int n, int64_t D, W* __restrict__ dw, W* __restrict__ db)
{
    __shared__ double acc[64][17];
    const int cl = threadIdx.x & 15, rg = threadIdx.x >> 4;
    W* out = blockIdx.y ? db : dw;
    if (!out) return;
    for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < D; c0 += (int64_t)gridDim.x * 16) {
        const int64_t c = c0 + cl;
        double s = 0.0;
        if (c < D) {
            const float* p = part + blockIdx.y * D + c;
#pragma unroll 8
            for (int k = rg; k < n; k += 64) s += (double)p[(size_t)k * 2 * D];
        }
        acc[rg][cl] = s;
        __syncthreads();
        for (int o = 32; o > 0; o >>= 1) {
            if (rg < o) acc[rg][cl] += acc[rg + o][cl];
            __syncthreads();
        }
        if (rg == 0 && c < D) out[c] = (W)(float)acc[0][cl];
        __syncthreads();
    }
}

constexpr int LN_WIDE_PARTS = 64;
constexpr int64_t LN_REDUCE_BLOCKS = 1 << 16;
// up to here dw / db are summed row by row by one thread a column: no partial sums, no second launch (32 x 1024 fp32: 4 us against 4 + 3)
constexpr int LN_FEW_ROWS = 64;

int esize(int dtype) { return dtype == MP_DTYPE_F32 ? 4 : 2; }
int64_t reg_limit(int dtype) { return 256 * 8 * (16 / esize(dtype)); }

// Threads a row and vectors a thread.  Up to 64 vectors the smallest power of two (from 8) that covers the row with one each; then the least
// waste of threads that leaves a CU several workgroups' registers (12 000 bf16 columns forward: 512 x 3 45 us, 1024 x 2 60).  The backward
// kernel holds two sums a column, 16 registers a vector of 16-bit values: one vector a thread while 512 threads cover the row (3000 bf16
// columns: 512 x 1 126 us, 256 x 2 141).  Calls of few rows (latency: more waves share a row): 256 threads.
struct LnShape { int tpr, nv; };
LnShape ln_shape(int64_t rows, int64_t D, int V, bool backward)
{
    const int64_t vecs = (D + V - 1) / V;
    if (vecs <= 8) return {8, 1};
    if (vecs <= 16) return {16, 1};
    if (vecs <= 32) return {32, 1};
    if (vecs <= 64) return {64, 1};
    const bool few = rows < 1024;
    if (!few && vecs <= 128) return {64, 2};
    if (!few && vecs <= 192) return {64, 3};
    if (vecs <= 256) return {256, 1};
    if (vecs <= 512) return backward ? LnShape{512, 1} : LnShape{256, 2};
    if (vecs <= 768 && !backward) return {256, 3};
    if (vecs <= 1024) return {512, 2};
    if (vecs <= 1536) return {512, 3};
    return {512, 4};
}

// Workgroups that walk the rows: about as many as the CUs hold at once.  Backward, every one writes a row of partial sums: 1280 of them cost
// 12 000 bf16 columns 220 us, 256 121.
int ln_fwd_blocks(LnShape s) { return s.tpr <= 256 ? 1024 : 512; }
int ln_bwd_blocks(LnShape s) { return s.tpr <= 256 ? (s.nv <= 2 ? 768 : 512) : s.nv == 1 ? 512 : 256; }

int ln_parts(int64_t rows, int64_t D, int dtype)
{
    if (D > reg_limit(dtype)) return (int)(rows < LN_WIDE_PARTS ? rows : LN_WIDE_PARTS);
    if (rows <= LN_FEW_ROWS) return 0;
    const LnShape s = ln_shape(rows, D, 16 / esize(dtype), true);
    const int64_t blocks = (rows + ln_block(s.tpr) / s.tpr - 1) / (ln_block(s.tpr) / s.tpr), most = ln_bwd_blocks(s);
    return (int)(blocks < most ? blocks : most);
}

#define LN_COMMON_SHAPES(GO)                          \
    if (s.tpr == 8) { GO(8, 1); }                     \
    else if (s.tpr == 16) { GO(16, 1); }              \
    else if (s.tpr == 32) { GO(32, 1); }              \
    else if (s.tpr == 64 && s.nv == 1) { GO(64, 1); } \
    else if (s.tpr == 64 && s.nv == 2) { GO(64, 2); } \
    else if (s.tpr == 64) { GO(64, 3); }              \
    else if (s.tpr == 256 && s.nv == 1) { GO(256, 1); } \
    else if (s.tpr == 512 && s.nv == 2) { GO(512, 2); } \
    else if (s.tpr == 512 && s.nv == 3) { GO(512, 3); } \
    else if (s.tpr == 512 && s.nv == 4) { GO(512, 4); }

template <typename T, typename W>
int ln_fwd(const void* x, int dtype, int64_t rows, int64_t D, int64_t xs, const void* w, const void* b, double eps, void* y, float* mean, float* rstd,
           hipStream_t stream)
{
    const double n = (double)rows * (double)D, bytes = 2.0 * n * sizeof(T);
    if (D > reg_limit(dtype)) {
        MP_LAUNCH("ln_fwd_wide_kernel", 8.0 * n, bytes, (ln_fwd_wide_kernel<T, W>), dim3((unsigned)rows), dim3(256), 0, stream, (const T*)x, rows, D,
                  xs, (const W*)w, (const W*)b, (float)eps, (T*)y, mean, rstd);
    } else {
        const LnShape s = ln_shape(rows, D, LnVec<T>::N, false);
        const int64_t blocks = (rows + ln_block(s.tpr) / s.tpr - 1) / (ln_block(s.tpr) / s.tpr);
        const unsigned grid = (unsigned)(blocks < ln_fwd_blocks(s) ? blocks : ln_fwd_blocks(s));
#define LN_GO(TPR, NV)                                                                                                                   \
    MP_LAUNCH("ln_fwd_kernel", 8.0 * n, bytes, (ln_fwd_kernel<T, W, TPR, NV>), dim3(grid), dim3(ln_block(TPR)), 0, stream, (const T*)x, rows, (int)D, \
              xs, (const W*)w, (const W*)b, (float)eps, (T*)y, mean, rstd)
        LN_COMMON_SHAPES(LN_GO)
        else if (s.nv == 2) { LN_GO(256, 2); }
        else { LN_GO(256, 3); }
#undef LN_GO
    }
    MP_CHECK_LAUNCH();
    return MP_OK;
}

template <typename T, typename W>
int ln_bwd(const void* dy, int64_t dys, const void* x, int64_t xs, int dtype, int64_t rows, int64_t D, const void* w, const float* mean,
           const float* rstd, void* dx, void* dw, void* db, float* part, hipStream_t stream)
{
    const double n = (double)rows * (double)D, bytes = 3.0 * n * sizeof(T);
    const int parts = ln_parts(rows, D, dtype);
    const bool pg = dw || db;
    if (rows > 0 && D > reg_limit(dtype)) {
        if (dx)
            MP_LAUNCH("ln_bwd_wide_kernel", 12.0 * n, bytes, (ln_bwd_wide_kernel<T, W>), dim3((unsigned)rows), dim3(256), 0, stream, (const T*)dy, dys,
                      (const T*)x, xs, rows, D, (const W*)w, mean, rstd, (T*)dx);
        if (pg)
            MP_LAUNCH("ln_param_grad_wide_kernel", 4.0 * n, 2.0 * n * sizeof(T), (ln_param_grad_wide_kernel<T>),
                      dim3((unsigned)((D + 255) / 256), (unsigned)parts), dim3(256), 0, stream, (const T*)dy, dys, (const T*)x, xs, rows, D, mean, rstd, part);
        MP_CHECK_LAUNCH();
    } else if (rows > 0 && rows <= LN_FEW_ROWS) {
        const unsigned grid = (unsigned)(rows + (pg ? (D + 255) / 256 : 0));
#define LN_GO(NV)                                                                                                                            \
    MP_LAUNCH("ln_bwd_few_kernel", 16.0 * n, bytes, (ln_bwd_few_kernel<T, W, NV>), dim3(grid), dim3(256), 0, stream, (const T*)dy, dys, (const T*)x, \
              xs, (int)rows, (int)D, (const W*)w, mean, rstd, (T*)dx, (W*)dw, (W*)db)
        const int64_t vecs = (D + LnVec<T>::N - 1) / LnVec<T>::N;
        if (vecs <= 256) LN_GO(1);
        else if (vecs <= 1024) LN_GO(4);
        else LN_GO(8);
#undef LN_GO
        MP_CHECK_LAUNCH();
        return MP_OK;
    } else if (rows > 0) {
        const LnShape s = ln_shape(rows, D, LnVec<T>::N, true);
#define LN_GO(TPR, NV)                                                                                                                     \
    MP_LAUNCH("ln_bwd_kernel", 16.0 * n, bytes, (ln_bwd_kernel<T, W, TPR, NV>), dim3((unsigned)parts), dim3(ln_block(TPR)), 0, stream, (const T*)dy, dys, \
              (const T*)x, xs, rows, (int)D, (const W*)w, mean, rstd, (T*)dx, pg ? part : nullptr)
        LN_COMMON_SHAPES(LN_GO)
        else { LN_GO(512, 1); }
#undef LN_GO
        MP_CHECK_LAUNCH();
    }
    if (pg) {      // (no rows: the sums are zero)
        const int64_t groups = (D + 15) / 16;
        hipLaunchKernelGGL((ln_param_reduce_kernel<W>), dim3((unsigned)(groups < LN_REDUCE_BLOCKS ? groups : LN_REDUCE_BLOCKS), 2), dim3(1024), 0, stream,
                           part, parts, D, (W*)dw, (W*)db);
        MP_CHECK_LAUNCH();
    }
    return MP_OK;
}

bool known(int dtype) { return dtype == MP_DTYPE_F32 || dtype == MP_DTYPE_F16 || dtype == MP_DTYPE_BF16; }

int ln_check(int64_t rows, int64_t cols, int dtype, int wdtype)
{
    if (rows < 0 || cols < 1) return MP_EINVAL;
    if (!known(dtype) || !known(wdtype) || (wdtype != MP_DTYPE_F32 && wdtype != dtype)) return MP_EUNSUPPORTED;
    if (rows > 0x7fffffff || cols > 0x7fffffff) return MP_EUNSUPPORTED;
    return MP_OK;
}

}  // namespace

extern "C" int mp_layer_norm_fwd(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_row_stride, const void* weight, const void* bias,
                                 int param_dtype, double eps, void* y, float* mean, float* rstd, mp_stream_t stream_)
{
    const int rc = ln_check(rows, cols, dtype, param_dtype);
    if (rc) return rc;
    if (rows == 0) return MP_OK;
    if (!x || !y || x_row_stride < 0 || !mean != !rstd || !(eps >= 0.0)) return MP_EINVAL;
    hipStream_t s = mp_stream(stream_);
#define LN_ARGS x, dtype, rows, cols, x_row_stride, weight, bias, eps, y, mean, rstd, s
    if (dtype == MP_DTYPE_F32) return ln_fwd<float, float>(LN_ARGS);
    if (dtype == MP_DTYPE_F16) return param_dtype == MP_DTYPE_F32 ? ln_fwd<_Float16, float>(LN_ARGS) : ln_fwd<_Float16, _Float16>(LN_ARGS);
    return param_dtype == MP_DTYPE_F32 ? ln_fwd<__bf16, float>(LN_ARGS) : ln_fwd<__bf16, __bf16>(LN_ARGS);
#undef LN_ARGS
}

extern "C" size_t mp_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols, int dtype)
{
    if (rows <= 0 || cols <= 0 || !known(dtype)) return 0;
    return (size_t)ln_parts(rows, cols, dtype) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int mp_layer_norm_bwd(const void* dy, int64_t dy_row_stride, const void* x, int64_t x_row_stride, int dtype, int64_t rows, int64_t cols,
                                 const void* weight, int param_dtype, const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                                 void* workspace, size_t workspace_bytes, mp_stream_t stream_)
{
    const int rc = ln_check(rows, cols, dtype, param_dtype);
    if (rc) return rc;
    if (!dx && !dweight && !dbias) return MP_OK;
    if (rows > 0 && (!dy || !x || !mean || !rstd || dy_row_stride < 0 || x_row_stride < 0)) return MP_EINVAL;
    if ((dweight || dbias) && rows > 0) {
        const size_t need = mp_layer_norm_bwd_workspace_bytes(rows, cols, dtype);
        if (need && (!workspace || workspace_bytes < need)) return MP_EWORKSPACE;
        if (reinterpret_cast<uintptr_t>(workspace) & 3) return MP_EINVAL;
    }
    hipStream_t s = mp_stream(stream_);
    float* part = static_cast<float*>(workspace);
#define LN_ARGS dy, dy_row_stride, x, x_row_stride, dtype, rows, cols, weight, mean, rstd, dx, dweight, dbias, part, s
    if (dtype == MP_DTYPE_F32) return ln_bwd<float, float>(LN_ARGS);
    if (dtype == MP_DTYPE_F16) return param_dtype == MP_DTYPE_F32 ? ln_bwd<_Float16, float>(LN_ARGS) : ln_bwd<_Float16, _Float16>(LN_ARGS);
    return param_dtype == MP_DTYPE_F32 ? ln_bwd<__bf16, float>(LN_ARGS) : ln_bwd<__bf16, __bf16>(LN_ARGS);
#undef LN_ARGS
}
