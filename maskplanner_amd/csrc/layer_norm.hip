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
// Rows wider than the register form (NV = 8) loop over the row in memory: the second and third reading come from the caches, and dw / db
// take a kernel of their own over column strips.
#include "common.h"

namespace {

template <typename T> struct LnVec {     // 16 bytes that may lie at any element address: rows of odd width are not aligned
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

template <typename T>
__device__ __forceinline__ void ln_load(const T* __restrict__ p, int left, float (&out)[LnVec<T>::N])
{
    constexpr int V = LnVec<T>::N;
    if (left >= V) {
        LnVec<T> t;
        __builtin_memcpy(&t, p, 16);
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = (float)t.v[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = e < left ? (float)p[e] : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void ln_store(T* __restrict__ p, int left, const float (&in)[LnVec<T>::N])
{
    constexpr int V = LnVec<T>::N;
    if (left >= V) {
        LnVec<T> t;
#pragma unroll
        for (int e = 0; e < V; ++e) t.v[e] = (T)in[e];       // the one rounding of the result: to nearest, ties to even
        __builtin_memcpy(p, &t, 16);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < left) p[e] = (T)in[e];
    }
}

// V parameters of columns c .. c + V - 1 (W may be wider than T: then two 16-byte loads)
template <typename W, int V>
__device__ __forceinline__ void ln_param(const W* __restrict__ p, int c, int D, float def, float (&out)[V])
{
    if (!p) {
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = def;
    } else if (c + V <= D) {
        W t[V];
        __builtin_memcpy(t, p + c, sizeof(t));
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = c + e < D ? (float)p[c + e] : 0.0f;
    }
}

// Sums of A values over the TPR threads of a row, left in all of them.  TPR <= 64: lanes of one wave (xor butterfly, the same order in
// every lane); TPR = 256: four waves through LDS (buf: 4 x A floats; the two barriers make it reusable).
template <int TPR, int A>
__device__ __forceinline__ void row_sum(float (&v)[A], float* buf)
{
    constexpr int L = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
        for (int a = 0; a < A; ++a) v[a] += __shfl_xor(v[a], o, 64);
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int a = 0; a < A; ++a) buf[w * A + a] = v[a];
        __syncthreads();
#pragma unroll
        for (int a = 0; a < A; ++a) v[a] = (buf[a] + buf[A + a]) + (buf[2 * A + a] + buf[3 * A + a]);
        __syncthreads();
    }
}

template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, int64_t rows, int D, int64_t xs, const W* __restrict__ w,
                                                     const W* __restrict__ b, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                                                     float* __restrict__ rstd_out)
{
    constexpr int V = LnVec<T>::N;
    __shared__ float buf[4];
    const int t = threadIdx.x % TPR;
    const int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool live = r < rows;
    const T* xr = x + (live ? r : 0) * xs;
    float v[NV][V];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * V;
        ln_load(xr + c, D - c, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += v[i][e];
    row_sum<TPR>(s, buf);
    const float mean = s[0] / (float)D;
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = v[i][e] - mean;
            s[0] += (i * TPR + t) * V + e < D ? d * d : 0.0f;
        }
    row_sum<TPR>(s, buf);
    const float rstd = 1.0f / sqrtf(s[0] / (float)D + eps);
    if (!live) return;
    if (t == 0 && mean_out) {
        mean_out[r] = mean;
        rstd_out[r] = rstd;
    }
    T* yr = y + r * D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * V;
        if (c < D) {
            float ww[V], bb[V];
            ln_param<W, V>(w, c, D, 1.0f, ww);
            ln_param<W, V>(b, c, D, 0.0f, bb);
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = fmaf((v[i][e] - mean) * rstd, ww[e], bb[e]);
            ln_store(yr + c, D - c, v[i]);
        }
    }
}

// part: [gridDim.x][2][D] fp32 (dw row, db row), or NULL when neither is wanted
template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs, int64_t rows,
                                                     int D, const W* __restrict__ w, const float* __restrict__ mean_in,
                                                     const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ part)
{
    constexpr int V = LnVec<T>::N, RPB = 256 / TPR;
    __shared__ float buf[8];
    __shared__ float fold[TPR < 256 ? 256 * V : 1];
    const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    float ww[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ln_param<W, V>(w, (i * TPR + t) * V, D, 1.0f, ww[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) aw[i][e] = ab[i][e] = 0.0f;
    }
    const float inv = 1.0f / (float)D;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {     // (uniform: row_sum has barriers)
        const int64_t r = r0 + slot;
        const bool live = r < rows;
        const int64_t rr = live ? r : 0;
        float z[NV][V], g[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
            ln_load(x + rr * xs + c, D - c, z[i]);
            ln_load(dy + rr * dys + c, live ? D - c : 0, g[i]);
        }
        const float mean = mean_in[rr], rstd = rstd_in[rr];
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                // columns behind D and rows behind the last stay out of the sums by selection: 0 * inf would not
                const bool in = live && (i * TPR + t) * V + e < D;
                z[i][e] = in ? (z[i][e] - mean) * rstd : 0.0f;
                aw[i][e] += g[i][e] * z[i][e];
                ab[i][e] += g[i][e];
                g[i][e] *= ww[i][e];
                s[0] += g[i][e];
                s[1] += g[i][e] * z[i][e];
            }
        row_sum<TPR>(s, buf);
        if (live && dx) {
            const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + t) * V;
                if (c < D) {
#pragma unroll
                    for (int e = 0; e < V; ++e) g[i][e] = rstd * (g[i][e] - c1 - z[i][e] * c2);
                    ln_store(dx + r * D + c, D - c, g[i]);
                }
            }
        }
    }
    if (!part) return;
    float* pw = part + (size_t)blockIdx.x * 2 * D;
    if constexpr (TPR == 256) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + t) * V;
            if (c < D) {
                ln_store(pw + c, D - c, *reinterpret_cast<float(*)[4]>(&aw[i][0]));
                ln_store(pw + D + c, D - c, *reinterpret_cast<float(*)[4]>(&ab[i][0]));
                if constexpr (V == 8) {
                    ln_store(pw + c + 4, D - c - 4, *reinterpret_cast<float(*)[4]>(&aw[i][4]));
                    ln_store(pw + D + c + 4, D - c - 4, *reinterpret_cast<float(*)[4]>(&ab[i][4]));
                }
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
                for (int q = threadIdx.x; q < TPR * V; q += 256) {     // q = e * TPR + thread of the row
                    const int e = q / TPR, tt = q % TPR, c = (i * TPR + tt) * V + e;
                    float sum = 0.0f;
#pragma unroll
                    for (int sl = 0; sl < RPB; ++sl) sum += fold[e * 256 + sl * TPR + tt];
                    if (c < D) pw[(size_t)k * D + c] = sum;
                }
            }
    }
}

// ---- rows wider than the register form: one workgroup walks a row three times (twice from the caches) -------------------------------
template <typename T, typename W>
__global__ __launch_bounds__(256) void ln_fwd_wide_kernel(const T* __restrict__ x, int64_t rows, int64_t D, int64_t xs, const W* __restrict__ w,
                                                          const W* __restrict__ b, float eps, T* __restrict__ y,
                                                          float* __restrict__ mean_out, float* __restrict__ rstd_out)
{
    __shared__ float buf[4];
    const int64_t r = blockIdx.x;
    const T* xr = x + r * xs;
    float s[1] = {0.0f};
    for (int64_t c = threadIdx.x; c < D; c += 256) s[0] += (float)xr[c];
    row_sum<256>(s, buf);
    const float mean = s[0] / (float)D;
    s[0] = 0.0f;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
        const float d = (float)xr[c] - mean;
        s[0] += d * d;
    }
    row_sum<256>(s, buf);
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
    float s[2] = {0.0f, 0.0f};
    for (int64_t c = threadIdx.x; c < D; c += 256) {
        const float g = (float)gr[c] * (w ? (float)w[c] : 1.0f);
        s[0] += g;
        s[1] += g * (((float)xr[c] - mean) * rstd);
    }
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
    float aw = 0.0f, ab = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float g = (float)dy[r * dys + c];
        aw += g * (((float)x[r * xs + c] - mean_in[r]) * rstd_in[r]);
        ab += g;
    }
    part[(size_t)blockIdx.y * 2 * D + c] = aw;
    part[(size_t)blockIdx.y * 2 * D + D + c] = ab;
}

// dw, db = sums of the n partial rows, fp64, in a fixed order: 16 columns x 16 row groups a workgroup, y: dw or db
template <typename W>
__global__ __launch_bounds__(256) void ln_param_reduce_kernel(const float* __restrict__ part, int n, int64_t D, W* __restrict__ dw, W* __restrict__ db)
{
    __shared__ double acc[16][17];
    const int cl = threadIdx.x & 15, rg = threadIdx.x >> 4;
    const int64_t c = (int64_t)blockIdx.x * 16 + cl;
    W* out = blockIdx.y ? db : dw;
    double s = 0.0;
    if (c < D && out) {
        const float* p = part + blockIdx.y * D + c;
#pragma unroll 8
        for (int k = rg; k < n; k += 16) s += (double)p[(size_t)k * 2 * D];
    }
    acc[rg][cl] = s;
    __syncthreads();
    if (rg == 0 && c < D && out) {
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < 16; ++k) v += acc[k][cl];
        out[c] = (W)(float)v;
    }
}

constexpr int LN_MAX_PARTS = 1024;       // partial rows of dw / db (4 workgroups a CU)
constexpr int LN_WIDE_PARTS = 64;

int esize(int dtype) { return dtype == MP_DTYPE_F32 ? 4 : 2; }
int64_t reg_limit(int dtype) { return 256 * 8 * (16 / esize(dtype)); }

// Threads a row: the smallest power of two (from 8) whose one vector each covers it, 64 with up to four; from there on, and for calls of
// few rows (latency: more waves share a row), 256.  [TPR, NV]
struct LnShape { int tpr, nv; };
LnShape ln_shape(int64_t rows, int64_t D, int V)
{
    const int64_t vecs = (D + V - 1) / V;
    if (vecs <= 8) return {8, 1};
    if (vecs <= 16) return {16, 1};
    if (vecs <= 32) return {32, 1};
    if (vecs <= 64) return {64, 1};
    const bool few = rows < 1024;
    if (!few && vecs <= 128) return {64, 2};
    if (!few && vecs <= 256) return {64, 4};
    if (vecs <= 256) return {256, 1};
    if (vecs <= 512) return {256, 2};
    if (vecs <= 1024) return {256, 4};
    return {256, 8};
}

int ln_parts(int64_t rows, int64_t D, int dtype)
{
    if (D > reg_limit(dtype)) return (int)(rows < LN_WIDE_PARTS ? rows : LN_WIDE_PARTS);
    const LnShape s = ln_shape(rows, D, 16 / esize(dtype));
    const int64_t blocks = (rows + 256 / s.tpr - 1) / (256 / s.tpr);
    return (int)(blocks < LN_MAX_PARTS ? blocks : LN_MAX_PARTS);
}

#define LN_EACH_SHAPE(GO)                                                          \
    if (s.tpr == 8) { GO(8, 1); }                                                  \
    else if (s.tpr == 16) { GO(16, 1); }                                           \
    else if (s.tpr == 32) { GO(32, 1); }                                           \
    else if (s.tpr == 64 && s.nv == 1) { GO(64, 1); }                              \
    else if (s.tpr == 64 && s.nv == 2) { GO(64, 2); }                              \
    else if (s.tpr == 64) { GO(64, 4); }                                           \
    else if (s.nv == 1) { GO(256, 1); }                                            \
    else if (s.nv == 2) { GO(256, 2); }                                            \
    else if (s.nv == 4) { GO(256, 4); }                                            \
    else { GO(256, 8); }

template <typename T, typename W>
int ln_fwd(const void* x, int dtype, int64_t rows, int64_t D, int64_t xs, const void* w, const void* b, double eps, void* y, float* mean, float* rstd,
           hipStream_t stream)
{
    const double n = (double)rows * (double)D, bytes = 2.0 * n * sizeof(T);
    if (D > reg_limit(dtype)) {
        MP_LAUNCH("ln_fwd_wide_kernel", 8.0 * n, bytes, (ln_fwd_wide_kernel<T, W>), dim3((unsigned)rows), dim3(256), 0, stream, (const T*)x, rows, D,
                  xs, (const W*)w, (const W*)b, (float)eps, (T*)y, mean, rstd);
    } else {
        const LnShape s = ln_shape(rows, D, LnVec<T>::N);
        const unsigned grid = (unsigned)((rows + 256 / s.tpr - 1) / (256 / s.tpr));
#define LN_GO(TPR, NV)                                                                                                                   \
    MP_LAUNCH("ln_fwd_kernel", 8.0 * n, bytes, (ln_fwd_kernel<T, W, TPR, NV>), dim3(grid), dim3(256), 0, stream, (const T*)x, rows, (int)D, \
              xs, (const W*)w, (const W*)b, (float)eps, (T*)y, mean, rstd)
        LN_EACH_SHAPE(LN_GO)
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
    } else if (rows > 0) {
        const LnShape s = ln_shape(rows, D, LnVec<T>::N);
#define LN_GO(TPR, NV)                                                                                                                     \
    MP_LAUNCH("ln_bwd_kernel", 16.0 * n, bytes, (ln_bwd_kernel<T, W, TPR, NV>), dim3((unsigned)parts), dim3(256), 0, stream, (const T*)dy, dys, \
              (const T*)x, xs, rows, (int)D, (const W*)w, mean, rstd, (T*)dx, pg ? part : nullptr)
        LN_EACH_SHAPE(LN_GO)
#undef LN_GO
        MP_CHECK_LAUNCH();
    }
    if (pg) {      // (no rows: the sums are zero)
        hipLaunchKernelGGL((ln_param_reduce_kernel<W>), dim3((unsigned)((D + 15) / 16), 2), dim3(256), 0, stream, part, parts, D, (W*)dw, (W*)db);
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
        if (!workspace || workspace_bytes < mp_layer_norm_bwd_workspace_bytes(rows, cols, dtype)) return MP_EWORKSPACE;
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
