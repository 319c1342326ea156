// Layer norm over the last dimension, forward and backward, with the reduction of the weights' gradients.
//
//   mean = sum(x) / C,  var = sum((x - mean)^2) / C,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd,  y = h gamma + beta
//   backward: e = dy gamma,  dx = rstd (e - mean(e) - h mean(e h)),  dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both passes are bound by memory: x in and y out (forward), x and dy in and dx out (backward).  A row is read ONCE into the
// registers of its group of lanes -- 16, 64, 256 or 1024 lanes, the fewest that hold it in at most four 16-byte pieces each -- and
// the variance is the second pass over those registers (a one-pass sum of squares would cancel where the mean is large).  Rows
// beyond 1024 x 4 pieces are streamed: each pass over the row reads it again, from L2.  A group walks the rows r, r + groups, ...
// and keeps its slice of gamma (and beta) in registers.
//
// Weight gradients: every lane owns the same columns in all its rows, so dgamma and dbeta are sums in its registers; the groups of a
// workgroup are added in LDS in a fixed order, workgroups through partials [P][2][C] in the workspace and a second launch: no
// atomics, the same bits every time.
#include "avsi_common.h"
#include "avsi_wave.h"

namespace {

constexpr int NV = 4;       // 16-byte pieces of a row per lane

// Sum over the L lanes of a group (L <= 64: inside a wave; else the whole workgroup, through LDS).
template <int L> __device__ __forceinline__ float group_sum(float v, float* lds) {
    if (L <= 64) return avsi_group<L < 64 ? L : 64>(v);
    v = avsi_group<64>(v);
    __syncthreads();                        // the sums of the previous call have been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) s += lds[i];
    return s;
}

template <typename T, typename W, int L>
__global__ __launch_bounds__(L < 256 ? 256 : L) void ln_fwd_kernel(const T* __restrict__ x, int64_t xs, const W* __restrict__ gamma,
                                                                    const W* __restrict__ beta, T* __restrict__ y, int64_t ys,
                                                                    float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                                                                    int C, float eps) {
    constexpr int V = 16 / sizeof(T);
    constexpr int PER_WG = (L < 256 ? 256 : L) / L;
    __shared__ float lds[L > 64 ? L / 64 : 1];
    const int lane = threadIdx.x % L;
    const float fc = (float)C;
    avsi_raw<W, V> gr[NV], br[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * L + lane) * V;
        if (gamma) gr[j] = avsi_load_raw<W, V>(gamma + c, C - c);
        if (beta) br[j] = avsi_load_raw<W, V>(beta + c, C - c);
    }
    for (int64_t r = (int64_t)blockIdx.x * PER_WG + threadIdx.x / L; r < rows; r += (int64_t)gridDim.x * PER_WG) {
        float v[NV][V];
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * L + lane) * V;
            avsi_load<T, V>(x + r * xs + c, C - c, v[j]);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) s += v[j][i];           // (columns behind the row's end are zero)
        const float mu = group_sum<L>(s, lds) / fc;
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = (j * L + lane) * V + i < C ? v[j][i] - mu : 0.f;
                q = fmaf(d, d, q);
            }
        const float rs = 1.f / sqrtf(group_sum<L>(q, lds) / fc + eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * L + lane) * V;
            if (c >= C) continue;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o[i] = (v[j][i] - mu) * rs;
                if (gamma) o[i] *= (float)gr[j].v[i];
                if (beta) o[i] += (float)br[j].v[i];
            }
            avsi_store<T, V>(y + r * ys + c, C - c, o);
        }
        if (lane == 0) {
            mean[r] = mu;
            rstd[r] = rs;
        }
    }
}

// Rows that do not fit the registers: one workgroup of 1024 per row, three passes over it.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(const T* __restrict__ x, int64_t xs, const W* __restrict__ gamma,
                                                           const W* __restrict__ beta, T* __restrict__ y, int64_t ys,
                                                           float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int C,
                                                           float eps) {
    constexpr int V = 16 / sizeof(T), L = 1024;
    __shared__ float lds[L / 64];
    const float fc = (float)C;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * xs;
        float s = 0.f, q = 0.f, v[V];
        for (int c = threadIdx.x * V; c < C; c += L * V) {
            avsi_load<T, V>(xr + c, C - c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) s += v[i];
        }
        const float mu = group_sum<L>(s, lds) / fc;
        for (int c = threadIdx.x * V; c < C; c += L * V) {
            avsi_load<T, V>(xr + c, C - c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = c + i < C ? v[i] - mu : 0.f;
                q = fmaf(d, d, q);
            }
        }
        const float rs = 1.f / sqrtf(group_sum<L>(q, lds) / fc + eps);
        for (int c = threadIdx.x * V; c < C; c += L * V) {
            float g[V], b[V];
            avsi_load<T, V>(xr + c, C - c, v);
            if (gamma) avsi_load<W, V>(gamma + c, C - c, g);
            if (beta) avsi_load<W, V>(beta + c, C - c, b);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[i] = (v[i] - mu) * rs;
                if (gamma) v[i] *= g[i];
                if (beta) v[i] += b[i];
            }
            avsi_store<T, V>(y + r * ys + c, C - c, v);
        }
        if (threadIdx.x == 0) {
            mean[r] = mu;
            rstd[r] = rs;
        }
    }
}

template <typename T, typename W, int L, bool WGRAD>
__global__ __launch_bounds__(L < 256 ? 256 : L) void ln_bwd_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x,
                                                                    int64_t xs, const float* __restrict__ mean,
                                                                    const float* __restrict__ rstd, const W* __restrict__ gamma,
                                                                    T* __restrict__ dx, int64_t dxs, float* __restrict__ part,
                                                                    int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T);
    constexpr int NT = L < 256 ? 256 : L, PER_WG = NT / L;
    __shared__ float lds[L > 64 ? L / 64 : 1];
    __shared__ float acc[WGRAD && PER_WG > 1 ? 2 * L * V * NV : 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const float inv = 1.f / (float)C;
    avsi_raw<W, V> gr[NV];
    float dg[NV][V], db[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * L + lane) * V;
        if (gamma) gr[j] = avsi_load_raw<W, V>(gamma + c, C - c);
#pragma unroll
        for (int i = 0; i < V; ++i) dg[j][i] = db[j][i] = 0.f;
    }
    for (int64_t r = (int64_t)blockIdx.x * PER_WG + group; r < rows; r += (int64_t)gridDim.x * PER_WG) {
        float h[NV][V], g[NV][V];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * L + lane) * V;
            avsi_load<T, V>(x + r * xs + c, C - c, h[j]);
            avsi_load<T, V>(dy + r * dys + c, C - c, g[j]);
        }
        const float mu = mean[r], rs = rstd[r];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[j][i] = (h[j][i] - mu) * rs;          // (behind the row's end dy is zero, and with it every term)
                if (WGRAD) {
                    dg[j][i] = fmaf(g[j][i], h[j][i], dg[j][i]);
                    db[j][i] += g[j][i];
                }
                if (gamma) g[j][i] *= (float)gr[j].v[i];
                s1 += g[j][i];
                s2 = fmaf(g[j][i], h[j][i], s2);
            }
        const float m1 = group_sum<L>(s1, lds) * inv, m2 = group_sum<L>(s2, lds) * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * L + lane) * V;
            if (c >= C) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) g[j][i] = (g[j][i] - m1 - h[j][i] * m2) * rs;
            avsi_store<T, V>(dx + r * dxs + c, C - c, g[j]);
        }
    }
    if (!WGRAD) return;
    // the groups of this workgroup, one after the other
    for (int k = 0; k < PER_WG; ++k) {
        if (PER_WG > 1) __syncthreads();
        if (group != k) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * L + lane) * V;
            if (c >= C) continue;
            if (PER_WG > 1) {
                float* a = acc + 2 * c;
                if (k > 0)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        dg[j][i] += a[i];
                        db[j][i] += a[V + i];
                    }
                if (k < PER_WG - 1)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        a[i] = dg[j][i];
                        a[V + i] = db[j][i];
                    }
            }
            if (k == PER_WG - 1) {
                float* p = part + (int64_t)blockIdx.x * 2 * C + c;
                avsi_store<float, V>(p, C - c, dg[j]);
                avsi_store<float, V>(p + C, C - c, db[j]);
            }
        }
    }
}

// Rows that do not fit the registers: dx by one workgroup per row in two passes over it, the weights' gradients by column (below).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           const W* __restrict__ gamma, T* __restrict__ dx, int64_t dxs, int64_t rows,
                                                           int C) {
    constexpr int V = 16 / sizeof(T), L = 1024;
    __shared__ float lds[L / 64];
    const float inv = 1.f / (float)C;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mu = mean[r], rs = rstd[r];
        float s1 = 0.f, s2 = 0.f, h[V], g[V], w[V];
        for (int pass = 0; pass < 2; ++pass) {
            const float m1 = pass ? group_sum<L>(s1, lds) * inv : 0.f, m2 = pass ? group_sum<L>(s2, lds) * inv : 0.f;
            for (int c = threadIdx.x * V; c < C; c += L * V) {
                avsi_load<T, V>(x + r * xs + c, C - c, h);
                avsi_load<T, V>(dy + r * dys + c, C - c, g);
                if (gamma) avsi_load<W, V>(gamma + c, C - c, w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    h[i] = (h[i] - mu) * rs;
                    if (gamma) g[i] *= w[i];
                    if (pass == 0) {
                        s1 += g[i];
                        s2 = fmaf(g[i], h[i], s2);
                    } else {
                        g[i] = (g[i] - m1 - h[i] * m2) * rs;
                    }
                }
                if (pass) avsi_store<T, V>(dx + r * dxs + c, C - c, g);
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_wgrad_wide_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                                                            const float* __restrict__ mean, const float* __restrict__ rstd,
                                                            float* __restrict__ part, int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T);
    const int c = (blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= C) return;
    float dg[V], db[V], h[V], g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) dg[i] = db[i] = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        avsi_load<T, V>(x + r * xs + c, C - c, h);
        avsi_load<T, V>(dy + r * dys + c, C - c, g);
        const float mu = mean[r], rs = rstd[r];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            dg[i] = fmaf(g[i], (h[i] - mu) * rs, dg[i]);
            db[i] += g[i];
        }
    }
    float* p = part + (int64_t)blockIdx.y * 2 * C + c;
    avsi_store<float, V>(p, C - c, dg);
    avsi_store<float, V>(p + C, C - c, db);
}

// out[c] = sum over p of part[p][c], c < 2 C: 16 columns x 16 slices of the partials per workgroup.
__global__ __launch_bounds__(256) void ln_wgrad_sum_kernel(const float* __restrict__ part, int P, int C, float* __restrict__ dgamma,
                                                           float* __restrict__ dbeta) {
    __shared__ float lds[256];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15);
    float s = 0.f;
    if (c < 2 * C)
        for (int p = threadIdx.x >> 4; p < P; p += 16) s += part[(int64_t)p * 2 * C + c];
    lds[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < 2 * C) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += lds[i * 16 + threadIdx.x];
        if (c < C) dgamma[c] = s;
        else dbeta[c - C] = s;
    }
}

// Lanes of a row's group: the fewest of 16, 64, 256, 1024 that hold C columns; 0: none does.
int group_lanes(int C, int dtype) {
    const int piece = 16 / avsi_dtype_size(dtype) * NV;
    return C <= 16 * piece ? 16 : C <= 64 * piece ? 64 : C <= 256 * piece ? 256 : C <= 1024 * piece ? 1024 : 0;
}

int fwd_groups(int64_t rows, int L) {
    const int per_wg = L && L < 256 ? 256 / L : 1;
    const int64_t wgs = avsi_ceil_div(rows, per_wg), most = (L == 1024 || L == 0 ? 2 : 8) * AVSI_NUM_CU;
    return (int)(wgs < most ? wgs : most);
}

// Workgroups of the backward pass = partials of the weights' gradients.
int bwd_groups(int64_t rows, int C, int dtype) {
    const int L = group_lanes(C, dtype);
    if (!L) return (int)(rows < 64 ? rows : 64);
    const int per_wg = L < 256 ? 256 / L : 1;
    const int64_t wgs = avsi_ceil_div(rows, per_wg), most = 2 * AVSI_NUM_CU;
    return (int)(wgs < most ? wgs : most);
}

template <typename T, typename W>
int launch_fwd(const void* x, int64_t xs, const void* gamma, const void* beta, void* y, int64_t ys, float* mean, float* rstd,
               int64_t rows, int C, float eps, int L, hipStream_t s) {
    const dim3 grid(fwd_groups(rows, L));
#define AVSI_LN_FWD(LANES, NT)                                                                                                       \
    hipLaunchKernelGGL((ln_fwd_kernel<T, W, LANES>), grid, dim3(NT), 0, s, (const T*)x, xs, (const W*)gamma, (const W*)beta, (T*)y, \
                       ys, mean, rstd, rows, C, eps)
    if (L == 16) AVSI_LN_FWD(16, 256);
    else if (L == 64) AVSI_LN_FWD(64, 256);
    else if (L == 256) AVSI_LN_FWD(256, 256);
    else if (L == 1024) AVSI_LN_FWD(1024, 1024);
    else
        hipLaunchKernelGGL((ln_fwd_wide_kernel<T, W>), grid, dim3(1024), 0, s, (const T*)x, xs, (const W*)gamma, (const W*)beta, (T*)y,
                           ys, mean, rstd, rows, C, eps);
#undef AVSI_LN_FWD
    return avsi_launch_status();
}

template <typename T, typename W>
int launch_bwd(const void* dy, int64_t dys, const void* x, int64_t xs, const float* mean, const float* rstd, const void* gamma,
               void* dx, int64_t dxs, float* dgamma, float* dbeta, float* part, int64_t rows, int C, int dtype, hipStream_t s) {
    const int L = group_lanes(C, dtype), P = bwd_groups(rows, C, dtype);
#define AVSI_LN_BWD(LANES, NT, WG)                                                                                                  \
    hipLaunchKernelGGL((ln_bwd_kernel<T, W, LANES, WG>), dim3(P), dim3(NT), 0, s, (const T*)dy, dys, (const T*)x, xs, mean, rstd,  \
                       (const W*)gamma, (T*)dx, dxs, part, rows, C)
#define AVSI_LN_BWD_L(WG)                           \
    if (L == 16) AVSI_LN_BWD(16, 256, WG);          \
    else if (L == 64) AVSI_LN_BWD(64, 256, WG);     \
    else if (L == 256) AVSI_LN_BWD(256, 256, WG);   \
    else AVSI_LN_BWD(1024, 1024, WG)
    if (!L) {
        hipLaunchKernelGGL((ln_bwd_wide_kernel<T, W>), dim3(fwd_groups(rows, 0)), dim3(1024), 0, s, (const T*)dy, dys, (const T*)x, xs,
                           mean, rstd, (const W*)gamma, (T*)dx, dxs, rows, C);
        if (dgamma)
            hipLaunchKernelGGL((ln_wgrad_wide_kernel<T>), dim3(avsi_ceil_div(C, 256 * (16 / sizeof(T))), P), dim3(256), 0, s,
                               (const T*)dy, dys, (const T*)x, xs, mean, rstd, part, rows, C);
    } else if (dgamma) {
        AVSI_LN_BWD_L(true);
    } else {
        AVSI_LN_BWD_L(false);
    }
#undef AVSI_LN_BWD_L
#undef AVSI_LN_BWD
    if (dgamma)
        hipLaunchKernelGGL(ln_wgrad_sum_kernel, dim3(avsi_ceil_div(2 * C, 16)), dim3(256), 0, s, part, P, C, dgamma, dbeta);
    return avsi_launch_status();
}

bool args_ok(const void* x, int64_t xs, int dtype, int wdtype, int64_t rows, int C) {
    return x && rows > 0 && C > 0 && C <= (1 << 30) && xs >= C && avsi_dtype_ok(dtype) && (wdtype == AVSI_F32 || wdtype == dtype);
}

}  // namespace

extern "C" int avsi_layer_norm(const void* x, int64_t x_stride, int dtype, const void* gamma, const void* beta, int wdtype, void* y,
                               int64_t y_stride, float* mean, float* rstd, int64_t rows, int cols, float eps, void* stream) {
    if (!args_ok(x, x_stride, dtype, wdtype, rows, cols) || !y || y_stride < cols || !mean || !rstd || !(eps >= 0.f))
        return AVSI_ERR_INVALID_ARG;
    avsi_clear_error();
    const int L = group_lanes(cols, dtype);
    hipStream_t s = (hipStream_t)stream;
#define AVSI_GO(T, W) return launch_fwd<T, W>(x, x_stride, gamma, beta, y, y_stride, mean, rstd, rows, cols, eps, L, s)
    if (dtype == AVSI_F32) AVSI_GO(float, float);
    if (dtype == AVSI_BF16) {
        if (wdtype == AVSI_F32) AVSI_GO(__bf16, float);
        AVSI_GO(__bf16, __bf16);
    }
    if (wdtype == AVSI_F32) AVSI_GO(_Float16, float);
    AVSI_GO(_Float16, _Float16);
#undef AVSI_GO
}

extern "C" size_t avsi_layer_norm_bwd_workspace_bytes(int64_t rows, int cols, int dtype) {
    if (rows <= 0 || cols <= 0 || !avsi_dtype_ok(dtype)) return 0;
    return (size_t)bwd_groups(rows, cols, dtype) * 2 * cols * sizeof(float);
}

extern "C" int avsi_layer_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int dtype, const float* mean,
                                   const float* rstd, const void* gamma, int wdtype, void* dx, int64_t dx_stride, float* dgamma,
                                   float* dbeta, int64_t rows, int cols, void* workspace, size_t workspace_bytes, void* stream) {
    if (!args_ok(x, x_stride, dtype, wdtype, rows, cols) || !dy || dy_stride < cols || !mean || !rstd || !dx || dx_stride < cols ||
        !dgamma != !dbeta)
        return AVSI_ERR_INVALID_ARG;
    if (dgamma && (!workspace || workspace_bytes < avsi_layer_norm_bwd_workspace_bytes(rows, cols, dtype))) return AVSI_ERR_WORKSPACE;
    avsi_clear_error();
    hipStream_t s = (hipStream_t)stream;
#define AVSI_GO(T, W)                                                                                                            \
    return launch_bwd<T, W>(dy, dy_stride, x, x_stride, mean, rstd, gamma, dx, dx_stride, dgamma, dbeta, (float*)workspace, rows, \
                            cols, dtype, s)
    if (dtype == AVSI_F32) AVSI_GO(float, float);
    if (dtype == AVSI_BF16) {
        if (wdtype == AVSI_F32) AVSI_GO(__bf16, float);
        AVSI_GO(__bf16, __bf16);
    }
    if (wdtype == AVSI_F32) AVSI_GO(_Float16, float);
    AVSI_GO(_Float16, _Float16);
#undef AVSI_GO
}
