// Layer norm over the last dimension, forward and backward, with the reduction of the weights' gradients.
//
//   mean = sum(x) / C,  var = sum((x - mean)^2) / C,  rstd = 1 / sqrt(var + eps),  h = (x - mean) rstd,  y = h gamma + beta
//   backward: e = dy gamma,  dx = rstd (e - mean(e) - h mean(e h)),  dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both passes are bound by memory: x in and y out (forward), x and dy in and dx out (backward).  A row is read ONCE into the
// registers of its group of lanes -- 16, 64, 256 or 1024 lanes with one to four 16-byte pieces each --
// and the variance is the second pass over those registers (a one-pass sum of squares would cancel where the mean is large).  The
// next row's loads are issued before this row's sums.  Rows beyond 1024 x 2 pieces are streamed: each pass over the row reads it
// again, from L2.  A group walks the rows r, r + groups, ... and keeps its slice of gamma (and beta) in registers.
//
// Widths in no whole pieces: the lane that the row's end cuts takes the last whole piece of the row instead, which overlaps its
// neighbour's; what both hold is counted once and written twice, with the same value.  (A branch around the load would wait for it.)
//
// 16384 x 2048 bf16: forward 22.7 us (5.9 TB/s, part of it the Infinity Cache's), backward 39 us (5.2 TB/s; a copy of that size 5.4) and
// 4 us for the partials; 8000 x 512 f32 backward 11.4 + 3.9 us; 32 x 512 f32 2.7 us.
//
// Weight gradients: every lane owns the same columns in all its rows, so dgamma and dbeta are sums in its registers; the groups of a
// workgroup are added in LDS in a fixed order, workgroups through partials [P][2][C] in the workspace and a second launch: no
// atomics, the same bits every time.
#include "avsi_common.h"
#include "avsi_wave.h"

namespace {

// Sums over the L lanes of a group: inside a wave, or over the whole workgroup through LDS.  Two buffers in turn: a wave that writes
// one again has passed the barrier behind which the other was read.  (The barrier waits for LDS only: loads stay in flight.)
template <int L> struct Sums {
    avsi_f2 lds[L > 64 ? 2 : 1][L > 64 ? L / 64 : 1];
};
template <int L> __device__ __forceinline__ avsi_f2 group_sums(float v, float w, Sums<L>& sums, int& turn) {
    v = avsi_group<L < 64 ? L : 64>(v);
    w = avsi_group<L < 64 ? L : 64>(w);
    if (L <= 64) return avsi_f2{v, w};
    if ((threadIdx.x & 63) == 0) sums.lds[turn][threadIdx.x >> 6] = avsi_f2{v, w};
    AVSI_LDS_BARRIER();
    avsi_f2 s = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < L / 64; ++i) {
        s[0] += sums.lds[turn][i][0];
        s[1] += sums.lds[turn][i][1];
    }
    turn ^= 1;
    return s;
}

// Where a lane's pieces lie: piece j starts at column c[j] and its elements from skip[j] on are its own.
template <typename T, int L, int NV, bool SMALL> struct Pieces {
    static constexpr int V = 16 / sizeof(T);
    int c[NV], skip[NV];
    __device__ __forceinline__ Pieces(int lane, int C) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * L + lane) * V;
            c[j] = SMALL ? at : (at < C - V ? at : C - V);
            skip[j] = SMALL ? 0 : at - c[j];
        }
    }
    __device__ __forceinline__ bool own(int j, int i, int C) const { return SMALL ? c[j] + i < C : i >= skip[j]; }
    __device__ __forceinline__ bool any(int j, int C) const { return SMALL ? c[j] < C : skip[j] < V; }
    // a piece of a row, or of a weight, in the elements' type
    template <typename E> __device__ __forceinline__ void load(const E* row, int j, int C, avsi_pack<E, V>& v) const {
        if (!SMALL) {
            v.load(row + c[j]);
        } else {                        // (fewer columns than a piece has)
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = (float)row[c[j] + i < C ? c[j] + i : C - 1];
            v.set(f);
        }
    }
    template <typename E> __device__ __forceinline__ void store(E* row, int j, int C, const float (&f)[V]) const {
        if (!any(j, C)) return;
        if (!SMALL) {
            avsi_pack<E, V> v;
            v.set(f);
            v.store(row + c[j]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c[j] + i < C) row[c[j] + i] = (E)f[i];
        }
    }
};

template <int L> constexpr int threads() { return L < 256 ? 256 : L; }

template <typename T, typename W, int L, int NV, bool SMALL>
__global__ __launch_bounds__(threads<L>()) void ln_fwd_kernel(const T* __restrict__ x, int64_t xs, const W* __restrict__ gamma,
                                                               const W* __restrict__ beta, T* __restrict__ y, int64_t ys,
                                                               float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int C,
                                                               float eps) {
    constexpr int V = 16 / sizeof(T), PER_WG = threads<L>() / L;
    __shared__ Sums<L> sums;
    int turn = 0;
    const int lane = threadIdx.x % L;
    const Pieces<T, L, NV, SMALL> at(lane, C);
    const float fc = (float)C;
    avsi_pack<W, V> gr[NV], br[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (gamma) at.load(gamma, j, C, gr[j]);
        if (beta) at.load(beta, j, C, br[j]);
    }
    const int64_t step = (int64_t)gridDim.x * PER_WG;
    int64_t r = (int64_t)blockIdx.x * PER_WG + threadIdx.x / L;
    avsi_pack<T, V> next[NV];
    if (r < rows)
#pragma unroll
        for (int j = 0; j < NV; ++j) at.load(x + r * xs, j, C, next[j]);
    for (; r < rows; r += step) {
        float v[NV][V], s = 0.f, q = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = next[j].at(i);
        const int64_t ahead = r + step < rows ? r + step : r;
#pragma unroll
        for (int j = 0; j < NV; ++j) at.load(x + ahead * xs, j, C, next[j]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) s += at.own(j, i, C) ? v[j][i] : 0.f;
        const float mu = group_sums<L>(s, 0.f, sums, turn)[0] / fc;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[j][i] -= mu;
                const float d = at.own(j, i, C) ? v[j][i] : 0.f;
                q = fmaf(d, d, q);
            }
        const float rs = 1.f / sqrtf(group_sums<L>(q, 0.f, sums, turn)[0] / fc + eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o[i] = v[j][i] * rs;
                if (gamma) o[i] *= gr[j].at(i);
                if (beta) o[i] += br[j].at(i);
            }
            at.store(y + r * ys, j, C, o);
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
    __shared__ Sums<L> sums;
    int turn = 0;
    const float fc = (float)C;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * xs;
        float s = 0.f, q = 0.f, v[V];
        for (int c = threadIdx.x * V; c < C; c += L * V) {
            avsi_load<T, V>(xr + c, C - c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) s += v[i];
        }
        const float mu = group_sums<L>(s, 0.f, sums, turn)[0] / fc;
        for (int c = threadIdx.x * V; c < C; c += L * V) {
            avsi_load<T, V>(xr + c, C - c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = c + i < C ? v[i] - mu : 0.f;
                q = fmaf(d, d, q);
            }
        }
        const float rs = 1.f / sqrtf(group_sums<L>(q, 0.f, sums, turn)[0] / fc + eps);
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

template <typename T, typename W, int L, int NV, bool SMALL, bool WGRAD>
__global__ __launch_bounds__(threads<L>()) void ln_bwd_kernel(const T* __restrict__ dy, int64_t dys, const T* __restrict__ x, int64_t xs,
                                                               const float* __restrict__ mean, const float* __restrict__ rstd,
                                                               const W* __restrict__ gamma, T* __restrict__ dx, int64_t dxs,
                                                               float* __restrict__ part, int64_t rows, int C) {
    constexpr int V = 16 / sizeof(T), PER_WG = threads<L>() / L;
    __shared__ Sums<L> sums;
    int turn = 0;
    __shared__ float acc[WGRAD && PER_WG > 1 ? 2 * L * V * NV : 1];
    const int lane = threadIdx.x % L, group = threadIdx.x / L;
    const Pieces<T, L, NV, SMALL> at(lane, C);
    const float inv = 1.f / (float)C;
    avsi_pack<W, V> gr[NV];
    float dg[NV][V], db[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (gamma) at.load(gamma, j, C, gr[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) dg[j][i] = db[j][i] = 0.f;
    }
    const int64_t step = (int64_t)gridDim.x * PER_WG;
    int64_t r = (int64_t)blockIdx.x * PER_WG + group;
    avsi_pack<T, V> nx[NV], ng[NV];
    float nmu = 0.f, nrs = 0.f;
    auto load = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            at.load(x + row * xs, j, C, nx[j]);
            at.load(dy + row * dys, j, C, ng[j]);
        }
        nmu = mean[row];
        nrs = rstd[row];
    };
    if (r < rows) load(r);
    for (; r < rows; r += step) {
        float h[NV][V], g[NV][V], s1 = 0.f, s2 = 0.f;
        const float mu = nmu, rs = nrs;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[j][i] = (nx[j].at(i) - mu) * rs;
                g[j][i] = ng[j].at(i);
            }
        load(r + step < rows ? r + step : r);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (WGRAD) {
                    dg[j][i] = fmaf(g[j][i], h[j][i], dg[j][i]);
                    db[j][i] += g[j][i];
                }
                if (gamma) g[j][i] *= gr[j].at(i);
                const float e = at.own(j, i, C) ? g[j][i] : 0.f;
                s1 += e;
                s2 += at.own(j, i, C) ? e * h[j][i] : 0.f;
            }
        const avsi_f2 both = group_sums<L>(s1, s2, sums, turn);
        const float m1 = both[0] * inv, m2 = both[1] * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int i = 0; i < V; ++i) g[j][i] = (g[j][i] - m1 - h[j][i] * m2) * rs;
            at.store(dx + r * dxs, j, C, g[j]);
        }
    }
    if (!WGRAD) return;
    // the groups of this workgroup, one after the other
    for (int k = 0; k < PER_WG; ++k) {
        if (PER_WG > 1) __syncthreads();
        if (group != k) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (PER_WG > 1) {
                float* a = acc + 2 * V * (j * L + lane);
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
                at.store(part + (int64_t)blockIdx.x * 2 * C, j, C, dg[j]);
                at.store(part + (int64_t)blockIdx.x * 2 * C + C, j, C, db[j]);
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
    __shared__ Sums<L> sums;
    int turn = 0;
    const float inv = 1.f / (float)C;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mu = mean[r], rs = rstd[r];
        float s1 = 0.f, s2 = 0.f, h[V], g[V], w[V];
        for (int pass = 0; pass < 2; ++pass) {
            float m1 = 0.f, m2 = 0.f;
            if (pass) {
                const avsi_f2 both = group_sums<L>(s1, s2, sums, turn);
                m1 = both[0] * inv, m2 = both[1] * inv;
            }
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

// dgamma, dbeta = sums of part[P][2][C].
__global__ __launch_bounds__(1024) void ln_wgrad_sum_kernel(const float* __restrict__ part, int P, int C, float* __restrict__ dgamma,
                                                            float* __restrict__ dbeta) {
    avsi_column_sums(part, P, 2 * (int64_t)C, 2 * (int64_t)C, [&](int64_t c, float s) {
        if (c < C) dgamma[c] = s;
        else dbeta[c - C] = s;
    });
}

// The group of lanes that a row of C columns takes, and its pieces per lane; 0 lanes: none holds it.  Four pieces only in the
// forward pass: the backward pass holds two rows and two sums per column.
struct Group { int L, NV; };
Group group_of(int C, int dtype, bool back) {
    const int V = 16 / avsi_dtype_size(dtype);
    const int64_t n = avsi_ceil_div(C, V);
    if (n <= 16) return {16, 1};
    if (n <= 128) return {64, n <= 64 ? 1 : 2};
    if (n <= 256) return back ? Group{256, 1} : Group{64, 4};
    if (n <= 512) return {256, 2};
    if (n <= 1024) return back ? Group{1024, 1} : Group{256, 4};
    return n <= 2048 ? Group{1024, 2} : Group{0, 0};
}

int fwd_groups(int64_t rows, int L) {
    const int per_wg = L && L < 256 ? 256 / L : 1;
    const int64_t wgs = avsi_ceil_div(rows, per_wg), most = (L == 1024 || L == 0 ? 2 : 8) * AVSI_NUM_CU;
    return (int)(wgs < most ? wgs : most);
}

// Workgroups of the backward pass = partials of the weights' gradients.
int bwd_groups(int64_t rows, int C, int dtype) {
    const int L = group_of(C, dtype, true).L;
    if (!L) return (int)(rows < 64 ? rows : 64);
    const int per_wg = L < 256 ? 256 / L : 1;
    const int64_t wgs = avsi_ceil_div(rows, per_wg), most = 2 * AVSI_NUM_CU;
    return (int)(wgs < most ? wgs : most);
}

#define AVSI_LN_SHAPES(GO, BIG)                         \
    if (C < 16 / (int)sizeof(T)) GO(16, 1, true);       \
    else if (g.L == 16) GO(16, 1, false);               \
    else if (g.L == 64 && g.NV == 1) GO(64, 1, false);  \
    else if (g.L == 64 && g.NV == 2) GO(64, 2, false);  \
    else if (g.L == 256 && g.NV == 2) GO(256, 2, false); \
    else if (g.L == 1024 && g.NV == 2) GO(1024, 2, false); \
    else BIG(GO)
#define AVSI_LN_BIG_FWD(GO) if (g.L == 64) GO(64, 4, false); else GO(256, 4, false)
#define AVSI_LN_BIG_BWD(GO) if (g.L == 256) GO(256, 1, false); else GO(1024, 1, false)

template <typename T, typename W>
int launch_fwd(const void* x, int64_t xs, const void* gamma, const void* beta, void* y, int64_t ys, float* mean, float* rstd,
               int64_t rows, int C, float eps, int dtype, hipStream_t s) {
    const Group g = group_of(C, dtype, false);
    const dim3 grid(fwd_groups(rows, g.L));
#define AVSI_LN_FWD(LANES, PIECES, SMALL)                                                                                            \
    hipLaunchKernelGGL((ln_fwd_kernel<T, W, LANES, PIECES, SMALL>), grid, dim3(threads<LANES>()), 0, s, (const T*)x, xs,             \
                       (const W*)gamma, (const W*)beta, (T*)y, ys, mean, rstd, rows, C, eps)
    if (!g.L)
        hipLaunchKernelGGL((ln_fwd_wide_kernel<T, W>), grid, dim3(1024), 0, s, (const T*)x, xs, (const W*)gamma, (const W*)beta, (T*)y,
                           ys, mean, rstd, rows, C, eps);
    else { AVSI_LN_SHAPES(AVSI_LN_FWD, AVSI_LN_BIG_FWD); }
#undef AVSI_LN_FWD
    return avsi_launch_status();
}

template <typename T, typename W>
int launch_bwd(const void* dy, int64_t dys, const void* x, int64_t xs, const float* mean, const float* rstd, const void* gamma,
               void* dx, int64_t dxs, float* dgamma, float* dbeta, float* part, int64_t rows, int C, int dtype, hipStream_t s) {
    const Group g = group_of(C, dtype, true);
    const int P = bwd_groups(rows, C, dtype);
#define AVSI_LN_BWD(LANES, PIECES, SMALL, WG)                                                                                        \
    hipLaunchKernelGGL((ln_bwd_kernel<T, W, LANES, PIECES, SMALL, WG>), dim3(P), dim3(threads<LANES>()), 0, s, (const T*)dy, dys,    \
                       (const T*)x, xs, mean, rstd, (const W*)gamma, (T*)dx, dxs, part, rows, C)
#define AVSI_LN_BWD_W(LANES, PIECES, SMALL) AVSI_LN_BWD(LANES, PIECES, SMALL, true)
#define AVSI_LN_BWD_X(LANES, PIECES, SMALL) AVSI_LN_BWD(LANES, PIECES, SMALL, false)
    if (!g.L) {
        hipLaunchKernelGGL((ln_bwd_wide_kernel<T, W>), dim3(fwd_groups(rows, 0)), dim3(1024), 0, s, (const T*)dy, dys, (const T*)x, xs,
                           mean, rstd, (const W*)gamma, (T*)dx, dxs, rows, C);
        if (dgamma)
            hipLaunchKernelGGL((ln_wgrad_wide_kernel<T>), dim3(avsi_ceil_div(C, 256 * (16 / sizeof(T))), P), dim3(256), 0, s,
                               (const T*)dy, dys, (const T*)x, xs, mean, rstd, part, rows, C);
    } else if (dgamma) {
        AVSI_LN_SHAPES(AVSI_LN_BWD_W, AVSI_LN_BIG_BWD);
    } else {
        AVSI_LN_SHAPES(AVSI_LN_BWD_X, AVSI_LN_BIG_BWD);
    }
#undef AVSI_LN_BWD_X
#undef AVSI_LN_BWD_W
#undef AVSI_LN_BWD
    if (dgamma)
        hipLaunchKernelGGL(ln_wgrad_sum_kernel, avsi_column_sum_grid(2 * (int64_t)C), dim3(1024), 0, s, part, P, C, dgamma, dbeta);
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
    hipStream_t s = (hipStream_t)stream;
#define AVSI_GO(T, W) return launch_fwd<T, W>(x, x_stride, gamma, beta, y, y_stride, mean, rstd, rows, cols, eps, dtype, s)
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
