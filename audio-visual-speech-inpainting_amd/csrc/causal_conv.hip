// Short causal convolution along time, one filter of K = 2 .. 8 taps per channel, for prompts, training and single tokens.
//
//   pre[b, t, d] = bias[d] + sum over k of w[d, k] x[b, t - K + 1 + k, d],   y = pre sigmoid(pre)  (or y = pre)
//   backward: dpre = dy * slope(pre),  dx[t] = sum over k of w[K - 1 - k] dpre[t + k],  dw[k] = sum dpre[t] x[t - K + 1 + k]
//
// x[-1], ..., x[1 - K] are the state (the last K - 1 inputs of the piece before, oldest first), or zero.  Behind lengths[b] outputs
// and gradients are zero, and nothing is read.
//
// All of it is bound by memory: one read of x (and dy), one write.  A thread owns four channels and a run of consecutive
// time steps, which it takes four at a time: the loads of the next four are in flight while these are computed, and the K - 1 inputs in
// front of them stay in registers, so an input is read once per run and K - 1 inputs again at its start.  In the backward pass the
// run is followed by K - 1 steps of the next one (dx needs their dpre); the weights' gradients stay in registers over all runs of a
// thread, are added over a workgroup in LDS and over the workgroups by a second launch, in a fixed order.
// 8 x 2048 x 2048 bf16, four taps: forward 28 us (4.8 TB/s), backward 49 us (4.1 TB/s) and 5 us for the partials; a copy 5.4 TB/s.
// Channels in no whole pieces: the last thread takes the last whole piece, which overlaps its neighbour's; both write the same values.
#include "avsi_common.h"
#include "avsi_wave.h"

namespace {

struct Conv {
    const void *x, *dy, *state;
    void *y, *state_out;                 // y: dx in the backward pass
    const float *w, *bias;
    const int32_t* lengths;
    int64_t xb, xt, yb, yt, gb, gt;      // strides of batch and time: x, y (dx), dy
    int B, T, D, silu, run;
};

// Channels of a thread, in any type.  (Sixteen bytes of a 16-bit type, eight channels, halve the waves that a CU holds: 29.9 against 27.0
// us forward, 67 against 54 backward, same runs, for 8 x 2048 x 2048 bf16 with four taps.)
constexpr int V = 4;

__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : (n < T ? n : T);
}

// A thread's channels c .. c + V - 1; SMALL: fewer channels than V exist, and they go one by one.
template <typename T, bool SMALL> struct Lane {
    int c;
    __device__ __forceinline__ Lane(int piece, int D) { c = SMALL ? 0 : (piece * V < D - V ? piece * V : D - V); }
    __device__ __forceinline__ void load(const T* row, int D, avsi_pack<T, V>& v) const {
        if (!SMALL) {
            v.load(row + c);
        } else {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = (float)row[i < D ? i : D - 1];
            v.set(f);
        }
    }
    __device__ __forceinline__ void store(T* row, int D, const avsi_pack<T, V>& v) const {
        if (!SMALL) {
            v.store(row + c);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < D) row[i] = (T)v.at(i);
        }
    }
    __device__ __forceinline__ void store(T* row, int D, const float (&f)[V]) const {
        avsi_pack<T, V> v;
        v.set(f);
        store(row, D, v);
    }
    __device__ __forceinline__ int channel(int i, int D) const { return SMALL ? (i < D ? i : D - 1) : c + i; }
};

// Input t of the sequence, 1 - K <= t < 0: from the state, if there is one.
template <typename T, int K, bool SMALL>
__device__ __forceinline__ void early(const Conv& a, const Lane<T, SMALL>& at, int64_t b, int t, float (&f)[V]) {
    avsi_pack<T, V> v;
    if (a.state) at.load((const T*)a.state + (b * (K - 1) + K - 1 + t) * a.D, a.D, v);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = a.state ? v.at(i) : 0.f;
}
// The K - 1 inputs in front of t0 into x[0 .. K - 2].
template <typename T, int K, int N, bool SMALL>
__device__ __forceinline__ void history(const Conv& a, const Lane<T, SMALL>& at, const T* xb, int64_t b, int t0, float (&x)[N][V]) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int t = t0 - K + 1 + k;
        if (t >= 0) {
            avsi_pack<T, V> v;
            at.load(xb + (int64_t)t * a.xt, a.D, v);
#pragma unroll
            for (int i = 0; i < V; ++i) x[k][i] = v.at(i);
        } else {
            early<T, K, SMALL>(a, at, b, t, x[k]);
        }
    }
}

template <typename T, int K, bool SMALL>
__device__ __forceinline__ void weights(const Conv& a, const Lane<T, SMALL>& at, float (&w)[K][V], float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = at.channel(i, a.D);
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = a.w[(int64_t)c * K + k];
        bias[i] = a.bias ? a.bias[c] : 0.f;
    }
}

template <typename T, int K, bool SMALL> __global__ __launch_bounds__(256) void conv_fwd_kernel(Conv a, int runs) {
    const int nv = (a.D + V - 1) / V;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rest = id / nv, b = rest / runs;
    const Lane<T, SMALL> at((int)(id % nv), a.D);
    const int t0 = (int)(rest % runs) * a.run;
    if (b >= a.B) return;
    const int len = length_of(a.lengths, (int)b, a.T);
    const int t1 = t0 + a.run < a.T ? t0 + a.run : a.T, live = len < t1 ? len : t1;
    const T* xb = (const T*)a.x + b * a.xb;
    T* yb = (T*)a.y + b * a.yb;
    float x[K + 3][V];
    if (t0 < live) {
        float w[K][V], bias[V];
        avsi_pack<T, V> next[4];
        auto load = [&](int t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) at.load(xb + (int64_t)(t + j < live ? t + j : live - 1) * a.xt, a.D, next[j]);
        };
        load(t0);
        weights<T, K, SMALL>(a, at, w, bias);
        history<T, K, K + 3, SMALL>(a, at, xb, b, t0, x);
        for (int t = t0; t < live; t += 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) x[K - 1 + j][i] = next[j].at(i);
            load(t + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float p = bias[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) p = fmaf(w[k][i], x[j + k][i], p);
                    const float s = p * avsi_sigmoid<T>(p);
                    o[i] = a.silu ? s : p;
                }
                if (t + j < live) at.store(yb + (int64_t)(t + j) * a.yt, a.D, o);
            }
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) x[k][i] = x[k + 4][i];
        }
    }
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    for (int t = live > t0 ? live : t0; t < t1; ++t) at.store(yb + (int64_t)t * a.yt, a.D, zero);
    if (a.state_out && t0 == 0) {        // the last K - 1 inputs in front of `len`
        history<T, K, K + 3, SMALL>(a, at, xb, b, len, x);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) at.store((T*)a.state_out + (b * (K - 1) + k) * a.D, a.D, x[k]);
    }
}

// part: [gridDim.y][K + 1][D].  A workgroup: `wide` threads along the channels (a power of two), 256 / wide runs.
template <typename T, int K, bool SMALL>
__global__ __launch_bounds__(256) void conv_bwd_kernel(Conv a, int runs, int wide, float* __restrict__ part) {
    __shared__ float lds[256 * V];
    const int piece = blockIdx.x * wide + threadIdx.x % wide, slot = threadIdx.x / wide, slots = 256 / wide;
    const bool mine = piece * V < a.D;
    const Lane<T, SMALL> at(piece, a.D);
    float w[K][V], bias[V], dw[K][V], db[V];
    weights<T, K, SMALL>(a, at, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
    }
    if (mine)
        for (int64_t r = (int64_t)blockIdx.y * slots + slot; r < (int64_t)a.B * runs; r += (int64_t)gridDim.y * slots) {
            const int64_t b = r / runs;
            const int t0 = (int)(r % runs) * a.run, len = length_of(a.lengths, (int)b, a.T);
            const int t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
            const T* xb = (const T*)a.x + b * a.xb;
            const T* gb = (const T*)a.dy + b * a.gb;
            T* dxb = (T*)a.y + b * a.yb;
            // x[K - 1 + j] and d[K - 1 + j] are input and dpre of step t + j; dx[t - K + 1 + j] is complete with d[j .. j + K - 1]
            float x[K + 3][V], d[K + 3][V];
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) d[k][i] = 0.f;
            if (t0 < len) {
                const int stop = len < t1 + K - 1 ? len : t1 + K - 1;       // steps that are read
                avsi_pack<T, V> nx[4], ng[4];
                auto load = [&](int t) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int64_t u = t + j < stop ? t + j : stop - 1;
                        at.load(xb + u * a.xt, a.D, nx[j]);
                        at.load(gb + u * a.gt, a.D, ng[j]);
                    }
                };
                load(t0);
                history<T, K, K + 3, SMALL>(a, at, xb, b, t0, x);
                for (int t = t0; t < t1 + K - 1; t += 4) {
                    float g[4][V];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            x[K - 1 + j][i] = nx[j].at(i);
                            g[j][i] = ng[j].at(i);
                        }
                    load(t + 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool live = t + j < stop, own = t + j < t1 && live;
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            float p = bias[i];
#pragma unroll
                            for (int k = 0; k < K; ++k) p = fmaf(w[k][i], x[j + k][i], p);
                            const float s = avsi_sigmoid<T>(p), slope = s * fmaf(p, 1.f - s, 1.f);
                            d[K - 1 + j][i] = live ? g[j][i] * (a.silu ? slope : 1.f) : 0.f;
                        }
                        // (not with a factor of zero: an input that is infinite or NaN belongs to the steps that it is a tap of)
                        if (own)
#pragma unroll
                            for (int i = 0; i < V; ++i) {
                                db[i] += d[K - 1 + j][i];
#pragma unroll
                                for (int k = 0; k < K; ++k) dw[k][i] = fmaf(d[K - 1 + j][i], x[j + k][i], dw[k][i]);
                            }
                        float o[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            float s = 0.f;
#pragma unroll
                            for (int k = 0; k < K; ++k) s = fmaf(w[K - 1 - k][i], d[j + k][i], s);
                            o[i] = s;
                        }
                        const int u = t + j - K + 1;
                        if (u >= t0 && u < t1) at.store(dxb + (int64_t)u * a.yt, a.D, o);
                    }
#pragma unroll
                    for (int k = 0; k < K - 1; ++k)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            x[k][i] = x[k + 4][i];
                            d[k][i] = d[k + 4][i];
                        }
                }
            } else {
                for (int t = t0; t < t1; ++t) at.store(dxb + (int64_t)t * a.yt, a.D, d[0]);
            }
        }
    if (!part) return;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) lds[threadIdx.x * V + i] = k < K ? dw[k < K ? k : 0][i] : db[i];
        __syncthreads();
        for (int i = threadIdx.x; i < wide * V; i += 256) {
            const int of = blockIdx.x * wide + i / V;
            const int c = Lane<T, SMALL>(of, a.D).c + i % V;
            float s = 0.f;
            for (int j = 0; j < slots; ++j) s += lds[j * wide * V + i];
            if (of * V < a.D && c < a.D) part[((int64_t)blockIdx.y * (K + 1) + k) * a.D + c] = s;
        }
    }
}

// dw[d][k], dbias[d] = sums of part[P][K + 1][D].
__global__ __launch_bounds__(1024) void conv_wgrad_sum_kernel(const float* __restrict__ part, int P, int K, int D, float* __restrict__ dw,
                                                              float* __restrict__ dbias) {
    const int64_t cols = (int64_t)(K + 1) * D;
    avsi_column_sums(part, P, cols, cols, [&](int64_t c, float s) {
        int k = 0;                  // (at most 8 turns, where a division of 64 bits behind the sum takes half a microsecond)
        int64_t d = c;
        for (; d >= D; d -= D) ++k;
        if (k < K) dw[d * K + k] = s;
        else if (dbias) dbias[d] = s;
    });
}

template <typename T, int K> __global__ __launch_bounds__(256) void conv_step_kernel(Conv a) {
    const int nv = (a.D + V - 1) / V;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, b = id / nv;
    if (b >= a.B) return;
    // (no overlap here, where state is read and written: the thread that the last channel cuts goes one by one)
    const int c = (int)(id % nv) * V, n = a.D - c;
    T* st = (T*)a.state_out + b * (K - 1) * a.D + c;
    const T* x = (const T*)a.x + b * a.xb + c;
    avsi_pack<T, V> win[K];
    auto fetch = [&](const T* p, avsi_pack<T, V>& v) {
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)p[i < n ? i : n - 1];
        v.set(f);
    };
    if (n >= V) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[k].load(st + (int64_t)k * a.D);
        win[K - 1].load(x);
    } else {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) fetch(st + (int64_t)k * a.D, win[k]);
        fetch(x, win[K - 1]);
    }
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int ch = c + (i < n ? i : n - 1);
        float p = a.bias ? a.bias[ch] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) p = fmaf(a.w[(int64_t)ch * K + k], win[k].at(i), p);
        const float s = p * avsi_sigmoid<T>(p);
        o[i] = a.silu ? s : p;
    }
    T* y = (T*)a.y + b * a.yb + c;
    if (n >= V) {
        avsi_pack<T, V> v;
        v.set(o);
        v.store(y);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[k + 1].store(st + (int64_t)k * a.D);
    } else {
        for (int i = 0; i < n; ++i) {
            y[i] = (T)o[i];
#pragma unroll
            for (int k = 0; k < K - 1; ++k) st[(int64_t)k * a.D + i] = (T)win[k + 1].at(i);
        }
    }
}

// Steps per run, a multiple of four.  Forward: 4 .. 32, the longest that leaves 2^18 threads (4 waves per SIMD).  1 x 8191 x 1536 bf16 in us
// with 4, 8, 12, 16, 32 steps: 16.5, 14.1, 13.3, 13.2, 14.8 (12 by this rule); 8 x 2048 x 2048: 35.1, 27.6, 27.1, 27.0, 27.6 (32).
int run_fwd(int64_t B, int T, int D) {
    const int64_t r = (B * T * avsi_ceil_div(D, V) >> 18) / 4 * 4;
    return (int)(r < 4 ? 4 : r > 32 ? 32 : r);
}
// Backward: 8 .. 64, the shortest with which three workgroups to each CU, which is what its registers hold, take all runs at once: a run
// costs K - 1 more steps, and a fourth workgroup comes after the others.  The same two with 8, 16, 32, 64 steps: 34.0, 26.3, 27.7,
// 33.3 (16 by this rule) and 64.4, 54.2, 49.6, 45.7 (44: 46).
constexpr int BACK_WGS = 3 * AVSI_NUM_CU;
int run_bwd(int64_t B, int T, int D) {
    const int64_t r = avsi_round_up(avsi_ceil_div(B * T * avsi_ceil_div(D, V), 256 * BACK_WGS), 4);
    return (int)(r < 8 ? 8 : r > 64 ? 64 : r);
}

// The backward pass' grid: threads along the channels, and workgroups over the runs = partials of the weights' gradients.
void bwd_shape(int64_t B, int T, int D, int* wide, int* groups) {
    const int nv = (int)avsi_ceil_div(D, V);
    *wide = 1;
    while (*wide < 64 && *wide < nv) *wide *= 2;
    const int64_t runs = B * avsi_ceil_div(T, run_bwd(B, T, D)), along = avsi_ceil_div(nv, *wide);
    int64_t g = avsi_ceil_div(runs, 256 / *wide), most = avsi_ceil_div(BACK_WGS, along);
    *groups = (int)(g < most ? g : most);
}

// (time up to 2^30: a step in front of or behind a sequence still has a number; channels likewise, behind the last one)
bool shape_ok(int dtype, int B, int T, int D, int taps) {
    return avsi_dtype_ok(dtype) && B > 0 && T > 0 && T <= (1 << 30) && D > 0 && D <= 0x7fffffff - 1023 && taps >= 2 && taps <= 8;
}

}  // namespace

#define AVSI_CONV_K(T, GO)                                \
    if (dim < V) {                                        \
        switch (taps) { AVSI_CONV_TAPS(T, GO, true) }     \
    } else {                                              \
        switch (taps) { AVSI_CONV_TAPS(T, GO, false) }    \
    }
#define AVSI_CONV_TAPS(T, GO, SMALL) \
    case 2: GO(T, 2, SMALL); break;  \
    case 3: GO(T, 3, SMALL); break;  \
    case 4: GO(T, 4, SMALL); break;  \
    case 5: GO(T, 5, SMALL); break;  \
    case 6: GO(T, 6, SMALL); break;  \
    case 7: GO(T, 7, SMALL); break;  \
    default: GO(T, 8, SMALL); break;
#define AVSI_CONV_T(GO)                                         \
    if (dtype == AVSI_F32) { AVSI_CONV_K(float, GO) }           \
    else if (dtype == AVSI_BF16) { AVSI_CONV_K(__bf16, GO) }    \
    else { AVSI_CONV_K(_Float16, GO) }

extern "C" int avsi_causal_conv(const void* x, int64_t x_stride_b, int64_t x_stride_t, int dtype, const float* w, const float* bias,
                                int silu, const void* state, const int32_t* lengths, void* y, int64_t y_stride_b, int64_t y_stride_t,
                                void* state_out, int batch, int time, int dim, int taps, void* stream) {
    if (!shape_ok(dtype, batch, time, dim, taps) || !x || !w || !y) return AVSI_ERR_INVALID_ARG;
    const int run = run_fwd(batch, time, dim), runs = (int)avsi_ceil_div(time, run);
    const int64_t wgs = avsi_ceil_div((int64_t)batch * runs * avsi_ceil_div(dim, V), 256);
    if (!avsi_grid_ok(wgs, 256)) return AVSI_ERR_UNSUPPORTED;
    Conv a = {x, nullptr, state, y, state_out, w, bias, lengths, x_stride_b, x_stride_t, y_stride_b, y_stride_t, 0, 0, batch, time, dim, silu, run};
    avsi_clear_error();
#define AVSI_GO(T, K, SMALL) hipLaunchKernelGGL((conv_fwd_kernel<T, K, SMALL>), dim3(wgs), dim3(256), 0, (hipStream_t)stream, a, runs)
    AVSI_CONV_T(AVSI_GO)
#undef AVSI_GO
    return avsi_launch_status();
}

extern "C" size_t avsi_causal_conv_bwd_workspace_bytes(int dtype, int batch, int time, int dim, int taps) {
    if (!shape_ok(dtype, batch, time, dim, taps)) return 0;
    int wide, groups;
    bwd_shape(batch, time, dim, &wide, &groups);
    return (size_t)groups * (taps + 1) * dim * sizeof(float);
}

extern "C" int avsi_causal_conv_bwd(const void* dy, int64_t dy_stride_b, int64_t dy_stride_t, const void* x, int64_t x_stride_b,
                                    int64_t x_stride_t, int dtype, const float* w, const float* bias, int silu, const void* state,
                                    const int32_t* lengths, void* dx, int64_t dx_stride_b, int64_t dx_stride_t, float* dw, float* dbias,
                                    int batch, int time, int dim, int taps, void* workspace, size_t workspace_bytes, void* stream) {
    if (!shape_ok(dtype, batch, time, dim, taps) || !dy || !x || !w || !dx || (dbias && !dw)) return AVSI_ERR_INVALID_ARG;
    if (dw && (!workspace || workspace_bytes < avsi_causal_conv_bwd_workspace_bytes(dtype, batch, time, dim, taps)))
        return AVSI_ERR_WORKSPACE;
    int wide, groups;
    bwd_shape(batch, time, dim, &wide, &groups);
    const int run = run_bwd(batch, time, dim), runs = (int)avsi_ceil_div(time, run);
    Conv a = {x, dy, state, dx, nullptr, w, bias, lengths, x_stride_b, x_stride_t, dx_stride_b, dx_stride_t, dy_stride_b, dy_stride_t,
              batch, time, dim, silu, run};
    const dim3 grid(avsi_ceil_div(avsi_ceil_div(dim, V), wide), groups);
    float* part = dw ? (float*)workspace : nullptr;
    avsi_clear_error();
#define AVSI_GO(T, K, SMALL) hipLaunchKernelGGL((conv_bwd_kernel<T, K, SMALL>), grid, dim3(256), 0, (hipStream_t)stream, a, runs, wide, part)
    AVSI_CONV_T(AVSI_GO)
#undef AVSI_GO
    if (dw)
        hipLaunchKernelGGL(conv_wgrad_sum_kernel, avsi_column_sum_grid((int64_t)(taps + 1) * dim), dim3(1024), 0, (hipStream_t)stream,
                           part, groups, taps, dim, dw, dbias);
    return avsi_launch_status();
}

extern "C" int avsi_causal_conv_step(const void* x, int64_t x_stride_b, int dtype, const float* w, const float* bias, int silu,
                                     void* state, void* y, int64_t y_stride_b, int batch, int dim, int taps, void* stream) {
    if (!shape_ok(dtype, batch, 1, dim, taps) || !x || !w || !state || !y) return AVSI_ERR_INVALID_ARG;
    Conv a = {x, nullptr, nullptr, y, state, w, bias, nullptr, x_stride_b, 0, y_stride_b, 0, 0, 0, batch, 1, dim, silu, 1};
    const int64_t wgs = avsi_ceil_div(batch * avsi_ceil_div(dim, V), 256);
    if (!avsi_grid_ok(wgs, 256)) return AVSI_ERR_UNSUPPORTED;
    avsi_clear_error();
#define AVSI_GO(T, K, SMALL) hipLaunchKernelGGL((conv_step_kernel<T, K>), dim3(wgs), dim3(256), 0, (hipStream_t)stream, a)
    AVSI_CONV_T(AVSI_GO)
#undef AVSI_GO
    return avsi_launch_status();
}
