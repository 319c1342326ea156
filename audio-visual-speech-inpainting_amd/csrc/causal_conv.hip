// Short causal convolution along time, one filter of K = 2 .. 8 taps per channel, for prompts, training and single tokens.
//
//   pre[b, t, d] = bias[d] + sum over k of w[d, k] x[b, t - K + 1 + k, d],   y = pre sigmoid(pre)  (or y = pre)
//   backward: dpre = dy * slope(pre),  dx[t] = sum over k of w[K - 1 - k] dpre[t + k],  dw[k] = sum dpre[t] x[t - K + 1 + k]
//
// x[-1], ..., x[1 - K] are the state (the last K - 1 inputs of the piece before, oldest first), or zero.  Behind lengths[b] outputs
// and gradients are zero, and nothing is read.
//
// All of it is bound by memory: one read of x (and dy), one write.  A thread owns 16 bytes of channels and a run of consecutive
// time steps, whose window slides through its registers, so an input is read once per run and K - 1 inputs again at its start.  In
// the backward pass the run is followed by K - 1 steps of the next one (dx needs their dpre); the weights' gradients stay in
// registers over all runs of a thread, are added over a workgroup in LDS and over the workgroups by a second launch, in a fixed order.
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

// Channels of a thread: 16 bytes; 8 where more than four taps of 16-bit values would not fit the registers of the backward pass.
template <typename T, int K> constexpr int channels() { return sizeof(T) == 4 || K > 4 ? 4 : 8; }

__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : (n < T ? n : T);
}

// Input t of the sequence, t >= 1 - K: from the state where t < 0.
template <typename T, int K, int V>
__device__ __forceinline__ void input(const Conv& a, const T* xb, int b, int t, int c, int n, float (&f)[V]) {
    if (t >= 0) {
        avsi_load<T, V>(xb + (int64_t)t * a.xt + c, n, f);
    } else if (a.state) {
        avsi_load<T, V>((const T*)a.state + ((int64_t)b * (K - 1) + K - 1 + t) * a.D + c, n, f);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = 0.f;
    }
}

template <typename T, int K, int V>
__device__ __forceinline__ void weights(const Conv& a, int c, int n, float (&w)[K][V], float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = i < n ? a.w[(int64_t)(c + i) * K + k] : 0.f;
        bias[i] = a.bias && i < n ? a.bias[c + i] : 0.f;
    }
}

template <typename T, int K> __global__ __launch_bounds__(256) void conv_fwd_kernel(Conv a, int runs) {
    constexpr int V = channels<T, K>();
    const int nv = (a.D + V - 1) / V;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(id % nv) * V;
    const int64_t rest = id / nv;
    const int b = (int)(rest / runs), t0 = (int)(rest % runs) * a.run;
    if (b >= a.B) return;
    const int n = a.D - c, len = length_of(a.lengths, b, a.T);
    const int t1 = t0 + a.run < a.T ? t0 + a.run : a.T, live = len < t1 ? len : t1;
    const T* xb = (const T*)a.x + (int64_t)b * a.xb;
    T* yb = (T*)a.y + (int64_t)b * a.yb + c;
    float w[K][V], bias[V], win[K][V], nx[V];
    if (t0 < live) {
        weights<T, K, V>(a, c, n, w, bias);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) input<T, K, V>(a, xb, b, t0 - K + 1 + k, c, n, win[k + 1]);
        avsi_load<T, V>(xb + (int64_t)t0 * a.xt + c, n, nx);
    }
    for (int t = t0; t < live; ++t) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int k = 0; k < K - 1; ++k) win[k][i] = win[k + 1][i];
            win[K - 1][i] = nx[i];
        }
        if (t + 1 < live) avsi_load<T, V>(xb + (int64_t)(t + 1) * a.xt + c, n, nx);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float p = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) p = fmaf(w[k][i], win[k][i], p);
            o[i] = a.silu ? p * avsi_sigmoid(p) : p;
        }
        avsi_store<T, V>(yb + (int64_t)t * a.yt, n, o);
    }
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    for (int t = live > t0 ? live : t0; t < t1; ++t) avsi_store<T, V>(yb + (int64_t)t * a.yt, n, zero);
    if (a.state_out && t0 == 0) {        // the last K - 1 inputs in front of `len`
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            input<T, K, V>(a, xb, b, len - K + 1 + k, c, n, nx);
            avsi_store<T, V>((T*)a.state_out + ((int64_t)b * (K - 1) + k) * a.D + c, n, nx);
        }
    }
}

// part: [gridDim.y][K + 1][D].  A workgroup: `wide` threads along the channels (a power of two), 256 / wide runs.
template <typename T, int K> __global__ __launch_bounds__(256) void conv_bwd_kernel(Conv a, int runs, int wide, float* __restrict__ part) {
    constexpr int V = channels<T, K>();
    __shared__ float lds[256 * V];
    const int lane = threadIdx.x % wide, slot = threadIdx.x / wide, slots = 256 / wide;
    const int c = (blockIdx.x * wide + lane) * V, n = a.D - c;
    float w[K][V], bias[V], dw[K][V], db[V];
    weights<T, K, V>(a, c, n, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
    }
    if (n > 0)
        for (int64_t r = (int64_t)blockIdx.y * slots + slot; r < (int64_t)a.B * runs; r += (int64_t)gridDim.y * slots) {
            const int b = (int)(r / runs), t0 = (int)(r % runs) * a.run, len = length_of(a.lengths, b, a.T);
            const int t1 = t0 + a.run < a.T ? t0 + a.run : a.T;
            const T* xb = (const T*)a.x + (int64_t)b * a.xb;
            const T* gb = (const T*)a.dy + (int64_t)b * a.gb + c;
            T* dxb = (T*)a.y + (int64_t)b * a.yb + c;
            float win[K][V], dp[K][V], nx[V], ng[V];
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int k = 0; k < K; ++k) dp[k][i] = win[k][i] = 0.f;
            if (t0 < len) {
#pragma unroll
                for (int k = 0; k < K - 1; ++k) input<T, K, V>(a, xb, b, t0 - K + 1 + k, c, n, win[k + 1]);
                avsi_load<T, V>(xb + (int64_t)t0 * a.xt + c, n, nx);
                avsi_load<T, V>(gb + (int64_t)t0 * a.gt, n, ng);
            }
            // dp[j] is dpre[t - K + 1 + j]; from t = t0 + K - 1 on dx[t - K + 1] is complete
            for (int t = t0; t < t1 + K - 1; ++t) {
                const bool live = t < len;
#pragma unroll
                for (int i = 0; i < V; ++i) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) {
                        win[k][i] = win[k + 1][i];
                        dp[k][i] = dp[k + 1][i];
                    }
                    win[K - 1][i] = live ? nx[i] : 0.f;
                    float p = bias[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) p = fmaf(w[k][i], win[k][i], p);
                    float slope = 1.f;
                    if (a.silu) {
                        const float s = avsi_sigmoid(p);
                        slope = s * fmaf(p, 1.f - s, 1.f);
                    }
                    dp[K - 1][i] = live ? ng[i] * slope : 0.f;
                }
                if (t + 1 < len && t + 1 < t1 + K - 1) {
                    avsi_load<T, V>(xb + (int64_t)(t + 1) * a.xt + c, n, nx);
                    avsi_load<T, V>(gb + (int64_t)(t + 1) * a.gt, n, ng);
                }
                if (t < t1) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        db[i] += dp[K - 1][i];
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][i] = fmaf(dp[K - 1][i], win[k][i], dw[k][i]);
                    }
                }
                if (t - K + 1 >= t0) {
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float s = 0.f;
#pragma unroll
                        for (int k = 0; k < K; ++k) s = fmaf(w[K - 1 - k][i], dp[k][i], s);
                        o[i] = s;
                    }
                    avsi_store<T, V>(dxb + (int64_t)(t - K + 1) * a.yt, n, o);
                }
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
            const int at = blockIdx.x * wide * V + i;
            float s = 0.f;
            for (int j = 0; j < slots; ++j) s += lds[j * wide * V + i];
            if (at < a.D) part[((int64_t)blockIdx.y * (K + 1) + k) * a.D + at] = s;
        }
    }
}

// dw[d][k], dbias[d] = sums of part[P][K + 1][D].
__global__ __launch_bounds__(1024) void conv_wgrad_sum_kernel(const float* __restrict__ part, int P, int K, int D, float* __restrict__ dw,
                                                              float* __restrict__ dbias) {
    const int64_t cols = (int64_t)(K + 1) * D, c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    const float s = avsi_column_sum(part, P, cols, cols);
    if (threadIdx.x < 32 && c < cols) {
        const int k = (int)(c / D), d = (int)(c % D);
        if (k < K) dw[(int64_t)d * K + k] = s;
        else if (dbias) dbias[d] = s;
    }
}

template <typename T, int K> __global__ __launch_bounds__(256) void conv_step_kernel(Conv a) {
    constexpr int V = channels<T, K>();
    const int nv = (a.D + V - 1) / V;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int c = (int)(id % nv) * V;
    const int64_t b = id / nv;
    if (b >= a.B) return;
    const int n = a.D - c;
    T* st = (T*)a.state_out + b * (K - 1) * a.D + c;
    avsi_raw<T, V> win[K];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) win[k] = avsi_load_raw<T, V>(st + (int64_t)k * a.D, n);
    win[K - 1] = avsi_load_raw<T, V>((const T*)a.x + b * a.xb + c, n);
    float w[K][V], bias[V], o[V];
    weights<T, K, V>(a, c, n, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float p = bias[i];
#pragma unroll
        for (int k = 0; k < K; ++k) p = fmaf(w[k][i], (float)win[k].v[i], p);
        o[i] = a.silu ? p * avsi_sigmoid(p) : p;
    }
    avsi_store<T, V>((T*)a.y + b * a.yb + c, n, o);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)win[k + 1].v[i];
        avsi_store<T, V>(st + (int64_t)k * a.D, n, f);
    }
}

int channels_of(int dtype, int taps) { return dtype == AVSI_F32 || taps > 4 ? 4 : 8; }
int vectors(int D, int dtype, int taps) { return (int)avsi_ceil_div(D, channels_of(dtype, taps)); }

// Steps per run: 4 .. 32, the longest that leaves 2^17 threads (2 waves per SIMD).
int run_length(int64_t B, int T, int D, int dtype, int taps) {
    int64_t r = B * T * vectors(D, dtype, taps) >> 17;
    return (int)(r < 4 ? 4 : r > 32 ? 32 : r);
}

// The backward pass' grid: threads along the channels, and workgroups over the runs = partials of the weights' gradients.
void bwd_shape(int64_t B, int T, int D, int dtype, int taps, int* wide, int* groups) {
    const int nv = vectors(D, dtype, taps);
    *wide = 1;
    while (*wide < 64 && *wide < nv) *wide *= 2;
    const int64_t runs = B * avsi_ceil_div(T, run_length(B, T, D, dtype, taps)), along = avsi_ceil_div(nv, *wide);
    int64_t g = avsi_ceil_div(runs, 256 / *wide), most = avsi_ceil_div(4 * AVSI_NUM_CU, along);
    *groups = (int)(g < most ? g : most);
}

bool shape_ok(int dtype, int B, int T, int D, int taps) { return avsi_dtype_ok(dtype) && B > 0 && T > 0 && D > 0 && taps >= 2 && taps <= 8; }

}  // namespace

#define AVSI_CONV_K(T, GO)        \
    switch (taps) {               \
        case 2: GO(T, 2); break;  \
        case 3: GO(T, 3); break;  \
        case 4: GO(T, 4); break;  \
        case 5: GO(T, 5); break;  \
        case 6: GO(T, 6); break;  \
        case 7: GO(T, 7); break;  \
        default: GO(T, 8); break; \
    }
#define AVSI_CONV_T(GO)                                         \
    if (dtype == AVSI_F32) { AVSI_CONV_K(float, GO) }           \
    else if (dtype == AVSI_BF16) { AVSI_CONV_K(__bf16, GO) }    \
    else { AVSI_CONV_K(_Float16, GO) }

extern "C" int avsi_causal_conv(const void* x, int64_t x_stride_b, int64_t x_stride_t, int dtype, const float* w, const float* bias,
                                int silu, const void* state, const int32_t* lengths, void* y, int64_t y_stride_b, int64_t y_stride_t,
                                void* state_out, int batch, int time, int dim, int taps, void* stream) {
    if (!shape_ok(dtype, batch, time, dim, taps) || !x || !w || !y) return AVSI_ERR_INVALID_ARG;
    const int run = run_length(batch, time, dim, dtype, taps), runs = (int)avsi_ceil_div(time, run);
    const int64_t wgs = avsi_ceil_div((int64_t)batch * runs * vectors(dim, dtype, taps), 256);
    if (wgs > 0x7fffffff) return AVSI_ERR_UNSUPPORTED;
    Conv a = {x, nullptr, state, y, state_out, w, bias, lengths, x_stride_b, x_stride_t, y_stride_b, y_stride_t, 0, 0, batch, time, dim, silu, run};
    avsi_clear_error();
#define AVSI_GO(T, K) hipLaunchKernelGGL((conv_fwd_kernel<T, K>), dim3(wgs), dim3(256), 0, (hipStream_t)stream, a, runs)
    AVSI_CONV_T(AVSI_GO)
#undef AVSI_GO
    return avsi_launch_status();
}

extern "C" size_t avsi_causal_conv_bwd_workspace_bytes(int dtype, int batch, int time, int dim, int taps) {
    if (!shape_ok(dtype, batch, time, dim, taps)) return 0;
    int wide, groups;
    bwd_shape(batch, time, dim, dtype, taps, &wide, &groups);
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
    bwd_shape(batch, time, dim, dtype, taps, &wide, &groups);
    const int run = run_length(batch, time, dim, dtype, taps), runs = (int)avsi_ceil_div(time, run);
    Conv a = {x, dy, state, dx, nullptr, w, bias, lengths, x_stride_b, x_stride_t, dx_stride_b, dx_stride_t, dy_stride_b, dy_stride_t,
              batch, time, dim, silu, run};
    const dim3 grid(avsi_ceil_div(vectors(dim, dtype, taps), wide), groups);
    float* part = dw ? (float*)workspace : nullptr;
    avsi_clear_error();
#define AVSI_GO(T, K) hipLaunchKernelGGL((conv_bwd_kernel<T, K>), grid, dim3(256), 0, (hipStream_t)stream, a, runs, wide, part)
    AVSI_CONV_T(AVSI_GO)
#undef AVSI_GO
    if (dw)
        hipLaunchKernelGGL(conv_wgrad_sum_kernel, dim3(avsi_ceil_div((int64_t)(taps + 1) * dim, 32)), dim3(1024), 0, (hipStream_t)stream,
                           part, groups, taps, dim, dw, dbias);
    return avsi_launch_status();
}

extern "C" int avsi_causal_conv_step(const void* x, int64_t x_stride_b, int dtype, const float* w, const float* bias, int silu,
                                     void* state, void* y, int64_t y_stride_b, int batch, int dim, int taps, void* stream) {
    if (!shape_ok(dtype, batch, 1, dim, taps) || !x || !w || !state || !y) return AVSI_ERR_INVALID_ARG;
    Conv a = {x, nullptr, nullptr, y, state, w, bias, nullptr, x_stride_b, 0, y_stride_b, 0, 0, 0, batch, 1, dim, silu, 1};
    const int64_t wgs = avsi_ceil_div((int64_t)batch * vectors(dim, dtype, taps), 256);
    if (wgs > 0x7fffffff) return AVSI_ERR_UNSUPPORTED;
    avsi_clear_error();
#define AVSI_GO(T, K) hipLaunchKernelGGL((conv_step_kernel<T, K>), dim3(wgs), dim3(256), 0, (hipStream_t)stream, a)
    AVSI_CONV_T(AVSI_GO)
#undef AVSI_GO
    return avsi_launch_status();
}
