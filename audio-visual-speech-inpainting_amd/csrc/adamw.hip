// One AdamW step over many tensors in few launches, moments in 32 or in 8 bits.
//
//   g = grad grad_scale,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   w -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay w),  copy = w rounded to the copy's type
//
// In 8 bits a block of 256 consecutive values of a tensor shares a scale: m is held as e4m3 of m / (max|m| / 448), and v as e4m3 of
// r = sqrt(v), likewise: the square root halves the range that eight bits have to hold, and it is what the step divides by.  A
// positive r keeps at least the smallest code: rounded to zero it would divide the next step by eps alone.  All arithmetic, and the
// weights, are fp32; the step itself uses the moments before they are rounded.
//
// Bound by memory: 28 bytes per value (w, m, v read and written, grad read), 16 with 8-bit moments, a 16-bit gradient and a 16-bit
// copy.  A workgroup takes 4096 consecutive values of one tensor, a wave four blocks of 256, a lane four consecutive values of each:
// loads of 16 bytes, all of a lane's issued before the first is used.  The tensors of a launch (up to 48) come in its arguments,
// so nothing is uploaded and a captured launch holds its table; a workgroup finds its tensor by halving over the first chunks.
// 151 M values, 8-bit moments, bf16 gradients and copies: 475 us (5.1 TB/s, a copy's rate at that size); 4.1 M values in 32 bits: 18.9 us
// (6.2 TB/s, part of it the Infinity Cache's).
#include "avsi_common.h"
#include "avsi_wave.h"

namespace {

constexpr int MOST = 48;                // tensors per launch: their table and the rest of the arguments stay below 4 KiB
constexpr int BLOCK = 256, PER_LANE = 4;
constexpr int CHUNK = 4 * PER_LANE * BLOCK;       // values of a workgroup
constexpr int64_t LAUNCH = ((int64_t)1 << 24) - 1;       // workgroups of a launch, which has fewer than 2^32 threads

struct Table {
    avsi_adamw_tensor t[MOST];
    int first[MOST];                    // chunk
    int count;
};
struct Hyper {
    float lr, b1, ob1, b2, ob2, eps, c1, root_c2, scale;
    int n_skip;
    const float* skip;
};
static_assert(sizeof(Table) + sizeof(Hyper) <= 4096, "kernel arguments");

// Maximum of absolute values by their bits: a NaN is above everything and stays.
struct top_bits {
    static __device__ __forceinline__ float of(float a, float b) {
        const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
        return __builtin_bit_cast(float, x > y ? x : y);
    }
};

// Four codes of x * inv, the block's scale.  `top`: the block's largest absolute value.
__device__ __forceinline__ float block_inv(float top) { return top != 0.f ? fminf(1.f / top * 448.f, 3.402823466e38f) : 0.f; }
__device__ __forceinline__ unsigned pack4(const float (&y)[4]) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], p, true);
}
__device__ __forceinline__ void unpack4(unsigned c, float s, float (&f)[4]) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    f[0] = a[0] * s, f[1] = a[1] * s, f[2] = b[0] * s, f[3] = b[1] * s;
}
__device__ __forceinline__ unsigned load_codes(const uint8_t* p, int n) {
    unsigned c = 0;
    if (n >= 4) __builtin_memcpy(&c, p, 4);
    else
        for (int i = 0; i < n; ++i) c |= (unsigned)p[i] << (8 * i);
    return c;
}
__device__ __forceinline__ void store_codes(uint8_t* p, int n, unsigned c) {
    if (n >= 4) __builtin_memcpy(p, &c, 4);
    else
        for (int i = 0; i < n; ++i) p[i] = (uint8_t)(c >> (8 * i));
}

// The moments, their scales and codes take one rounding per operation, in the order in which they stand here: a code next to a border
// goes to the same side as in any other evaluation of the formula in elementary fp32 operations.  (A fused one would differ in one code
// of some millions, by up to a sixteenth of its value, and where such a code is its block's largest in a later step the whole block
// follows.)  The weights, which no border hangs on, take fused operations.
template <int BITS> __global__ __launch_bounds__(256) void adamw_kernel(Table tab, Hyper h) {
    for (int i = 0; i < h.n_skip; ++i)
        if (!(h.skip[i] == 0.f)) return;
    int lo = 0, hi = tab.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (tab.first[mid] <= (int)blockIdx.x) lo = mid;
        else hi = mid;
    }
    const avsi_adamw_tensor& t = tab.t[lo];
    const int64_t base = (int64_t)((int)blockIdx.x - tab.first[lo]) * CHUNK + (threadIdx.x >> 6) * (PER_LANE * BLOCK);
    const int64_t left = t.numel - base - 4 * (threadIdx.x & 63);
    const int64_t at = base + 4 * (threadIdx.x & 63);
    float w[PER_LANE][4], g[PER_LANE][4], m[PER_LANE][4], v[PER_LANE][4];
    unsigned mc[PER_LANE], vc[PER_LANE];
    float ms[PER_LANE], vs[PER_LANE];
    int n[PER_LANE];
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
        const int64_t r = left - k * BLOCK, i = at + k * BLOCK;
        n[k] = r < 0 ? 0 : r > 4 ? 4 : (int)r;
        avsi_load<float, 4>(t.w + i, n[k], w[k]);
        if (BITS == 32) {
            avsi_load<float, 4>((const float*)t.m + i, n[k], m[k]);
            avsi_load<float, 4>((const float*)t.v + i, n[k], v[k]);
        } else {
            mc[k] = load_codes((const uint8_t*)t.m + i, n[k]);
            vc[k] = load_codes((const uint8_t*)t.v + i, n[k]);
            const bool on = base + k * BLOCK < t.numel;
            ms[k] = on ? t.m_scale[base / BLOCK + k] : 0.f;
            vs[k] = on ? t.v_scale[base / BLOCK + k] : 0.f;
        }
    }
    if (t.grad_dtype == AVSI_F32) {
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) avsi_load<float, 4>((const float*)t.grad + at + k * BLOCK, n[k], g[k]);
    } else if (t.grad_dtype == AVSI_BF16) {
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) avsi_load<__bf16, 4>((const __bf16*)t.grad + at + k * BLOCK, n[k], g[k]);
    } else {
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) avsi_load<_Float16, 4>((const _Float16*)t.grad + at + k * BLOCK, n[k], g[k]);
    }
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
        const int64_t i = at + k * BLOCK;
        float r[4], topm = 0.f, topr = 0.f;
        if (BITS == 8) {
            unpack4(mc[k], ms[k], m[k]);
            unpack4(vc[k], vs[k], v[k]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k][j] *= v[k][j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma clang fp contract(off)
            const float gj = g[k][j] * h.scale;
            m[k][j] = h.b1 * m[k][j] + h.ob1 * gj;
            v[k][j] = h.b2 * v[k][j] + h.ob2 * gj * gj;
            r[j] = sqrtf(v[k][j]);
            const float d = fmaf(r[j], h.root_c2, h.eps);
            w[k][j] = fmaf(-h.lr, fmaf(t.weight_decay, w[k][j], (m[k][j] * h.c1) / d), w[k][j]);
            if (BITS == 8) {
                topm = top_bits::of(topm, fabsf(m[k][j]));
                topr = top_bits::of(topr, fabsf(r[j]));
            }
        }
        avsi_store<float, 4>(t.w + i, n[k], w[k]);
        if (t.copy) {
            if (t.copy_dtype == AVSI_BF16) avsi_store<__bf16, 4>((__bf16*)t.copy + i, n[k], w[k]);
            else if (t.copy_dtype == AVSI_F16) avsi_store<_Float16, 4>((_Float16*)t.copy + i, n[k], w[k]);
            else avsi_store<float, 4>((float*)t.copy + i, n[k], w[k]);
        }
        if (BITS == 32) {
            avsi_store<float, 4>((float*)t.m + i, n[k], m[k]);
            avsi_store<float, 4>((float*)t.v + i, n[k], v[k]);
        } else {
            topm = avsi_group<64, top_bits>(topm);
            topr = avsi_group<64, top_bits>(topr);
            const float im = block_inv(topm), ir = block_inv(topr);
            const float least = ir > 0.f ? 0x1p-9f : 0.f;        // (an infinite scale: codes of zero decode to NaN)
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = m[k][j] * im;
            store_codes((uint8_t*)t.m + i, n[k], pack4(y));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y[j] = r[j] * ir;
                if (r[j] > 0.f && y[j] < least) y[j] = least;
            }
            store_codes((uint8_t*)t.v + i, n[k], pack4(y));
            if ((threadIdx.x & 63) == 0 && base + k * BLOCK < t.numel) {
                t.m_scale[base / BLOCK + k] = topm * (1.f / 448.f);
                t.v_scale[base / BLOCK + k] = topr * (1.f / 448.f);
            }
        }
    }
}

}  // namespace

extern "C" int avsi_adamw(const avsi_adamw_tensor* tensors, int count, int bits, double lr, double beta1, double beta2, double eps,
                          int64_t step, double grad_scale, const float* skip, int n_skip, void* stream) {
    if (!tensors || count < 0 || (bits != 8 && bits != 32) || step < 1 || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) ||
        !(eps >= 0) || n_skip < 0 || n_skip > 8 || (n_skip && !skip))
        return AVSI_ERR_INVALID_ARG;
    for (int i = 0; i < count; ++i) {
        const avsi_adamw_tensor& t = tensors[i];
        if (t.numel < 0 || t.numel > LAUNCH * CHUNK) return AVSI_ERR_INVALID_ARG;
        if (t.numel == 0) continue;
        if (!t.w || !t.grad || !t.m || !t.v || !avsi_dtype_ok(t.grad_dtype) || (t.copy && !avsi_dtype_ok(t.copy_dtype)) ||
            (bits == 8 && (!t.m_scale || !t.v_scale)))
            return AVSI_ERR_INVALID_ARG;
    }
    Hyper h;
    h.lr = (float)lr, h.b1 = (float)beta1, h.ob1 = (float)(1 - beta1), h.b2 = (float)beta2, h.ob2 = (float)(1 - beta2), h.eps = (float)eps;
    h.c1 = (float)(1 / (1 - pow(beta1, (double)step)));
    h.root_c2 = (float)sqrt(1 / (1 - pow(beta2, (double)step)));
    h.scale = (float)grad_scale, h.skip = skip, h.n_skip = n_skip;
    avsi_clear_error();
    Table tab;
    tab.count = 0;
    int64_t chunks = 0;
    for (int i = 0; i <= count; ++i) {
        const int64_t more = i < count ? avsi_ceil_div(tensors[i].numel, CHUNK) : 0;
        if (tab.count && (i == count || tab.count == MOST || chunks + more > LAUNCH)) {
            if (bits == 32) hipLaunchKernelGGL(adamw_kernel<32>, dim3(chunks), dim3(256), 0, (hipStream_t)stream, tab, h);
            else hipLaunchKernelGGL(adamw_kernel<8>, dim3(chunks), dim3(256), 0, (hipStream_t)stream, tab, h);
            tab.count = 0;
            chunks = 0;
        }
        if (i == count || tensors[i].numel == 0) continue;
        tab.t[tab.count] = tensors[i];
        tab.first[tab.count++] = (int)chunks;
        chunks += more;
    }
    return avsi_launch_status();
}
