// Element types and lane sums shared by the kernels that take float32, bfloat16 and float16 tensors
// (layer_norm.hip, scan.hip, causal_conv.hip, adamw.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef __attribute__((ext_vector_type(2))) float avsi_f2;
typedef __attribute__((ext_vector_type(4))) float avsi_f4;

// One element type behind the codes avsi_dtype of the C ABI: rounding from fp32 is to nearest even in all of them.
template <int CODE> struct avsi_type;
template <> struct avsi_type<AVSI_F32> { typedef float T; };
template <> struct avsi_type<AVSI_BF16> { typedef __bf16 T; };
template <> struct avsi_type<AVSI_F16> { typedef _Float16 T; };

static inline bool avsi_dtype_ok(int code) { return code == AVSI_F32 || code == AVSI_BF16 || code == AVSI_F16; }
static inline int avsi_dtype_size(int code) { return code == AVSI_F32 ? 4 : 2; }

// V consecutive elements as fp32.  gfx950 takes loads and stores of 16 bytes at any address that is aligned to the element, so rows
// of odd width or pitch need no kernel of their own; `n` < V elements exist at the end of a row: those are taken one by one.
template <typename T, int V> struct avsi_raw { T v[V]; };
template <typename T, int V> __device__ __forceinline__ avsi_raw<T, V> avsi_load_raw(const T* __restrict__ p, int n) {
    avsi_raw<T, V> r;
    if (n >= V) {
        __builtin_memcpy(&r, p, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
    }
    return r;
}
template <typename T, int V> __device__ __forceinline__ void avsi_load(const T* __restrict__ p, int n, float (&f)[V]) {
    const avsi_raw<T, V> r = avsi_load_raw<T, V>(p, n);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = (float)r.v[i];
}
template <typename T, int V> __device__ __forceinline__ void avsi_store(T* __restrict__ p, int n, const float (&f)[V]) {
    avsi_raw<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)f[i];
    if (n >= V) {
        __builtin_memcpy(p, &r, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = r.v[i];
    }
}

// Four elements as they lie in memory, in 32-bit words: a load of them that is in flight stays one register group, where an array of
// 16-bit elements is taken apart (and waited for) at once.
template <typename T> struct avsi_quad {
    typedef __attribute__((ext_vector_type(sizeof(T)))) unsigned V;
    V v;
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&v, p, sizeof(v)); }
    __device__ __forceinline__ void get(float (&f)[4]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(float, (unsigned)v[i]);
        } else if constexpr (__is_same(T, __bf16)) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[2 * i] = __builtin_bit_cast(float, (unsigned)v[i] << 16);
                f[2 * i + 1] = __builtin_bit_cast(float, (unsigned)v[i] & 0xffff0000u);
            }
        } else {
            typedef __attribute__((ext_vector_type(2))) _Float16 half2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const half2 h = __builtin_bit_cast(half2, (unsigned)v[i]);
                f[2 * i] = (float)h[0], f[2 * i + 1] = (float)h[1];
            }
        }
    }
    __device__ __forceinline__ void set(const float (&f)[4]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(unsigned, f[i]);
        } else {
            typedef __attribute__((ext_vector_type(2))) T Pair;
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = __builtin_bit_cast(unsigned, Pair{(T)f[2 * i], (T)f[2 * i + 1]});
        }
    }
    // the first n of them
    __device__ __forceinline__ void store(T* p, int n) const {
        if (n >= 4) {
            __builtin_memcpy(p, &v, sizeof(v));
            return;
        }
        T e[4];
        __builtin_memcpy(e, &v, sizeof(v));
        if (n > 0) p[0] = e[0];
        if (n > 1) p[1] = e[1];
        if (n > 2) p[2] = e[2];
    }
};

// V elements as words: the same for pieces of V * sizeof(T) bytes.
template <typename T, int V> struct avsi_pack {
    static constexpr int WORDS = V * sizeof(T) / 4;
    typedef __attribute__((ext_vector_type(WORDS))) unsigned W;
    W v;
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(&v, p, sizeof(v)); }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, &v, sizeof(v)); }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, (unsigned)v[i]);
        const unsigned w = v[i / 2];
        if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
        typedef __attribute__((ext_vector_type(2))) _Float16 half2;
        return (float)__builtin_bit_cast(half2, w)[i & 1];
    }
    __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __builtin_bit_cast(unsigned, f[i]);
            } else {
                typedef __attribute__((ext_vector_type(2))) T Pair;
                v[i] = __builtin_bit_cast(unsigned, Pair{(T)f[2 * i], (T)f[2 * i + 1]});
            }
        }
    }
};

// A lane permutation inside rows of 16 as a VALU operand (no LDS).
template <int CTRL> __device__ __forceinline__ float avsi_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// a[lanes 32 .. 63] <-> b[lanes 0 .. 31], and the same of the odd rows of a with the even rows of b.
__device__ __forceinline__ void avsi_swap32(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned x = r[0], y = r[1];
    a = __builtin_bit_cast(float, x);
    b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ void avsi_swap16(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b), false, false);
    const unsigned x = r[0], y = r[1];
    a = __builtin_bit_cast(float, x);
    b = __builtin_bit_cast(float, y);
}

// Sum (or maximum) over every aligned group of G lanes, left in all of them; the order is fixed.
struct avsi_add { static __device__ __forceinline__ float of(float a, float b) { return a + b; } };
template <int G, typename OP = avsi_add> __device__ __forceinline__ float avsi_group(float v) {
    if (G >= 2) v = OP::of(v, avsi_dpp<0xB1>(v));       // quad_perm [1, 0, 3, 2]
    if (G >= 4) v = OP::of(v, avsi_dpp<0x4E>(v));       // quad_perm [2, 3, 0, 1]
    if (G >= 8) v = OP::of(v, avsi_dpp<0x141>(v));      // row_half_mirror: the other quad of the eight
    if (G >= 16) v = OP::of(v, avsi_dpp<0x140>(v));     // row_mirror: the other eight of the row
    if (G >= 32) { float a = v, b = v; avsi_swap16(a, b); v = OP::of(a, b); }
    if (G >= 64) { float a = v, b = v; avsi_swap32(a, b); v = OP::of(a, b); }
    return v;
}

// Sums of P rows of partials by columns, handed to `put(column, sum)`, by workgroups of 1024 in a grid of avsi_column_sum_grid(cols):
// 32 columns at a time in 32 slices of the rows, eight loads of a slice in flight, then the slices, all in a fixed order.
// (A launch has fewer than 2^32 threads: of more than 2^26 columns a workgroup takes several blocks.)
static inline dim3 avsi_column_sum_grid(int64_t cols) {
    const int64_t blocks = (cols + 31) / 32, most = 1 << 21;
    return dim3((unsigned)(blocks < most ? blocks : most));
}
template <typename Put> __device__ __forceinline__ void avsi_column_sums(const float* __restrict__ part, int P, int64_t stride, int64_t cols,
                                                                         Put put) {
    __shared__ float lds[32][33];
    const int slice = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < cols; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + lane;
        float s = 0.f;
        if (c < cols) {
            const float* at = part + c;
            int r = slice;
            for (; r + 7 * 32 < P; r += 8 * 32) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = at[(int64_t)(r + 32 * i) * stride];
#pragma unroll
                for (int i = 0; i < 8; ++i) s += v[i];
            }
            for (; r < P; r += 32) s += at[(int64_t)r * stride];
        }
        if (c0 != (int64_t)blockIdx.x * 32) __syncthreads();        // (the block before has been read)
        lds[slice][lane] = s;
        __syncthreads();
        if (threadIdx.x < 32 && c < cols) {
            s = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) s += lds[i][lane];
            put(c, s);
        }
    }
}

// Functions of the gates on the hardware's base-2 exponential (off by one ulp, as its reciprocal).  e^y takes y log2 e rounded to one word
// and puts back what that left out, r = y - (that) ln 2, as 1 + r: the relative error stays that of the exponential and one
// rounding whatever y (in one word alone it would be |y| half-ulps, 60 for a gate at -60).  So counted in half-ulps: e^y 3.1, the sigmoid
// at most 7.1.  In softplus log(1 + e) for 0 <= e <= 1 is 2 atanh(s), s = e / (2 + e) <= 1 / 3, by a polynomial in r = (2 s)^2 whose
// largest error over that range, 5e-9 of the value, was made least; small e keep their relative accuracy (1 + e would round them
// away).  A NaN comes out of softplus, and of x sigmoid(x), as one.  `slope`: the derivative, sigmoid(x), out of the same exponential.
__device__ __forceinline__ float avsi_exp_of(float y) {       // -120 <= y <= 0
    const float hi = y * 1.44269504088896340736f, a = __builtin_amdgcn_exp2f(hi);
    return fmaf(a, fmaf(-hi, -1.90465429995776804525e-9f, fmaf(-hi, 0.693147182464599609375f, y)), a);
}
// T: the type that what comes of it is rounded to.  For 16 bits the exponential takes y log2 e in one word: at most 2^-17.5 off, where
// half a step is 2^-12 (fp16) or 2^-9, and seven operations less (8 x 2048 x 2048 bf16, convolution forward 26 us against 32).
template <typename T> __device__ __forceinline__ float avsi_sigmoid(float x) {
    if (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
    const float e = avsi_exp_of(fmaxf(-fabsf(x), -120.f));
    return (x < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e);
}
__device__ __forceinline__ float avsi_softplus(float x, float& slope) {
    const float e = avsi_exp_of(fmaxf(-fabsf(x), -120.f));
    const float s = e * __builtin_amdgcn_rcpf(fmaf(e, 0.5f, 1.f)), r = s * s;
    float q = fmaf(r, 0.14008851f / 256.f, 0.14000203f / 64.f);
    q = fmaf(r, q, 0.20010814f / 16.f);
    q = fmaf(r, q, 0.33333207f / 4.f);
    slope = (x < 0.f ? e : 1.f) * __builtin_amdgcn_rcpf(1.f + e);
    return (x < 0.f ? 0.f : x) + fmaf(s * r, q, s);
}
