// Selective state-space scan: per channel d a diagonal recurrence of N states whose step size, input and output vectors come from
// the token itself.
//
//   delta = softplus(dt + dt_bias)   (or dt + dt_bias),   a[t, d, n] = exp(delta[t, d] A[d, n])
//   h[t] = a[t] h[t - 1] + delta[t] u[t] B[t, n],   y = sum over n of C[t, n] h[t, n] + D u,   out = y z sigmoid(z)
//   backward, with dy = dout z sigmoid(z) and the adjoint state g[t] = C[t] dy[t] + a[t + 1] g[t + 1]:
//     dC = sum over d of dy h,  dB = sum over d of g delta u,  dA = sum over t of g a h[t - 1] delta,  dD = sum dy u
//     ddelta = sum over n of g (a h[t - 1] A + u B),  du = D dy + delta sum over n of g B,  dz = dout y slope(z)
// Behind lengths[b] a step has delta = 0: a = 1, nothing comes in, the state passes through unchanged and every gradient is zero;
// nothing is read there.
//
// Bound: N exponentials per channel and step (quarter rate) and four (forward) to twelve (backward) plain operations each; the
// bytes of u, dt, z and out come close to that for N = 16.  So the recurrence is laid out for the vector unit: a lane owns 4 states
// of one channel, LN = N / 4 lanes a channel, and a sum over the states is log2(LN) lane permutations inside an operand.  A
// workgroup of up to four waves takes CH = min(64, 256 / LN) channels and goes through time in tiles of 16 steps, staged in LDS: the
// softplus and the gate are computed once per channel and step, where the tile is loaded, in 16-byte pieces along the channels; the
// loads of the next tile are in flight during the recurrence of this one.
//
// Time is cut into chunks only where batch and channels do not fill the chip (chunk_count): then a first launch runs every chunk from a
// zero state, a second one joins the chunk ends (h_end = exp(A sum delta) h_start + h_local), and the main launch starts from those.
//
// Training: the forward pass keeps the state at the start of every tile, so the backward pass redoes 16 steps at a time in registers
// (64 decays and 64 states per lane) and goes back over them.  dB and dC are sums over the channels: over a wave by lane exchanges
// that halve the number of values at each level, over the workgroup's waves in LDS, over the workgroups through partials and a last
// launch.  All sums have a fixed order; there are no atomics.
#include "avsi_common.h"
#include "avsi_wave.h"

namespace {

constexpr int TT = 16;          // steps per tile
constexpr int MAX_STATE = 64;   // states per channel: 16 lanes
constexpr float LOG2E = 1.44269504088896340736f;

struct Scan {
    const void *u, *dt, *z, *B, *C, *dout;
    int64_t ub, ut, tb, tt, zb, zt, Bb, Bt, Bg, Cb, Ct, Cg, ob, ot, gb, gt;     // strides: batch, time, group
    const float *A, *D, *bias, *state;
    float* state_out;
    const int32_t* lengths;
    void* out;
    float* kept;                     // [batch][tiles][dim][4 LN]
    void *du, *ddt, *dz;             // [batch][time][dim]
    float *part_bc, *part_w;         // [batch][time][groups][blocks][2][4 LN], [batch * chunks][partial_stride]
    float *ends, *sums;              // [batch][chunks][dim][4 LN], [batch][chunks][dim]
    int batch, T, dim, N, groups, softplus, chunk, chunks, blocks;     // chunk: steps, a multiple of TT; blocks: per group
};

__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : (n < T ? n : T);
}

template <int LN> struct Shape {
    static constexpr int CH = LN <= 4 ? 64 : 256 / LN;      // channels of a workgroup
    static constexpr int NT = CH * LN;                      // its threads
    static constexpr int QR = CH / 4;                       // quads of channels per step
    static constexpr int ROWS = NT / QR < TT ? NT / QR : TT;
    static constexpr int PASSES = TT / ROWS;                // of the workgroup over a tile's [TT][CH]
    static constexpr int BPASSES = (TT * LN + NT - 1) / NT;  // over a tile's [TT][4 LN] of B and C
    static constexpr int NP = 4 * LN;
};

// Where a workgroup is: its group of channels, its first channel (of all), how many of CH exist.
template <int LN> struct Place {
    int g, d0, n, b, c;
    __device__ __forceinline__ Place(const Scan& p) {
        const int per = p.dim / p.groups, blk = blockIdx.x % p.blocks;
        g = blockIdx.x / p.blocks;
        d0 = g * per + blk * Shape<LN>::CH;
        n = per - blk * Shape<LN>::CH;
        n = n < Shape<LN>::CH ? n : Shape<LN>::CH;
        c = blockIdx.y;
        b = blockIdx.z;
    }
};

// A [TT][CH] tile of one tensor in the registers of the threads that stage it: quad `q` of row pass * ROWS + row.
template <typename T, int LN> struct Tile {
    avsi_raw<T, 4> v[Shape<LN>::PASSES];
    __device__ __forceinline__ void load(const void* base, int64_t bs, int64_t ts, const Place<LN>& at, int t0, int end) {
        typedef Shape<LN> S;
        const int q = threadIdx.x % S::QR, row = threadIdx.x / S::QR;
        const T* p = (const T*)base + at.b * bs + at.d0 + 4 * q;
#pragma unroll
        for (int i = 0; i < S::PASSES; ++i) {
            const int t = t0 + i * S::ROWS + row;
            v[i] = avsi_load_raw<T, 4>(p + (int64_t)t * ts, row < S::ROWS && t < end ? at.n - 4 * q : 0);
        }
    }
};
template <typename T, int LN> struct TileBC {
    avsi_raw<T, 4> v[Shape<LN>::BPASSES];
    __device__ __forceinline__ void load(const void* base, int64_t bs, int64_t ts, int64_t gs, const Place<LN>& at, int N, int t0, int end) {
        typedef Shape<LN> S;
#pragma unroll
        for (int i = 0; i < S::BPASSES; ++i) {
            const int id = i * S::NT + threadIdx.x, t = t0 + id / LN, n = 4 * (id % LN);
            v[i] = avsi_load_raw<T, 4>((const T*)base + at.b * bs + at.g * gs + (int64_t)t * ts + n, id < TT * LN && t < end ? N - n : 0);
        }
    }
    __device__ __forceinline__ void put(avsi_f4* lds) const {       // [TT][LN]
        typedef Shape<LN> S;
#pragma unroll
        for (int i = 0; i < S::BPASSES; ++i) {
            const int id = i * S::NT + threadIdx.x;
            if (id < TT * LN) lds[id] = avsi_f4{(float)v[i].v[0], (float)v[i].v[1], (float)v[i].v[2], (float)v[i].v[3]};
        }
    }
};

__device__ __forceinline__ float step_size(float x, int softplus) { return softplus ? avsi_softplus(x) : x; }

// dt_bias of this thread's quad of channels
template <int LN> __device__ __forceinline__ void quad_of(const float* v, const Place<LN>& at, float other, float (&f)[4]) {
    const int q = threadIdx.x % Shape<LN>::QR;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v && 4 * q + i < at.n ? v[at.d0 + 4 * q + i] : other;
}

// The four values of this lane in a [..][dim][NP] array at row d0 + channel; and A, times log2 e
template <int LN> __device__ __forceinline__ int64_t lane_at(const Scan& p, const Place<LN>& at, int64_t lead) {
    return ((lead * p.dim + at.d0 + threadIdx.x / LN) * LN + threadIdx.x % LN) * 4;
}
template <int LN> __device__ __forceinline__ void lane_A(const Scan& p, const Place<LN>& at, float (&A)[4]) {
    const int c = threadIdx.x / LN, n = 4 * (threadIdx.x % LN);
#pragma unroll
    for (int j = 0; j < 4; ++j) A[j] = c < at.n && n + j < p.N ? p.A[(int64_t)(at.d0 + c) * p.N + n + j] : 0.f;
}
template <int LN> __device__ __forceinline__ void lane_start(const Scan& p, const Place<LN>& at, float (&h)[4]) {
    const int c = threadIdx.x / LN, n = 4 * (threadIdx.x % LN);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = 0.f;
    if (c >= at.n) return;
    if (at.c > 0) {
        const avsi_f4 v = *(const avsi_f4*)(p.ends + lane_at<LN>(p, at, (int64_t)at.b * p.chunks + at.c));
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = v[j];
    } else if (p.state) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n + j < p.N) h[j] = p.state[((int64_t)at.b * p.dim + at.d0 + c) * p.N + n + j];
    }
}

// One partial of the weights' gradients: dA [dim][NP], dD [dim], ddt_bias [dim], to a multiple of 16 bytes.
__host__ __device__ __forceinline__ int64_t partial_stride(int dim, int NP) { return ((int64_t)dim * (NP + 2) + 3) / 4 * 4; }

// ------------------------------------------------------------------------------------------------------------- forward
template <typename T, int LN> __global__ __launch_bounds__(Shape<LN>::NT) void scan_fwd_kernel(Scan p) {
    typedef Shape<LN> S;
    __shared__ avsi_f2 s_in[TT][S::CH];             // delta, delta u
    __shared__ avsi_f4 s_B[TT * LN], s_C[TT * LN];
    __shared__ float s_y[TT][S::CH];
    const Place<LN> at(p);
    const int len = length_of(p.lengths, at.b, p.T), begin = at.c * p.chunk;
    const int end = begin + p.chunk < p.T ? begin + p.chunk : p.T, live = len < end ? len : end;
    const int q = threadIdx.x % S::QR, row = threadIdx.x / S::QR, ch = threadIdx.x / LN, ql = threadIdx.x % LN;
    float A[4], h[4], bias[4], Dq[4];
    lane_A<LN>(p, at, A);
    lane_start<LN>(p, at, h);
    quad_of<LN>(p.bias, at, 0.f, bias);
    quad_of<LN>(p.D, at, 0.f, Dq);
#pragma unroll
    for (int j = 0; j < 4; ++j) A[j] *= LOG2E;
    T* out = (T*)p.out + at.b * p.ob + at.d0 + 4 * q;
    const int tiles = (p.T + TT - 1) / TT;

    Tile<T, LN> u, dt, z;
    TileBC<T, LN> Bt, Ct;
    if (begin < live) {
        u.load(p.u, p.ub, p.ut, at, begin, live);
        dt.load(p.dt, p.tb, p.tt, at, begin, live);
        if (p.z) z.load(p.z, p.zb, p.zt, at, begin, live);
        Bt.load(p.B, p.Bb, p.Bt, p.Bg, at, p.N, begin, live);
        Ct.load(p.C, p.Cb, p.Ct, p.Cg, at, p.N, begin, live);
    }
    int t0 = begin;
    for (; t0 < live; t0 += TT) {
        float through[S::PASSES][4], gate[S::PASSES][4];        // D u, and the gate
#pragma unroll
        for (int i = 0; i < S::PASSES; ++i) {
            const int r = i * S::ROWS + row;
            if (row < S::ROWS) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float uf = (float)u.v[i].v[k];
                    const float d = t0 + r < live ? step_size((float)dt.v[i].v[k] + bias[k], p.softplus) : 0.f;
                    s_in[r][4 * q + k] = avsi_f2{d, d * uf};
                    through[i][k] = Dq[k] * uf;
                    const float zf = p.z ? (float)z.v[i].v[k] : 0.f;
                    gate[i][k] = p.z ? zf * avsi_sigmoid(zf) : 1.f;
                }
            }
        }
        Bt.put(s_B);
        Ct.put(s_C);
        AVSI_LDS_BARRIER();
        if (p.kept && ch < at.n)
            *(avsi_f4*)(p.kept + lane_at<LN>(p, at, (int64_t)at.b * tiles + t0 / TT)) = avsi_f4{h[0], h[1], h[2], h[3]};
        if (t0 + TT < live) {
            u.load(p.u, p.ub, p.ut, at, t0 + TT, live);
            dt.load(p.dt, p.tb, p.tt, at, t0 + TT, live);
            if (p.z) z.load(p.z, p.zb, p.zt, at, t0 + TT, live);
            Bt.load(p.B, p.Bb, p.Bt, p.Bg, at, p.N, t0 + TT, live);
            Ct.load(p.C, p.Cb, p.Ct, p.Cg, at, p.N, t0 + TT, live);
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const avsi_f2 in = s_in[t][ch];
            const avsi_f4 Bv = s_B[t * LN + ql], Cv = s_C[t * LN + ql];
            float y = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[j] = fmaf(__builtin_amdgcn_exp2f(in[0] * A[j]), h[j], in[1] * Bv[j]);
                y = fmaf(h[j], Cv[j], y);
            }
            y = avsi_group<LN>(y);
            if (ql == t % LN) s_y[t][ch] = y;
        }
        AVSI_LDS_BARRIER();
#pragma unroll
        for (int i = 0; i < S::PASSES; ++i) {
            const int t = t0 + i * S::ROWS + row;
            if (row < S::ROWS && t < end) {
                float o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    o[k] = t < live ? (s_y[i * S::ROWS + row][4 * q + k] + through[i][k]) * gate[i][k] : 0.f;
                avsi_store<T, 4>(out + (int64_t)t * p.ot, at.n - 4 * q, o);
            }
        }
    }
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    if (row < S::ROWS)
        for (int t = t0 + row; t < end; t += S::ROWS) avsi_store<T, 4>(out + (int64_t)t * p.ot, at.n - 4 * q, zero);
    if (p.state_out && at.c == p.chunks - 1 && ch < at.n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (4 * ql + j < p.N) p.state_out[((int64_t)at.b * p.dim + at.d0 + ch) * p.N + 4 * ql + j] = h[j];
}

// A chunk from a zero state: its end state and the sum of its step sizes.  BACK: the adjoint state, from behind.
template <typename T, int LN, bool BACK> __global__ __launch_bounds__(Shape<LN>::NT) void scan_chunk_kernel(Scan p) {
    typedef Shape<LN> S;
    __shared__ avsi_f2 s_in[TT][S::CH];             // delta, delta u (BACK: dy)
    __shared__ avsi_f4 s_B[TT * LN];                // (BACK: C)
    Place<LN> at(p);
    if (BACK) ++at.c;                               // (the first chunk's is not needed; forward: the last one's)
    const int len = length_of(p.lengths, at.b, p.T), begin = at.c * p.chunk;
    const int end = begin + p.chunk < p.T ? begin + p.chunk : p.T, live = len < end ? len : end;
    const int q = threadIdx.x % S::QR, row = threadIdx.x / S::QR, ch = threadIdx.x / LN, ql = threadIdx.x % LN;
    float A[4], h[4] = {0.f, 0.f, 0.f, 0.f}, bias[4], sum = 0.f;
    lane_A<LN>(p, at, A);
    quad_of<LN>(p.bias, at, 0.f, bias);
#pragma unroll
    for (int j = 0; j < 4; ++j) A[j] *= LOG2E;
    const int n_tiles = begin < live ? (live - begin + TT - 1) / TT : 0;
    Tile<T, LN> u, dt, z;                           // BACK: u is dout
    TileBC<T, LN> Bt;
    auto load = [&](int t0) {
        dt.load(p.dt, p.tb, p.tt, at, t0, live);
        if (BACK) {
            u.load(p.dout, p.gb, p.gt, at, t0, live);
            if (p.z) z.load(p.z, p.zb, p.zt, at, t0, live);
            Bt.load(p.C, p.Cb, p.Ct, p.Cg, at, p.N, t0, live);
        } else {
            u.load(p.u, p.ub, p.ut, at, t0, live);
            Bt.load(p.B, p.Bb, p.Bt, p.Bg, at, p.N, t0, live);
        }
    };
    auto tile_at = [&](int i) { return begin + (BACK ? n_tiles - 1 - i : i) * TT; };
    if (n_tiles) load(tile_at(0));
    for (int i = 0; i < n_tiles; ++i) {
        const int t0 = tile_at(i);
#pragma unroll
        for (int k = 0; k < S::PASSES; ++k) {
            const int r = k * S::ROWS + row;
            if (row < S::ROWS) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float d = t0 + r < live ? step_size((float)dt.v[k].v[j] + bias[j], p.softplus) : 0.f;
                    float x = (float)u.v[k].v[j];
                    if (BACK) {
                        if (p.z) x *= (float)z.v[k].v[j] * avsi_sigmoid((float)z.v[k].v[j]);
                    } else {
                        x *= d;
                    }
                    s_in[r][4 * q + j] = avsi_f2{d, x};
                }
            }
        }
        Bt.put(s_B);
        AVSI_LDS_BARRIER();
        if (i + 1 < n_tiles) load(tile_at(i + 1));
#pragma unroll
        for (int k = 0; k < TT; ++k) {
            const int t = BACK ? TT - 1 - k : k;
            const avsi_f2 in = s_in[t][ch];
            const avsi_f4 Bv = s_B[t * LN + ql];
            sum += in[0];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = __builtin_amdgcn_exp2f(in[0] * A[j]);
                h[j] = BACK ? a * fmaf(Bv[j], in[1], h[j]) : fmaf(a, h[j], in[1] * Bv[j]);
            }
        }
        AVSI_LDS_BARRIER();
    }
    if (ch < at.n) {
        // the chunk's row of `ends` is read as the start of the chunk behind it (in front of it)
        const int64_t lead = (int64_t)at.b * p.chunks + (BACK ? at.c - 1 : at.c + 1);
        *(avsi_f4*)(p.ends + lane_at<LN>(p, at, lead)) = avsi_f4{h[0], h[1], h[2], h[3]};
        if (ql == 0) p.sums[lead * p.dim + at.d0 + ch] = sum;
    }
}

// start[c] = local end of c - 1 + exp(A sum of c - 1) start[c - 1] (BACK: with c + 1), in place.  One thread per four states.
template <int LN, bool BACK> __global__ __launch_bounds__(256) void scan_join_kernel(Scan p) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)p.batch * p.dim * LN) return;
    const int ql = (int)(id % LN), d = (int)(id / LN % p.dim), b = (int)(id / LN / p.dim);
    float A[4], h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = 4 * ql + j;
        A[j] = n < p.N ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
        h[j] = !BACK && p.state && n < p.N ? p.state[((int64_t)b * p.dim + d) * p.N + n] : 0.f;
    }
    for (int i = 1; i < p.chunks; ++i) {
        const int64_t lead = (int64_t)b * p.chunks + (BACK ? p.chunks - 1 - i : i);
        avsi_f4* e = (avsi_f4*)(p.ends + ((lead * p.dim + d) * LN + ql) * 4);
        const float s = p.sums[lead * p.dim + d];
        avsi_f4 v = *e;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = h[j] = fmaf(__builtin_amdgcn_exp2f(s * A[j]), h[j], v[j]);
        *e = v;
    }
}

// ------------------------------------------------------------------------------------------------------------ backward
// Sum over the channels of a wave (the lanes that share a quad of states) of b[0 .. 3] and c[0 .. 3], at *out = [2][NP] of one step.
// While a level halves the lanes it halves the values too: the upper half of the lanes takes c, then the odd rows values 2 and 3.
template <int LN> __device__ __forceinline__ void channel_sums(float (&b)[4], float (&c)[4], float* out) {
    const int lane = threadIdx.x & 63, q = lane % LN;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        avsi_swap32(b[j], c[j]);
        b[j] += c[j];
    }
    float* o = out + (lane >> 5) * 4 * LN + 4 * q;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        avsi_swap16(b[j], b[j + 2]);
        b[j] += b[j + 2];
        if (LN <= 8) b[j] += avsi_dpp<0x128>(b[j]);         // row_ror 8
        if (LN <= 4) b[j] += avsi_dpp<0x124>(b[j]);         // row_ror 4
        if (LN <= 2) b[j] += avsi_dpp<0x4E>(b[j]);
        if (LN <= 1) b[j] += avsi_dpp<0xB1>(b[j]);
    }
    if ((lane & 15) < LN) {
        o += ((lane >> 4) & 1) * 2;
        o[0] = b[0];
        o[1] = b[1];
    }
}

template <typename T, int LN> __global__ __launch_bounds__(Shape<LN>::NT) void scan_bwd_kernel(Scan p) {
    typedef Shape<LN> S;
    constexpr int NW = S::NT / 64;
    __shared__ avsi_f4 s_in[TT][S::CH];             // delta, delta u, dy
    __shared__ avsi_f4 s_B[TT * LN], s_C[TT * LN];
    __shared__ float s_y[TT][S::CH], s_gB[TT][S::CH], s_gA[TT][S::CH];
    __shared__ float s_bc[NW][TT][2 * S::NP];
    const Place<LN> at(p);
    const int len = length_of(p.lengths, at.b, p.T), begin = at.c * p.chunk;
    const int end = begin + p.chunk < p.T ? begin + p.chunk : p.T, live = len < end ? len : end;
    const int q = threadIdx.x % S::QR, row = threadIdx.x / S::QR, ch = threadIdx.x / LN, ql = threadIdx.x % LN;
    float A[4], Al[4], g[4] = {0.f, 0.f, 0.f, 0.f}, dA[4] = {0.f, 0.f, 0.f, 0.f}, bias[4], Dq[4], dD[4], dbias[4];
    lane_A<LN>(p, at, A);
    quad_of<LN>(p.bias, at, 0.f, bias);
    quad_of<LN>(p.D, at, 0.f, Dq);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        Al[j] = A[j] * LOG2E;
        dD[j] = dbias[j] = 0.f;
    }
    if (at.c < p.chunks - 1 && ch < at.n) {
        const avsi_f4 v = *(const avsi_f4*)(p.ends + lane_at<LN>(p, at, (int64_t)at.b * p.chunks + at.c));
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = v[j];
    }
    const int tiles = (p.T + TT - 1) / TT, n_tiles = begin < live ? (live - begin + TT - 1) / TT : 0;
    const int64_t flat = ((int64_t)at.b * p.T) * p.dim + at.d0 + 4 * q;
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    if (row < S::ROWS)
        for (int t = begin + n_tiles * TT + row; t < end; t += S::ROWS) {
            avsi_store<T, 4>((T*)p.du + flat + (int64_t)t * p.dim, at.n - 4 * q, zero);
            avsi_store<T, 4>((T*)p.ddt + flat + (int64_t)t * p.dim, at.n - 4 * q, zero);
            if (p.z) avsi_store<T, 4>((T*)p.dz + flat + (int64_t)t * p.dim, at.n - 4 * q, zero);
        }
    Tile<T, LN> u, dt, z, go;
    TileBC<T, LN> Bt, Ct;
    avsi_f4 start = {0.f, 0.f, 0.f, 0.f};
    auto load = [&](int t0) {
        u.load(p.u, p.ub, p.ut, at, t0, live);
        dt.load(p.dt, p.tb, p.tt, at, t0, live);
        go.load(p.dout, p.gb, p.gt, at, t0, live);
        if (p.z) z.load(p.z, p.zb, p.zt, at, t0, live);
        Bt.load(p.B, p.Bb, p.Bt, p.Bg, at, p.N, t0, live);
        Ct.load(p.C, p.Cb, p.Ct, p.Cg, at, p.N, t0, live);
        if (ch < at.n) start = *(const avsi_f4*)(p.kept + lane_at<LN>(p, at, (int64_t)at.b * tiles + t0 / TT));
    };
    if (n_tiles) load(begin + (n_tiles - 1) * TT);
    for (int t0 = begin + (n_tiles - 1) * TT; t0 >= begin; t0 -= TT) {
        float uf[S::PASSES][4], delta[S::PASSES][4], slope[S::PASSES][4], dy[S::PASSES][4], gz[S::PASSES][4];
#pragma unroll
        for (int i = 0; i < S::PASSES; ++i) {
            const int r = i * S::ROWS + row;
            if (row < S::ROWS) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float x = (float)dt.v[i].v[k] + bias[k];
                    const bool on = t0 + r < live;
                    uf[i][k] = (float)u.v[i].v[k];
                    delta[i][k] = on ? step_size(x, p.softplus) : 0.f;
                    slope[i][k] = on ? (p.softplus ? avsi_sigmoid(x) : 1.f) : 0.f;
                    dy[i][k] = (float)go.v[i].v[k];
                    if (p.z) {
                        const float zf = (float)z.v[i].v[k], s = avsi_sigmoid(zf);
                        gz[i][k] = dy[i][k] * s * fmaf(zf, 1.f - s, 1.f);
                        dy[i][k] *= zf * s;
                    }
                    s_in[r][4 * q + k] = avsi_f4{delta[i][k], delta[i][k] * uf[i][k], dy[i][k], 0.f};
                }
            }
        }
        Bt.put(s_B);
        Ct.put(s_C);
        float h[4] = {start[0], start[1], start[2], start[3]};
        AVSI_LDS_BARRIER();
        if (t0 > begin) load(t0 - TT);
        float a[TT][4], before[TT][4];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const avsi_f4 in = s_in[t][ch], Bv = s_B[t * LN + ql];
            float y = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                before[t][j] = h[j];
                a[t][j] = __builtin_amdgcn_exp2f(in[0] * Al[j]);
                h[j] = fmaf(a[t][j], h[j], in[1] * Bv[j]);
            }
            if (p.z) {
                const avsi_f4 Cv = s_C[t * LN + ql];
#pragma unroll
                for (int j = 0; j < 4; ++j) y = fmaf(h[j], Cv[j], y);
                y = avsi_group<LN>(y);
                if (ql == t % LN) s_y[t][ch] = y;
            }
        }
        float dAt[4] = {0.f, 0.f, 0.f, 0.f};        // (a tile's own sum: the long sum over time keeps its low bits)
#pragma unroll
        for (int t = TT - 1; t >= 0; --t) {
            const avsi_f4 in = s_in[t][ch], Bv = s_B[t * LN + ql], Cv = s_C[t * LN + ql];
            float vb[4], vc[4], gB = 0.f, gA = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float gj = fmaf(Cv[j], in[2], g[j]);
                vb[j] = gj * in[1];
                vc[j] = in[2] * (t == TT - 1 ? h[j] : before[t == TT - 1 ? t : t + 1][j]);
                gB = fmaf(gj, Bv[j], gB);
                g[j] = a[t][j] * gj;
                const float x = g[j] * before[t][j];
                gA = fmaf(x, A[j], gA);
                dAt[j] = fmaf(x, in[0], dAt[j]);
            }
            gB = avsi_group<LN>(gB);
            gA = avsi_group<LN>(gA);
            if (ql == t % LN) {
                s_gB[t][ch] = gB;
                s_gA[t][ch] = gA;
            }
            channel_sums<LN>(vb, vc, s_bc[threadIdx.x >> 6][t]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) dA[j] += dAt[j];
        AVSI_LDS_BARRIER();
        for (int i = threadIdx.x; i < TT * 2 * S::NP; i += S::NT) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) s += s_bc[w][i / (2 * S::NP)][i % (2 * S::NP)];
            const int t = t0 + i / (2 * S::NP);
            if (t < live)
                p.part_bc[((((int64_t)at.b * p.T + t) * p.groups + at.g) * p.blocks + blockIdx.x % p.blocks) * 2 * S::NP + i % (2 * S::NP)] = s;
        }
#pragma unroll
        for (int i = 0; i < S::PASSES; ++i) {
            const int r = i * S::ROWS + row, t = t0 + r;
            if (row < S::ROWS && t < end) {
                float o[4], od[4], oz[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gB = s_gB[r][4 * q + k];
                    const bool on = t < live;
                    o[k] = on ? fmaf(Dq[k], dy[i][k], delta[i][k] * gB) : 0.f;
                    od[k] = on ? fmaf(uf[i][k], gB, s_gA[r][4 * q + k]) * slope[i][k] : 0.f;
                    dD[k] = fmaf(dy[i][k], uf[i][k], dD[k]);
                    dbias[k] += od[k];
                    oz[k] = on && p.z ? gz[i][k] * fmaf(Dq[k], uf[i][k], s_y[r][4 * q + k]) : 0.f;
                }
                const int64_t o_at = flat + (int64_t)t * p.dim;
                avsi_store<T, 4>((T*)p.du + o_at, at.n - 4 * q, o);
                avsi_store<T, 4>((T*)p.ddt + o_at, at.n - 4 * q, od);
                if (p.z) avsi_store<T, 4>((T*)p.dz + o_at, at.n - 4 * q, oz);
            }
        }
    }
    // the weights' gradients of this workgroup's channels, over its chunk
    float* pw = p.part_w + ((int64_t)at.b * p.chunks + at.c) * partial_stride(p.dim, S::NP);
    if (ch < at.n) *(avsi_f4*)(pw + ((int64_t)(at.d0 + ch) * LN + ql) * 4) = avsi_f4{dA[0], dA[1], dA[2], dA[3]};
    AVSI_LDS_BARRIER();
    if (row < S::ROWS)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s_gB[row][4 * q + k] = dD[k];
            s_gA[row][4 * q + k] = dbias[k];
        }
    AVSI_LDS_BARRIER();
    if (threadIdx.x < at.n) {
        float sD = 0.f, sb = 0.f;
        for (int r = 0; r < S::ROWS; ++r) {
            sD += s_gB[r][threadIdx.x];
            sb += s_gA[r][threadIdx.x];
        }
        pw += (int64_t)p.dim * S::NP + at.d0 + threadIdx.x;
        pw[0] = sD;
        pw[p.dim] = sb;
    }
}

// dA [dim][N], dD, ddt_bias [dim] = sums over P partials of [dim][NP], [dim], [dim]: 16 columns x 16 slices per workgroup.
__global__ __launch_bounds__(256) void scan_wgrad_sum_kernel(const float* __restrict__ part, int P, int dim, int NP, int N,
                                                             float* __restrict__ dA, float* __restrict__ dD, float* __restrict__ dbias) {
    __shared__ float lds[256];
    const int64_t cols = (int64_t)dim * (NP + 2), c = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
    float s = 0.f;
    if (c < cols)
        for (int k = threadIdx.x >> 4; k < P; k += 16) s += part[k * partial_stride(dim, NP) + c];
    lds[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 16 && c < cols) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += lds[i * 16 + threadIdx.x];
        if (c < (int64_t)dim * NP) {
            if (c % NP < N) dA[c / NP * N + c % NP] = s;
        } else if (c < (int64_t)dim * (NP + 1)) {
            if (dD) dD[c - (int64_t)dim * NP] = s;
        } else if (dbias) {
            dbias[c - (int64_t)dim * (NP + 1)] = s;
        }
    }
}

// dB, dC [batch][time][groups][N] = sums over the blocks of part_bc; zero behind a length.
template <typename T> __global__ __launch_bounds__(256) void scan_bc_sum_kernel(Scan p, int NP, T* __restrict__ dB, T* __restrict__ dC) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, tokens = (int64_t)p.batch * p.T;
    if (id >= tokens * p.groups * 2 * NP) return;
    const int n = (int)(id % NP), which = (int)(id / NP % 2);
    const int64_t tg = id / (2 * NP);
    const int t = (int)(tg / p.groups % p.T), b = (int)(tg / p.groups / p.T);
    if (n >= p.N) return;
    float s = 0.f;
    if (t < length_of(p.lengths, b, p.T))
        for (int k = 0; k < p.blocks; ++k) s += p.part_bc[(tg * p.blocks + k) * 2 * NP + which * NP + n];
    (which ? dC : dB)[tg * p.N + n] = (T)s;
}

// ---------------------------------------------------------------------------------------------------------- one token
template <typename T, int LN> __global__ __launch_bounds__(256) void scan_step_kernel(Scan p) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int ql = (int)(id % LN), d = (int)(id / LN % p.dim);
    const int64_t b = id / LN / p.dim;
    if (b >= p.batch) return;               // (whole groups of LN lanes leave: dim LN per sequence)
    const int n0 = 4 * ql, n = p.N - n0, grp = d / (p.dim / p.groups);
    float A[4], Bv[4], Cv[4], h[4];
    avsi_load<float, 4>(p.A + (int64_t)d * p.N + n0, n, A);
    avsi_load<T, 4>((const T*)p.B + b * p.Bb + grp * p.Bg + n0, n, Bv);
    avsi_load<T, 4>((const T*)p.C + b * p.Cb + grp * p.Cg + n0, n, Cv);
    float* st = p.state_out + (b * p.dim + d) * p.N + n0;
    avsi_load<float, 4>(st, n, h);
    const float u = (float)((const T*)p.u)[b * p.ub + d];
    const float x = (float)((const T*)p.dt)[b * p.tb + d] + (p.bias ? p.bias[d] : 0.f);
    const float delta = step_size(x, p.softplus), du = delta * u;
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(__builtin_amdgcn_exp2f(delta * (A[j] * LOG2E)), h[j], du * Bv[j]);
        y = fmaf(h[j], Cv[j], y);
    }
    avsi_store<float, 4>(st, n, h);
    y = avsi_group<LN>(y);
    if (ql == 0) {
        if (p.D) y = fmaf(p.D[d], u, y);
        if (p.z) {
            const float z = (float)((const T*)p.z)[b * p.zb + d];
            y *= z * avsi_sigmoid(z);
        }
        ((T*)p.out)[b * p.ob + d] = (T)y;
    }
}

int lanes_of(int N) {
    int l = 1;
    while (4 * l < N) l *= 2;
    return l;
}
int block_channels(int LN) { return LN <= 4 ? 64 : 256 / LN; }

// Chunks of time: none where the batch and the channels leave a wave for each of the 1024 SIMDs -- the first launch over the chunks
// costs three quarters of the main one --, else as many as make two, of at least 64 steps.
void chunks_of(const avsi_scan_args* a, int* chunk, int* chunks) {
    const int LN = lanes_of(a->state), CH = block_channels(LN);
    const int64_t waves = (int64_t)a->batch * a->groups * avsi_ceil_div(a->dim / a->groups, CH) * (CH * LN / 64);
    int64_t n = waves >= 1024 ? 1 : avsi_ceil_div(2048, waves);
    const int64_t most = avsi_ceil_div(a->time, 64);
    n = n < most ? n : most;
    *chunk = (int)avsi_round_up(avsi_ceil_div(a->time, n), TT);
    *chunks = (int)avsi_ceil_div(a->time, *chunk);
}

bool shape_ok(const avsi_scan_args* a) {
    return a && avsi_dtype_ok(a->dtype) && a->batch > 0 && a->batch <= 65535 && a->time > 0 && a->dim > 0 && a->state > 0 &&
           a->groups > 0 && a->dim % a->groups == 0;
}

Scan params(const avsi_scan_args* a) {
    Scan p = {};
    p.u = a->u, p.dt = a->dt, p.z = a->z, p.B = a->B, p.C = a->C, p.dout = a->dout;
    p.ub = a->u_stride[0], p.ut = a->u_stride[1], p.tb = a->dt_stride[0], p.tt = a->dt_stride[1];
    p.zb = a->z_stride[0], p.zt = a->z_stride[1], p.gb = a->dout_stride[0], p.gt = a->dout_stride[1];
    p.Bb = a->B_stride[0], p.Bt = a->B_stride[1], p.Bg = a->B_stride[2];
    p.Cb = a->C_stride[0], p.Ct = a->C_stride[1], p.Cg = a->C_stride[2];
    p.ob = a->out_stride[0], p.ot = a->out_stride[1];
    p.A = a->A, p.D = a->D, p.bias = a->dt_bias, p.state = a->state_in, p.state_out = a->state_out;
    p.lengths = a->lengths, p.out = a->out, p.kept = a->kept, p.du = a->du, p.ddt = a->ddt, p.dz = a->dz;
    p.batch = a->batch, p.T = a->time, p.dim = a->dim, p.N = a->state, p.groups = a->groups, p.softplus = a->softplus;
    chunks_of(a, &p.chunk, &p.chunks);
    p.blocks = (int)avsi_ceil_div(a->dim / a->groups, block_channels(lanes_of(a->state)));
    return p;
}

size_t chunk_floats(const avsi_scan_args* a, int chunks) {
    return chunks < 2 ? 0 : (size_t)a->batch * chunks * a->dim * (4 * lanes_of(a->state) + 1);
}

template <typename T, int LN> void go_fwd(const Scan& p, hipStream_t s) {
    const dim3 wg(Shape<LN>::NT);
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_chunk_kernel<T, LN, false>), dim3(p.groups * p.blocks, p.chunks - 1, p.batch), wg, 0, s, p);
        hipLaunchKernelGGL((scan_join_kernel<LN, false>), dim3(avsi_ceil_div((int64_t)p.batch * p.dim * LN, 256)), dim3(256), 0, s, p);
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, LN>), dim3(p.groups * p.blocks, p.chunks, p.batch), wg, 0, s, p);
}
template <typename T, int LN> void go_bwd(const Scan& p, hipStream_t s) {
    const dim3 wg(Shape<LN>::NT);
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_chunk_kernel<T, LN, true>), dim3(p.groups * p.blocks, p.chunks - 1, p.batch), wg, 0, s, p);
        hipLaunchKernelGGL((scan_join_kernel<LN, true>), dim3(avsi_ceil_div((int64_t)p.batch * p.dim * LN, 256)), dim3(256), 0, s, p);
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, LN>), dim3(p.groups * p.blocks, p.chunks, p.batch), wg, 0, s, p);
}
template <typename T, int LN> void go_step(const Scan& p, hipStream_t s) {
    hipLaunchKernelGGL((scan_step_kernel<T, LN>), dim3(avsi_ceil_div((int64_t)p.batch * p.dim * LN, 256)), dim3(256), 0, s, p);
}

}  // namespace

#define AVSI_SCAN_LN(T, GO)         \
    switch (lanes_of(a->state)) {   \
        case 1: GO<T, 1>(p, s); break;   \
        case 2: GO<T, 2>(p, s); break;   \
        case 4: GO<T, 4>(p, s); break;   \
        case 8: GO<T, 8>(p, s); break;   \
        default: GO<T, 16>(p, s); break; \
    }
#define AVSI_SCAN_T(GO)                                         \
    if (a->dtype == AVSI_F32) { AVSI_SCAN_LN(float, GO) }       \
    else if (a->dtype == AVSI_BF16) { AVSI_SCAN_LN(__bf16, GO) } \
    else { AVSI_SCAN_LN(_Float16, GO) }

extern "C" size_t avsi_selective_scan_kept_floats(const avsi_scan_args* a) {
    if (!shape_ok(a) || a->state > MAX_STATE) return 0;
    return (size_t)a->batch * avsi_ceil_div(a->time, TT) * a->dim * 4 * lanes_of(a->state);
}

extern "C" size_t avsi_selective_scan_workspace_bytes(const avsi_scan_args* a) {
    if (!shape_ok(a) || a->state > MAX_STATE) return 0;
    int chunk, chunks;
    chunks_of(a, &chunk, &chunks);
    return chunk_floats(a, chunks) * sizeof(float);
}

extern "C" int avsi_selective_scan(const avsi_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!shape_ok(a) || !a->u || !a->dt || !a->A || !a->B || !a->C || !a->out) return AVSI_ERR_INVALID_ARG;
    if (a->state > MAX_STATE) return AVSI_ERR_UNSUPPORTED;
    const size_t need = avsi_selective_scan_workspace_bytes(a);
    if (need && (!workspace || workspace_bytes < need)) return AVSI_ERR_WORKSPACE;
    Scan p = params(a);
    p.ends = (float*)workspace;
    p.sums = p.ends ? p.ends + (size_t)p.batch * p.chunks * p.dim * 4 * lanes_of(p.N) : nullptr;
    hipStream_t s = (hipStream_t)stream;
    avsi_clear_error();
    AVSI_SCAN_T(go_fwd)
    return avsi_launch_status();
}

extern "C" size_t avsi_selective_scan_bwd_workspace_bytes(const avsi_scan_args* a) {
    if (!shape_ok(a) || a->state > MAX_STATE) return 0;
    const Scan p = params(a);
    const size_t NP = 4 * lanes_of(p.N);
    return (chunk_floats(a, p.chunks) + (size_t)p.batch * p.T * p.groups * p.blocks * 2 * NP +
            (size_t)p.batch * p.chunks * partial_stride(p.dim, NP)) * sizeof(float);
}

extern "C" int avsi_selective_scan_bwd(const avsi_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!shape_ok(a) || !a->u || !a->dt || !a->A || !a->B || !a->C || !a->dout || !a->kept || !a->du || !a->ddt || !a->dA || !a->dB ||
        !a->dC || !a->z != !a->dz)
        return AVSI_ERR_INVALID_ARG;
    if (a->state > MAX_STATE) return AVSI_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < avsi_selective_scan_bwd_workspace_bytes(a)) return AVSI_ERR_WORKSPACE;
    Scan p = params(a);
    const int NP = 4 * lanes_of(p.N);
    // (every part is a multiple of four floats but the sums of the chunks: they come last)
    p.part_bc = (float*)workspace;
    p.part_w = p.part_bc + (size_t)p.batch * p.T * p.groups * p.blocks * 2 * NP;
    p.ends = p.part_w + (size_t)p.batch * p.chunks * partial_stride(p.dim, NP);
    p.sums = p.ends + (size_t)p.batch * p.chunks * p.dim * NP;
    hipStream_t s = (hipStream_t)stream;
    avsi_clear_error();
    AVSI_SCAN_T(go_bwd)
    const int64_t bc = (int64_t)p.batch * p.T * p.groups * 2 * NP;
    const dim3 grid(avsi_ceil_div(bc, 256));
    if (a->dtype == AVSI_F32)
        hipLaunchKernelGGL((scan_bc_sum_kernel<float>), grid, dim3(256), 0, s, p, NP, (float*)a->dB, (float*)a->dC);
    else if (a->dtype == AVSI_BF16)
        hipLaunchKernelGGL((scan_bc_sum_kernel<__bf16>), grid, dim3(256), 0, s, p, NP, (__bf16*)a->dB, (__bf16*)a->dC);
    else
        hipLaunchKernelGGL((scan_bc_sum_kernel<_Float16>), grid, dim3(256), 0, s, p, NP, (_Float16*)a->dB, (_Float16*)a->dC);
    hipLaunchKernelGGL(scan_wgrad_sum_kernel, dim3(avsi_ceil_div((int64_t)p.dim * (NP + 2), 16)), dim3(256), 0, s, p.part_w,
                       p.batch * p.chunks, p.dim, NP, p.N, a->dA, a->dD, a->ddt_bias);
    return avsi_launch_status();
}

extern "C" int avsi_selective_scan_step(const avsi_scan_args* a, void* stream) {
    if (!shape_ok(a) || a->time != 1 || !a->u || !a->dt || !a->A || !a->B || !a->C || !a->out || !a->state_out) return AVSI_ERR_INVALID_ARG;
    if (a->state > MAX_STATE) return AVSI_ERR_UNSUPPORTED;
    Scan p = params(a);
    hipStream_t s = (hipStream_t)stream;
    avsi_clear_error();
    AVSI_SCAN_T(go_step)
    return avsi_launch_status();
}
