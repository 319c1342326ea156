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
// Bound: the vector unit.  A state and step costs one exponential (10.5 cycles of its SIMD for a wave, 3.2 for a plain operation) and
// four (forward) to twelve (backward) plain operations; the bytes of u, dt, z and out come second for N = 16.  A lane owns 4 states
// of one channel, N / 4 lanes a channel: four independent chains and one exchange of the sum over the states, in LDS.  Time goes by in
// tiles of 16 steps, between two kinds of waves (below).  8 sequences of 2048 steps and channels, N = 16, bfloat16: forward 166 us
// (2.4 TB/s with the states it keeps, the vector unit's counter at 80 %), backward 463 us (81 %); one kind of waves that staged, ran and
// wrote in turn took 316 and 770 us.  (float32 operands carry the gates' exponents in two words: 32 x 250 x 512, 23.5 us against 23.0.)
//
// Time is cut into chunks only where batch and channels do not fill the chip (chunks_of): then a first launch runs every chunk from a
// zero state, a second one joins the chunk ends (h_end = exp(A sum delta) h_start + h_local), and the main launch starts from those.
//
// Training: the forward pass keeps the state at the start of every tile, so the backward pass redoes 16 steps at a time in registers
// (64 decays and 64 states per lane) and goes back over them.  dB and dC are sums over the channels: over a wave's channels by lane
// exchanges, over the workgroup's waves in LDS, over the workgroups through partials and a last launch.  All sums have a fixed order;
// there are no atomics.
#include "avsi_common.h"
#include "avsi_wave.h"

#include <type_traits>

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
    float* kept;                     // [batch][tiles][dim][NP]
    void *du, *ddt, *dz;             // [batch][time][dim]
    float *part_bc, *part_w;         // [batch][time][groups][blocks][2][NP], [batch * chunks][partial_stride]
    float *ends, *sums;              // [batch][chunks][dim][NP], [batch][chunks][dim]
    int batch, T, dim, N, NP, groups, softplus, gated, chunk, chunks, blocks;     // chunk: steps, a multiple of TT; blocks: per group
};

__device__ __forceinline__ int length_of(const int32_t* lengths, int b, int T) {
    if (!lengths) return T;
    const int n = lengths[b];
    return n < 0 ? 0 : (n < T ? n : T);
}

// ------------------------------------------------------------------------------------------------- what the kernels share
// A workgroup is two kinds of waves.  The consumers own the states: a lane NS states of a channel, LN lanes a channel.  The producers
// stage the tile behind the one the consumers are at (softplus, gates, conversion, once per channel and step) into the other half of
// the buffers and finish the tile in front of it (sums over the lanes of a channel, outputs): a recurrence alone is a chain of
// dependent operations that one wave per SIMD cannot fill, and the waves fill each other's gaps.  One barrier per tile; loads are a
// tile ahead of their use.
template <int LN_, int NS_, bool EL = false> struct Shape {
    static constexpr int LN = LN_, NS = NS_;
    static constexpr bool ELEMENTS = EL;                    // load one by one: fewer than four channels, or states in no whole quads
    static constexpr int NP = LN * NS;                      // states with their padding
    static constexpr int CH = LN <= 4 ? 64 : 256 / LN;      // channels of a workgroup
    static constexpr int NC = CH * LN, NW = NC / 64;        // consumers: threads, waves
    static constexpr int QR = CH / 4, PT = 256;             // quads of channels per step; producers
    static constexpr bool SPARE = PT > QR * TT;             // more of them than quads in a tile: they stage B and C and add dB and dC
    static constexpr int PL = LN > 4 ? 4 : LN;              // parts in which a sum over a channel's lanes is handed to the producers
    static constexpr int QB = NP / 4;                       // quads of states per step
    static constexpr int BPASSES = (TT * QB + PT - 1) / PT;  // of the producers over a tile's [TT][NP] of B and C
    typedef __attribute__((ext_vector_type(NS_))) float Vec;   // the states of a lane
};

// Where a workgroup is: its group of channels, its first channel (of all), how many of CH exist; its sequence, chunk and steps.
template <typename S> struct Place {
    int g, d0, n, b, c, begin, end, live, tiles, block;
    bool ragged;                // groups of channels in no whole quads
    __device__ __forceinline__ Place(const Scan& p, int chunk) {
        const int per = p.dim / p.groups;
        block = blockIdx.x % p.blocks;
        g = blockIdx.x / p.blocks;
        d0 = g * per + block * S::CH;
        n = per - block * S::CH;
        n = n < S::CH ? n : S::CH;
        ragged = per & 3;
        c = chunk;
        b = blockIdx.z;
        const int len = length_of(p.lengths, b, p.T);
        begin = c * p.chunk;
        end = begin + p.chunk < p.T ? begin + p.chunk : p.T;
        live = len < end ? len : end;
        tiles = begin < live ? (live - begin + TT - 1) / TT : 0;
    }
};

// A producer's part of a tile: quad q of the channels in step `row`.
// Nothing that loads may branch by lane (the join behind such a branch waits for the load): rows from `live` on read the last row, a
// quad that goes over the last of all channels takes the last four and is shifted when it is used; what a group does not own is
// masked where it is used.
template <typename S> struct Stage {
    int id, q, row, c;          // c: the channel (of all) at which the quad is loaded
    bool works;                 // whether it has a quad of its own (without one it goes through the same steps on another's)
    bool on[4];                 // which of its channels exist
    __device__ __forceinline__ Stage(const Scan& p, const Place<S>& at, int thread) {
        id = thread;
        q = id % S::QR, row = id / S::QR % TT;
        works = !S::SPARE || id < S::QR * TT;
        c = at.d0 + 4 * q;
        if (!S::ELEMENTS) c = c < p.dim - 4 ? c : p.dim - 4;
#pragma unroll
        for (int k = 0; k < 4; ++k) on[k] = 4 * q + k < at.n;
    }
};
// Row `i`'s place inside a tile that has `rows` rows left: bytes in 32 bits, on top of the tile's uniform address.
template <typename T> __device__ __forceinline__ unsigned row_at(int i, int rows, int64_t ts) {
    const unsigned step = (unsigned)ts * sizeof(T), at = i * step, last = ((rows < TT ? rows : TT) - 1) * step;
    return at < last ? at : last;
}
template <typename T> __device__ __forceinline__ T* at_byte(T* p, unsigned offset) {
    return (T*)((typename std::conditional<std::is_const<T>::value, const char, char>::type*)p + offset);
}

template <typename T, typename S> struct Tile {
    avsi_quad<T> v;
    __device__ __forceinline__ void load(const void* base, int64_t bs, int64_t ts, const Scan& p, const Place<S>& at, const Stage<S>& st, int t0) {
        const T* b = (const T*)base + at.b * bs + t0 * ts;
        const unsigned r = row_at<T>(st.row, at.live - t0, ts);
        if (!S::ELEMENTS) {
            v.load(at_byte(b, r + st.c * (unsigned)sizeof(T)));
        } else {
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = (float)*at_byte(b, r + (st.c + k < p.dim ? st.c + k : p.dim - 1) * (unsigned)sizeof(T));
            v.set(f);
        }
    }
    __device__ __forceinline__ void get(const Place<S>& at, const Stage<S>& st, float (&f)[4]) const {
        v.get(f);
        if (!S::ELEMENTS && at.ragged) {            // (a branch of the whole launch)
            const int shift = at.d0 + 4 * st.q - st.c;
            if (shift & 1) f[0] = f[1], f[1] = f[2], f[2] = f[3];
            if (shift & 2) f[0] = f[2], f[1] = f[3];
        }
    }
};
template <typename T, typename S> struct TileBC {
    avsi_quad<T> v[S::BPASSES];
    __device__ __forceinline__ void load(const void* base, int64_t bs, int64_t ts, int64_t gs, const Scan& p, const Place<S>& at,
                                         const Stage<S>& st, int t0) {
        const T* b = (const T*)base + at.b * bs + at.g * gs + t0 * ts;
#pragma unroll
        for (int i = 0; i < S::BPASSES; ++i) {
            const int id = i * S::PT + st.id, n = 4 * (id % S::QB);
            const unsigned r = row_at<T>(id / S::QB % TT, at.live - t0, ts);
            if (!S::ELEMENTS) {
                v[i].load(at_byte(b, r + (n < p.N ? n : p.N - 4) * (unsigned)sizeof(T)));
            } else {
                float f[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = (float)*at_byte(b, r + (n + k < p.N ? n + k : p.N - 1) * (unsigned)sizeof(T));
                v[i].set(f);
            }
        }
    }
    __device__ __forceinline__ void put(avsi_f4* lds, const Scan& p, const Place<S>& at, const Stage<S>& st, int t0) const {   // [TT][NP]
#pragma unroll
        for (int i = 0; i < S::BPASSES; ++i) {
            const int id = i * S::PT + st.id, n = 4 * (id % S::QB);
            float f[4];
            v[i].get(f);
            if (t0 + TT > at.live || p.N < S::NP)       // (uniform)
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = n + k < p.N && t0 + id / S::QB < at.live ? f[k] : 0.f;
            if (S::BPASSES * S::PT == TT * S::QB || id < TT * S::QB) lds[id] = avsi_f4{f[0], f[1], f[2], f[3]};
        }
    }
};
template <typename T> __device__ __forceinline__ void put_quad(T* p, int n, const float (&f)[4]) {
    avsi_quad<T> v;
    v.set(f);
    v.store(p, n);
}

// (both values and a choice: a branch, though one of the whole launch, would fence the schedule)
__device__ __forceinline__ float step_size(float x, int softplus, float& slope) {
    const float s = avsi_softplus(x, slope);
    slope = softplus ? slope : 1.f;
    return softplus ? s : x;
}
__device__ __forceinline__ float step_size(float x, int softplus) {
    float slope;
    return step_size(x, softplus, slope);
}

// dt_bias, D of this thread's quad of channels
template <typename S> __device__ __forceinline__ void quad_of(const float* v, const Place<S>& at, const Stage<S>& st, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v && st.on[i] ? v[at.d0 + 4 * st.q + i] : 0.f;
}

// A consumer's states in a [..][dim][NP] array at row `lead`, its A, and the state it starts from.
template <typename S> __device__ __forceinline__ int64_t lane_at(const Scan& p, const Place<S>& at, int64_t lead) {
    return ((lead * p.dim + at.d0 + threadIdx.x / S::LN) * S::LN + threadIdx.x % S::LN) * S::NS;
}
template <typename S> __device__ __forceinline__ void store_lane(float* p, const float (&f)[S::NS]) {
    typename S::Vec v;
#pragma unroll
    for (int j = 0; j < S::NS; ++j) v[j] = f[j];
    *(typename S::Vec*)p = v;
}
template <typename S> __device__ __forceinline__ void lane_A(const Scan& p, const Place<S>& at, float (&A)[S::NS]) {
    const int c = threadIdx.x / S::LN, n = S::NS * (threadIdx.x % S::LN);
#pragma unroll
    for (int j = 0; j < S::NS; ++j) A[j] = c < at.n && n + j < p.N ? p.A[(int64_t)(at.d0 + c) * p.N + n + j] : 0.f;
}
template <typename S> __device__ __forceinline__ void lane_start(const Scan& p, const Place<S>& at, float (&h)[S::NS]) {
    const int c = threadIdx.x / S::LN, n = S::NS * (threadIdx.x % S::LN);
#pragma unroll
    for (int j = 0; j < S::NS; ++j) h[j] = 0.f;
    if (c >= at.n) return;
    if (at.c > 0) {
        const typename S::Vec v = *(const typename S::Vec*)(p.ends + lane_at<S>(p, at, (int64_t)at.b * p.chunks + at.c));
#pragma unroll
        for (int j = 0; j < S::NS; ++j) h[j] = v[j];
    } else if (p.state) {
#pragma unroll
        for (int j = 0; j < S::NS; ++j)
            if (n + j < p.N) h[j] = p.state[((int64_t)at.b * p.dim + at.d0 + c) * p.N + n + j];
    }
}

// Where a channel's 16 (8) bytes lie in a row of LDS: sixteen producers in a row read or write the same channel of their quads at 64 (32)
// bytes from each other, which is one bank in four (two); so the channels inside a quad are permuted from quad to quad.  (With them in
// order the backward pass spent a quarter of its LDS cycles on conflicts.)
template <typename S> __device__ __forceinline__ int place16(int row, int ch) { return ch ^ ((row * S::QR + (ch >> 2)) >> 2 & 3); }
template <typename S> __device__ __forceinline__ int place8(int row, int ch) { return ch ^ ((row * S::QR + (ch >> 2)) >> 3 & 1) << 1; }

// A sum over a channel's lanes: one value per lane into LDS, [channel][PL], and four channels' sums out of it.  More than four lanes
// hand over four values (the buffers would not fit otherwise); the lanes that then hold the same one all write it.
template <typename S> __device__ __forceinline__ void put_part(avsi_f4 (*rows)[S::CH * S::PL / 4], int t, float v) {
    int part = threadIdx.x % S::LN;
    if (S::LN == 8) {
        v += avsi_dpp<0x141>(v);            // row_half_mirror
        part = part < 4 ? part : 7 - part;
    }
    if (S::LN == 16) {
        v += avsi_dpp<0x128>(v);            // row_ror 8
        v += avsi_dpp<0x124>(v);            // row_ror 4
        part &= 3;
    }
    const int ch = threadIdx.x / S::LN;
    ((float*)rows[t])[(S::PL == 4 ? place16<S>(t, ch) : ch) * S::PL + part] = v;
}
template <typename S> __device__ __forceinline__ void lane_sums(const avsi_f4 (*rows)[S::CH * S::PL / 4], int t, int q, float (&f)[4]) {
    constexpr int PL = S::PL, V = PL < 4 ? PL : 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float* p = (const float*)rows[t] + (PL == 4 ? place16<S>(t, 4 * q + k) : 4 * q + k) * PL;
        f[k] = 0.f;
#pragma unroll
        for (int l = 0; l < PL; l += V) {
            const avsi_raw<float, V> r = *(const avsi_raw<float, V>*)__builtin_assume_aligned(p + l, 4 * V);
#pragma unroll
            for (int i = 0; i < V; ++i) f[k] += r.v[i];
        }
    }
}

// One partial of the weights' gradients: dA [dim][NP], dD [dim], ddt_bias [dim], to a multiple of 16 bytes.
__host__ __device__ __forceinline__ int64_t partial_stride(int dim, int NP) { return ((int64_t)dim * (NP + 2) + 3) / 4 * 4; }

// ------------------------------------------------------------------------------------------------------------- forward
// The consumers' decays are a group of two steps ahead of the states, and the operands of a group are read from LDS during the one
// before; the fences keep the compiler from moving the reads back to their use.
template <typename T, typename S> __global__ __launch_bounds__(S::NC + S::PT) void scan_fwd_kernel(Scan p) {
    typedef typename S::Vec Vec;
    __shared__ avsi_f2 s_in[2][TT][S::CH];             // delta, delta u
    __shared__ avsi_f4 s_B[2][TT * S::QB], s_C[2][TT * S::QB];
    __shared__ avsi_f4 s_y[2][TT][S::CH * S::PL / 4];          // C . h of each lane's states
    const Place<S> at(p, blockIdx.y);
    if (threadIdx.x < S::NC) {
        __builtin_amdgcn_s_setprio(3);          // (they are the longer of the two: 60.4 -> 59.0 us for 8191 steps of 1536 channels)
        const int ch = threadIdx.x / S::LN, ql = threadIdx.x % S::LN;
        float A[S::NS], h[S::NS];
        lane_A<S>(p, at, A);
        lane_start<S>(p, at, h);
#pragma unroll
        for (int j = 0; j < S::NS; ++j) A[j] *= LOG2E;
        float* kept = p.kept && ch < at.n ? p.kept + lane_at<S>(p, at, (int64_t)at.b * ((p.T + TT - 1) / TT) + at.begin / TT) : nullptr;
        AVSI_LDS_BARRIER();
        for (int n = 0; n < at.tiles; ++n) {
            const int buf = n & 1;
            avsi_f2 in[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) in[t] = s_in[buf][t][place8<S>(t, ch)];
            Vec Bv[2], Cv[2], Bn[2], Cn[2];
            auto fetch = [&](int t) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    Bn[j] = ((const Vec*)s_B[buf])[(t + j) * S::LN + ql];
                    Cn[j] = ((const Vec*)s_C[buf])[(t + j) * S::LN + ql];
                }
            };
            float a[2][S::NS], next[2][S::NS];
            auto decays = [&](int t) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) next[k][j] = __builtin_amdgcn_exp2f(in[t + k][0] * A[j]);
            };
            if (kept) store_lane<S>(kept + (int64_t)n * p.dim * S::NP, h);
            fetch(0);
            decays(0);
#pragma unroll
            for (int t = 0; t < TT; t += 2) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    Bv[k] = Bn[k], Cv[k] = Cn[k];
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) a[k][j] = next[k][j];
                }
                if (t + 2 < TT) fetch(t + 2);
                __builtin_amdgcn_sched_barrier(0);
                if (t + 2 < TT) decays(t + 2);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float y = 0.f;
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) {
                        h[j] = fmaf(a[k][j], h[j], in[t + k][1] * Bv[k][j]);
                        y = fmaf(h[j], Cv[k][j], y);
                    }
                    put_part<S>(s_y[buf], t + k, y);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            AVSI_LDS_BARRIER();
        }
        if (p.state_out && at.c == p.chunks - 1 && ch < at.n)
#pragma unroll
            for (int j = 0; j < S::NS; ++j)
                if (S::NS * ql + j < p.N) p.state_out[((int64_t)at.b * p.dim + at.d0 + ch) * p.N + S::NS * ql + j] = h[j];
        return;
    }
    const Stage<S> st(p, at, threadIdx.x - S::NC);
    float bias[4], Dq[4];
    quad_of<S>(p.bias, at, st, bias);
    quad_of<S>(p.D, at, st, Dq);
    T* out = (T*)p.out + at.b * p.ob + at.d0;
    const unsigned place = (st.row * (unsigned)p.ot + 4 * st.q) * (unsigned)sizeof(T);          // in a tile
    struct Ahead {              // a tile's operands in flight, two tiles ahead of their use
        Tile<T, S> u, dt, z;
        TileBC<T, S> B, C;
    } x;
    auto load = [&](int n) {
        const int t0 = at.begin + (n < at.tiles ? n : at.tiles - 1) * TT;
        x.u.load(p.u, p.ub, p.ut, p, at, st, t0);
        x.dt.load(p.dt, p.tb, p.tt, p, at, st, t0);
        x.z.load(p.z, p.zb, p.zt, p, at, st, t0);
        x.B.load(p.B, p.Bb, p.Bt, p.Bg, p, at, st, t0);
        x.C.load(p.C, p.Cb, p.Ct, p.Cg, p, at, st, t0);
    };
    struct Held {                // D u and the gate of a tile
        float thru[4], gate[4];
    } even, odd;
    float uf[4], df[4], zf[4];
    auto take = [&](int n) {
        const int t0 = at.begin + n * TT, buf = n & 1;
        x.u.get(at, st, uf);
        x.dt.get(at, st, df);
        x.z.get(at, st, zf);
        x.B.put(s_B[buf], p, at, st, t0);
        x.C.put(s_C[buf], p, at, st, t0);
        load(n + 1);
    };
    auto stage = [&](int n, Held& w) {
        const int t0 = at.begin + n * TT, buf = n & 1;
        float d[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float g = zf[k] * avsi_sigmoid<T>(zf[k]);
            d[k] = step_size(df[k] + bias[k], p.softplus);
            w.thru[k] = Dq[k] * uf[k];
            w.gate[k] = p.gated ? g : 1.f;
        }
        if (t0 + TT > at.live) {         // (uniform; what lanes without a channel compute goes nowhere)
            const bool on = t0 + st.row < at.live;
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] = on ? d[k] : 0.f, uf[k] = on ? uf[k] : 0.f;
        }
        if (!st.works) return;
        avsi_f4* to = (avsi_f4*)s_in[buf][st.row];
        to[place8<S>(st.row, 4 * st.q) / 2] = avsi_f4{d[0], d[0] * uf[0], d[1], d[1] * uf[1]};
        to[place8<S>(st.row, 4 * st.q + 2) / 2] = avsi_f4{d[2], d[2] * uf[2], d[3], d[3] * uf[3]};
    };
    auto write = [&](int n, const Held& w) {
        const int t = at.begin + n * TT + st.row;
        if (t < at.end && st.works) {
            float o[4];
            lane_sums<S>(s_y[n & 1], st.row, st.q, o);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = (o[k] + w.thru[k]) * w.gate[k];
            if (at.begin + (n + 1) * TT > at.live)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = t < at.live ? o[k] : 0.f;
            put_quad<T>(at_byte(out + (at.begin + n * TT) * p.ot, place), at.n - 4 * st.q, o);
        }
    };
    // While the consumers are at tile n: tile n + 1 is staged, n - 1 finished (`w`: what is held of n - 1, then of n + 1).  The loads and
    // then the stores are issued in front of the arithmetic, and no branch lies between a load and its use: a wait behind one is for all
    // that is in flight.
    auto turn = [&](int n, Held& w) {
        take(n + 1);
        write(n - 1, w);
        stage(n + 1, w);
        AVSI_LDS_BARRIER();
    };
    if (at.tiles) {
        load(0);
        take(0);
        stage(0, even);
    }
    AVSI_LDS_BARRIER();
    if (at.tiles > 1) {
        take(1);
        stage(1, odd);
        AVSI_LDS_BARRIER();
        for (int n = 1; n + 1 < at.tiles; n += 2) {
            turn(n, even);
            if (n + 2 >= at.tiles) break;
            turn(n + 1, odd);
        }
        Held before, last;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            before.thru[k] = at.tiles % 2 ? odd.thru[k] : even.thru[k], last.thru[k] = at.tiles % 2 ? even.thru[k] : odd.thru[k];
            before.gate[k] = at.tiles % 2 ? odd.gate[k] : even.gate[k], last.gate[k] = at.tiles % 2 ? even.gate[k] : odd.gate[k];
        }
        write(at.tiles - 2, before);
        AVSI_LDS_BARRIER();
        write(at.tiles - 1, last);
    } else if (at.tiles) {
        AVSI_LDS_BARRIER();
        write(0, even);
    }
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    if (st.works)
        for (int t0 = at.begin + at.tiles * TT; t0 + st.row < at.end; t0 += TT)
            put_quad<T>(at_byte(out + t0 * p.ot, place), at.n - 4 * st.q, zero);
}

// A chunk from a zero state: its end state and the sum of its step sizes.  BACK: the adjoint state, from behind.
template <typename T, typename S, bool BACK> __global__ __launch_bounds__(S::NC + S::PT) void scan_chunk_kernel(Scan p) {
    typedef typename S::Vec Vec;
    __shared__ avsi_f2 s_in[2][TT][S::CH];             // delta, delta u (BACK: dy)
    __shared__ avsi_f4 s_B[2][TT * S::QB];             // (BACK: C)
    const Place<S> at(p, blockIdx.y + (BACK ? 1 : 0));  // (the first chunk's is not needed; forward: the last one's)
    if (threadIdx.x < S::NC) {
        __builtin_amdgcn_s_setprio(3);
        const int ch = threadIdx.x / S::LN, ql = threadIdx.x % S::LN;
        float A[S::NS], h[S::NS] = {}, sum = 0.f;
        lane_A<S>(p, at, A);
#pragma unroll
        for (int j = 0; j < S::NS; ++j) A[j] *= LOG2E;
        AVSI_LDS_BARRIER();
        for (int n = 0; n < at.tiles; ++n) {
            const int buf = n & 1;
            avsi_f2 in[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) in[t] = s_in[buf][BACK ? TT - 1 - t : t][place8<S>(BACK ? TT - 1 - t : t, ch)];
            Vec Bv[2], Bn[2];
            auto fetch = [&](int t) {
#pragma unroll
                for (int j = 0; j < 2; ++j) Bn[j] = ((const Vec*)s_B[buf])[(BACK ? TT - 1 - t - j : t + j) * S::LN + ql];
            };
            float a[2][S::NS], next[2][S::NS];
            auto decays = [&](int t) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) next[k][j] = __builtin_amdgcn_exp2f(in[t + k][0] * A[j]);
            };
            fetch(0);
            decays(0);
            float part = 0.f;               // (a tile's own sum: the long one keeps its low bits)
#pragma unroll
            for (int t = 0; t < TT; t += 2) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    Bv[k] = Bn[k];
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) a[k][j] = next[k][j];
                }
                if (t + 2 < TT) fetch(t + 2);
                __builtin_amdgcn_sched_barrier(0);
                if (t + 2 < TT) decays(t + 2);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    part += in[t + k][0];
#pragma unroll
                    for (int j = 0; j < S::NS; ++j)
                        h[j] = BACK ? a[k][j] * fmaf(Bv[k][j], in[t + k][1], h[j]) : fmaf(a[k][j], h[j], in[t + k][1] * Bv[k][j]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            sum += part;
            AVSI_LDS_BARRIER();
        }
        if (ch < at.n) {
            // the chunk's row of `ends` is read as the start of the chunk behind it (in front of it)
            const int64_t lead = (int64_t)at.b * p.chunks + (BACK ? at.c - 1 : at.c + 1);
            store_lane<S>(p.ends + lane_at<S>(p, at, lead), h);
            if (ql == 0) p.sums[lead * p.dim + at.d0 + ch] = sum;
        }
        return;
    }
    const Stage<S> st(p, at, threadIdx.x - S::NC);
    float bias[4];
    quad_of<S>(p.bias, at, st, bias);
    Tile<T, S> u, dt, z;                               // BACK: u is dout
    TileBC<T, S> Bt;
    auto tile_at = [&](int n) { return at.begin + (BACK ? at.tiles - 1 - n : n) * TT; };
    auto load = [&](int n) {
        const int t0 = tile_at(n < at.tiles ? n : at.tiles - 1);
        dt.load(p.dt, p.tb, p.tt, p, at, st, t0);
        if (BACK) {
            u.load(p.dout, p.gb, p.gt, p, at, st, t0);
            z.load(p.z, p.zb, p.zt, p, at, st, t0);
            Bt.load(p.C, p.Cb, p.Ct, p.Cg, p, at, st, t0);
        } else {
            u.load(p.u, p.ub, p.ut, p, at, st, t0);
            Bt.load(p.B, p.Bb, p.Bt, p.Bg, p, at, st, t0);
        }
    };
    auto stage = [&](int n) {
        const int t0 = tile_at(n), buf = n & 1;
        float x[4], df[4], zf[4] = {}, d[4];
        u.get(at, st, x);
        dt.get(at, st, df);
        if (BACK) z.get(at, st, zf);
        Bt.put(s_B[buf], p, at, st, t0);
        load(n + 1);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            d[k] = step_size(df[k] + bias[k], p.softplus);
            const float gate = zf[k] * avsi_sigmoid<T>(zf[k]);
            x[k] *= BACK ? (p.gated ? gate : 1.f) : d[k];
        }
        if (t0 + TT > at.live) {
            const bool on = t0 + st.row < at.live;
#pragma unroll
            for (int k = 0; k < 4; ++k) d[k] = on ? d[k] : 0.f, x[k] = on ? x[k] : 0.f;
        }
        if (!st.works) return;
        avsi_f4* to = (avsi_f4*)s_in[buf][st.row];
        to[place8<S>(st.row, 4 * st.q) / 2] = avsi_f4{d[0], x[0], d[1], x[1]};
        to[place8<S>(st.row, 4 * st.q + 2) / 2] = avsi_f4{d[2], x[2], d[3], x[3]};
    };
    if (at.tiles) {
        load(0);
        stage(0);
    }
    AVSI_LDS_BARRIER();
    for (int n = 0; n < at.tiles; ++n) {
        if (n + 1 < at.tiles) stage(n + 1);
        AVSI_LDS_BARRIER();
    }
}

// start[c] = local end of c - 1 + exp(A sum of c - 1) start[c - 1] (BACK: with c + 1), in place.  One thread per four states.
// The exponential of a whole chunk may leave the range of a float where the states, which its steps multiply one by one, do not
// (growth from zero or a tiny state, an infinite one that decays): its power of two goes onto the state by itself.
template <bool BACK> __global__ __launch_bounds__(256) void scan_join_kernel(Scan p, int QB) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)p.batch * p.dim * QB) return;
    const int ql = (int)(id % QB), d = (int)(id / QB % p.dim), b = (int)(id / QB / p.dim);
    float A[4], h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int n = 4 * ql + j;
        A[j] = n < p.N ? p.A[(int64_t)d * p.N + n] * LOG2E : 0.f;
        h[j] = !BACK && p.state && n < p.N ? p.state[((int64_t)b * p.dim + d) * p.N + n] : 0.f;
    }
    // (the rows do not depend on each other: eight of them in flight)
    for (int i0 = 1; i0 < p.chunks; i0 += 8) {
        avsi_f4 v[8];
        float sum[8];
        auto row = [&](int i) {
            i = i < p.chunks ? i : p.chunks - 1;
            return ((int64_t)b * p.chunks + (BACK ? p.chunks - 1 - i : i)) * p.dim + d;
        };
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = *(const avsi_f4*)(p.ends + (row(i0 + k) * QB + ql) * 4);
            sum[k] = p.sums[row(i0 + k)];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i0 + k < p.chunks) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = fmaxf(fminf(sum[k] * A[j], 1000.f), -1000.f), n = floorf(x);     // (2^+-1000 takes any state to its end)
                    v[k][j] = h[j] = fmaf(__builtin_amdgcn_exp2f(x - n), ldexpf(h[j], (int)n), v[k][j]);
                }
                *(avsi_f4*)(p.ends + (row(i0 + k) * QB + ql) * 4) = v[k];
            }
    }
}

// ------------------------------------------------------------------------------------------------------------ backward
// Sum over the channels of a wave (the lanes that share a place among the states) of b and c, at *out = [2][NP] of one step.
// While a level halves the lanes it halves the values too: the upper half of the lanes takes c, then the odd rows the upper states.
template <typename S> __device__ __forceinline__ void channel_sums(float (&b)[S::NS], float (&c)[S::NS], float* out) {
    constexpr int LN = S::LN, H = S::NS / 2;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < S::NS; ++j) {
        avsi_swap32(b[j], c[j]);
        b[j] += c[j];
    }
#pragma unroll
    for (int j = 0; j < H; ++j) {
        avsi_swap16(b[j], b[j + H]);
        b[j] += b[j + H];
        if (LN <= 8) b[j] += avsi_dpp<0x128>(b[j]);         // row_ror 8
        if (LN <= 4) b[j] += avsi_dpp<0x124>(b[j]);         // row_ror 4
        if (LN <= 2) b[j] += avsi_dpp<0x4E>(b[j]);
        if (LN <= 1) b[j] += avsi_dpp<0xB1>(b[j]);
    }
    // (the lanes of a row that hold the same sums all write them: a branch here would fence the schedule of every step)
    float* o = out + (lane >> 5) * S::NP + S::NS * (lane % LN) + ((lane >> 4) & 1) * H;
#pragma unroll
    for (int j = 0; j < H; ++j) o[j] = b[j];
}

// A tile is 16 steps forward from its kept state, decays and states staying in the registers of the consumers, and 16 steps back
// over them.
template <typename T, typename S> __global__ __launch_bounds__(S::NC + S::PT) void scan_bwd_kernel(Scan p) {
    typedef typename S::Vec Vec;
    __shared__ avsi_f4 s_in[2][TT][S::CH];             // delta, delta u, dy
    __shared__ avsi_f4 s_B[2][TT * S::QB], s_C[2][TT * S::QB];
    __shared__ avsi_f4 s_y[2][TT][S::CH * S::PL / 4], s_gB[2][TT][S::CH * S::PL / 4], s_gA[2][TT][S::CH * S::PL / 4];      // sums over each lane's states
    __shared__ alignas(16) float s_bc[2][S::NW][TT][2 * S::NP];
    const Place<S> at(p, blockIdx.y);
    auto tile_at = [&](int n) { return at.begin + (at.tiles - 1 - n) * TT; };
    float* pw = p.part_w + ((int64_t)at.b * p.chunks + at.c) * partial_stride(p.dim, S::NP);
    if (threadIdx.x < S::NC) {
        const int ch = threadIdx.x / S::LN, ql = threadIdx.x % S::LN;
        float A[S::NS], Al[S::NS], g[S::NS] = {}, dA[S::NS] = {};
        lane_A<S>(p, at, A);
#pragma unroll
        for (int j = 0; j < S::NS; ++j) Al[j] = A[j] * LOG2E;
        if (at.c < p.chunks - 1 && ch < at.n) {
            const Vec v = *(const Vec*)(p.ends + lane_at<S>(p, at, (int64_t)at.b * p.chunks + at.c));
#pragma unroll
            for (int j = 0; j < S::NS; ++j) g[j] = v[j];
        }
        // (lanes without a channel read the last one's)
        const float* kept = p.kept + lane_at<S>(p, at, (int64_t)at.b * ((p.T + TT - 1) / TT)) - (ch < at.n ? 0 : (int64_t)(ch - at.n + 1) * S::NP);
        Vec start;
        auto load = [&](int n) { start = *(const Vec*)(kept + (int64_t)(tile_at(n < at.tiles ? n : at.tiles - 1) / TT) * p.dim * S::NP); };
        if (at.tiles) load(0);
        AVSI_LDS_BARRIER();
        for (int n = 0; n < at.tiles; ++n) {
            const int buf = n & 1;
            float h[S::NS];
#pragma unroll
            for (int j = 0; j < S::NS; ++j) h[j] = start[j];
            load(n + 1);
            float a[TT][S::NS], before[TT][S::NS];
            avsi_f4 in[2], in2[2];
            Vec Bv[2], Cv[2], Bn[2], Cn[2];
            auto fetch = [&](int t) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    in2[j] = s_in[buf][t + j][place16<S>(t + j, ch)];
                    Bn[j] = ((const Vec*)s_B[buf])[(t + j) * S::LN + ql];
                    Cn[j] = ((const Vec*)s_C[buf])[(t + j) * S::LN + ql];
                }
            };
            auto take = [&]() {
#pragma unroll
                for (int j = 0; j < 2; ++j) in[j] = in2[j], Bv[j] = Bn[j], Cv[j] = Cn[j];
            };
            fetch(0);
#pragma unroll
            for (int t = 0; t < TT; t += 2) {
                take();
                fetch(t + 2 < TT ? t + 2 : TT - 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float y = 0.f;                          // (for dz; without a gate it is not read)
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) {
                        before[t + k][j] = h[j];
                        a[t + k][j] = __builtin_amdgcn_exp2f(in[k][0] * Al[j]);
                        h[j] = fmaf(a[t + k][j], h[j], in[k][1] * Bv[k][j]);
                        y = fmaf(h[j], Cv[k][j], y);
                    }
                    put_part<S>(s_y[buf], t + k, y);
                }
            }
            float dAt[S::NS] = {};        // (a tile's own sum: the long sum over time keeps its low bits)
#pragma unroll
            for (int t2 = TT - 2; t2 >= 0; t2 -= 2) {
                take();
                if (t2 > 0) fetch(t2 - 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 1; k >= 0; --k) {
                    const int t = t2 + k;
                    float vb[S::NS], vc[S::NS], gB = 0.f, gA = 0.f;
#pragma unroll
                    for (int j = 0; j < S::NS; ++j) {
                        const float gj = fmaf(Cv[k][j], in[k][2], g[j]);
                        vb[j] = gj * in[k][1];
                        vc[j] = in[k][2] * (t == TT - 1 ? h[j] : before[t == TT - 1 ? t : t + 1][j]);
                        gB = fmaf(gj, Bv[k][j], gB);
                        g[j] = a[t][j] * gj;
                        const float x = g[j] * before[t][j];
                        gA = fmaf(x, A[j], gA);
                        dAt[j] = fmaf(x, in[k][0], dAt[j]);
                    }
                    put_part<S>(s_gB[buf], t, gB);
                    put_part<S>(s_gA[buf], t, gA);
                    channel_sums<S>(vb, vc, s_bc[buf][threadIdx.x >> 6][t]);
                }
            }
#pragma unroll
            for (int j = 0; j < S::NS; ++j) dA[j] += dAt[j];
            AVSI_LDS_BARRIER();
        }
        if (ch < at.n) store_lane<S>(pw + ((int64_t)(at.d0 + ch) * S::LN + ql) * S::NS, dA);
        AVSI_LDS_BARRIER();
        AVSI_LDS_BARRIER();
        return;
    }
    const Stage<S> st(p, at, threadIdx.x - S::NC);
    float bias[4], Dq[4], dD[4] = {}, dbias[4] = {};
    quad_of<S>(p.bias, at, st, bias);
    quad_of<S>(p.D, at, st, Dq);
    const int64_t flat = (int64_t)at.b * p.T * p.dim + at.d0;
    const unsigned place = (st.row * (unsigned)p.dim + 4 * st.q) * (unsigned)sizeof(T);         // in a tile
    const int left = at.n - 4 * st.q;
    auto put = [&](int t0, const float (&du)[4], const float (&ddt)[4], const float (&dz)[4]) {
        const int64_t i = flat + (int64_t)t0 * p.dim;
        put_quad<T>(at_byte((T*)p.du + i, place), left, du);
        put_quad<T>(at_byte((T*)p.ddt + i, place), left, ddt);
        if (p.gated) put_quad<T>(at_byte((T*)p.dz + i, place), left, dz);
    };
    struct Ahead {
        Tile<T, S> u, dt, z, go;
        TileBC<T, S> B, C;
    } x;
    auto load = [&](int n) {
        const int t0 = tile_at(n < at.tiles ? n : at.tiles - 1);
        x.u.load(p.u, p.ub, p.ut, p, at, st, t0);
        x.dt.load(p.dt, p.tb, p.tt, p, at, st, t0);
        x.go.load(p.dout, p.gb, p.gt, p, at, st, t0);
        x.z.load(p.z, p.zb, p.zt, p, at, st, t0);
        x.B.load(p.B, p.Bb, p.Bt, p.Bg, p, at, st, t0);
        x.C.load(p.C, p.Cb, p.Ct, p.Cg, p, at, st, t0);
    };
    struct Held {                // what a tile's gradients need besides the consumers' sums
        float u[4], delta[4], slope[4], dy[4], gz[4];
    } even, odd;
    float uf[4], df[4], zf[4], of[4];
    auto take = [&](int n) {
        const int t0 = tile_at(n), buf = n & 1;
        x.u.get(at, st, uf);
        x.dt.get(at, st, df);
        x.z.get(at, st, zf);
        x.go.get(at, st, of);
        x.B.put(s_B[buf], p, at, st, t0);
        x.C.put(s_C[buf], p, at, st, t0);
        load(n + 1);
    };
    auto stage = [&](int n, Held& w) {
        const int t0 = tile_at(n), buf = n & 1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float e = avsi_sigmoid<T>(zf[k]);
            w.u[k] = uf[k];
            w.delta[k] = step_size(df[k] + bias[k], p.softplus, w.slope[k]);
            w.dy[k] = of[k] * (p.gated ? zf[k] * e : 1.f);
            w.gz[k] = of[k] * (e * fmaf(zf[k], 1.f - e, 1.f));
        }
        if (t0 + TT > at.live || at.n < S::CH) {         // (uniform; the sums over channels and time take them all)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool on = st.on[k] && t0 + st.row < at.live;
                w.u[k] = on ? w.u[k] : 0.f, w.delta[k] = on ? w.delta[k] : 0.f, w.dy[k] = on ? w.dy[k] : 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (st.works) s_in[buf][st.row][place16<S>(st.row, 4 * st.q + k)] = avsi_f4{w.delta[k], w.delta[k] * w.u[k], w.dy[k], 0.f};
        }
    };
    auto finish = [&](int n, const Held& w) {
        const int t0 = tile_at(n), buf = n & 1;
        constexpr int ROW = 2 * S::NP;
#pragma unroll
        for (int i0 = 0; i0 < TT * ROW; i0 += 2 * S::PT) {
            const int i = i0 + 2 * st.id, t = t0 + i / ROW;
            if (TT * ROW % (2 * S::PT) && i >= TT * ROW) break;
            avsi_f2 s = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < S::NW; ++k) s += *(const avsi_f2*)&s_bc[buf][k][i / ROW][i % ROW];
            if (t < at.live)
                *(avsi_f2*)(p.part_bc + ((((int64_t)at.b * p.T + t) * p.groups + at.g) * p.blocks + at.block) * ROW + i % ROW) = s;
        }
        const int t = t0 + st.row;
        if (t < at.end && st.works) {
            float du[4], ddt[4], dz[4], gB[4], gA[4], y[4];
            lane_sums<S>(s_gB[buf], st.row, st.q, gB);
            lane_sums<S>(s_gA[buf], st.row, st.q, gA);
            lane_sums<S>(s_y[buf], st.row, st.q, y);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                du[k] = fmaf(Dq[k], w.dy[k], w.delta[k] * gB[k]);
                ddt[k] = fmaf(w.u[k], gB[k], gA[k]) * w.slope[k];
                dz[k] = w.gz[k] * fmaf(Dq[k], w.u[k], y[k]);
                dD[k] = fmaf(w.dy[k], w.u[k], dD[k]);
            }
            if (t0 + TT > at.live)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (t >= at.live) du[k] = ddt[k] = dz[k] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) dbias[k] += ddt[k];
            put(t0, du, ddt, dz);
        }
    };
    // While the consumers are at tile n: tile n + 1 is staged, n - 1 finished (`w`: what is held of n - 1, then of n + 1).  The loads and
    // then the stores are issued in front of the arithmetic, and no branch lies between a load and its use: a wait behind one is for all
    // that is in flight.
    auto turn = [&](int n, Held& w) {
        take(n + 1);
        finish(n - 1, w);
        stage(n + 1, w);
        AVSI_LDS_BARRIER();
    };
    if (at.tiles) {
        load(0);
        take(0);
        stage(0, even);
    }
    AVSI_LDS_BARRIER();
    if (at.tiles > 1) {
        take(1);
        stage(1, odd);
        AVSI_LDS_BARRIER();
        for (int n = 1; n + 1 < at.tiles; n += 2) {
            turn(n, even);
            if (n + 2 >= at.tiles) break;
            turn(n + 1, odd);
        }
        Held before, last;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            before.u[k] = at.tiles % 2 ? odd.u[k] : even.u[k], last.u[k] = at.tiles % 2 ? even.u[k] : odd.u[k];
            before.delta[k] = at.tiles % 2 ? odd.delta[k] : even.delta[k], last.delta[k] = at.tiles % 2 ? even.delta[k] : odd.delta[k];
            before.slope[k] = at.tiles % 2 ? odd.slope[k] : even.slope[k], last.slope[k] = at.tiles % 2 ? even.slope[k] : odd.slope[k];
            before.dy[k] = at.tiles % 2 ? odd.dy[k] : even.dy[k], last.dy[k] = at.tiles % 2 ? even.dy[k] : odd.dy[k];
            before.gz[k] = at.tiles % 2 ? odd.gz[k] : even.gz[k], last.gz[k] = at.tiles % 2 ? even.gz[k] : odd.gz[k];
        }
        finish(at.tiles - 2, before);
        AVSI_LDS_BARRIER();
        finish(at.tiles - 1, last);
    } else if (at.tiles) {
        AVSI_LDS_BARRIER();
        finish(0, even);
    }
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    if (st.works)
        for (int t0 = at.begin + at.tiles * TT; t0 + st.row < at.end; t0 += TT) put(t0, zero, zero, zero);
    // D's and the bias' gradients of this workgroup's channels, over its chunk: the rows of the producers
    AVSI_LDS_BARRIER();
    if (st.works)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ((float*)s_gB[0][st.row])[4 * st.q + k] = dD[k];
            ((float*)s_gA[0][st.row])[4 * st.q + k] = dbias[k];
        }
    AVSI_LDS_BARRIER();
    if (st.id < at.n) {
        float sD = 0.f, sb = 0.f;
#pragma unroll
        for (int r = 0; r < TT; ++r) {
            sD += ((const float*)s_gB[0][r])[st.id];
            sb += ((const float*)s_gA[0][r])[st.id];
        }
        pw += (int64_t)p.dim * S::NP + at.d0 + st.id;
        pw[0] = sD;
        pw[p.dim] = sb;
    }
}

// dA [dim][N], dD, ddt_bias [dim] = sums over P partials of [dim][NP], [dim], [dim].
__global__ __launch_bounds__(1024) void scan_wgrad_sum_kernel(const float* __restrict__ part, int P, int dim, int NP, int N,
                                                              float* __restrict__ dA, float* __restrict__ dD, float* __restrict__ dbias) {
    avsi_column_sums(part, P, partial_stride(dim, NP), (int64_t)dim * (NP + 2), [&](int64_t c, float s) {
        if (c < (int64_t)dim * NP) {
            if (c % NP < N) dA[c / NP * N + c % NP] = s;
        } else if (c < (int64_t)dim * (NP + 1)) {
            if (dD) dD[c - (int64_t)dim * NP] = s;
        } else if (dbias) {
            dbias[c - (int64_t)dim * (NP + 1)] = s;
        }
    });
}

// dB, dC [batch][time][groups][N] = sums over the blocks of part_bc; zero behind a length.  A thread: four states of one of the two,
// the partials of eight blocks in flight.  `first`: where this launch begins (one has fewer than 2^32 threads).
template <typename T>
__global__ __launch_bounds__(256) void scan_bc_sum_kernel(Scan p, int NP, int64_t first, T* __restrict__ dB, T* __restrict__ dC) {
    const int Q = NP / 2;                   // quads of dB and dC of a token and group
    const int64_t id = first + (int64_t)blockIdx.x * 256 + threadIdx.x, tg = id / Q;
    if (tg >= (int64_t)p.batch * p.T * p.groups) return;
    const int q = (int)(id % Q), n = 4 * (q % (NP / 4)), t = (int)(tg / p.groups % p.T), b = (int)(tg / p.groups / p.T);
    if (n >= p.N) return;
    avsi_f4 s = {0.f, 0.f, 0.f, 0.f};
    if (t < length_of(p.lengths, b, p.T)) {
        const avsi_f4* at = (const avsi_f4*)p.part_bc + tg * p.blocks * Q + q;
        int k = 0;
        for (; k + 8 <= p.blocks; k += 8) {
            avsi_f4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = at[(int64_t)(k + i) * Q];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; k < p.blocks; ++k) s += at[(int64_t)k * Q];
    }
    const float f[4] = {s[0], s[1], s[2], s[3]};
    put_quad<T>((q < NP / 4 ? dB : dC) + tg * p.N + n, p.N - n, f);
}

// ---------------------------------------------------------------------------------------------------------- one token
// Bound by the states, read and written once (256 sequences of 2048 channels, N = 16: 16 us, 4.9 TB/s).  A lane: four states of one
// channel, over the sequences b, b + gridDim.y, ..., with the next sequence's operands in flight.  EL: states in no whole quads, one by
// one.
template <typename T, int LN, bool EL> __global__ __launch_bounds__(256) void scan_step_kernel(Scan p) {
    const int id = blockIdx.x * 256 + threadIdx.x, ql = id % LN, d = id / LN, n0 = 4 * ql, left = p.N - n0;
    if (d >= p.dim) return;                 // (whole groups of LN lanes leave)
    const int grp = d / (p.dim / p.groups), c0 = n0 < p.N - 4 ? n0 : (p.N < 4 ? 0 : p.N - 4);    // (lanes without states read the last four)
    float A[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) A[j] = j < left ? p.A[(int64_t)d * p.N + n0 + j] * LOG2E : 0.f;
    const float Dd = p.D ? p.D[d] : 0.f, bias = p.bias ? p.bias[d] : 0.f;
    avsi_quad<T> Bq, Cq;
    avsi_quad<float> hq;
    T u, dt, z;
    auto load = [&](int64_t b) {
        const T* Bp = (const T*)p.B + b * p.Bb + grp * p.Bg;
        const T* Cp = (const T*)p.C + b * p.Cb + grp * p.Cg;
        const float* st = p.state_out + (b * p.dim + d) * p.N;
        if (!EL) {
            hq.load(st + c0);
            Bq.load(Bp + c0);
            Cq.load(Cp + c0);
        } else {
            float f[4], g[4], h[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + j < p.N ? n0 + j : p.N - 1;
                f[j] = (float)Bp[n], g[j] = (float)Cp[n], h[j] = st[n];
            }
            Bq.set(f), Cq.set(g), hq.set(h);
        }
        u = ((const T*)p.u)[b * p.ub + d];
        dt = ((const T*)p.dt)[b * p.tb + d];
        z = ((const T*)p.z)[b * p.zb + d];
    };
    int64_t b = blockIdx.y;
    load(b);
    for (; b < p.batch; b += gridDim.y) {
        float Bv[4], Cv[4], h[4];
        Bq.get(Bv);
        Cq.get(Cv);
        hq.get(h);
        const float uf = (float)u, x = (float)dt + bias, zf = (float)z;
        load(b + gridDim.y < p.batch ? b + gridDim.y : b);       // (another sequence's states than those written below, or unused)
        const float delta = step_size(x, p.softplus), du = delta * uf;
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(__builtin_amdgcn_exp2f(delta * A[j]), h[j], du * Bv[j]);
            y += j < left ? h[j] * Cv[j] : 0.f;
        }
        put_quad<float>(p.state_out + (b * p.dim + d) * p.N + n0, left, h);
        y = avsi_group<LN>(y);
        if (ql == 0) {
            y = fmaf(Dd, uf, y);
            ((T*)p.out)[b * p.ob + d] = (T)(p.gated ? y * (zf * avsi_sigmoid<T>(zf)) : y);
        }
    }
}

// States with their padding: a power of two from 4 on; MAX_STATE where elements are loaded one by one (fewer than four channels,
// or states in no whole quads: one form of the kernels for all of those).
bool by_elements(const avsi_scan_args* a) { return a->dim < 4 || a->state % 4; }
int padded(const avsi_scan_args* a) {
    int n = by_elements(a) ? MAX_STATE : 4;
    while (n < a->state) n *= 2;
    return n;
}
int lanes_of(const avsi_scan_args* a) { return padded(a) / 4; }
int step_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }
int block_channels(int LN) { return LN <= 4 ? 64 : 256 / LN; }

// Chunks of time, of at least 64 steps: as many as give two workgroups to each CU and not one more; none where batch and channels leave
// one for three of four CUs -- the launch over the chunks costs three quarters of the main one.  (The forward kernel has room for two
// workgroups on a CU, so that none gets a third; the backward kernel's LDS, 151552 bytes at 16 states, has room for one, and its two take
// turns.) 2048 steps, N = 16, a whole forward / backward call in us: 2 sequences of 2048 channels (64 workgroups) 146 / 431 uncut, 67 /
// 158 in 8 chunks (85 / 204 in 6, 79 / 188 in 10); 4 (128) 147 / 439 uncut, 120 / 291 in 4; 6 (192) 152 / 445 uncut, 185 / 514 in 2, 175 /
// 428 in 4. Fewer states make smaller workgroups, but no more of them: 8191 steps of 1536 channels with 4 / 8 states in 21 chunks 75 / 217
// and 94 / 226; in as many as make the waves of 16 states, 85 and 42, 83 / 236 and 98 / 242.
void chunks_of(const avsi_scan_args* a, int* chunk, int* chunks) {
    const int64_t wgs = (int64_t)a->batch * a->groups * avsi_ceil_div(a->dim / a->groups, block_channels(lanes_of(a)));
    int64_t n = wgs >= 3 * AVSI_NUM_CU / 4 ? 1 : 2 * AVSI_NUM_CU / wgs;
    const int64_t most = avsi_ceil_div(a->time, 64);
    n = n < most ? n : most;
    *chunk = (int)avsi_round_up(avsi_ceil_div(a->time, n), TT);
    *chunks = (int)avsi_ceil_div(a->time, *chunk);
}

bool shape_ok(const avsi_scan_args* a) {
    return a && avsi_dtype_ok(a->dtype) && a->batch > 0 && a->batch <= 65535 && a->time > 0 && a->time <= (1 << 30) && a->dim > 0 &&
           a->dim <= (1 << 26) && a->state > 0 && a->groups > 0 && a->dim % a->groups == 0;
}

// The workgroups of a sequence, of 16 channels of a group or more and up to 512 threads, are one launch.
bool grid_ok(const avsi_scan_args* a) { return avsi_grid_ok(a->groups * avsi_ceil_div(a->dim / a->groups, 16), 512); }

// A tile's rows are addressed with 32 bits from its first one.  (A single step has no second row: any stride will do.)
bool strides_ok(const avsi_scan_args* a) {
    if (a->time == 1) return true;
    const int64_t most = (int64_t)1 << 26;
    for (int64_t s : {a->u_stride[1], a->dt_stride[1], a->z_stride[1], a->dout_stride[1], a->out_stride[1], a->B_stride[1], a->C_stride[1]})
        if (s < 0 || s > most) return false;
    return true;
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
    p.gated = a->z != nullptr;
    if (!p.gated) p.z = p.u, p.zb = p.ub, p.zt = p.ut;         // (read in its place, and not used)
    p.lengths = a->lengths, p.out = a->out, p.kept = a->kept, p.du = a->du, p.ddt = a->ddt, p.dz = a->dz;
    p.batch = a->batch, p.T = a->time, p.dim = a->dim, p.N = a->state, p.NP = padded(a), p.groups = a->groups, p.softplus = a->softplus;
    chunks_of(a, &p.chunk, &p.chunks);
    p.blocks = (int)avsi_ceil_div(a->dim / a->groups, block_channels(lanes_of(a)));
    return p;
}

size_t chunk_floats(const avsi_scan_args* a, int chunks) {
    return chunks < 2 ? 0 : (size_t)a->batch * chunks * a->dim * (padded(a) + 1);
}

template <bool BACK> void go_join(const Scan& p, hipStream_t s) {
    const int QB = p.NP / 4;
    hipLaunchKernelGGL(scan_join_kernel<BACK>, dim3(avsi_ceil_div((int64_t)p.batch * p.dim * QB, 256)), dim3(256), 0, s, p, QB);
}
template <typename T, typename S> void go_fwd(const Scan& p, hipStream_t s) {
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_chunk_kernel<T, S, false>), dim3(p.groups * p.blocks, p.chunks - 1, p.batch), dim3(S::NC + S::PT), 0, s, p);
        go_join<false>(p, s);
    }
    hipLaunchKernelGGL((scan_fwd_kernel<T, S>), dim3(p.groups * p.blocks, p.chunks, p.batch), dim3(S::NC + S::PT), 0, s, p);
}
template <typename T, typename S> void go_bwd(const Scan& p, hipStream_t s) {
    if (p.chunks > 1) {
        hipLaunchKernelGGL((scan_chunk_kernel<T, S, true>), dim3(p.groups * p.blocks, p.chunks - 1, p.batch), dim3(S::NC + S::PT), 0, s, p);
        go_join<true>(p, s);
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, S>), dim3(p.groups * p.blocks, p.chunks, p.batch), dim3(S::NC + S::PT), 0, s, p);
}
template <typename T, int LN> void go_step(const Scan& p, hipStream_t s) {
    // as many workgroups as stay on the chip (eight a CU), each over several sequences
    const int64_t along = avsi_ceil_div((int64_t)p.dim * LN, 256), most = avsi_ceil_div(8 * AVSI_NUM_CU, along);
    const dim3 grid(along, p.batch < most ? p.batch : most);
    if (p.N % 4) hipLaunchKernelGGL((scan_step_kernel<T, LN, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((scan_step_kernel<T, LN, false>), grid, dim3(256), 0, s, p);
}

}  // namespace

#define AVSI_SCAN_N(T, GO)                               \
    switch (by_elements(a) ? 0 : padded(a)) {            \
        case 0: GO<T, Shape<16, 4, true>>(p, s); break;  \
        case 4: GO<T, Shape<1, 4>>(p, s); break;         \
        case 8: GO<T, Shape<2, 4>>(p, s); break;         \
        case 16: GO<T, Shape<4, 4>>(p, s); break;        \
        case 32: GO<T, Shape<8, 4>>(p, s); break;        \
        default: GO<T, Shape<16, 4>>(p, s); break;       \
    }
#define AVSI_STEP_N(T, GO)               \
    switch (step_states(a->state)) { \
        case 4: GO<T, 1>(p, s); break;   \
        case 8: GO<T, 2>(p, s); break;   \
        case 16: GO<T, 4>(p, s); break;  \
        case 32: GO<T, 8>(p, s); break;  \
        default: GO<T, 16>(p, s); break; \
    }
#define AVSI_SCAN_T(BY_N, GO)                          \
    if (a->dtype == AVSI_F32) { BY_N(float, GO) }      \
    else if (a->dtype == AVSI_BF16) { BY_N(__bf16, GO) } \
    else { BY_N(_Float16, GO) }

extern "C" size_t avsi_selective_scan_kept_floats(const avsi_scan_args* a) {
    if (!shape_ok(a) || a->state > MAX_STATE) return 0;
    return (size_t)a->batch * avsi_ceil_div(a->time, TT) * a->dim * padded(a);
}

extern "C" size_t avsi_selective_scan_workspace_bytes(const avsi_scan_args* a) {
    if (!shape_ok(a) || a->state > MAX_STATE) return 0;
    int chunk, chunks;
    chunks_of(a, &chunk, &chunks);
    return chunk_floats(a, chunks) * sizeof(float);
}

extern "C" int avsi_selective_scan(const avsi_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!shape_ok(a) || !a->u || !a->dt || !a->A || !a->B || !a->C || !a->out) return AVSI_ERR_INVALID_ARG;
    if (a->state > MAX_STATE || !strides_ok(a) || !grid_ok(a)) return AVSI_ERR_UNSUPPORTED;
    const size_t need = avsi_selective_scan_workspace_bytes(a);
    if (need && (!workspace || workspace_bytes < need)) return AVSI_ERR_WORKSPACE;
    Scan p = params(a);
    p.ends = (float*)workspace;
    p.sums = p.ends ? p.ends + (size_t)p.batch * p.chunks * p.dim * p.NP : nullptr;
    hipStream_t s = (hipStream_t)stream;
    avsi_clear_error();
    AVSI_SCAN_T(AVSI_SCAN_N, go_fwd)
    return avsi_launch_status();
}

extern "C" size_t avsi_selective_scan_bwd_workspace_bytes(const avsi_scan_args* a) {
    if (!shape_ok(a) || a->state > MAX_STATE) return 0;
    const Scan p = params(a);
    const size_t NP = p.NP;
    return (chunk_floats(a, p.chunks) + (size_t)p.batch * p.T * p.groups * p.blocks * 2 * NP +
            (size_t)p.batch * p.chunks * partial_stride(p.dim, NP)) * sizeof(float);
}

extern "C" int avsi_selective_scan_bwd(const avsi_scan_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (!shape_ok(a) || !a->u || !a->dt || !a->A || !a->B || !a->C || !a->dout || !a->kept || !a->du || !a->ddt || !a->dA || !a->dB ||
        !a->dC || !a->z != !a->dz)
        return AVSI_ERR_INVALID_ARG;
    if (a->state > MAX_STATE || !strides_ok(a) || !grid_ok(a)) return AVSI_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < avsi_selective_scan_bwd_workspace_bytes(a)) return AVSI_ERR_WORKSPACE;
    Scan p = params(a);
    const int NP = p.NP;
    // (every part is a multiple of four floats but the sums of the chunks: they come last)
    p.part_bc = (float*)workspace;
    p.part_w = p.part_bc + (size_t)p.batch * p.T * p.groups * p.blocks * 2 * NP;
    p.ends = p.part_w + (size_t)p.batch * p.chunks * partial_stride(p.dim, NP);
    p.sums = p.ends + (size_t)p.batch * p.chunks * p.dim * NP;
    hipStream_t s = (hipStream_t)stream;
    avsi_clear_error();
    AVSI_SCAN_T(AVSI_SCAN_N, go_bwd)
    const int64_t bc = (int64_t)p.batch * p.T * p.groups * NP / 2, most = (int64_t)1 << 31;
    for (int64_t first = 0; first < bc; first += most) {
        const dim3 grid((unsigned)avsi_ceil_div(bc - first < most ? bc - first : most, 256));
        if (a->dtype == AVSI_F32)
            hipLaunchKernelGGL((scan_bc_sum_kernel<float>), grid, dim3(256), 0, s, p, NP, first, (float*)a->dB, (float*)a->dC);
        else if (a->dtype == AVSI_BF16)
            hipLaunchKernelGGL((scan_bc_sum_kernel<__bf16>), grid, dim3(256), 0, s, p, NP, first, (__bf16*)a->dB, (__bf16*)a->dC);
        else
            hipLaunchKernelGGL((scan_bc_sum_kernel<_Float16>), grid, dim3(256), 0, s, p, NP, first, (_Float16*)a->dB, (_Float16*)a->dC);
    }
    hipLaunchKernelGGL(scan_wgrad_sum_kernel, avsi_column_sum_grid((int64_t)p.dim * (NP + 2)), dim3(1024), 0, s, p.part_w,
                       p.batch * p.chunks, p.dim, NP, p.N, a->dA, a->dD, a->ddt_bias);
    return avsi_launch_status();
}

extern "C" int avsi_selective_scan_step(const avsi_scan_args* a, void* stream) {
    if (!shape_ok(a) || a->time != 1 || !a->u || !a->dt || !a->A || !a->B || !a->C || !a->out || !a->state_out) return AVSI_ERR_INVALID_ARG;
    if (a->state > MAX_STATE || !strides_ok(a)) return AVSI_ERR_UNSUPPORTED;
    Scan p = params(a);
    hipStream_t s = (hipStream_t)stream;
    avsi_clear_error();
    AVSI_SCAN_T(AVSI_STEP_N, go_step)
    return avsi_launch_status();
}
