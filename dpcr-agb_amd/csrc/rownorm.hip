// rownorm.hip — row norms (layer: centred, rms: not) around a residual block, fused with everything that touches the same rows
// (norm_ops.row_norm_act / row_norm_join):
//     zhat = (z - mean z) rstd            n = zhat w + b          f[p] = keep[p] gate[p] scale   (p: the row's plot)
//     u = r + f[p] n                      y = act(u)              h = norm(y) of the next block (optional)
// and backwards, from dy and dh, with everything recomputed from z and r (one row lives in registers, so a second look at it
// costs no traffic; nothing but z and r is kept by the forward pass):
//     dy += rstd2 (dh w2 - [mean] - yhat mean(dh w2 yhat))        du = dy act'(u)      dr = du
//     dz = rstd (g - [mean g] - zhat mean(g zhat)),  g = du f w
//     S0[p] = sum du, S1[p] = sum du zhat over the rows of plot p; every parameter gradient follows from these two:
//     dgate = keep scale (w S1 + b S0), dscale = sum_p keep gate (w S1 + b S0), dw = sum_p f S1, db = sum_p f S0.
// Bound: HBM.  Forward 3 N C e bytes (z, r, y; + h), backward 5 N C e (z, r, dy, dz, dr; + dh).
// A row belongs to G lanes (8 .. 64 of one wave, 256 for the widest rows) that hold V pieces of 16 bytes each where widths,
// strides and addresses allow, single channels otherwise; the next row is in flight while one is worked on.  A workgroup owns a
// contiguous run of rows and walks it plot segment by plot segment; each (run, plot) pair leaves ONE partial column sum in slot
// run + plot — both only grow along the rows, so the slots are distinct and runs + plots + 1 of them are enough — folded in slot
// order: no atomics, results repeat bit for bit.
// Measured: norm + GELU of 211000 x 64 fp32 21 us forward, 31 backward (5.2 TB/s both); RMS norm + ReLU of 61007 x 512 bf16 23
// and 36 (5.5, 5.3); join of 211000 x 256 bf16 78 and 111 (4.2, 4.9), folds 20; 50021 x 203 fp32, single channels, with the next
// norm 32 and 57 (5.1, 4.3).
// What a bf16 element may cost beside HBM is about 60 vector instructions (37 T lane-instructions/s against 1 T elements/s at 5
// to 6 bytes): hence the fused parameters f w and f b, the one exponential that value and slope of the GELU share, no compares.
#include "agb_common.h"
#include "../../include/agb_hip.h"      // struct agb_rownorm_call

#define RN_THREADS 256
#define RN_MAX_C 4096
#define RN_MAX_N 2000000000      // (a row number and a turn further still fit)
#define RN_MAX_B 10000000

struct RnArgs {
    const void *z, *r, *dy, *dh;
    void *y, *h, *dz, *dr;
    long long ldz, ldr, ldy, ldh, lddy, lddh, lddz, lddr;
    const float *w, *b, *gate, *keep, *scale, *w2, *b2;
    const int32_t* ptr;
    float* part;
    int n, C, B, rows;       // rows: rows of a workgroup's run
    float eps, eps2;
    int rms, act, next;
};

// ---- sum over the G lanes of a row (every lane gets it).  Up to 16 lanes by DPP (quad swaps, half-row and row mirrors: the
// partners hold equal sums by then), 32 and 64 by the half-wave swaps, 256 through LDS with two buffers in turn.
template <int CTRL>
__device__ __forceinline__ float rn_mov(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int G>
__device__ __forceinline__ float rn_sum(float v, float* red, int& turn) {
    v += rn_mov<0xB1>(v);
    v += rn_mov<0x4E>(v);
    v += rn_mov<0x141>(v);
    if (G > 8) v += rn_mov<0x140>(v);
    if (G > 16) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (G > 32) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (G > 64) {
        float* t = red + 4 * turn;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) t[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (t[0] + t[1]) + (t[2] + t[3]);
    }
    return v;
}

typedef unsigned rn_u32x4 __attribute__((ext_vector_type(4)));
// a piece of W channels as it lies in memory: 16 bytes (W = 4 fp32, 8 bf16) or one channel
template <typename T, int W>
struct RnPiece {
    rn_u32x4 raw;
    __device__ __forceinline__ void load(const T* p) { raw = *(const rn_u32x4*)p; }
    __device__ __forceinline__ void clear() { raw = rn_u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void get(float* v) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(raw[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[2 * e] = __uint_as_float(raw[e] << 16);
                v[2 * e + 1] = __uint_as_float(raw[e] & 0xFFFF0000u);
            }
        }
    }
    static __device__ __forceinline__ void put(T* p, const float* v) {
        rn_u32x4 q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = sizeof(T) == 4 ? __float_as_uint(v[e]) : agb_pack2_bf16(v[2 * e], v[2 * e + 1]);
        *(rn_u32x4*)p = q;
    }
};
template <typename T>
struct RnPiece<T, 1> {
    float raw;
    __device__ __forceinline__ void load(const T* p) { raw = ld1(p); }
    __device__ __forceinline__ void clear() { raw = 0.f; }
    __device__ __forceinline__ void get(float* v) const { *v = raw; }
    static __device__ __forceinline__ void put(T* p, const float* v) { st1(p, *v); }
};

// This lane's piece 0 of a group's row of a matrix, and a walk down the rows a turn apart; pieces behind the last channel, rows
// that are not there (`on` false) and absent matrices read as zeros and are not written.
template <typename T, int W, int G, int V>
struct RnRow {
    T* at;
    long long step;
    RnPiece<T, W> piece[V ? V : 1];
    __device__ __forceinline__ void start(const void* base, long long ld, int row, int lane, int groups) {
        at = base ? (T*)base + row * ld + lane * W : nullptr;
        step = groups * ld;
    }
    __device__ __forceinline__ void load(int lane, int C, bool on) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (on && at && (j * G + lane) * W < C) piece[j].load(at + j * G * W);
            else piece[j].clear();
        }
        at += at ? step : 0;
    }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int j = 0; j < V; ++j) piece[j].get(v + j * W);
    }
    template <int VP>
    __device__ __forceinline__ void put(int lane, int C, bool on, const float* v) {
        if (!at) return;
#pragma unroll
        for (int j = 0; j < VP; ++j)
            if (on && (j * G + lane) * W < C) RnPiece<T, W>::put(at + j * G * W, v + j * W);
        at += step;
    }
};
// a parameter vector's values: `other` where there is none, 0 behind the last channel.  No branch between the loads: all are in
// flight together (a load, a branch and a use at a time they were most of a short call's time).
struct __attribute__((packed, aligned(4))) RnFour {
    float v[4];
};
template <int W, int G, int V>
__device__ __forceinline__ void rn_vec(const float* p, int lane, int C, float other, float* v) {
#pragma unroll
    for (int i = 0; i < V * W; ++i) v[i] = other;
    if (p) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float* q = p + min((j * G + lane) * W, C - W);      // (W > 1: C is a multiple of W)
            if constexpr (W == 1) {
                v[j] = *q;
            } else {
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    const RnFour f = *(const RnFour*)(q + e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[j * W + e + i] = f.v[i];
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V * W; ++i) v[i] = ((i / W) * G + lane) * W < C ? v[i] : 0.f;
}

// x <- xhat in place, returns rstd; 0 for both where `on` is false.  there[j]: 1 for a piece of channels, 0 behind the last
// channel (where x is 0 and stays 0)
template <int W, int G, int V>
__device__ __forceinline__ float rn_normalise(float* x, const float* there, float inv, bool rms, float eps, bool on, float* red, int& turn) {
    if (!rms) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V * W; ++i) s += x[i];
        const float mean = rn_sum<G>(s, red, turn) * inv;
#pragma unroll
        for (int i = 0; i < V * W; ++i) x[i] = __builtin_fmaf(-mean, there[i / W], x[i]);
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V * W; ++i) q = __builtin_fmaf(x[i], x[i], q);
    float rstd = rsqrtf(__builtin_fmaf(rn_sum<G>(q, red, turn), inv, eps));
    rstd = on ? rstd : 0.f;
#pragma unroll
    for (int i = 0; i < V * W; ++i) x[i] *= rstd;
    return rstd;
}

// d <- rstd (d - [mean d] - xhat mean(d xhat))
template <int W, int G, int V>
__device__ __forceinline__ void rn_norm_grad(float* d, const float* xhat, float rstd, float inv, bool rms, float* red, int& turn) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < V * W; ++i) { s0 += d[i]; s1 = __builtin_fmaf(d[i], xhat[i], s1); }
    s1 = rn_sum<G>(s1, red, turn) * inv * rstd;
    s0 = rms ? 0.f : rn_sum<G>(s0, red, turn) * inv * rstd;
#pragma unroll
    for (int i = 0; i < V * W; ++i) d[i] = __builtin_fmaf(-xhat[i], s1, __builtin_fmaf(d[i], rstd, -s0));
}

// GELU u Phi(u) and its slope Phi(u) + u phi(u).  Phi(-|u|) = erfc(|u| / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (error of
// erf at most 1.5e-7), whose exponential is phi's: 20 instructions for both, where the library's erff and an exponential take 60.
__device__ __forceinline__ void rn_gelu(float u, float& y, float& slope) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.23164189f, __builtin_fabsf(u), 1.f));      // 0.3275911 / sqrt 2
    const float e = __builtin_amdgcn_exp2f(u * u * -0.72134752f);
    float p = __builtin_fmaf(t, 0.5307027145f, -0.7265760135f);
    p = __builtin_fmaf(t, p, 0.7107068705f);
    p = __builtin_fmaf(t, p, -0.142248368f);
    p = __builtin_fmaf(t, p, 0.127414796f);
    const float tail = p * t * e, cdf = u > 0.f ? 1.f - tail : tail;
    y = u * cdf;
    slope = __builtin_fmaf(u * 0.39894228f, e, cdf);
}

// how many of 0 .. n - 1 `holds` holds for, if for none behind one that it does not hold for; 64 looks at once, a 64th of what is
// left between them (whatever `holds` says: it ends, between 0 and n)
template <typename F>
__device__ __forceinline__ int rn_count(int n, F holds) {
    int from = 0, end = n;
    while (from < end) {
        const int apart = (end - from + 63) >> 6, i = from + apart * (int)(threadIdx.x & 63) + apart - 1;
        const int yes = __popcll(__ballot(i < end && holds(min(i, n - 1))));
        from += yes * apart;
        end = min(end, from + apart - 1);
    }
    return __builtin_amdgcn_readfirstlane(from);
}
// the plot of a row: how many of ptr[1 .. B] are <= row (B: behind the last plot)
__device__ __forceinline__ int rn_plot(const int32_t* ptr, int B, int row) {
    return rn_count(B, [&](int i) { return ptr[i + 1] <= row; });
}

// f w and f b with f = keep[p] gate[p] scale of plot p; 0 behind the last plot (such a row is handed on as act(r))
template <int W, int G, int V>
__device__ __forceinline__ void rn_factor(const RnArgs& a, int p, int lane, float* fw, float* fb) {
    const float k = !a.ptr ? 1.f : p >= a.B ? 0.f : a.keep ? a.keep[p] : 1.f;
    float scale[V * W], gate[V * W];
    rn_vec<W, G, V>(a.w, lane, a.C, 1.f, fw);
    rn_vec<W, G, V>(a.b, lane, a.C, 0.f, fb);
    rn_vec<W, G, V>(a.scale, lane, a.C, 1.f, scale);
    rn_vec<W, G, V>(a.gate && p < a.B ? a.gate + (size_t)p * a.C : nullptr, lane, a.C, 1.f, gate);
#pragma unroll
    for (int i = 0; i < V * W; ++i) {
        const float f = k * scale[i] * gate[i];
        fw[i] *= f;
        fb[i] *= f;
    }
}

// One kernel for both directions: a run of rows, plot segment by plot segment.
template <typename T, int W, int G, int V, bool BWD, bool NEXT>
__global__ __launch_bounds__(RN_THREADS) void k_rownorm(const RnArgs a) {
    constexpr int N = V * W, GROUPS = RN_THREADS / G;
    constexpr int SUMS = NEXT ? 4 : 2;
    typedef RnRow<T, W, G, V> Row;
    __shared__ float red[8];
    __shared__ float fold[(BWD && GROUPS > 1) ? RN_THREADS * N : 1];
    const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G;
    int turn = 0;
    const int first = blockIdx.x * a.rows;
    const int last = min(a.n, first + a.rows);
    const float inv = 1.f / (float)a.C;
    float there[V], w2[NEXT ? N : 1], b2[(NEXT && !BWD) ? N : 1];
#pragma unroll
    for (int j = 0; j < V; ++j) there[j] = (j * G + lane) * W < a.C ? 1.f : 0.f;
    if constexpr (NEXT) {
        rn_vec<W, G, V>(a.w2, lane, a.C, 1.f, w2);
        if constexpr (!BWD) rn_vec<W, G, V>(a.b2, lane, a.C, 0.f, b2);
    }
    int row0 = first;
    while (row0 < last) {
        const int p = a.ptr ? rn_plot(a.ptr, a.B, row0) : 0;
        const int end = a.ptr && p < a.B ? min(last, max(a.ptr[p + 1], row0 + 1)) : last;      // (it ends, whatever ptr holds)
        const bool live = !a.ptr || p < a.B;      // (rows behind the last plot: y = act(r), dz = 0 whatever z holds)
        float fw[N], fb[N], sums[BWD ? SUMS : 1][N];
        rn_factor<W, G, V>(a, p, lane, fw, fb);
        if constexpr (BWD) {
#pragma unroll
            for (int s = 0; s < SUMS; ++s)
#pragma unroll
                for (int i = 0; i < N; ++i) sums[s][i] = 0.f;
        }
        Row z, r, dy, dh;
        RnRow<T, W, G, 0> to1, to2;      // y and h, or dr and dz
        z.start(a.z, a.ldz, row0 + group, lane, GROUPS);
        r.start(a.r, a.ldr, row0 + group, lane, GROUPS);
        if constexpr (BWD) {
            dy.start(a.dy, a.lddy, row0 + group, lane, GROUPS);
            dh.start(a.dh, a.lddh, row0 + group, lane, GROUPS);
        }
        to1.start(BWD ? a.dr : a.y, BWD ? a.lddr : a.ldy, row0 + group, lane, GROUPS);
        to2.start(BWD ? a.dz : a.h, BWD ? a.lddz : a.ldh, row0 + group, lane, GROUPS);
        auto fetch = [&](int at) {
            const bool on = at + group < end;
            z.load(lane, a.C, on);
            r.load(lane, a.C, on);
            if constexpr (BWD) dy.load(lane, a.C, on);
            if constexpr (BWD && NEXT) dh.load(lane, a.C, on);
        };
        fetch(row0);
        for (int at = row0; at < end; at += GROUPS) {      // (every lane takes every turn: the sums need whole groups)
            const bool on = at + group < end;
            float x[N], u[N], g[BWD ? N : 1], h[(BWD && NEXT) ? N : 1];
            z.get(x);
            r.get(u);
            if constexpr (BWD) dy.get(g);
            if constexpr (BWD && NEXT) dh.get(h);
            if (at + GROUPS < end) fetch(at + GROUPS);
            const float rstd = rn_normalise<W, G, V>(x, there, inv, a.rms, a.eps, on, red, turn);
            if (!live) {
#pragma unroll
                for (int i = 0; i < N; ++i) x[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] = __builtin_fmaf(fw[i], x[i], u[i] + fb[i]);
            if constexpr (!BWD) {
                if (a.act == ACT_GELU) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        float slope;
                        rn_gelu(u[i], u[i], slope);
                    }
                } else if (a.act == ACT_RELU) {
#pragma unroll
                    for (int i = 0; i < N; ++i) u[i] = act_fwd(u[i], ACT_RELU);
                }
                to1.template put<V>(lane, a.C, on, u);
                if constexpr (NEXT) {
                    rn_normalise<W, G, V>(u, there, inv, a.rms, a.eps2, on, red, turn);
#pragma unroll
                    for (int i = 0; i < N; ++i) u[i] = __builtin_fmaf(u[i], w2[i], b2[i]);
                    to2.template put<V>(lane, a.C, on, u);
                }
            } else {
                float slope[N];
                if (a.act == ACT_GELU) {
#pragma unroll
                    for (int i = 0; i < N; ++i) rn_gelu(u[i], u[i], slope[i]);
                } else if (a.act == ACT_RELU) {
#pragma unroll
                    for (int i = 0; i < N; ++i) act_fwd_grad(u[i], ACT_RELU, &u[i], &slope[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) slope[i] = 1.f;
                }
                if constexpr (NEXT) {
                    const float rstd2 = rn_normalise<W, G, V>(u, there, inv, a.rms, a.eps2, on, red, turn);
                    float d[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        sums[2][i] += h[i];
                        sums[3][i] = __builtin_fmaf(h[i], u[i], sums[3][i]);
                        d[i] = h[i] * w2[i];
                    }
                    rn_norm_grad<W, G, V>(d, u, rstd2, inv, a.rms, red, turn);
#pragma unroll
                    for (int i = 0; i < N; ++i) g[i] += d[i];
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    g[i] *= slope[i];
                    sums[0][i] += g[i];
                    sums[1][i] = __builtin_fmaf(g[i], x[i], sums[1][i]);
                }
                to1.template put<V>(lane, a.C, on, g);
                if (a.dz) {
#pragma unroll
                    for (int i = 0; i < N; ++i) g[i] *= fw[i];
                    rn_norm_grad<W, G, V>(g, x, live ? rstd : 0.f, inv, a.rms, red, turn);
                    to2.template put<V>(lane, a.C, on, g);
                }
            }
        }
        if constexpr (BWD) {
            float* out = a.part + (size_t)(blockIdx.x + p) * SUMS * a.C;
#pragma unroll
            for (int s = 0; s < SUMS; ++s) {
                if constexpr (GROUPS == 1) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int c = ((i / W) * G + lane) * W + i % W;
                        if (c < a.C) out[(size_t)s * a.C + c] = sums[s][i];
                    }
                } else {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < N; ++i) fold[group * (G * N) + ((i / W) * G + lane) * W + i % W] = sums[s][i];
                    __syncthreads();
                    for (int c = threadIdx.x; c < a.C; c += RN_THREADS) {
                        float v = 0.f;
#pragma unroll
                        for (int q = 0; q < GROUPS; ++q) v += fold[q * (G * N) + c];
                        out[(size_t)s * a.C + c] = v;
                    }
                }
            }
            if constexpr (GROUPS > 1) __syncthreads();
        }
        row0 = end;
    }
}

// ---- folds of the partial column sums: 32 channels x 32 slots at a time, in slot order per lane, lanes in order.  Many runs are
// folded to blocks of 64 slots first, whose sums lie by the same rule at block + plot.
struct RnFold {
    const float *part, *w, *b, *gate, *keep, *scale;
    const int32_t* ptr;
    float *blocks, *plots, *dgate, *dw, *db, *dscale, *dw2, *db2;
    int n, C, B, rows, sums, runs;
};
// first and last (exclusive) slot of plot p (B: the rows behind the last plot)
__device__ __forceinline__ void rn_slots(const RnFold& a, int p, int& s0, int& s1) {
    s0 = 0;
    s1 = a.runs;
    if (a.ptr) {
        const int lo = p == 0 ? 0 : min(max(a.ptr[p], 0), a.n), hi = p == a.B ? a.n : min(max(a.ptr[p + 1], 0), a.n);
        s0 = lo / a.rows + p;
        s1 = hi > lo ? (hi - 1) / a.rows + p + 1 : s0;
    }
}

// up to four sums over the 32 rows of lanes at once: row k is left with sum k
typedef float RnFoldBox[4][32][33];
__device__ __forceinline__ float rn_fold32(const float* v, int sums, RnFoldBox& t) {
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
    __syncthreads();
    for (int i = 0; i < sums; ++i) t[i][k][c] = v[i];
    __syncthreads();
    float s = 0.f;
    if (k < sums) {
#pragma unroll
        for (int i = 0; i < 32; ++i) s += t[k][i][c];
    }
    return s;
}
// ... and row 0 with all of them
__device__ __forceinline__ void rn_fold32_all(float* v, int sums, RnFoldBox& t) {
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
    const float s = rn_fold32(v, sums, t);
    __syncthreads();
    if (k < sums) t[k][0][c] = s;
    __syncthreads();
    for (int i = 0; i < sums; ++i) v[i] = t[i][0][c];
}

__device__ __forceinline__ void rn_finish(const RnFold& a, int c, const float* s) {
    const float sc = a.scale ? a.scale[c] : 1.f;
    if (a.dw) a.dw[c] = sc * s[1];
    if (a.db) a.db[c] = sc * s[0];
    if (a.dscale) a.dscale[c] = (a.w ? a.w[c] : 1.f) * s[1] + (a.b ? a.b[c] : 0.f) * s[0];
    if (a.sums == 4) {
        if (a.db2) a.db2[c] = s[2];
        if (a.dw2) a.dw2[c] = s[3];
    }
}

// slots [64 x, 64 x + 64), plot by plot; 32 columns of blockIdx.y
__global__ __launch_bounds__(1024) void k_rownorm_fold_slots(const RnFold a) {
    __shared__ RnFoldBox t;
    const int c = blockIdx.y * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5, first = blockIdx.x * 64;
    int s0, s1;
    int p = !a.ptr ? 0 : rn_count(a.B + 1, [&](int i) {      // the first plot that ends behind `first`
        rn_slots(a, i, s0, s1);
        return s1 <= first;
    });
    int look0 = 0, look1 = 0;      // lane i: the slots of plot p + i (of every 64 plots, one look)
    for (int i = 0; p <= a.B; ++p, i = (i + 1) & 63) {
        if (i == 0) rn_slots(a, min(p + (int)(threadIdx.x & 63), a.B), look0, look1);
        s0 = __builtin_amdgcn_readlane(look0, i);
        s1 = __builtin_amdgcn_readlane(look1, i);
        if (s0 >= first + 64) return;
        s0 = max(s0, first);
        s1 = min(s1, first + 64);
        if (s0 >= s1) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (c < a.C)
            for (int s = s0 + k; s < s1; s += 32)
                for (int i = 0; i < a.sums; ++i) v[i] += a.part[((size_t)s * a.sums + i) * a.C + c];
        const float sum = rn_fold32(v, a.sums, t);
        if (k < a.sums && c < a.C) a.blocks[((size_t)(blockIdx.x + p) * a.sums + k) * a.C + c] = sum;
    }
}

// per plot (blockIdx.x; there may be more than the other grid axes take): the sum of its blocks, or slots -> plots[p][sums][C] and the gate's gradient; without plots straight to
// the parameter gradients
__global__ __launch_bounds__(1024) void k_rownorm_fold_plots(const RnFold a) {
    __shared__ RnFoldBox t;
    const int c = blockIdx.y * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5, p = blockIdx.x;
    int s0, s1;
    rn_slots(a, p, s0, s1);
    const float* from = a.part;
    const bool any = s1 > s0;
    if (a.blocks) {
        from = a.blocks;
        s1 = any ? (s1 - 1) / 64 + p + 1 : 0;
        s0 = any ? s0 / 64 + p : 0;
    }
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C)
        for (int s = s0 + k; s < s1; s += 32)
            for (int i = 0; i < a.sums; ++i) v[i] += from[((size_t)s * a.sums + i) * a.C + c];
    rn_fold32_all(v, a.sums, t);
    if (k || c >= a.C) return;
    if (!a.ptr) { rn_finish(a, c, v); return; }
    for (int i = 0; i < a.sums; ++i) a.plots[((size_t)p * a.sums + i) * a.C + c] = v[i];
    if (a.dgate && p < a.B)
        a.dgate[(size_t)p * a.C + c] = !any ? 0.f : (a.keep ? a.keep[p] : 1.f) * (a.scale ? a.scale[c] : 1.f) *
                                       ((a.w ? a.w[c] : 1.f) * v[1] + (a.b ? a.b[c] : 0.f) * v[0]);
}

__global__ __launch_bounds__(1024) void k_rownorm_fold(const RnFold a) {
    __shared__ RnFoldBox t;
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C)
        for (int p = k; p <= a.B; p += 32) {
            int s0, s1;
            rn_slots(a, p, s0, s1);
            if (s0 >= s1) continue;      // (no rows: whatever its factors are, an average over no rows among them)
            const float* s = a.plots + (size_t)p * a.sums * a.C + c;
            const float f = p == a.B ? 0.f : (a.keep ? a.keep[p] : 1.f) * (a.gate ? a.gate[(size_t)p * a.C + c] : 1.f);
            if (p < a.B) { v[0] += f * s[0]; v[1] += f * s[a.C]; }
            if (a.sums == 4) { v[2] += s[2 * (size_t)a.C]; v[3] += s[3 * (size_t)a.C]; }
        }
    rn_fold32_all(v, a.sums, t);
    if (k == 0 && c < a.C) rn_finish(a, c, v);
}

// ---- host side
// lanes a row gets and pieces a lane: as few lanes as hold the row with one piece each (more rows in flight, shorter sums), then
// 16 channels a lane of a whole wave, then the whole workgroup
template <bool BWD, bool NEXT, typename T, int W>
static void rn_launch(const RnArgs& a, int runs, hipStream_t st) {
#define RN_GO(G, V)                                                                                         \
    do {                                                                                                    \
        hipLaunchKernelGGL((k_rownorm<T, W, G, V, BWD, NEXT>), dim3(runs), dim3(RN_THREADS), 0, st, a);      \
        return;                                                                                             \
    } while (0)
    const int pieces = agb_cdiv(a.C, W);
    if (pieces <= 8) RN_GO(8, 1);
    if (pieces <= 16) RN_GO(16, 1);
    if (pieces <= 32) RN_GO(32, 1);
    if (pieces <= 64) RN_GO(64, 1);
    if (pieces <= 128) RN_GO(64, 2);
    if constexpr (W == 1) {
        if (pieces <= 256) RN_GO(64, 4);
        if (pieces <= 512) RN_GO(64, 8);
        if (pieces <= 1024) RN_GO(256, 4);
        if (pieces <= 2048) RN_GO(256, 8);
        RN_GO(256, 16);
    } else if constexpr (W == 4) {
        if (pieces <= 256) RN_GO(64, 4);
        if (pieces <= 512) RN_GO(256, 2);
        RN_GO(256, 4);
    } else {
        if (pieces <= 256) RN_GO(256, 1);
        RN_GO(256, 2);
    }
#undef RN_GO
}

// rows that a workgroup takes at once (the fewest over the layouts above: what a run is cut by does not depend on alignment)
static int rn_groups(int C) {
    const int lanes = agb_cdiv(C, 8);
    return lanes <= 8 ? 32 : lanes <= 16 ? 16 : lanes <= 32 ? 8 : 4;
}

// rows of a run: at most RN_RUNS runs, whole turns
#define RN_RUNS 2048
static int rn_rows(int n, int C) {
    const int groups = rn_groups(C);
    return agb_cdiv(agb_cdiv(n > 0 ? n : 1, RN_RUNS), groups) * groups;
}
// (measured, 211000 x 64: 2048 slots folded at once 43 us, by blocks 5)
static int rn_blocks(int runs, int B) { return runs > 128 ? agb_cdiv((long long)runs + B + 1, 64) : 0; }

template <typename T>
static bool rn_vec_ok(const RnArgs& a) {
    const int W = 16 / (int)sizeof(T);
    if (a.C % W) return false;
    const void* p[] = {a.z, a.r, a.dy, a.dh, a.y, a.h, a.dz, a.dr};
    const long long ld[] = {a.ldz, a.ldr, a.lddy, a.lddh, a.ldy, a.ldh, a.lddz, a.lddr};
    for (int i = 0; i < 8; ++i)
        if (p[i] && ((uintptr_t)p[i] % 16 || ld[i] % W)) return false;
    return true;
}

template <typename T>
static int rn_run(const RnArgs& a, bool bwd, hipStream_t st) {
    const int runs = agb_cdiv(a.n, a.rows);
    const bool vec = rn_vec_ok<T>(a);
    constexpr int W = 16 / sizeof(T);
#define RN_DIR(BWD, NEXT)                                       \
    do {                                                        \
        if (vec) rn_launch<BWD, NEXT, T, W>(a, runs, st);       \
        else rn_launch<BWD, NEXT, T, 1>(a, runs, st);           \
    } while (0)
    if (bwd) {
        if (a.next) RN_DIR(true, true);
        else RN_DIR(true, false);
    } else {
        if (a.next) RN_DIR(false, true);
        else RN_DIR(false, false);
    }
#undef RN_DIR
    AGB_CHECK_LAUNCH(bwd ? "agb_rownorm_bwd" : "agb_rownorm_fwd");
    return AGB_OK;
}

static int rn_check(const char* name, int n, int C, int B, const int32_t* ptr, const float* gate, const float* keep, int rms,
                    int act, int bf16) {
    AGB_CHECK_ARG(n >= 0 && n <= RN_MAX_N && C >= 1 && C <= RN_MAX_C, "%s: bad shape n=%d C=%d (n <= %d, C <= %d)", name, n, C,
                  RN_MAX_N, RN_MAX_C);
    AGB_CHECK_ARG(!ptr || B <= RN_MAX_B, "%s: %d plots (up to %d)", name, B, RN_MAX_B);
    AGB_CHECK_ARG(act >= ACT_NONE && act <= ACT_GELU, "%s: act %d", name, act);
    AGB_CHECK_ARG((rms == 0 || rms == 1) && (bf16 == 0 || bf16 == 1), "%s: rms and bf16 are 0 or 1", name);
    AGB_CHECK_ARG(ptr ? B >= 1 : (!gate && !keep), "%s: a gate or a keep factor needs the plots' row ranges", name);
    return AGB_OK;
}

extern "C" {

int agb_rownorm_fwd(const void* Z, long long ldz, const void* R, long long ldr, int n, int C, const float* w, const float* b,
                    float eps, int rms, int act, const float* gate, const float* keep, const int32_t* ptr, int B,
                    const float* scale, const float* w2, const float* b2, float eps2, void* Y, long long ldy, void* H,
                    long long ldh, int bf16, void* stream) {
    if (int rc = rn_check("agb_rownorm_fwd", n, C, B, ptr, gate, keep, rms, act, bf16)) return rc;
    if (n == 0) return AGB_OK;
    AGB_CHECK_ARG(Z && (Y || H), "agb_rownorm_fwd: null pointer");
    AGB_CHECK_ARG(ldz >= C && (!R || ldr >= C) && (!Y || ldy >= C) && (!H || ldh >= C),
                  "agb_rownorm_fwd: a row stride is less than C=%d", C);
    RnArgs a = {};
    a.z = Z; a.ldz = ldz; a.r = R; a.ldr = ldr; a.y = Y; a.ldy = ldy; a.h = H; a.ldh = ldh;
    a.n = n; a.C = C; a.B = ptr ? B : 1; a.w = w; a.b = b; a.eps = eps; a.rms = rms; a.act = act;
    a.gate = gate; a.keep = keep; a.ptr = ptr; a.scale = scale;
    a.w2 = w2; a.b2 = b2; a.eps2 = eps2; a.next = H != nullptr;
    a.rows = rn_rows(n, C);
    return bf16 ? rn_run<bf16_t>(a, false, (hipStream_t)stream) : rn_run<float>(a, false, (hipStream_t)stream);
}

size_t agb_rownorm_bwd_workspace_bytes(int n, int C, int B, int next) {
    if (n < 0 || n > RN_MAX_N || C < 1 || C > RN_MAX_C || B < 0 || B > RN_MAX_B) return 0;
    const int runs = agb_cdiv(n, rn_rows(n, C)), blocks = rn_blocks(runs, B);
    const size_t slots = (size_t)runs + B + 1, more = blocks ? (size_t)blocks + B + 1 : 0;
    return (slots + more + B + 1) * (next ? 4 : 2) * (size_t)C * sizeof(float);
}

int agb_rownorm_bwd(const void* Z, long long ldz, const void* R, long long ldr, const void* dY, long long lddy, const void* dH,
                    long long lddh, int n, int C, const float* w, const float* b, float eps, int rms, int act,
                    const float* gate, const float* keep, const int32_t* ptr, int B, const float* scale, const float* w2,
                    const float* b2, float eps2, void* dZ, long long lddz, void* dR, long long lddr, float* dw, float* db,
                    float* dgate, float* dscale, float* dw2, float* db2, void* workspace, size_t workspace_bytes, int bf16,
                    void* stream) {
    if (int rc = rn_check("agb_rownorm_bwd", n, C, B, ptr, gate, keep, rms, act, bf16)) return rc;
    AGB_CHECK_ARG(ldz >= C && (!R || ldr >= C) && (!dY || lddy >= C) && (!dH || lddh >= C) && (!dZ || lddz >= C) &&
                      (!dR || lddr >= C),
                  "agb_rownorm_bwd: a row stride is less than C=%d", C);
    AGB_CHECK_ARG(n == 0 || (Z && (dY || dH)), "agb_rownorm_bwd: null pointer");
    AGB_CHECK_ARG(!dgate || gate, "agb_rownorm_bwd: a gradient of a gate that is not there");
    AGB_CHECK_ARG(n == 0 || dH || (!dw2 && !db2), "agb_rownorm_bwd: gradients of the next norm without its incoming gradient");
    const bool next = dH || dw2 || db2;      // (without rows an incoming gradient has no address)
    const size_t need = agb_rownorm_bwd_workspace_bytes(n, C, ptr ? B : 0, next);
    AGB_CHECK_ARG(workspace && workspace_bytes >= need, "agb_rownorm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
                  need);
    hipStream_t st = (hipStream_t)stream;
    RnArgs a = {};
    a.z = Z; a.ldz = ldz; a.r = R; a.ldr = ldr; a.dy = dY; a.lddy = lddy; a.dh = dH; a.lddh = lddh;
    a.dz = dZ; a.lddz = lddz; a.dr = dR; a.lddr = lddr;
    a.n = n; a.C = C; a.B = ptr ? B : 1; a.w = w; a.b = b; a.eps = eps; a.rms = rms; a.act = act;
    a.gate = gate; a.keep = keep; a.ptr = ptr; a.scale = scale;
    a.w2 = w2; a.b2 = b2; a.eps2 = eps2; a.next = next;
    a.part = (float*)workspace;
    a.rows = rn_rows(n, C);
    if (n > 0) {
        const int rc = bf16 ? rn_run<bf16_t>(a, true, st) : rn_run<float>(a, true, st);
        if (rc != AGB_OK) return rc;
    }
    if (!(dw || db || dgate || dscale || dw2 || db2)) return AGB_OK;
    RnFold f = {};
    f.part = a.part; f.w = w; f.b = b; f.gate = gate; f.keep = keep; f.scale = scale; f.ptr = ptr;
    f.n = n; f.C = C; f.B = ptr ? B : 0; f.rows = a.rows; f.sums = a.next ? 4 : 2; f.runs = agb_cdiv(n, a.rows);
    const int blocks = rn_blocks(f.runs, f.B);
    f.plots = a.part + ((size_t)f.runs + f.B + 1) * f.sums * C;
    if (blocks) {
        f.blocks = f.plots;
        f.plots = f.blocks + ((size_t)blocks + f.B + 1) * f.sums * C;
    }
    f.dw = dw; f.db = db; f.dgate = dgate; f.dscale = dscale; f.dw2 = dw2; f.db2 = db2;
    if (blocks) {
        hipLaunchKernelGGL(k_rownorm_fold_slots, dim3(blocks, agb_cdiv(C, 32)), dim3(1024), 0, st, f);
        AGB_CHECK_LAUNCH("agb_rownorm_fold_slots");
    }
    hipLaunchKernelGGL(k_rownorm_fold_plots, dim3(ptr ? B + 1 : 1, agb_cdiv(C, 32)), dim3(1024), 0, st, f);
    AGB_CHECK_LAUNCH("agb_rownorm_fold_plots");
    if (ptr && (dw || db || dscale || dw2 || db2)) {
        hipLaunchKernelGGL(k_rownorm_fold, dim3(agb_cdiv(C, 32)), dim3(1024), 0, st, f);
        AGB_CHECK_LAUNCH("agb_rownorm_fold");
    }
    return AGB_OK;
}

static int rn_check_call(const char* name, const agb_rownorm_call* c) {
    AGB_CHECK_ARG(c, "%s: null pointer", name);
    AGB_CHECK_ARG(c->n >= 0 && c->n <= RN_MAX_N && c->C >= 1 && c->C <= RN_MAX_C && c->B >= 0 && c->B <= RN_MAX_B,
                  "%s: bad shape n=%lld C=%lld B=%lld", name, c->n, c->C, c->B);
    AGB_CHECK_ARG((c->rms | c->bf16) >= 0 && (c->rms | c->bf16) <= 1 && c->act >= 0 && c->act <= ACT_GELU, "%s: rms, act or bf16",
                  name);
    return AGB_OK;
}

int agb_rownorm_fwd_call(const agb_rownorm_call* c, void* stream) {
    if (int rc = rn_check_call("agb_rownorm_fwd", c)) return rc;
    return agb_rownorm_fwd(c->Z, c->ldz, c->R, c->ldr, (int)c->n, (int)c->C, c->w, c->b, (float)c->eps, (int)c->rms, (int)c->act,
                           c->gate, c->keep, c->ptr, (int)c->B, c->scale, c->w2, c->b2, (float)c->eps2, c->Y, c->ldy, c->H, c->ldh,
                           (int)c->bf16, stream);
}

int agb_rownorm_bwd_call(const agb_rownorm_call* c, void* stream) {
    if (int rc = rn_check_call("agb_rownorm_bwd", c)) return rc;
    return agb_rownorm_bwd(c->Z, c->ldz, c->R, c->ldr, c->dY, c->lddy, c->dH, c->lddh, (int)c->n, (int)c->C, c->w, c->b,
                           (float)c->eps, (int)c->rms, (int)c->act, c->gate, c->keep, c->ptr, (int)c->B, c->scale, c->w2, c->b2,
                           (float)c->eps2, c->dZ, c->lddz, c->dR, c->lddr, c->dw, c->db, c->dgate, c->dscale, c->dw2, c->db2,
                           c->workspace, c->workspace_bytes, (int)c->bf16, stream);
}

}  // extern "C"
