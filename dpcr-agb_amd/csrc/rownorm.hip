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
// A row belongs to G lanes (8 .. 64 of one wave, 256 for the widest rows) that hold V pieces of W channels each: W = 4 where
// widths, strides and addresses allow 4-channel accesses, else 1.  A workgroup owns a contiguous run of rows and walks it plot
// segment by plot segment; each (run, plot) pair leaves ONE partial column sum in slot run + plot — both only grow along the
// rows, so the slots are distinct and runs + plots + 1 of them are enough — folded in slot order: no atomics, results repeat
// bit for bit.
#include "agb_common.h"

#define RN_THREADS 256
#define RN_MAX_C 4096

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

template <typename T, int W>
__device__ __forceinline__ void rn_load(const T* p, float* v) {
    if constexpr (W == 4) {
        const float4 q = ld4(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        v[0] = ld1(p);
    }
}
template <typename T, int W>
__device__ __forceinline__ void rn_store(T* p, const float* v) {
    if constexpr (W == 4) st4(p, make_float4(v[0], v[1], v[2], v[3]));
    else st1(p, v[0]);
}

// a row's pieces (0 behind the last channel or where `on` is false); parameters: `other` where there is no vector
template <typename T, int W, int G, int V>
__device__ __forceinline__ void rn_row(const void* base, long long ld, long long row, int lane, int C, bool on, float* v) {
    const T* p = (const T*)base + row * ld;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (j * G + lane) * W;
        if (on && c < C) {
            rn_load<T, W>(p + c, v + j * W);
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) v[j * W + e] = 0.f;
        }
    }
}
template <typename T, int W, int G, int V>
__device__ __forceinline__ void rn_put(void* base, long long ld, long long row, int lane, int C, bool on, const float* v) {
    T* p = (T*)base + row * ld;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = (j * G + lane) * W;
        if (on && c < C) rn_store<T, W>(p + c, v + j * W);
    }
}
template <int W, int G, int V>
__device__ __forceinline__ void rn_vec(const float* p, int lane, int C, float other, float* v) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const int c = (j * G + lane) * W + e;
            v[j * W + e] = c < C ? (p ? p[c] : other) : 0.f;
        }
}

// x <- xhat in place (0 behind the last channel: the sums below run over every piece), returns rstd
template <int W, int G, int V>
__device__ __forceinline__ float rn_normalise(float* x, int lane, int C, bool rms, float eps, float* red, int& turn) {
    const float inv = 1.f / (float)C;
    float mean = 0.f;
    if (!rms) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V * W; ++i) s += x[i];
        mean = rn_sum<G>(s, red, turn) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V * W; ++i) {
        const int c = ((i / W) * G + lane) * W + i % W;
        x[i] = c < C ? x[i] - mean : 0.f;
        q += x[i] * x[i];
    }
    const float rstd = 1.f / sqrtf(rn_sum<G>(q, red, turn) * inv + eps);
#pragma unroll
    for (int i = 0; i < V * W; ++i) x[i] *= rstd;
    return rstd;
}

// d <- rstd (d - [mean d] - xhat mean(d xhat))
template <int W, int G, int V>
__device__ __forceinline__ void rn_norm_grad(float* d, const float* xhat, float rstd, int C, bool rms, float* red, int& turn) {
    const float inv = 1.f / (float)C;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < V * W; ++i) { s0 += d[i]; s1 += d[i] * xhat[i]; }
    s1 = rn_sum<G>(s1, red, turn) * inv;
    s0 = rms ? 0.f : rn_sum<G>(s0, red, turn) * inv;
#pragma unroll
    for (int i = 0; i < V * W; ++i) d[i] = rstd * (d[i] - s0 - xhat[i] * s1);
}

// the plot of a row: how many of ptr[1 .. B] are <= row (B: behind the last plot)
__device__ __forceinline__ int rn_plot(const int32_t* ptr, int B, int row) {
    int lo = 0, hi = B;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ptr[mid + 1] <= row) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// keep[p] gate[p] scale of plot p; 0 behind the last plot (such a row is handed on as act(r))
template <int W, int G, int V>
__device__ __forceinline__ void rn_factor(const RnArgs& a, int p, int lane, float* f) {
    rn_vec<W, G, V>(a.scale, lane, a.C, 1.f, f);
    if (!a.ptr) return;
    const float k = p >= a.B ? 0.f : a.keep ? a.keep[p] : 1.f;
#pragma unroll
    for (int i = 0; i < V * W; ++i) {
        const int c = ((i / W) * G + lane) * W + i % W;
        const float g = (a.gate && p < a.B && c < a.C) ? a.gate[(size_t)p * a.C + c] : 1.f;
        f[i] *= k * g;
    }
}

// One kernel for both directions: a run of rows, plot segment by plot segment.
template <typename T, int W, int G, int V, bool BWD, bool NEXT>
__global__ __launch_bounds__(RN_THREADS) void k_rownorm(const RnArgs a) {
    constexpr int N = V * W, GROUPS = RN_THREADS / G;
    constexpr int SUMS = NEXT ? 4 : 2;
    __shared__ float red[8];
    __shared__ float fold[(BWD && GROUPS > 1) ? RN_THREADS * N : 1];
    const int lane = threadIdx.x & (G - 1), group = threadIdx.x / G;
    int turn = 0;
    const int first = blockIdx.x * a.rows;
    const int last = min(a.n, first + a.rows);
    float w[N], b[N], w2[NEXT ? N : 1], b2[NEXT ? N : 1];
    rn_vec<W, G, V>(a.w, lane, a.C, 1.f, w);
    rn_vec<W, G, V>(a.b, lane, a.C, 0.f, b);
    if constexpr (NEXT) {
        rn_vec<W, G, V>(a.w2, lane, a.C, 1.f, w2);
        rn_vec<W, G, V>(a.b2, lane, a.C, 0.f, b2);
    }
    int row0 = first;
    int p = a.ptr ? rn_plot(a.ptr, a.B, first) : 0;
    while (row0 < last) {
        int end = last;
        if (a.ptr) {
            while (p < a.B && a.ptr[p + 1] <= row0) ++p;
            if (p < a.B) end = min(last, a.ptr[p + 1]);
        }
        const bool live = !a.ptr || p < a.B;      // (rows behind the last plot: y = act(r), dz = 0 whatever z holds)
        float f[N], sums[BWD ? SUMS : 1][N];
        rn_factor<W, G, V>(a, p, lane, f);
        if constexpr (BWD) {
#pragma unroll
            for (int s = 0; s < SUMS; ++s)
#pragma unroll
                for (int i = 0; i < N; ++i) sums[s][i] = 0.f;
        }
        for (int at = row0; at < end; at += GROUPS) {      // (every lane takes every turn: the sums need whole groups)
            const long long row = at + group;
            const bool on = row < end;
            float x[N], u[N];
            rn_row<T, W, G, V>(a.z, a.ldz, row, lane, a.C, on, x);
            if (a.r) rn_row<T, W, G, V>(a.r, a.ldr, row, lane, a.C, on, u);
            else {
#pragma unroll
                for (int i = 0; i < N; ++i) u[i] = 0.f;
            }
            float dy[BWD ? N : 1], dh[(BWD && NEXT) ? N : 1];
            if constexpr (BWD) {
                if (a.dy) rn_row<T, W, G, V>(a.dy, a.lddy, row, lane, a.C, on, dy);
                else {
#pragma unroll
                    for (int i = 0; i < N; ++i) dy[i] = 0.f;
                }
                if constexpr (NEXT) rn_row<T, W, G, V>(a.dh, a.lddh, row, lane, a.C, on, dh);
            }
            const float rstd = rn_normalise<W, G, V>(x, lane, a.C, a.rms, a.eps, red, turn);
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] = live ? u[i] + f[i] * (x[i] * w[i] + b[i]) : u[i];
            if constexpr (!BWD) {
#pragma unroll
                for (int i = 0; i < N; ++i) u[i] = act_fwd(u[i], a.act);
                if (a.y) rn_put<T, W, G, V>(a.y, a.ldy, row, lane, a.C, on, u);
                if constexpr (NEXT) {
                    rn_normalise<W, G, V>(u, lane, a.C, a.rms, a.eps2, red, turn);
#pragma unroll
                    for (int i = 0; i < N; ++i) u[i] = u[i] * w2[i] + b2[i];
                    rn_put<T, W, G, V>(a.h, a.ldh, row, lane, a.C, on, u);
                }
            } else {
                float slope[N];
#pragma unroll
                for (int i = 0; i < N; ++i) act_fwd_grad(u[i], a.act, &u[i], &slope[i]);
                if constexpr (NEXT) {
                    const float rstd2 = rn_normalise<W, G, V>(u, lane, a.C, a.rms, a.eps2, red, turn);
                    float d[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        sums[2][i] += dh[i];
                        sums[3][i] += on ? dh[i] * u[i] : 0.f;
                        d[i] = dh[i] * w2[i];
                    }
                    rn_norm_grad<W, G, V>(d, u, rstd2, a.C, a.rms, red, turn);
#pragma unroll
                    for (int i = 0; i < N; ++i) dy[i] += d[i];
                }
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    dy[i] *= slope[i];
                    sums[0][i] += on ? dy[i] : 0.f;
                    sums[1][i] += on ? dy[i] * x[i] : 0.f;
                }
                if (a.dr) rn_put<T, W, G, V>(a.dr, a.lddr, row, lane, a.C, on, dy);
                if (a.dz) {
#pragma unroll
                    for (int i = 0; i < N; ++i) dy[i] *= f[i] * w[i];
                    rn_norm_grad<W, G, V>(dy, x, rstd, a.C, a.rms, red, turn);
#pragma unroll
                    for (int i = 0; i < N; ++i) dy[i] = live ? dy[i] : 0.f;
                    rn_put<T, W, G, V>(a.dz, a.lddz, row, lane, a.C, on, dy);
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
                        for (int g = 0; g < GROUPS; ++g) v += fold[g * (G * N) + c];
                        out[(size_t)s * a.C + c] = v;
                    }
                }
            }
            if constexpr (GROUPS > 1) __syncthreads();
        }
        row0 = end;
    }
}

// ---- folds of the partial column sums: 32 channels x 32 slots at a time, in slot order per lane, lanes in order.
struct RnFold {
    const float *part, *w, *b, *gate, *keep, *scale;
    const int32_t* ptr;
    float *plots, *dgate, *dw, *db, *dscale, *dw2, *db2;
    int n, C, B, rows, sums, runs;
};

__device__ __forceinline__ float rn_fold32(float v, float (*t)[33]) {
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
    __syncthreads();
    t[k][c] = v;
    __syncthreads();
    float s = 0.f;
    if (k == 0)
        for (int i = 0; i < 32; ++i) s += t[i][c];
    return s;          // (lane k == 0)
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

// per plot (blockIdx.y; B: the rows behind the last plot): the sum of its slots -> plots[p][sums][C] and the gate's gradient;
// without plots straight to the parameter gradients
__global__ __launch_bounds__(1024) void k_rownorm_fold_plots(const RnFold a) {
    __shared__ float t[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5, p = blockIdx.y;
    int s0 = 0, s1 = a.runs;
    if (a.ptr) {
        const int lo = p == 0 ? 0 : min(max(a.ptr[p], 0), a.n), hi = p == a.B ? a.n : min(max(a.ptr[p + 1], 0), a.n);
        s0 = lo / a.rows + p;
        s1 = hi > lo ? (hi - 1) / a.rows + p + 1 : s0;
    }
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C)
        for (int s = s0 + k; s < s1; s += 32)
            for (int i = 0; i < a.sums; ++i) v[i] += a.part[((size_t)s * a.sums + i) * a.C + c];
    for (int i = 0; i < a.sums; ++i) v[i] = rn_fold32(v[i], t);
    if (k || c >= a.C) return;
    if (!a.ptr) { rn_finish(a, c, v); return; }
    for (int i = 0; i < a.sums; ++i) a.plots[((size_t)p * a.sums + i) * a.C + c] = v[i];
    if (a.dgate && p < a.B)
        a.dgate[(size_t)p * a.C + c] = (a.keep ? a.keep[p] : 1.f) * (a.scale ? a.scale[c] : 1.f) *
                                       ((a.w ? a.w[c] : 1.f) * v[1] + (a.b ? a.b[c] : 0.f) * v[0]);
}

__global__ __launch_bounds__(1024) void k_rownorm_fold(const RnFold a) {
    __shared__ float t[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C)
        for (int p = k; p <= a.B; p += 32) {
            const float* s = a.plots + (size_t)p * a.sums * a.C + c;
            const float f = p == a.B ? 0.f : (a.keep ? a.keep[p] : 1.f) * (a.gate ? a.gate[(size_t)p * a.C + c] : 1.f);
            if (p < a.B) { v[0] += f * s[0]; v[1] += f * s[a.C]; }
            if (a.sums == 4) { v[2] += s[2 * (size_t)a.C]; v[3] += s[3 * (size_t)a.C]; }
        }
    for (int i = 0; i < a.sums; ++i) v[i] = rn_fold32(v[i], t);
    if (k == 0 && c < a.C) rn_finish(a, c, v);
}

// ---- host side
// lanes a row gets and pieces a lane: as few lanes as hold the row with one piece each (more rows in flight, shorter sums), up
// to four pieces of a whole wave, then the whole workgroup
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
    if (pieces <= 256) RN_GO(64, 4);
    if constexpr (W == 1) {
        if (pieces <= 512) RN_GO(64, 8);
        if (pieces <= 1024) RN_GO(256, 4);
        if (pieces <= 2048) RN_GO(256, 8);
        RN_GO(256, 16);
    } else {
        if (pieces <= 512) RN_GO(256, 2);
        RN_GO(256, 4);
    }
#undef RN_GO
}

static int rn_groups(int C, bool vec) {
    const int pieces = vec ? agb_cdiv(C, 4) : C;
    if (pieces <= 8) return 32;
    if (pieces <= 16) return 16;
    if (pieces <= 32) return 8;
    if (pieces <= (vec ? 256 : 512)) return 4;
    return 1;
}

// rows of a run: at least four turns of the workgroup's groups, at most RN_RUNS runs
#define RN_RUNS 2048
static int rn_rows(int n, int C) {
    const int least = 4 * rn_groups(C, C % 4 == 0), even = agb_cdiv(n, RN_RUNS);
    return even > least ? even : least;
}

static bool rn_vec_ok(const RnArgs& a, int esize) {
    if (a.C % 4) return false;
    const void* p[] = {a.z, a.r, a.dy, a.dh, a.y, a.h, a.dz, a.dr};
    const long long ld[] = {a.ldz, a.ldr, a.lddy, a.lddh, a.ldy, a.ldh, a.lddz, a.lddr};
    for (int i = 0; i < 8; ++i)
        if (p[i] && ((uintptr_t)p[i] % (4 * esize) || ld[i] % 4)) return false;
    return true;
}

template <typename T>
static int rn_run(const RnArgs& a, bool bwd, hipStream_t st) {
    const int runs = agb_cdiv(a.n, a.rows);
    const bool vec = rn_vec_ok(a, sizeof(T));
#define RN_DIR(BWD, NEXT)                                       \
    do {                                                        \
        if (vec) rn_launch<BWD, NEXT, T, 4>(a, runs, st);       \
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
    AGB_CHECK_ARG(n >= 0 && C >= 1 && C <= RN_MAX_C, "%s: bad shape n=%d C=%d (C <= %d)", name, n, C, RN_MAX_C);
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
    if (n < 0 || C < 1 || C > RN_MAX_C || B < 0) return 0;
    const size_t slots = (size_t)agb_cdiv(n, rn_rows(n, C)) + B + 1;
    return (slots + B + 1) * (next ? 4 : 2) * (size_t)C * sizeof(float);
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
    f.plots = a.part + ((size_t)f.runs + f.B + 1) * f.sums * C;
    f.dw = dw; f.db = db; f.dgate = dgate; f.dscale = dscale; f.dw2 = dw2; f.db2 = db2;
    hipLaunchKernelGGL(k_rownorm_fold_plots, dim3(agb_cdiv(C, 32), ptr ? B + 1 : 1), dim3(1024), 0, st, f);
    AGB_CHECK_LAUNCH("agb_rownorm_fold_plots");
    if (ptr && (dw || db || dscale || dw2 || db2)) {
        hipLaunchKernelGGL(k_rownorm_fold, dim3(agb_cdiv(C, 32)), dim3(1024), 0, st, f);
        AGB_CHECK_LAUNCH("agb_rownorm_fold");
    }
    return AGB_OK;
}

}  // extern "C"
