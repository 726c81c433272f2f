// muon.hip — orthogonalised updates (muon_ops.orthogonalize / muon_update, optim.Muon): Newton-Schulz iterations on a list of
// matrix stacks at once.  A matrix M [rows, cols] is taken by its shorter side k and its longer side n, as X [n, k]:
//     X = M / (|M|_F + eps);   repeat:  G = X^T X,   P = b G + c G G,   X <- a X + X P
// (an odd polynomial of every singular value), and the result is written out or, in an update, stepped along:
//     m <- mu m + (1 - mu) g,  M = m  or  (1 - mu) g + mu m,  p <- decay p - step X.
//
// Bound: matrix instructions.  Operands are PAIRS of fp16, x 2^13 = hi + lo (22 to 23 bits), a product is three MFMAs — lo hi +
// hi lo + hi hi, the dropped lo lo is 2^-24 of it — accumulated in fp32: the error of the result against 64 bits is that of
// fp32 products (1e-6; plain bf16 or fp16 operands: 1e-3 and more, since the polynomial lifts the small singular values'
// rounding noise up to 485-fold) at a ceiling of 2500 / 3 TFLOP/s instead of the 157 of fp32 MFMA.  2^13: entries are bounded
// by the singular values' bound (checked from the coefficients to stay below 7), so hi stays below 65504, and an entry of 2^-13
// still keeps its 22 bits.  a X is added in fp32 behind the products: folded into P's diagonal it would cost the small
// directions two more bits.
//
// Layout: X is held as [n][k] (the longer side down), so X P reads both operands along their rows (P is symmetric), and G = X^T X
// reads X down its columns: those fragments are transposed by the LDS reads.  Columns are cut into blocks of 32; a block holds
// row after row of 128 bytes, 32 hi then 32 lo, so that what a step takes of an operand is contiguous (in rows of all columns, the
// rows of a tile lay a power of two apart: in the same few L2 channels, and the products ran at their speed).  Rows and columns
// are padded to multiples of 64 with zeros, which the iteration keeps zero.  G and P are
// symmetric: only tiles on and above the diagonal are computed.  G has few tiles and a long sum: it is split over n into chunks,
// folded in order.
#include "agb_common.h"
#include <type_traits>

typedef _Float16 half_t;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
// pointers that come out of a table: global memory, as the compiler cannot know (its accesses would go by way of the LDS counter)
#define NS_GLOBAL __attribute__((address_space(1)))
typedef NS_GLOBAL void gvoid;
typedef NS_GLOBAL char gchar;
typedef NS_GLOBAL half_t ghalf;
typedef NS_GLOBAL half8 ghalf8;
typedef NS_GLOBAL half4 ghalf4;
typedef NS_GLOBAL float gfloat;
typedef NS_GLOBAL f32x4 gfloat4;
typedef NS_GLOBAL double gdouble;
typedef NS_GLOBAL unsigned short gshort;
typedef NS_GLOBAL u16x4 gshort4;
typedef NS_GLOBAL u32x4 guint4;

#define NS_THREADS 256
#define NS_WIDE 512           // threads of a product's workgroup
#define NS_SCALE 8192.f
#define NS_UNSCALE (1.f / 8192.f)
#define NS_CHUNK 4096       // elements that a workgroup squares at once
#define NS_SUMS 2048        // partial sums of squares at most (every workgroup of k_ns_planes adds them up)
#define NS_MAX_STEPS 64

struct __attribute__((aligned(16))) NsMat {
    const gvoid* in;
    gvoid* out;
    gfloat* mom;
    long long in_ld, in_bs, out_ld, out_bs;
    int rows, cols, batch, type;      // type of `in` (and of `out` where nothing is updated): 0 fp32, 1 bf16, 2 fp16
    int k, n, kp, np, tall;
    int vec, out_vec;                 // bits: input contiguous and aligned, four elements at a time; tall, and eight elements along
                                      // k at a time; output rows aligned: eight elements
    int tile, kt, tri, splits, chunk;          // tile of G: along k, on and above the diagonal; chunks of n
    int tile_p, kt_p, tri_p;                   // tile of P
    int tile_x, kt_x, nt_x;                    // tile of X
    int sums;                                  // partial sums of squares per matrix
    float step;
    ghalf *xt0, *xt1, *g, *p;                  // planes of matrix 0 of the stack
    gfloat4* part;
    gdouble* sq;
    int at[7];      // first workgroup in the launches over: NS_CHUNKs, 64 x 64 blocks of X, G tiles x splits, X tiles, P tiles,
                    // units of G tiles (fold), whole matrices
};

// ---- pairs of fp16: hi + lo = s, the value times 2^13 (everything between the first split and the output carries that factor;
// a product's sums carry its square).  fmaf with a converted half is one instruction (v_fma_mix_f32).
__device__ __forceinline__ void ns_split(float s, half_t& hi, half_t& lo) {
    hi = (half_t)s;
    lo = (half_t)__builtin_fmaf((float)hi, -1.f, s);
}
__device__ __forceinline__ float ns_pair_sum(half_t hi, half_t lo) { return __builtin_fmaf((float)hi, 1.f, (float)lo); }
__device__ __forceinline__ void ns_split8(const float* s, half8& hi, half8& lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        half_t h, l;
        ns_split(s[e], h, l);
        hi[e] = h;
        lo[e] = l;
    }
}
// element offset of (row, first column of a group of 8) of a plane pair with `rows` padded rows; lo: 32 further
__device__ __forceinline__ size_t ns_at(int row, int col, int rows) {
    return ((size_t)(col >> 5) * rows + row) * 64 + (col & 31);
}

// which matrix a workgroup belongs to: the last whose first workgroup is not behind it (64 candidates a look)
enum { NS_SQUARES, NS_PLANES, NS_GRAM, NS_APPLY, NS_POLY, NS_FOLD, NS_RESIDENT, NS_LAUNCHES };
// (The descriptor is copied whole, by scalar loads in one go.)
typedef const __attribute__((address_space(4))) NsMat* NsTab;
template <int WHICH>
__device__ __forceinline__ NsMat ns_find(NsTab tab, int count, int wg) {
    int found = 0;
    if (count > 1) {
        found = -1;
        for (int base = 0; base < count; base += 64) {
            const int i = base + (threadIdx.x & 63);
            found += __popcll(__ballot(i < count && tab[min(i, count - 1)].at[WHICH] <= wg));
        }
        found = __builtin_amdgcn_readfirstlane(found);
    }
    struct {
        u32x4 v[sizeof(NsMat) / 16];
    } raw;
#pragma unroll
    for (unsigned i = 0; i < sizeof(NsMat) / 16; ++i) raw.v[i] = ((const __attribute__((address_space(4))) u32x4*)(tab + found))[i];
    return __builtin_bit_cast(NsMat, raw);
}

// The table's way to the device: by value, in kernel arguments (a captured call keeps its own), copied by all lanes at once.
#define NS_TABLE 12
struct NsTable {
    NsMat m[NS_TABLE];
};
static_assert(sizeof(NsTable) < 3200 && sizeof(NsMat) % 16 == 0, "kernel arguments hold 4 KB");
__global__ __launch_bounds__(256) void k_ns_table(const NsTable t, u32x4* tab, int pieces) {
    const auto* from = (const __attribute__((address_space(4))) u32x4*)__builtin_amdgcn_kernarg_segment_ptr();      // (t: the first)
    if ((int)threadIdx.x < pieces) tab[threadIdx.x] = from[threadIdx.x];
}

// ---- the matrix that is orthogonalised
struct NsUpdate {
    int on, nesterov;
    float mu, omu, clip, decay;
};
__device__ __forceinline__ float ns_value(unsigned short v, int type) {      // (16 bits: bf16 or fp16)
    return type == 1 ? __uint_as_float((unsigned)v << 16) : (float)__builtin_bit_cast(half_t, v);
}
__device__ __forceinline__ float ns_in(const NsMat& m, size_t off) {
    return m.type == 0 ? ((const gfloat*)m.in)[off] : ns_value(((const gshort*)m.in)[off], m.type);
}
__device__ __forceinline__ void ns_in4(const NsMat& m, size_t off, float* v) {      // (aligned)
    if (m.type == 0) {
        const f32x4 q = *(const gfloat4*)((const gfloat*)m.in + off);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        const u16x4 q = *(const gshort4*)((const gshort*)m.in + off);
        v[0] = ns_value(q.x, m.type); v[1] = ns_value(q.y, m.type); v[2] = ns_value(q.z, m.type); v[3] = ns_value(q.w, m.type);
    }
}
__device__ __forceinline__ float ns_clip(float g, float clip) {      // (NaN stays)
    if (clip > 0.f) g = g > clip ? clip : g < -clip ? -clip : g;
    return g;
}

// sums of squares in 64 bits (neither huge nor tiny entries leave the range), and the momentum's update
__global__ __launch_bounds__(NS_THREADS) void k_ns_squares(const NsMat* tab, int count, const NsUpdate up) {
    const NsMat m = ns_find<NS_SQUARES>((NsTab)tab, count, blockIdx.x);
    const int at = blockIdx.x - m.at[NS_SQUARES], b = at / m.sums, part = at % m.sums;
    const long long total = (long long)m.rows * m.cols;
    const bool linear = m.in_ld == m.cols;
    const long long base = b * m.in_bs;
    // (all of a thread's loads first)
    constexpr int TURNS = NS_CHUNK / (4 * NS_THREADS);
    double s = 0;
    for (long long first = (long long)part * NS_CHUNK; first < total; first += (long long)m.sums * NS_CHUNK) {
        const long long last = first + NS_CHUNK < total ? first + NS_CHUNK : total;
        float v[TURNS][4], mom[TURNS][4];
#pragma unroll
        for (int l = 0; l < TURNS; ++l) {
            const long long i0 = first + (l * NS_THREADS + threadIdx.x) * 4;
            if ((m.vec & 1) && i0 + 4 <= last) {
                ns_in4(m, base + i0, v[l]);
                if (up.on) {
                    const f32x4 q = *(const gfloat4*)(m.mom + i0);
                    mom[l][0] = q.x; mom[l][1] = q.y; mom[l][2] = q.z; mom[l][3] = q.w;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const long long i = i0 + e;
                    v[l][e] = mom[l][e] = 0.f;
                    if (i < last) {
                        v[l][e] = ns_in(m, linear ? base + i : base + i / m.cols * m.in_ld + i % m.cols);
                        if (up.on) mom[l][e] = m.mom[i];
                    }
                }
            }
        }
#pragma unroll
        for (int l = 0; l < TURNS; ++l) {
            const long long i0 = first + (l * NS_THREADS + threadIdx.x) * 4;
            if (up.on) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[l][e] = ns_clip(v[l][e], up.clip);
                    mom[l][e] = mom[l][e] * up.mu + v[l][e] * up.omu;
                    v[l][e] = up.nesterov ? v[l][e] * up.omu + mom[l][e] * up.mu : mom[l][e];
                }
                if ((m.vec & 1) && i0 + 4 <= last) {
                    *(gfloat4*)(m.mom + i0) = f32x4{mom[l][0], mom[l][1], mom[l][2], mom[l][3]};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (i0 + e < last) m.mom[i0 + e] = mom[l][e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s += (double)v[l][e] * v[l][e];
        }
    }
    __shared__ double red[NS_THREADS];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int o = NS_THREADS / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) m.sq[(size_t)b * m.sums + part] = red[0];
}

// X = M / (|M| + eps) as plane pairs, 64 x 64 of [n][k] at a time
__global__ __launch_bounds__(NS_THREADS) void k_ns_planes(const NsMat* tab, int count, const NsUpdate up, double eps) {
    const NsMat m = ns_find<NS_PLANES>((NsTab)tab, count, blockIdx.x);
    const int kb = m.kp / 64, nb = m.np / 64;
    int at = blockIdx.x - m.at[NS_PLANES];
    const int b = at / (kb * nb);
    at %= kb * nb;
    const int n0 = at / kb * 64, k0 = at % kb * 64;
    __shared__ double red[NS_THREADS];
    __shared__ float tile[64][65];
    // rows of M along threadIdx / 64, columns along the lanes; all of a thread's loads first, from the last row or column where
    // there is none
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = (m.tall ? n0 : k0) + wave, c = (m.tall ? k0 : n0) + lane;
    float v[16], mom[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = min(r0 + 4 * i, m.rows - 1), q = min(c, m.cols - 1);
        v[i] = ns_in(m, b * m.in_bs + r * m.in_ld + q);
        if (up.on) mom[i] = m.mom[(size_t)r * m.cols + q];
    }
    double s = 0;
    for (int i = threadIdx.x; i < m.sums; i += NS_THREADS) s += m.sq[(size_t)b * m.sums + i];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int o = NS_THREADS / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    const double inverse = 1 / (sqrt(red[0]) + eps);      // (0 / 0, inf 0: NaN as by division)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = wave + 4 * i;
        float x = v[i];
        if (up.on) {
            x = ns_clip(x, up.clip);
            x = up.nesterov ? x * up.omu + mom[i] * up.mu : mom[i];
        }
        x = r0 + 4 * i < m.rows && c < m.cols ? (float)(x * inverse) * NS_SCALE : 0.f;
        if (m.tall) tile[j][lane] = x;
        else tile[lane][j] = x;
    }
    __syncthreads();
    ghalf* xt = m.xt0 + (size_t)b * m.np * m.kp * 2;
    for (int q = threadIdx.x; q < 512; q += NS_THREADS) {
        const int row = q >> 2 & 63, col = (q & 3) * 8 + (q >> 8) * 32;
        float x[8];
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = tile[row][col + e];
        ns_split8(x, hi, lo);
        const size_t o = ns_at(n0 + row, k0 + col, m.np);
        *(ghalf8*)(xt + o) = hi;
        *(ghalf8*)(xt + o + 32) = lo;
    }
}

// ---- a T x T tile of a product of plane pairs, by eight waves: two groups of four, a quarter of the tile each; a step takes 32
// of the summed index, 16 a group, so that every SIMD has two waves whatever the number of tiles.  Operands go straight from
// global memory to LDS, 16 bytes a lane, into four buffers in turn: transfers are issued four steps ahead (a step of 128 x 128
// takes 0.6 us, a transfer from the other XCDs' side of memory more than one), fragments are read one step ahead of their
// products.  One barrier a step: behind it everybody's transfers of the next step have landed and everybody has read this one's.
//   rows (TR = false): sum over columns [c0, c1) of A[a0 + i][.] B[b0 + j][.]; a block of 32 columns is T rows of 128 bytes, eight
//     pieces of 16, piece q of row r at place q ^ (r / 2 % 8): the 16 lanes that read one piece of 16 rows meet each bank once.
//     Rows behind the last are read as the last and never stored.
//   columns (TR = true): sum over rows [c0, c1) of A[.][a0 + i] B[.][b0 + j]; 32 rows of T columns, piece q of row r at place
//     q ^ 4 (r % 4); ds_read_b64_tr_b16 hands a lane four rows of its column: the four rows that 16 lanes read lie in different
//     quarters of the banks.  Column blocks behind the last are read as the last and never stored.
// Measured: X P of 2048 x 2048 54 us (950 TFLOP/s of fp16), of 13824 x 512 35 us (432 tiles, two turns: 618); a step of 128 x 128
// 0.63 us where its 24 MFMAs a SIMD alone take 0.51; before the first and behind the last together 6 us (descriptor 1.4, first
// operands 0.7, adding the groups 0.9, the rest output).
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half8 ns_read_tr(const char* p, int second) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + second));
    return __builtin_bit_cast(half8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 16 bytes a lane from `from` to LDS at `to` + 16 lane.  (Written out: the compiler would wait for every transfer in flight before
// any LDS read.  Nothing is returned in registers; the waits are NsTile::run's.)
__device__ __forceinline__ void ns_transfer(const gchar* from, unsigned to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory");
}

template <int T, bool TR>
struct NsTile {
    static constexpr int S = T / 64;           // 32 x 32 blocks of a wave along each side
    static constexpr int LOADS = T / 64;       // 16-byte transfers of a lane, per operand and step
    static constexpr int PART = T * 128;       // bytes of an operand's step
    static constexpr int BUFFERS = 4;
    f32x16 acc[S][S];

    __device__ __forceinline__ void run(const ghalf* A, int a0, int a_rows, const ghalf* B, int b0, int b_rows, int cols,
                                        int c0, int c1, char* lds) {
        const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all & 3, group = all >> 2;
        const int wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
        const gchar *pa[LOADS], *pb[LOADS];
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            if constexpr (TR) {
                const int row = (all * LOADS + l) * (256 / T) + lane / (T / 4), piece = lane % (T / 4) ^ (4 * (row & 3));
                pa[l] = (const gchar*)A + ((size_t)min(a0 / 32 + (piece >> 3), cols / 32 - 1) * a_rows + c0 + row) * 128 + (piece & 7) * 16;
                pb[l] = (const gchar*)B + ((size_t)min(b0 / 32 + (piece >> 3), cols / 32 - 1) * b_rows + c0 + row) * 128 + (piece & 7) * 16;
            } else {
                const int row = (all * LOADS + l) * 8 + (lane >> 3), piece = (lane & 7) ^ ((row >> 1) & 7);
                pa[l] = (const gchar*)A + ((size_t)(c0 / 32) * a_rows + min(a0 + row, a_rows - 1)) * 128 + piece * 16;
                pb[l] = (const gchar*)B + ((size_t)(c0 / 32) * b_rows + min(b0 + row, b_rows - 1)) * 128 + piece * 16;
            }
        }
        // a step further: 32 rows, or the next block of 32 columns
        const size_t stride_a = TR ? 32 * 128 : (size_t)a_rows * 128, stride_b = TR ? 32 * 128 : (size_t)b_rows * 128;
        const unsigned to = (unsigned)(size_t)(__attribute__((address_space(3))) char*)lds + all * LOADS * 1024;
        // transfer `l` of the 2 LOADS of a step; the second of a pair moves its pointers on
        auto fetch1 = [&](int step, int l) {
            const unsigned dst = to + (step % BUFFERS) * (2 * PART) + (l >> 1) * 1024;
            if (l & 1) {
                ns_transfer(pb[l >> 1], dst + PART);
                pb[l >> 1] += stride_b;
            } else {
                ns_transfer(pa[l >> 1], dst);
                pa[l >> 1] += stride_a;
            }
        };
        auto fetch = [&](int step) {
#pragma unroll
            for (int l = 0; l < 2 * LOADS; ++l) fetch1(step, l);
        };
        int at_a[S], at_b[S];      // hi; lo: bit 6 flipped
#pragma unroll
        for (int i = 0; i < S; ++i) {
            if constexpr (TR) {
                const int g = lane >> 4, q = (lane & 15) >> 2, p = lane & 3, chunk = 2 * (g & 1) + (p >> 1);
                const int row = (group * 16 + 8 * (g >> 1) + q) * (T * 4) + (p & 1) * 8;
                at_a[i] = row + ((((wr / 32 + i) * 8 + chunk) ^ (4 * q)) << 4);
                at_b[i] = PART + row + ((((wc / 32 + i) * 8 + chunk) ^ (4 * q)) << 4);
            } else {
                const int q = group * 2 + (lane >> 5), r = wr + i * 32 + (lane & 31), c = wc + i * 32 + (lane & 31);
                at_a[i] = r * 128 + ((q ^ ((r >> 1) & 7)) << 4);
                at_b[i] = PART + c * 128 + ((q ^ ((c >> 1) & 7)) << 4);
            }
        }
        struct Fragments {
            half8 ah[S], al[S], bh[S], bl[S];
        };
        // fragment `l` of the 4 S of a step, those of the first products first
        auto read1 = [&](Fragments& f, int step, int l) {
            const char* now = lds + (step % BUFFERS) * (2 * PART);
            const int i = l % (2 * S) / 2, lo = (l / (2 * S)) ^ !(l & 1);       // al, bh of every block, then ah, bl
            const char* p = now + ((l & 1 ? at_b[i] : at_a[i]) ^ (lo ? 64 : 0));
            half8& to = l & 1 ? (lo ? f.bl[i] : f.bh[i]) : (lo ? f.al[i] : f.ah[i]);
            to = TR ? ns_read_tr(p, T * 16) : *(const half8*)p;
        };
        auto multiply1 = [&](const Fragments& f, int l) {
            const int i = l / S % S, j = l % S, kind = l / (S * S);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kind == 0 ? f.al[i] : f.ah[i], kind == 1 ? f.bl[j] : f.bh[j], acc[i][j],
                                                               0, 0, 0);
        };
        // A step's products with the next step's reads and a later one's transfers between them, two to a product at first: what is
        // issued while the matrix pipe is busy costs nothing.  (The scheduler is held off: it gathers the reads, and carries
        // products over the meeting, to where those reads are waited for.)
        auto mixed = [&](const Fragments& now, Fragments& next, int step, bool more, bool further) {
            constexpr int READS = 4 * S, TRANSFERS = 2 * LOADS, PRODUCTS = 3 * S * S, EACH = (READS + TRANSFERS + PRODUCTS - 1) / PRODUCTS;
#pragma unroll
            for (int l = 0; l < PRODUCTS; ++l) {
                multiply1(now, l);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = l * EACH; e < (l + 1) * EACH; ++e) {
                    if (e < READS) {
                        if (more) read1(next, step + 1, e);
                    } else if (e < READS + TRANSFERS) {
                        if (further) fetch1(step + BUFFERS, e - READS);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const int steps = (c1 - c0) / 32;
        // this wave's LDS reads are done (0xC07F: lgkmcnt(0)) and its transfers but those of the last `behind` steps have landed;
        // then everybody's
        auto meet = [&](int behind) {
            __builtin_amdgcn_s_waitcnt(0xC07F);
            if (behind >= 3) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(6 * LOADS) : "memory");
            else if (behind == 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 * LOADS) : "memory");
            else if (behind == 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        };
        auto turn = [&](const Fragments& now, Fragments& next, int step) {
            meet(2);
            mixed(now, next, step, true, true);
        };
        auto last_turn = [&](const Fragments& now, Fragments& next, int step) {
            if (step + 1 < steps) meet(min(2, steps - 2 - step));
            mixed(now, next, step, step + 1 < steps, step + BUFFERS < steps);
        };
        Fragments f0, f1;
        for (int step = 0; step < min(steps, BUFFERS); ++step) fetch(step);
        meet(min(steps, BUFFERS) - 1);
#pragma unroll
        for (int l = 0; l < 4 * S; ++l) read1(f0, 0, l);
        int step = 0;
        for (; step + 3 + BUFFERS < steps; step += 4) {
            turn(f0, f1, step);
            turn(f1, f0, step + 1);
            turn(f0, f1, step + 2);
            turn(f1, f0, step + 3);
        }
        for (; step < steps; step += 2) {
            last_turn(f0, f1, step);
            if (step + 1 < steps) last_turn(f1, f0, step + 1);
        }
        __syncthreads();
    }
    // Adds the two groups' sums.  T = 128: group g is left with blocks j == g (32 rows of B x 64 of A a wave); T = 64: group 0 with
    // everything.  false: this wave is left with nothing.
    static constexpr int UC = 32 * S;          // a wave's unit: 32 rows of B by UC of A
    __device__ __forceinline__ bool merge(char* lds) {
        const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3, group = threadIdx.x >> 8;
        float4* box = (float4*)lds + (wave * S * 2) * 4 * 64 + lane;
        if constexpr (S == 2) {
            // (every wave puts the blocks of the other group; boxes: [wave][giver's blocks i][quad])
            float4* mine = box + group * S * 4 * 64;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float4 v;
                    v.x = group ? acc[i][0][4 * q] : acc[i][1][4 * q];
                    v.y = group ? acc[i][0][4 * q + 1] : acc[i][1][4 * q + 1];
                    v.z = group ? acc[i][0][4 * q + 2] : acc[i][1][4 * q + 2];
                    v.w = group ? acc[i][0][4 * q + 3] : acc[i][1][4 * q + 3];
                    mine[(i * 4 + q) * 64] = v;
                }
            __syncthreads();
            const float4* theirs = box + (group ^ 1) * S * 4 * 64;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = theirs[(i * 4 + q) * 64];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float own = group ? acc[i][1][4 * q + e] : acc[i][0][4 * q + e];
                        acc[i][0][4 * q + e] = own + (e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
                    }
                }
            __syncthreads();      // (the boxes are free for what follows)
            return true;
        } else {
            if (group) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    box[q * 64] = make_float4(acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]);
            }
            __syncthreads();
            if (!group) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = box[q * 64];
                    acc[0][0][4 * q] += v.x;
                    acc[0][0][4 * q + 1] += v.y;
                    acc[0][0][4 * q + 2] += v.z;
                    acc[0][0][4 * q + 3] += v.w;
                }
            }
            __syncthreads();
            return !group;
        }
    }
    // first row (of B's) and column (of A's) of this wave's unit in the tile, and its number
    __device__ __forceinline__ int unit_row() const {
        return (threadIdx.x >> 6 & 1) * (T / 2) + (S == 2 ? (threadIdx.x >> 8) * 32 : 0);
    }
    __device__ __forceinline__ int unit_col() const { return (threadIdx.x >> 7 & 1) * (T / 2); }
    static constexpr int UNITS = S == 2 ? 8 : 4;
    __device__ __forceinline__ int unit() const { return threadIdx.x >> 6; }
    // quad q of block i of the unit (four columns of one row), as the product left it: scaled by 2^26
    __device__ __forceinline__ float4 quad(int i, int q) const {
        return make_float4(acc[i][0][4 * q], acc[i][0][4 * q + 1], acc[i][0][4 * q + 2], acc[i][0][4 * q + 3]);
    }
    __device__ __forceinline__ void stage(float* unit) const;
};

#define NS_LDS(T) (T * 128 * 8)      // four steps' operands; the boxes and the staged units are smaller

// A unit in LDS: 32 rows of UC columns, rows UC + 4 floats apart (the lanes that write or read 16 bytes together meet each bank
// once).  It belongs to one wave (or, in the fold, to the workgroup).
template <int UC>
__device__ __forceinline__ void ns_put_quad(float* unit, int i, int q, int lane, float4 v) {
    const float s = NS_UNSCALE;
    *(float4*)(unit + (lane & 31) * (UC + 4) + i * 32 + q * 8 + (lane >> 5) * 4) = make_float4(v.x * s, v.y * s, v.z * s, v.w * s);
}
template <int T, bool TR>
__device__ __forceinline__ void NsTile<T, TR>::stage(float* unit) const {
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) ns_put_quad<UC>(unit, i, q, threadIdx.x & 63, quad(i, q));
    __builtin_amdgcn_wave_barrier();      // (LDS serves a wave in order)
}
// groups of eight of a unit: number `l` of a thread among `threads`; along a row (four lanes a block's row, sixteen rows) or down
// the rows (four lanes down a column, sixteen columns)
template <int UC>
__device__ __forceinline__ void ns_group(int q, int& row, int& col) {
    row = q >> 2 & 31;
    col = (q & 3) * 8 + (q >> 7) * 32;
}
template <int UC>
__device__ __forceinline__ void ns_along(const float* unit, int row, int col, float* v) {
    const float4 a = *(const float4*)(unit + row * (UC + 4) + col), b = *(const float4*)(unit + row * (UC + 4) + col + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <int UC>
__device__ __forceinline__ void ns_down(const float* unit, int q, int& row, int& col, float* v) {
    row = (q & 3) * 8;
    col = q >> 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = unit[(row + e) * (UC + 4) + col];
}
__device__ __forceinline__ void ns_write8(ghalf* out, size_t o, const float* v) {
    half8 hi, lo;
    ns_split8(v, hi, lo);
    *(ghalf8*)(out + o) = hi;
    *(ghalf8*)(out + o + 32) = lo;
}
// a unit at rows r0, columns c0 of a symmetric plane pair [kp][kp], and its mirror image unless it lies in a diagonal tile
template <int UC, int THREADS>
__device__ __forceinline__ void ns_symmetric(ghalf* out, int kp, int r0, int c0, bool diagonal, const float* unit, int t) {
    float v[8];
    int row, col;
#pragma unroll
    for (int q = t; q < 4 * UC; q += THREADS) {
        ns_group<UC>(q, row, col);
        ns_along<UC>(unit, row, col, v);
        if (r0 + row < kp && c0 + col < kp) ns_write8(out, ns_at(r0 + row, c0 + col, kp), v);
    }
    if (diagonal) return;
#pragma unroll
    for (int q = t; q < 4 * UC; q += THREADS) {
        ns_down<UC>(unit, q, row, col, v);
        if (r0 + row < kp && c0 + col < kp) ns_write8(out, ns_at(c0 + col, r0 + row, kp), v);
    }
}

// tile number -> (i, j), i <= j, of a triangle of `t` rows
__device__ __forceinline__ void ns_pair(int l, int t, int& i, int& j) {
    i = 0;
    while (l >= t - i) { l -= t - i; ++i; }
    j = i + l;
}
// workgroup number within a matrix's `count` -> number of its piece of work: consecutive pieces, which share operands, to
// workgroups 8 apart, which share an XCD and its L2
__device__ __forceinline__ int ns_order(int at, int count) {
    const int each = count >> 3, more = count & 7, xcd = at & 7;
    return xcd * each + min(xcd, more) + (at >> 3);
}

// G = X^T X, a chunk of n at a time
template <int T>
__device__ __forceinline__ void ns_gram(const NsMat& m, int from, char* lds) {
    typedef NsTile<T, true> Tile;
    int at = ns_order(blockIdx.x - m.at[NS_GRAM], m.tri * m.splits * m.batch);
    const int b = at / (m.tri * m.splits);
    at %= m.tri * m.splits;
    const int split = at / m.tri, l = at % m.tri;
    int i, j;
    ns_pair(l, m.kt, i, j);
    const ghalf* x = (from ? m.xt1 : m.xt0) + (size_t)b * m.np * m.kp * 2;
    const int c0 = split * m.chunk, c1 = min(m.np, c0 + m.chunk);
    Tile t;
    t.run(x, i * T, m.np, x, j * T, m.np, m.kp, c0, c1, lds);
    if (!t.merge(lds)) return;
    const int unit = t.unit(), lane = threadIdx.x & 63;
    if (m.splits == 1) {
        float* mine = (float*)lds + unit * 32 * (Tile::UC + 4);
        t.stage(mine);
        ns_symmetric<Tile::UC, 64>(m.g + (size_t)b * m.kp * m.kp * 2, m.kp, j * T + t.unit_row(), i * T + t.unit_col(), i == j, mine, lane);
    } else {      // [batch][split][tile][unit][quad][lane]
        gfloat4* out = m.part + ((((size_t)b * m.splits + split) * m.tri + l) * Tile::UNITS + unit) * (Tile::S * 4 * 64) + lane;
#pragma unroll
        for (int i = 0; i < Tile::S; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 v = t.quad(i, q);
                out[(i * 4 + q) * 64] = f32x4{v.x, v.y, v.z, v.w};
            }
    }
}
// (WIDE: some tile is 128 x 128.  Without, half the registers: two workgroups a CU.)
template <bool WIDE>
__global__ __launch_bounds__(NS_WIDE) void k_ns_gram(const NsMat* tab, int count, int from) {
    extern __shared__ __align__(16) char lds[];
    const NsMat m = ns_find<NS_GRAM>((NsTab)tab, count, blockIdx.x);
    if constexpr (WIDE) {
        if (m.tile == 128) return ns_gram<128>(m, from, lds);
    }
    ns_gram<64>(m, from, lds);
}

// the chunks' sums in order, a unit of a tile
template <int T>
__device__ __forceinline__ void ns_fold(const NsMat& m, float* unit) {
    typedef NsTile<T, true> Tile;
    int at = blockIdx.x - m.at[NS_FOLD];
    const int u = at % Tile::UNITS, l = at / Tile::UNITS % m.tri, b = at / Tile::UNITS / m.tri;
    int i, j;
    ns_pair(l, m.kt, i, j);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t next = (size_t)m.tri * Tile::UNITS * (Tile::S * 4 * 64);
#pragma unroll
    for (int s = 0; s < Tile::S; ++s) {
        const int quad = wave * Tile::S + s;      // (Tile::S * 4 of them by four waves)
        const gfloat4* in = m.part + (((size_t)b * m.splits * m.tri + l) * Tile::UNITS + u) * (Tile::S * 4 * 64) + quad * 64 + lane;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int p = 0; p < m.splits; ++p) {
            const f32x4 v = in[p * next];
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        ns_put_quad<Tile::UC>(unit, quad / 4, quad % 4, lane, sum);
    }
    __syncthreads();
    const int row = (u & 1) * (T / 2) + (Tile::S == 2 ? (u >> 2) * 32 : 0), col = (u >> 1 & 1) * (T / 2);
    ns_symmetric<Tile::UC, NS_THREADS>(m.g + (size_t)b * m.kp * m.kp * 2, m.kp, j * T + row, i * T + col, i == j, unit, threadIdx.x);
}
__global__ __launch_bounds__(NS_THREADS) void k_ns_fold(const NsMat* tab, int count) {
    const NsMat m = ns_find<NS_FOLD>((NsTab)tab, count, blockIdx.x);
    __shared__ __align__(16) float unit[32 * 68];
    if (m.tile == 128) ns_fold<128>(m, unit);
    else ns_fold<64>(m, unit);
}

// P = b G + c G G
template <int T>
__device__ __forceinline__ void ns_poly(const NsMat& m, float cb, float cc, char* lds) {
    typedef NsTile<T, false> Tile;
    const int at = ns_order(blockIdx.x - m.at[NS_POLY], m.tri_p * m.batch), b = at / m.tri_p;
    int i, j;
    ns_pair(at % m.tri_p, m.kt_p, i, j);
    const ghalf* g = m.g + (size_t)b * m.kp * m.kp * 2;
    Tile t;
    t.run(g, i * T, m.kp, g, j * T, m.kp, m.kp, 0, m.kp, lds);
    if (!t.merge(lds)) return;
    const int lane = threadIdx.x & 63, r0 = j * T + t.unit_row(), c0 = i * T + t.unit_col();
    float* mine = (float*)lds + t.unit() * 32 * (Tile::UC + 4);
    constexpr int EACH = Tile::UC / 16;
    half8 gh[EACH], gl[EACH];
    int row, col;
#pragma unroll
    for (int l = 0; l < EACH; ++l) {
        ns_group<Tile::UC>(l * 64 + lane, row, col);
        const size_t o = ns_at(min(r0 + row, m.kp - 1), min(c0 + col, m.kp - 8), m.kp);
        gh[l] = *(const ghalf8*)(g + o);
        gl[l] = *(const ghalf8*)(g + o + 32);
    }
    t.stage(mine);
#pragma unroll
    for (int l = 0; l < EACH; ++l) {
        ns_group<Tile::UC>(l * 64 + lane, row, col);
        float v[8];
        ns_along<Tile::UC>(mine, row, col, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(cc, v[e], cb * ns_pair_sum(gh[l][e], gl[l][e]));
        float4* p = (float4*)(mine + row * (Tile::UC + 4) + col);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __builtin_amdgcn_wave_barrier();
    ns_symmetric<Tile::UC, 64>(m.p + (size_t)b * m.kp * m.kp * 2, m.kp, r0, c0, i == j, mine, lane);
}
template <bool WIDE>
__global__ __launch_bounds__(NS_WIDE) void k_ns_poly(const NsMat* tab, int count, float cb, float cc) {
    extern __shared__ __align__(16) char lds[];
    const NsMat m = ns_find<NS_POLY>((NsTab)tab, count, blockIdx.x);
    if constexpr (WIDE) {
        if (m.tile_p == 128) return ns_poly<128>(m, cb, cc, lds);
    }
    ns_poly<64>(m, cb, cc, lds);
}

// two values as 16-bit ones
__device__ __forceinline__ unsigned ns_pack(float a, float b, int type) {
    if (type == 1) return agb_pack2_bf16(a, b);
    return __builtin_bit_cast(unsigned short, (half_t)a) | (unsigned)__builtin_bit_cast(unsigned short, (half_t)b) << 16;
}
// eight adjacent elements of an output row (those behind its end are not there)
__device__ __forceinline__ void ns_out8(const NsMat& m, const NsUpdate& up, int b, int r, int c, const float* v) {
    if (r >= m.rows || c >= m.cols) return;
    const size_t o = b * m.out_bs + (size_t)r * m.out_ld + c;
    const bool whole = m.out_vec && c + 8 <= m.cols;
    if (up.on || m.type == 0) {
        gfloat* p = (gfloat*)m.out + o;
        if (whole) {
            f32x4 a = {v[0], v[1], v[2], v[3]}, d = {v[4], v[5], v[6], v[7]};
            if (up.on) {
                a = *(gfloat4*)p * up.decay - m.step * a;
                d = *(gfloat4*)(p + 4) * up.decay - m.step * d;
            }
            *(gfloat4*)p = a;
            *(gfloat4*)(p + 4) = d;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < m.cols) p[e] = up.on ? p[e] * up.decay - m.step * v[e] : v[e];
        }
    } else {
        gshort* p = (gshort*)m.out + o;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ns_pack(v[2 * e], v[2 * e + 1], m.type);
        if (whole) {
            *(guint4*)p = w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < m.cols) p[e] = (unsigned short)(w[e / 2] >> 16 * (e & 1));
        }
    }
}

// X <- a X + X P
template <int T>
__device__ __forceinline__ void ns_apply(const NsMat& m, int wg, int from, float ca, bool last, const NsUpdate& up, char* lds) {
    typedef NsTile<T, false> Tile;
    int at = ns_order(wg - m.at[NS_APPLY], m.nt_x * m.kt_x * m.batch);
    const int b = at / (m.nt_x * m.kt_x);
    at %= m.nt_x * m.kt_x;
    const size_t plane = (size_t)b * m.np * m.kp * 2;
    const ghalf* x = (from ? m.xt1 : m.xt0) + plane;
    ghalf* out = (from ? m.xt0 : m.xt1) + plane;
    Tile t;
    t.run(m.p + (size_t)b * m.kp * m.kp * 2, at % m.kt_x * T, m.kp, x, at / m.kt_x * T, m.np, m.kp, 0, m.kp, lds);
    const int lane = threadIdx.x & 63, n0 = at / m.kt_x * T + t.unit_row(), k0 = at % m.kt_x * T + t.unit_col();
    constexpr int EACH = Tile::UC / 16;
    half8 xh[EACH], xl[EACH];
    int row, col;
#pragma unroll
    for (int l = 0; l < EACH; ++l) {
        ns_group<Tile::UC>(l * 64 + lane, row, col);
        const size_t o = ns_at(min(n0 + row, m.np - 1), min(k0 + col, m.kp - 8), m.np);
        xh[l] = *(const ghalf8*)(x + o);
        xl[l] = *(const ghalf8*)(x + o + 32);
    }
    if (!t.merge(lds)) return;
    float* mine = (float*)lds + t.unit() * 32 * (Tile::UC + 4);
    t.stage(mine);
#pragma unroll
    for (int l = 0; l < EACH; ++l) {
        ns_group<Tile::UC>(l * 64 + lane, row, col);
        float v[8];
        ns_along<Tile::UC>(mine, row, col, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(ca, ns_pair_sum(xh[l][e], xl[l][e]), v[e]) * (last ? NS_UNSCALE : 1.f);
        if (!last) {
            if (n0 + row < m.np && k0 + col < m.kp) ns_write8(out, ns_at(n0 + row, k0 + col, m.np), v);
        } else if (m.tall) {
            ns_out8(m, up, b, n0 + row, k0 + col, v);
        } else {
            float4* p = (float4*)(mine + row * (Tile::UC + 4) + col);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
    if (!last || m.tall) return;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int l = 0; l < EACH; ++l) {
        float v[8];
        ns_down<Tile::UC>(mine, l * 64 + lane, row, col, v);
        ns_out8(m, up, b, k0 + col, n0 + row, v);
    }
}
// ---- small matrices: everything in one workgroup, X, G and P in LDS (one launch instead of 17)
// kp = 64 with np <= 512 (one matrix alone: 256), or kp = np = 128.  Products by 16 x 16 blocks of the result spread over eight
// waves: what an iteration takes is latency — the products' chains, the splitting of what they leave, five meetings — and small
// blocks shorten each.
// X and G stay in registers beside their planes in LDS.  Measured: 64 x 64 13 us, 27 x 128 x 128 (27 CUs) 46: a step of 128 is 7.
// kp = 64 adds lo lo: its short sums round so little that the dropped term would show.
// LDS: X [block of 32 columns][n][128 bytes], then G / P [block][k][128 bytes], piece q of row r at place q ^ (r / 2 % 8).
#define NS_RES_ROWS 512
struct NsCoef {
    float v[3 * NS_MAX_STEPS];
};

__device__ __forceinline__ int ns_place(int rows, int row, int piece, int blk) {
    return (blk * rows + row) * 128 + ((piece ^ ((row >> 1) & 7)) << 4);
}
// Operands of 16 x 16 x 32 products out of planes of ROWS rows.  Rows block * 16 .. + 15, columns of block `s` of 32: `at` as
// ns_row_at says, s * ROWS * 128 further (an immediate).
__device__ __forceinline__ int ns_row_at(int rows, int block) {
    const int lane = threadIdx.x & 63;
    return ns_place(rows, block * 16 + (lane & 15), lane >> 4, 0);
}
__device__ __forceinline__ void ns_row16(const char* planes, int at, int offset, half8& hi, half8& lo) {
    hi = *(const half8*)(planes + at + offset);
    lo = *(const half8*)(planes + (at ^ 64) + offset);
}
// ... columns block * 16 .. + 15, rows s * 32 .. + 31: s * 32 * 128 further
__device__ __forceinline__ int ns_column_at(int rows, int block, int second) {
    const int lane = threadIdx.x & 63, q = (lane & 15) >> 2, p = lane & 3;
    return ns_place(rows, 8 * (lane >> 4) + q + 4 * second, 2 * (block & 1) + (p >> 1), block >> 1) + (p & 1) * 8;
}
__device__ __forceinline__ void ns_column16(const char* planes, int first, int second, int offset, half8& hi, half8& lo) {
    auto read = [&](int flip) {
        const s16x4 u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(planes + (first ^ flip) + offset));
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(planes + (second ^ flip) + offset));
        return __builtin_bit_cast(half8, __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    hi = read(0);
    lo = read(64);
}
// LOLO: the fourth product too
template <bool LOLO>
__device__ __forceinline__ void ns_mfma(f32x4& acc, half8 ah, half8 al, half8 bh, half8 bl) {
    if constexpr (LOLO) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bl, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, acc, 0, 0, 0);
}
// A lane's four sums of a 16 x 16 product: columns ia * 16 + 4 (lane / 16) .. + 3 of row ib * 16 + lane % 16
__device__ __forceinline__ int ns_quad_at(int rows, int ia, int ib) {
    const int lane = threadIdx.x & 63;
    return ns_place(rows, ib * 16 + (lane & 15), 2 * (ia & 1) + (lane >> 5), ia >> 1) + (lane >> 4 & 1) * 8;
}
__device__ __forceinline__ void ns_quad_put(char* planes, int rows, int ia, int ib, const float* v) {
    const int at = ns_quad_at(rows, ia, ib);
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        half_t h, l;
        ns_split(v[e], h, l);
        hi[e] = h;
        lo[e] = l;
    }
    *(half4*)(planes + at) = hi;
    *(half4*)(planes + (at ^ 64)) = lo;
}
__device__ __forceinline__ void ns_quad_get(const char* planes, int rows, int ia, int ib, float* v) {
    const int at = ns_quad_at(rows, ia, ib);
    const half4 hi = *(const half4*)(planes + at), lo = *(const half4*)(planes + (at ^ 64));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ns_pair_sum(hi[e], lo[e]);
}

template <int KP, int NP>
__device__ __forceinline__ void ns_resident(const NsMat& m, int b, const NsUpdate& up, double eps, const float* abc, int steps,
                                            char* X, double* red) {
    // G and P: a wave's blocks of 16 x 16 are TA by TB; X: PAIRS pairs of blocks along k, a wave keeps to one pair
    constexpr int GROUPS8 = KP / 8, TA = KP == 64 ? 1 : 2, TB = KP == 64 ? 2 : 4, PAIRS = KP / 32, SUM = KP / 32;
    constexpr bool LOLO = KP == 64;
    constexpr int GROUPS = (NP / 64 * GROUPS8 + 7) / 8, UNITS = (NP / 16 * PAIRS + 7) / 8;      // of a wave, rounded up
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* G = X + NP * KP * 4;
    // M, its momentum's update, its norm: a wave takes 64 rows n of eight columns k.  (Loads without branches, from the last row
    // or column where there is none: all in flight together.)
    float u[GROUPS][8];
    const int groups = NP / 64 * GROUPS8;      // of a matrix; this wave's: wave, wave + 8, ...
    auto first_of = [&](int group, long long ld) { return min(group / GROUPS8 * 64 + lane, m.n - 1) * (m.tall ? ld : 1); };
    auto column_of = [&](int group, int e, long long ld) { return min(group % GROUPS8 * 8 + e, m.k - 1) * (m.tall ? 1 : ld); };
    const bool eights = m.vec & 2;      // (rows of M are rows n, and their ends are groups' ends)
    auto eight_at = [&](int group, long long ld) { return first_of(group, ld) + min(group % GROUPS8 * 8, m.k - 8); };
    if (eights && m.type == 0) {
        const gfloat* in = (const gfloat*)m.in + b * m.in_bs;
#pragma unroll
        for (int l = 0; l < GROUPS; ++l)
            if (l * 8 + wave < groups) {
                const gfloat4* p = (const gfloat4*)(in + eight_at(l * 8 + wave, m.in_ld));
                const f32x4 q = p[0], r = p[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) { u[l][e] = q[e]; u[l][4 + e] = r[e]; }
            }
    } else if (eights) {
        const gshort* in = (const gshort*)m.in + b * m.in_bs;
        u32x4 raw[GROUPS];
#pragma unroll
        for (int l = 0; l < GROUPS; ++l)
            if (l * 8 + wave < groups) raw[l] = *(const guint4*)(in + eight_at(l * 8 + wave, m.in_ld));
#pragma unroll
        for (int l = 0; l < GROUPS; ++l)
#pragma unroll
            for (int e = 0; e < 8; ++e) u[l][e] = ns_value((unsigned short)(raw[l][e / 2] >> 16 * (e & 1)), m.type);
    } else if (m.type == 0) {
        const gfloat* in = (const gfloat*)m.in + b * m.in_bs;
#pragma unroll
        for (int l = 0; l < GROUPS; ++l)
            if (l * 8 + wave < groups) {
                const gfloat* p = in + first_of(l * 8 + wave, m.in_ld);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[l][e] = p[column_of(l * 8 + wave, e, m.in_ld)];
            }
    } else {
        const gshort* in = (const gshort*)m.in + b * m.in_bs;
        unsigned short raw[GROUPS][8];
#pragma unroll
        for (int l = 0; l < GROUPS; ++l)
            if (l * 8 + wave < groups) {
                const gshort* p = in + first_of(l * 8 + wave, m.in_ld);
#pragma unroll
                for (int e = 0; e < 8; ++e) raw[l][e] = p[column_of(l * 8 + wave, e, m.in_ld)];
            }
#pragma unroll
        for (int l = 0; l < GROUPS; ++l)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                u[l][e] = ns_value(raw[l][e], m.type);
    }
    double s = 0;
#pragma unroll
    for (int l = 0; l < GROUPS; ++l) {
        const int group = l * 8 + wave, n = group / GROUPS8 * 64 + lane, k = group % GROUPS8 * 8;
        if (group >= groups) continue;
        float mom[8];
        gfloat* pm = m.mom + first_of(group, m.cols);
        gfloat4* pm8 = (gfloat4*)(m.mom + eight_at(group, m.cols));
        if (up.on && eights) {
            const f32x4 q = pm8[0], r = pm8[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) { mom[e] = q[e]; mom[4 + e] = r[e]; }
        } else if (up.on) {
#pragma unroll
            for (int e = 0; e < 8; ++e) mom[e] = pm[column_of(group, e, m.cols)];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool there = n < m.n && k + e < m.k;
            float v = u[l][e];
            if (up.on) {
                v = ns_clip(v, up.clip);
                mom[e] = mom[e] * up.mu + v * up.omu;
                if (there && !eights) pm[column_of(group, e, m.cols)] = mom[e];
                v = up.nesterov ? v * up.omu + mom[e] * up.mu : mom[e];
            }
            u[l][e] = there ? v : 0.f;
            s += (double)u[l][e] * u[l][e];
        }
        if (up.on && eights && n < m.n && k < m.k) {
            pm8[0] = f32x4{mom[0], mom[1], mom[2], mom[3]};
            pm8[1] = f32x4{mom[4], mom[5], mom[6], mom[7]};
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = ((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]));
    const double inverse = 1 / (sqrt(s) + eps);
#pragma unroll
    for (int l = 0; l < GROUPS; ++l) {
        const int group = l * 8 + wave;
        if (group >= groups) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[l][e] = (float)(u[l][e] * inverse) * NS_SCALE;
        half8 hi, lo;
        ns_split8(u[l], hi, lo);
        const int at = ns_place(NP, group / GROUPS8 * 64 + lane, group % GROUPS8 & 3, group % GROUPS8 >> 2);
        *(half8*)(X + at) = hi;
        *(half8*)(X + (at ^ 64)) = lo;
    }
    __syncthreads();
    const int ia0 = (wave >> 1) * TA, ib0 = (wave & 1) * TB, pair = wave & (PAIRS - 1);
    f32x4 x[UNITS][2];      // this wave's blocks of X, as the last step left them
#pragma unroll
    for (int l = 0; l < UNITS; ++l) {
        const int n = (l * 8 + wave) / PAIRS;
        if (n < NP / 16) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v[4];
                ns_quad_get(X, NP, pair * 2 + i, n, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[l][i][e] = v[e];
            }
        }
    }
    for (int step = 0; step < steps; ++step) {
        const float ca = abc[3 * step], cb = abc[3 * step + 1], cc = abc[3 * step + 2] * NS_UNSCALE;
        f32x4 acc[TA][TB], g[TA][TB];
        auto clear = [&]() {
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        // Operands are read one block of B ahead of the products that take them (all of a step ahead: too many registers).
        auto product = [&](auto count, auto read_a, auto read_b) {
            half8 ah[2][TA], al[2][TA], bh[2], bl[2];
#pragma unroll
            for (int i = 0; i < TA; ++i) read_a(0, i, ah[0][i], al[0][i]);
            read_b(0, 0, bh[0], bl[0]);
#pragma unroll
            for (int l = 0; l < count * TB; ++l) {
                const int s = l / TB, j = l % TB, n = l + 1;
                if (n < count * TB) read_b(n / TB, n % TB, bh[n & 1], bl[n & 1]);
                if (s + 1 < count) {
#pragma unroll
                    for (int i = j * TA / TB; i < (j + 1) * TA / TB; ++i) read_a(s + 1, i, ah[(s + 1) & 1][i], al[(s + 1) & 1][i]);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = LOLO ? 0 : 1; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < TA; ++i)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k < 2 ? al[s & 1][i] : ah[s & 1][i],
                                                                           k == 0 || k == 2 ? bl[l & 1] : bh[l & 1], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // G = X^T X
        {
            int a1[TA], a2[TA], b1[TB], b2[TB];
#pragma unroll
            for (int i = 0; i < TA; ++i) { a1[i] = ns_column_at(NP, ia0 + i, 0); a2[i] = ns_column_at(NP, ia0 + i, 1); }
#pragma unroll
            for (int j = 0; j < TB; ++j) { b1[j] = ns_column_at(NP, ib0 + j, 0); b2[j] = ns_column_at(NP, ib0 + j, 1); }
            clear();
            product(std::integral_constant<int, NP / 32>(),
                    [&](int s, int i, half8& hi, half8& lo) { ns_column16(X, a1[i], a2[i], s * 4096, hi, lo); },
                    [&](int s, int j, half8& hi, half8& lo) { ns_column16(X, b1[j], b2[j], s * 4096, hi, lo); });
        }
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) g[i][j][e] = v[e] = acc[i][j][e] * NS_UNSCALE;
                ns_quad_put(G, KP, ia0 + i, ib0 + j, v);
            }
        __syncthreads();
        // P = b G + c G G, in G's place
        clear();
        {
            int a1[TA], b1[TB];
#pragma unroll
            for (int i = 0; i < TA; ++i) a1[i] = ns_row_at(KP, ia0 + i);
#pragma unroll
            for (int j = 0; j < TB; ++j) b1[j] = ns_row_at(KP, ib0 + j);
            product(std::integral_constant<int, SUM>(),
                    [&](int s, int i, half8& hi, half8& lo) { ns_row16(G, a1[i], s * KP * 128, hi, lo); },
                    [&](int s, int j, half8& hi, half8& lo) { ns_row16(G, b1[j], s * KP * 128, hi, lo); });
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(cc, acc[i][j][e], cb * g[i][j][e]);
                ns_quad_put(G, KP, ia0 + i, ib0 + j, v);
            }
        __syncthreads();
        // X <- a X + X P: every product first, then every block in its place (behind the last step nobody reads it)
        {
            half8 ph[2][SUM], pl[2][SUM];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int s = 0; s < SUM; ++s) ns_row16(G, ns_row_at(KP, pair * 2 + i), s * KP * 128, ph[i][s], pl[i][s]);
#pragma unroll
            for (int l = 0; l < UNITS; ++l) {
                const int n = (l * 8 + wave) / PAIRS;
                if (n < NP / 16) {
                    f32x4 xp[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
                    const int at = ns_row_at(NP, n);
#pragma unroll
                    for (int s = 0; s < SUM; ++s) {
                        half8 xh, xl;
                        ns_row16(X, at, s * NP * 128, xh, xl);
#pragma unroll
                        for (int i = 0; i < 2; ++i) ns_mfma<LOLO>(xp[i], ph[i][s], pl[i][s], xh, xl);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[l][i][e] = __builtin_fmaf(xp[i][e], NS_UNSCALE, ca * x[l][i][e]);
                }
            }
        }
        if (step == steps - 1) break;
        __syncthreads();
#pragma unroll
        for (int l = 0; l < UNITS; ++l) {
            const int n = (l * 8 + wave) / PAIRS;
            if (n < NP / 16) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = x[l][i][e];
                    ns_quad_put(X, NP, pair * 2 + i, n, v);
                }
            }
        }
        __syncthreads();
    }
    // out of the registers of the last step: row n, four columns k
    const long long row = m.tall ? m.out_ld : 1, col = m.tall ? 1 : m.out_ld;
#pragma unroll
    for (int l = 0; l < UNITS; ++l) {
        const int n = (l * 8 + wave) / PAIRS * 16 + (lane & 15);
        if ((l * 8 + wave) / PAIRS >= NP / 16) continue;
        const long long base = b * m.out_bs + min(n, m.n - 1) * row;
        x[l][0] *= NS_UNSCALE;
        x[l][1] *= NS_UNSCALE;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k0 = (pair * 2 + i) * 16 + 4 * (lane >> 4);
            if (m.tall && m.out_vec && k0 + 4 <= m.k) {
                if (n >= m.n) continue;
                if (up.on || m.type == 0) {
                    gfloat4* p = (gfloat4*)((gfloat*)m.out + base + k0);
                    *p = up.on ? *p * up.decay - m.step * x[l][i] : x[l][i];
                } else {
                    const unsigned long long w = ns_pack(x[l][i][0], x[l][i][1], m.type) |
                                                 (unsigned long long)ns_pack(x[l][i][2], x[l][i][3], m.type) << 32;
                    *(NS_GLOBAL unsigned long long*)((gshort*)m.out + base + k0) = w;
                }
            } else if (up.on || m.type == 0) {
                gfloat* p = (gfloat*)m.out + base;
                float old[4];
                if (up.on) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) old[e] = p[min(k0 + e, m.k - 1) * col];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n < m.n && k0 + e < m.k) p[(k0 + e) * col] = up.on ? old[e] * up.decay - m.step * x[l][i][e] : x[l][i][e];
            } else {
                gshort* p = (gshort*)m.out + base;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n < m.n && k0 + e < m.k) p[(k0 + e) * col] = (unsigned short)ns_pack(x[l][i][e], x[l][i][e], m.type);
            }
        }
    }
}
__device__ __forceinline__ void ns_resident_any(const NsMat& m, int b, const NsUpdate& up, double eps, const NsCoef& coef, int steps,
                                                char* lds) {
    __shared__ double red[8];
    __shared__ float abc[3 * NS_MAX_STEPS];
    if ((int)threadIdx.x < 3 * steps) abc[threadIdx.x] = coef.v[threadIdx.x];
    if (m.kp == 128) ns_resident<128, 128>(m, b, up, eps, abc, steps, lds, red);
    else if (m.np == 64) ns_resident<64, 64>(m, b, up, eps, abc, steps, lds, red);
    else if (m.np == 128) ns_resident<64, 128>(m, b, up, eps, abc, steps, lds, red);
    else if (m.np == 192) ns_resident<64, 192>(m, b, up, eps, abc, steps, lds, red);
    else if (m.np == 256) ns_resident<64, 256>(m, b, up, eps, abc, steps, lds, red);
    else ns_resident<64, 512>(m, b, up, eps, abc, steps, lds, red);
}
__global__ __launch_bounds__(NS_WIDE) void k_ns_resident(const NsTable args, const NsMat* tab, int count, const NsUpdate up, double eps,
                                                         const NsCoef coef, int steps) {
    extern __shared__ __align__(16) char lds[];
    // (a list that fits travels in the arguments alone; those are far away: everything is read at once, at the start)
    const NsMat m = ns_find<NS_RESIDENT>(tab ? (NsTab)tab : (NsTab)__builtin_amdgcn_kernarg_segment_ptr(), count, blockIdx.x);
    ns_resident_any(m, blockIdx.x - m.at[NS_RESIDENT], up, eps, coef, steps, lds);
}

template <bool WIDE>
__device__ __forceinline__ void ns_apply_any(const NsMat& m, int wg, int from, float ca, bool last, const NsUpdate& up, char* lds) {
    if constexpr (WIDE) {
        if (m.tile_x == 128) return ns_apply<128>(m, wg, from, ca, last, up, lds);
    }
    ns_apply<64>(m, wg, from, ca, last, up, lds);
}
template <bool WIDE>
__global__ __launch_bounds__(NS_WIDE) void k_ns_apply(const NsMat* tab, int count, int from, float ca, int last,
                                                      const NsUpdate up) {
    extern __shared__ __align__(16) char lds[];
    const NsMat m = ns_find<NS_APPLY>((NsTab)tab, count, blockIdx.x);
    ns_apply_any<WIDE>(m, blockIdx.x, from, ca, last, up, lds);
}
// The last step of a list that also has matrices that are taken whole: those, by the first workgroups, beside the others' tiles
// (SENet14: seven of its matrices, on seven CUs, in the 80 us that its last products and the parameters take).
template <bool WIDE>
__global__ __launch_bounds__(NS_WIDE) void k_ns_last(const NsMat* tab, int count, int from, float ca, const NsUpdate up, int whole,
                                                     double eps, const NsCoef coef, int steps) {
    extern __shared__ __align__(16) char lds[];
    if ((int)blockIdx.x < whole) {
        const NsMat m = ns_find<NS_RESIDENT>((NsTab)tab, count, blockIdx.x);
        ns_resident_any(m, blockIdx.x - m.at[NS_RESIDENT], up, eps, coef, steps, lds);
    } else {
        const int wg = blockIdx.x - whole;
        const NsMat m = ns_find<NS_APPLY>((NsTab)tab, count, wg);
        ns_apply_any<WIDE>(m, wg, from, ca, true, up, lds);
    }
}

// ---- host side
// fields of a matrix stack in the callers' table (int64 each)
enum { NS_IN, NS_OUT, NS_MOM, NS_ROWS, NS_COLS, NS_BATCH, NS_IN_LD, NS_IN_BS, NS_OUT_LD, NS_OUT_BS, NS_TYPE, NS_FIELDS };
#define NS_MAX_SIDE (1 << 24)

struct NsPlan {
    size_t bytes;
    int grid[NS_LAUNCHES];
    bool wide, wide_p, wide_x;      // a tile of 128 among those of G, P, X
    int lds;                // bytes of the largest matrix that is taken whole
};

// One matrix stack's part of the workspace and of the launches.  false: a size that is not taken.
static bool ns_plan(const long long* f, NsMat& m, char* ws, NsPlan& plan) {
    const long long rows = f[NS_ROWS], cols = f[NS_COLS], batch = f[NS_BATCH];
    if (rows < 1 || cols < 1 || batch < 1 || rows > NS_MAX_SIDE || cols > NS_MAX_SIDE || batch > (1 << 20)) return false;
    m.in = (const gvoid*)f[NS_IN]; m.out = (gvoid*)f[NS_OUT]; m.mom = (gfloat*)f[NS_MOM];
    m.in_ld = f[NS_IN_LD]; m.in_bs = f[NS_IN_BS]; m.out_ld = f[NS_OUT_LD]; m.out_bs = f[NS_OUT_BS];
    m.rows = (int)rows; m.cols = (int)cols; m.batch = (int)batch; m.type = (int)f[NS_TYPE];
    m.tall = rows >= cols;
    const int esize = m.type == 0 ? 4 : 2;
    const bool aligned = f[NS_IN] % 16 == 0 && f[NS_MOM] % 16 == 0;
    m.vec = (m.in_ld == cols && m.in_bs % 4 == 0 && aligned ? 1 : 0) |
            (m.tall && cols % 8 == 0 && m.in_ld * esize % 16 == 0 && m.in_bs * esize % 16 == 0 && aligned ? 2 : 0);
    m.out_vec = m.out_ld * esize % 16 == 0 && m.out_bs * esize % 16 == 0 && f[NS_OUT] % 16 == 0;
    m.k = m.tall ? m.cols : m.rows;
    m.n = m.tall ? m.rows : m.cols;
    if (m.k > 16384) return false;
    m.kp = agb_cdiv(m.k, 64) * 64;
    m.np = agb_cdiv(m.n, 64) * 64;
    // (measured: 64 x 64 13 us whole, 64 x 1728 in tiles 110; the limits: LDS, and what a thread holds of X)
    // (one 64 x 512 takes 70 us a call whole and 97 in tiles, but in a list those come with the others' launches, and of the last
    // launch it would be the longest part; a stack of 27 takes 74 whole, 102 in tiles)
    const bool whole = (m.kp == 64 && m.np <= (m.batch > 1 ? NS_RES_ROWS : NS_RES_ROWS / 2)) || (m.kp == 128 && m.np == 128);
    // Products, measured: a workgroup of T = 128 has a CU to itself, for about 6 us and 0.65 for each 32 of the sum; of T = 64 a CU
    // holds two, which share what one alone reaches: 6 us and 0.22 for each 32 (a quarter of the work).  So 64 x 64 where the
    // tiles are few and 128 x 128 where they are many.
    auto cost = [](int T, long long wgs, int sum) {      // us; `sum`: of how many products
        const double rounds = (double)((wgs + 255) / 256), steps = sum / 32;
        return T == 128 ? rounds * (6 + 0.65 * steps) : 5 + rounds * (1 + 0.22 * steps);
    };
    auto tiles_of = [&](int T) { return agb_cdiv(m.np, T) * (long long)agb_cdiv(m.kp, T) * m.batch; };
    auto triangle_of = [&](int T) { const long long kt = agb_cdiv(m.kp, T); return kt * (kt + 1) / 2 * m.batch; };
    // (X P of 1500 x 1500 by 128 x 128: 424 us a call instead of 491; of 3 x 515 x 1029 by 64 x 64: 238 instead of 251)
    m.tile_x = m.kp >= 256 && cost(128, tiles_of(128), m.kp) <= cost(64, tiles_of(64), m.kp) ? 128 : 64;
    m.kt_x = agb_cdiv(m.kp, m.tile_x);
    m.nt_x = agb_cdiv(m.np, m.tile_x);
    // G: the tile and the number of chunks of n (none shorter than 256) that take least by those figures and the fold's, which
    // more than one chunk needs: 3 us and what the chunks' sums take through memory.  (By the matrix alone: what else is in the
    // list does not change a result.  3 x 515 x 1029: 135 tiles of 64 x 64 take 200 us in all; 45 of 128 x 128 in three chunks
    // each 231.  2048 x 2048: 136 of 128 x 128 698, 528 of 64 x 64 736.)
    double best = 1e30;
    m.tile = 64;
    m.chunk = m.np;
    for (int T = 64; !whole && T <= (m.kp >= 256 ? 128 : 64); T *= 2) {
        const long long tiles = triangle_of(T);
        for (int splits = 1; splits <= 64 && (splits == 1 || m.np / splits >= 256); ++splits) {
            const int chunk = agb_cdiv(agb_cdiv(m.np, splits), 64) * 64, real = agb_cdiv(m.np, chunk);
            const double us = cost(T, tiles * real, chunk) + (real > 1 ? 3 + (double)tiles * real * (T == 128 ? 0.04 : 0.02) : 0);
            if (us < best) {
                best = us;
                m.tile = T;
                m.chunk = chunk;
            }
        }
    }
    m.kt = agb_cdiv(m.kp, m.tile);
    m.tri = m.kt * (m.kt + 1) / 2;
    const long long tiles = (long long)m.tri * m.batch;
    m.splits = agb_cdiv(m.np, m.chunk);
    m.tile_p = m.kp >= 256 && cost(128, triangle_of(128), m.kp) <= cost(64, triangle_of(64), m.kp) ? 128 : 64;
    m.kt_p = agb_cdiv(m.kp, m.tile_p);
    m.tri_p = m.kt_p * (m.kt_p + 1) / 2;
    m.sums = agb_cdiv((long long)rows * cols, NS_CHUNK);
    m.sums = m.sums < NS_SUMS ? m.sums : NS_SUMS;
    if (whole) {
        const int lds = (m.np > 256 ? NS_RES_ROWS : m.np) * m.kp * 4 + m.kp * m.kp * 4;
        if (lds > plan.lds) plan.lds = lds;
    } else {
        plan.wide |= m.tile == 128;
        plan.wide_x |= m.tile_x == 128;
        plan.wide_p |= m.tile_p == 128;
    }
    const size_t x = whole ? 0 : (size_t)m.np * m.kp * 4 * batch, g = whole ? 0 : (size_t)m.kp * m.kp * 4 * batch;
    auto take = [&](size_t n) {
        char* p = ws ? ws + plan.bytes : nullptr;
        plan.bytes += (n + 255) / 256 * 256;
        return p;
    };
    m.xt0 = (ghalf*)take(x);
    m.xt1 = (ghalf*)take(x);
    m.g = (ghalf*)take(g);
    m.p = (ghalf*)take(g);
    m.part = (gfloat4*)take(m.splits > 1 && !whole ? (size_t)m.splits * tiles * m.tile * m.tile * 4 : 0);
    m.sq = (gdouble*)take(whole ? 0 : (size_t)m.sums * batch * 8);
    const long long units = m.tile == 128 ? 8 : 4;
    const long long wgs[NS_LAUNCHES] = {(long long)m.sums * batch, (long long)(m.kp / 64) * (m.np / 64) * batch, tiles * m.splits,
                                        (long long)m.kt_x * m.nt_x * batch, (long long)m.tri_p * batch,
                                        m.splits > 1 ? tiles * units : 0, batch};
    for (int i = 0; i < NS_LAUNCHES; ++i) {
        m.at[i] = plan.grid[i];
        const long long more = whole == (i == NS_RESIDENT) ? wgs[i] : 0;
        if (plan.grid[i] + more > 0x7fffffff) return false;
        plan.grid[i] += (int)more;
    }
    return true;
}

// Largest |sigma| along the iterations from [0, 1], and largest |b s^2 + c s^4|: both are entries' bounds of what is held as
// fp16 pairs.  In t = s^2: the former is largest at an end or where a + 3 b t + 5 c t^2 = 0, the latter at an end or at -b / 2 c.
static bool ns_bounded(const float* coef, int steps) {
    double hi = 1.0;
    for (int i = 0; i < steps; ++i) {
        const double a = coef[3 * i], b = coef[3 * i + 1], c = coef[3 * i + 2], end = hi * hi;
        if (!(end < 7)) return false;
        double at[4] = {end, 0, 0, 0};
        if (c != 0) {
            at[1] = -b / (2 * c);
            const double root = sqrt(9 * b * b - 20 * a * c);      // (NaN: there are none)
            at[2] = (-3 * b + root) / (10 * c);
            at[3] = (-3 * b - root) / (10 * c);
        } else if (b != 0) {
            at[1] = -a / (3 * b);
        }
        double next = 0;
        for (double t : at) {
            if (!(t > 0 && t <= end)) continue;
            const double q = t * (b + c * t), v = fabs(sqrt(t) * (a + q));
            if (!(fabs(q) < 7 && v <= 7)) return false;
            next = v > next ? v : next;
        }
        if (!(a == a && b == b && c == c)) return false;
        hi = next * 1.001 + 1e-3;
    }
    return true;
}

static int ns_run(const char* name, const long long* fields, int count, int steps, const float* coef, double eps, const float* step,
                  const NsUpdate& up, void* workspace, size_t workspace_bytes, hipStream_t st) {
    AGB_CHECK_ARG(count >= 0 && (count == 0 || fields), "%s: %d matrices", name, count);
    AGB_CHECK_ARG(steps >= 1 && steps <= NS_MAX_STEPS && coef, "%s: %d steps (1 to %d)", name, steps, NS_MAX_STEPS);
    AGB_CHECK_ARG(ns_bounded(coef, steps), "%s: the coefficients let singular values grow past 7 (or hi^2 past 7)", name);
    AGB_CHECK_ARG(eps >= 0, "%s: eps", name);
    if (count == 0) return AGB_OK;
    NsPlan plan = {};
    const size_t table = ((size_t)count * sizeof(NsMat) + 255) / 256 * 256;
    plan.bytes = table;
    NsTable t;
    NsMat* m = t.m;
    // sizes first: nothing is enqueued before everything has been looked at
    for (int i = 0; i < count; ++i) {
        const long long* f = fields + (size_t)i * NS_FIELDS;
        AGB_CHECK_ARG(ns_plan(f, m[0], nullptr, plan), "%s: matrix %d: [%lld, %lld, %lld] is not taken", name, i, f[NS_BATCH],
                      f[NS_ROWS], f[NS_COLS]);
        AGB_CHECK_ARG(m[0].in && m[0].out && (!up.on || m[0].mom), "%s: matrix %d: null pointer", name, i);
        AGB_CHECK_ARG(m[0].type >= 0 && m[0].type <= 2, "%s: matrix %d: type %d", name, i, m[0].type);
        AGB_CHECK_ARG(m[0].in_ld >= m[0].cols && m[0].out_ld >= m[0].cols, "%s: matrix %d: row stride", name, i);
        AGB_CHECK_ARG(!up.on || m[0].batch == 1, "%s: matrix %d: updates take one matrix each", name, i);
    }
    AGB_CHECK_ARG(workspace && workspace_bytes >= plan.bytes, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                  plan.bytes);
    NsMat* tab = (NsMat*)workspace;
    plan = {};
    plan.bytes = table;
    for (int base = 0; base < count; base += NS_TABLE) {
        const int some = count - base < NS_TABLE ? count - base : NS_TABLE;
        t = {};
        for (int i = 0; i < some; ++i) {
            ns_plan(fields + (size_t)(base + i) * NS_FIELDS, m[i], (char*)workspace, plan);
            m[i].step = step ? step[base + i] : 0.f;
        }
        if (count <= NS_TABLE && !plan.grid[NS_SQUARES]) tab = nullptr;      // (every matrix is taken whole: no table)
        else hipLaunchKernelGGL(k_ns_table, dim3(1), dim3(256), 0, st, t, (u32x4*)(tab + base), (int)(some * sizeof(NsMat) / 16));
    }
    const int* grid = plan.grid;
    NsCoef all = {};
    for (int i = 0; i < 3 * steps; ++i) all.v[i] = coef[i];
    if (!grid[NS_SQUARES]) {
        const hipError_t e = hipFuncSetAttribute((const void*)k_ns_resident, hipFuncAttributeMaxDynamicSharedMemorySize, plan.lds);
        if (e != hipSuccess) { agb_set_error("%s: %s", name, hipGetErrorString(e)); return AGB_ELAUNCH; }
        if (tab) t = {};
        hipLaunchKernelGGL(k_ns_resident, dim3(grid[NS_RESIDENT]), dim3(NS_WIDE), plan.lds, st, t, tab, count, up, eps, all, steps);
        AGB_CHECK_LAUNCH(name);
        return AGB_OK;
    }
    for (const void* k : {(const void*)k_ns_gram<true>, (const void*)k_ns_poly<true>, (const void*)k_ns_apply<true>, (const void*)k_ns_last<true>,
                          (const void*)k_ns_last<false>}) {
        const hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, plan.lds > NS_LDS(128) ? plan.lds : NS_LDS(128));
        if (e != hipSuccess) { agb_set_error("%s: %s", name, hipGetErrorString(e)); return AGB_ELAUNCH; }
    }
#define NS_PRODUCT(kernel, which, wide, ...)                                                                                \
    do {                                                                                                                    \
        if (wide) hipLaunchKernelGGL(kernel<true>, dim3(grid[which]), dim3(NS_WIDE), NS_LDS(128), st, tab, count, __VA_ARGS__); \
        else hipLaunchKernelGGL(kernel<false>, dim3(grid[which]), dim3(NS_WIDE), NS_LDS(64), st, tab, count, __VA_ARGS__);      \
    } while (0)
    hipLaunchKernelGGL(k_ns_squares, dim3(grid[NS_SQUARES]), dim3(NS_THREADS), 0, st, tab, count, up);
    hipLaunchKernelGGL(k_ns_planes, dim3(grid[NS_PLANES]), dim3(NS_THREADS), 0, st, tab, count, up, eps);
    for (int i = 0; i < steps; ++i) {
        const float* c = coef + 3 * i;
        NS_PRODUCT(k_ns_gram, NS_GRAM, plan.wide, i & 1);
        if (grid[NS_FOLD]) hipLaunchKernelGGL(k_ns_fold, dim3(grid[NS_FOLD]), dim3(NS_THREADS), 0, st, tab, count);
        NS_PRODUCT(k_ns_poly, NS_POLY, plan.wide_p, c[1], c[2]);
        if (i < steps - 1 || !grid[NS_RESIDENT]) {
            NS_PRODUCT(k_ns_apply, NS_APPLY, plan.wide_x, i & 1, c[0], i == steps - 1, up);
            continue;
        }
        const int whole = grid[NS_RESIDENT], lds = plan.wide_x ? NS_LDS(128) : NS_LDS(64);
        const dim3 both(whole + grid[NS_APPLY]);
        if (plan.wide_x)
            hipLaunchKernelGGL(k_ns_last<true>, both, dim3(NS_WIDE), lds > plan.lds ? lds : plan.lds, st, tab, count, i & 1, c[0], up,
                               whole, eps, all, steps);
        else
            hipLaunchKernelGGL(k_ns_last<false>, both, dim3(NS_WIDE), lds > plan.lds ? lds : plan.lds, st, tab, count, i & 1, c[0], up,
                               whole, eps, all, steps);
    }
#undef NS_PRODUCT
    AGB_CHECK_LAUNCH(name);
    return AGB_OK;
}

extern "C" {

int agb_ns_fields(void) { return NS_FIELDS; }

size_t agb_ns_workspace_bytes(const long long* fields, int count) {
    if (count < 1 || !fields) return 0;
    NsPlan plan = {};
    plan.bytes = ((size_t)count * sizeof(NsMat) + 255) / 256 * 256;
    NsMat m;
    for (int i = 0; i < count; ++i)
        if (!ns_plan(fields + (size_t)i * NS_FIELDS, m, nullptr, plan)) return 0;
    return plan.bytes;
}

int agb_orthogonalize(const long long* fields, int count, int steps, const float* coef, double eps, void* workspace,
                      size_t workspace_bytes, void* stream) {
    const NsUpdate up = {};
    return ns_run("agb_orthogonalize", fields, count, steps, coef, eps, nullptr, up, workspace, workspace_bytes,
                  (hipStream_t)stream);
}

int agb_muon_update(const long long* fields, int count, int steps, const float* coef, double eps, const float* step, double decay,
                    double momentum, int nesterov, float clip, void* workspace, size_t workspace_bytes, void* stream) {
    AGB_CHECK_ARG(count == 0 || step, "agb_muon_update: null pointer");
    AGB_CHECK_ARG(momentum >= 0 && momentum < 1, "agb_muon_update: momentum %g", momentum);
    NsUpdate up;
    up.on = 1;
    up.nesterov = nesterov != 0;
    up.mu = (float)momentum;
    up.omu = (float)(1 - momentum);      // (1 - momentum in double: 1 - 0.95f is not 0.05f)
    up.clip = clip;
    up.decay = (float)decay;
    return ns_run("agb_muon_update", fields, count, steps, coef, eps, step, up, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
