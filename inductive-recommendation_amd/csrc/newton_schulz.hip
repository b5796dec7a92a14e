// newton_schulz.hip - orthogonalising a weight's update by Newton-Schulz products (gfx950 matrix cores).
//
//   X_0 = G / (|G|_F + eps),   A = X X^T,   X <- a X + (b A + c A A) X        steps times
// on the side with fewer rows (G^T for a tall G).  The iteration pushes X's singular values towards
// 1 and amplifies the small ones by a each step, so its products need fp32's accuracy: every matrix
// is held as pairs of halves (half_split.h) and multiplied in three 16-bit products.  X's
// singular values stay below about 1.2 and A's and b A + c A A's entries below 3, so one
// fixed scale 2^11 serves all of them: entries up to 32, down to steps of 2^-35.
// Where |G| is not above eps, X_0 is small: X is held times 2^k, with k of each step from a bound on its norm n
// (n <- n (|a| + |b| n^2 + |c| n^4) a step, at most 1 where k > 0), and the powers go into b, c and the result.
//
// A and Q = b A + c A A are symmetric: only tiles on and below the diagonal are computed.
//
// A matrix is kept as MFMA fragments (32 rows x 16 columns, 64 lanes of 16 bytes, two planes), so a tile
// is loaded as it lies.  A product needs both operands along the contraction: X as rows (for A) and X^T as
// rows (for Q X), which the update writes together, one straight from the MFMA layout (a
// lane holds four consecutive rows of a column), the other turned in LDS.
//
// Small matrices (up to 64 x 256, a recommender's dense layers) run all steps in one workgroup, X in
// LDS: six of 64 x 64 take 18 us, the latency of fifteen dependent products.  Above that a step is three
// launches; 2 x 1024 x 256 takes 115 us, 5 to 8 us a launch, bound by their latency.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "half_split.h"

namespace igr {
namespace {

constexpr int kThreads = 256;
constexpr int kScale = 11;
typedef Frags<SplitF32> Frag2;

struct Mat {  // a strided batch of matrices, oriented so that rows <= cols: element (r, c) at r sr + c sc
    int64_t S, L, sr, sc, sb;
};

__device__ __forceinline__ void load2(const u32x4_t *p, int64_t frag, int lane, Frag2 &f) {
    f.p[0] = __builtin_bit_cast(half8_t, p[(frag * 2) * 64 + lane]);
    f.p[1] = __builtin_bit_cast(half8_t, p[(frag * 2 + 1) * 64 + lane]);
}

// 1 / (|G| + eps); a matrix of zeros stays one, also with an eps of 0 or too small for its inverse.
__device__ __forceinline__ double inverse_norm(double ss, double eps) { return ss == 0. ? 0. : 1. / (sqrt(ss) + eps); }
// k of step 0: |X_0| 2^k in [0.5, 1); 0 for |X_0| of that size, zeros and what is not finite.
__device__ __forceinline__ int first_power(double ss, double inv) {
    const double n = sqrt(ss) * inv;
    if (!(n > 0. && n < 0.5)) return 0;
    int e;
    frexp(n, &e);
    return -e;
}
struct Growth {  // |a|, |b|, |c|
    double a, b, c;
};
// k after s steps: a bound on |X| 2^k is at most 1, or k is 0.
__device__ __forceinline__ int power_of(int k0, int s, Growth g) {
    if (k0 == 0 && g.a >= 1.) return 0;  // as mostly
    double n = ldexp(1. - 1e-9, -k0);    // (k0 again for s = 0)
    for (int i = 0; i < s; ++i) {
        n *= (g.a + n * n * (g.b + n * n * g.c)) * (1. + 1e-5);  // (roundings)
        if (n >= 1.) return 0;
    }
    int e;
    frexp(n, &e);
    return n > 0. && n < 1. ? -e : 0;
}

// Four values as (hi, lo) halves.
struct Quad {
    uint2 hi, lo;
};
__device__ __forceinline__ Quad split4(float a, float b, float c, float d) {
    const half2_t h0 = __builtin_convertvector((float2_t{a, b}), half2_t);
    const half2_t h1 = __builtin_convertvector((float2_t{c, d}), half2_t);
    const half2_t l0 = __builtin_convertvector((float2_t{rest_of<0>(h0, a), rest_of<1>(h0, b)}), half2_t);
    const half2_t l1 = __builtin_convertvector((float2_t{rest_of<0>(h1, c), rest_of<1>(h1, d)}), half2_t);
    return {make_uint2(__builtin_bit_cast(uint32_t, h0), __builtin_bit_cast(uint32_t, h1)),
            make_uint2(__builtin_bit_cast(uint32_t, l0), __builtin_bit_cast(uint32_t, l1))};
}
__device__ __forceinline__ float half_at(uint2 v, int i) {
    const uint32_t w = i < 2 ? v.x : v.y;
    return (float)__builtin_bit_cast(half2_t, w)[i & 1];
}

// A 32 x 32 result block (lane: column n % 32, register 4 g + i: row 8 g + 4 h + i) as part of a
// fragment matrix whose rows are the block's columns: 8 bytes a group of four rows.
__device__ __forceinline__ int64_t quad_index(int64_t row_block, int64_t KS, int64_t k0, int g, int lane, int plane) {
    const int64_t frag = row_block * KS + (k0 >> 4) + (g >> 1);
    return ((frag * 2 + plane) * 64 + (lane & 31) + 32 * (g & 1)) * 2 + (lane >> 5);
}
__device__ __forceinline__ void put_block(u32x4_t *dst, int64_t row_block, int64_t KS, int64_t k0,
                                          const float (&v)[16], int lane) {
    uint2 *d = reinterpret_cast<uint2 *>(dst);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const Quad q = split4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        d[quad_index(row_block, KS, k0, g, lane, 0)] = q.hi;
        d[quad_index(row_block, KS, k0, g, lane, 1)] = q.lo;
    }
}
__device__ __forceinline__ void get_block(const u32x4_t *src, int64_t row_block, int64_t KS, int64_t k0, float (&v)[16],
                                          int lane) {
    const uint2 *s = reinterpret_cast<const uint2 *>(src);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint2 hi = s[quad_index(row_block, KS, k0, g, lane, 0)];
        const uint2 lo = s[quad_index(row_block, KS, k0, g, lane, 1)];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * g + i] = half_at(hi, i) + half_at(lo, i);
    }
}

// ------------------------------------------------------------------ one workgroup a matrix

// X: 64 x 64 NW in two blocks of rows and 2 NW of columns; wave w holds row block w & 1 of column
// blocks (w >> 1) + 2 j in registers, in fp32, and block (w >> 1, w & 1) of A.
template <class T, int NW>
__global__ __launch_bounds__(kThreads) void ns_small(Mat in, Mat out, const T *g, T *y, int32_t steps, float ca,
                                                     float cb, float cc, double eps, Growth gr) {
    constexpr int KL = 4 * NW;  // 16-column steps of X's rows
    __shared__ u32x4_t xs[2 * KL * 2 * 64], xt[2 * NW * 4 * 2 * 64], am[2 * 4 * 2 * 64], qm[2 * 4 * 2 * 64];
    double *red = reinterpret_cast<double *>(qm);  // qm is first written two barriers later
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 31, h = lane >> 5;
    const int mb = wave & 1, nb0 = wave >> 1;
    const T *src = g + blockIdx.x * in.sb;
    float x[NW][16];
    double ss = 0.;
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t r = mb * 32 + 8 * (i >> 2) + 4 * h + (i & 3), c = (nb0 + 2 * j) * 32 + col;
            x[j][i] = r < in.S && c < in.L ? (float)src[r * in.sr + c * in.sc] : 0.f;
            ss += (double)x[j][i] * x[j][i];
        }
#pragma unroll
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if (lane == 0) red[wave] = ss;
    __syncthreads();
    ss = (red[0] + red[1]) + (red[2] + red[3]);
    const double inv = inverse_norm(ss, eps);
    const int k0 = first_power(ss, inv);
    constexpr float up = 1 << kScale, down = 1.f / (1 << kScale);
    // values in x are X 2^11, as the fragments hold them
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[j][i] = (float)ldexp(x[j][i] * inv, k0) * up;

    auto store_x = [&]() {
        _Float16 *rows = reinterpret_cast<_Float16 *>(xs);
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const int nb = nb0 + 2 * j;
            put_block(xt, nb, 4, mb * 32, x[j], lane);
            // the rows' fragments: this lane's column is one half of 16 different lanes' 16 bytes
            const int at = ((mb * KL + nb * 2 + (col >> 4)) * 2 * 64 + 32 * ((col >> 3) & 1)) * 8 + (col & 7);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 8 * (i >> 2) + 4 * h + (i & 3);
                const _Float16 hi = (_Float16)x[j][i];
                rows[at + r * 8] = hi;
                rows[at + r * 8 + 64 * 8] = (_Float16)(x[j][i] - (float)hi);
            }
        }
    };
    // K steps of two fragment rows; the three parts of the product in sums of their own, so that
    // the MFMAs, 3 K in a row otherwise, wait for each other a third as long
    auto product = [&](const u32x4_t *p, int p0, const u32x4_t *q, int q0, auto ks) {
        constexpr int K = decltype(ks)::value;
        f32x16_t c0, c1, c2;
#pragma unroll
        for (int i = 0; i < 16; ++i) c0[i] = c1[i] = c2[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Frag2 fp, fq;
            load2(p, p0 + k, lane, fp);
            load2(q, q0 + k, lane, fq);
            c0 = mfma32(fp.p[0], fq.p[1], c0);
            c1 = mfma32(fp.p[1], fq.p[0], c1);
            c2 = mfma32(fp.p[0], fq.p[0], c2);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) c2[i] += c0[i] + c1[i];
        return c2;
    };
    store_x();
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const int k = power_of(k0, s, gr), next = power_of(k0, s + 1, gr) - k;
        const float kb = ldexpf(cb, -2 * k), kc = ldexpf(cc, -4 * k);
        float av[16], v[16];
        f32x16_t acc = product(xs, nb0 * KL, xs, mb * KL, std::integral_constant<int, KL>());
#pragma unroll
        for (int i = 0; i < 16; ++i) av[i] = acc[i] * down;
        put_block(am, mb, 4, nb0 * 32, av, lane);
        __syncthreads();
        acc = product(am, nb0 * 4, am, mb * 4, std::integral_constant<int, 4>());
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = fmaf(kb, av[i], kc * (acc[i] * down));
        put_block(qm, mb, 4, nb0 * 32, v, lane);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            acc = product(qm, mb * 4, xt, (nb0 + 2 * j) * 4, std::integral_constant<int, 4>());
#pragma unroll
            for (int i = 0; i < 16; ++i) x[j][i] = ldexpf(fmaf(ca, x[j][i], acc[i] * down), next);
        }
        if (s + 1 < steps) {
            __syncthreads();
            store_x();
            __syncthreads();
        }
    }
    T *dst = y + blockIdx.x * out.sb;
    const int last = power_of(k0, steps, gr);
#pragma unroll
    for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t r = mb * 32 + 8 * (i >> 2) + 4 * h + (i & 3), c = (nb0 + 2 * j) * 32 + col;
            if (r < out.S && c < out.L) dst[r * out.sr + c * out.sc] = (T)ldexpf(x[j][i] * down, -last);
        }
}

// ------------------------------------------------------------------ tiles over the whole chip

constexpr int kSumBlocks = 255;  // partial sums of squares a matrix; a matrix's 256th value is its first power

template <class T>
__global__ __launch_bounds__(kThreads) void ns_sumsq(Mat in, const T *g, double *part) {
    __shared__ double red[4];
    const T *src = g + (int64_t)blockIdx.y * in.sb;
    // the unit-stride side is walked by the threads
    const bool flip = in.sr == 1;
    const int64_t rows = flip ? in.L : in.S, cols = flip ? in.S : in.L, ld = flip ? in.sc : in.sr;
    int wide = 256;  // threads along a row
    while (wide > 1 && wide / 2 >= cols) wide >>= 1;
    const int t = threadIdx.x, across = kThreads / wide;
    double s = 0.;
    for (int64_t r = (int64_t)blockIdx.x * across + t / wide; r < rows; r += (int64_t)gridDim.x * across) {
        const T *row = src + r * ld;
        int64_t c = t % wide;
        for (; c + 7 * wide < cols; c += 8 * wide) {  // eight loads in flight
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)row[c + i * wide];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += (double)v[i] * v[i];
        }
        for (; c < cols; c += wide) {
            const float v = (float)row[c];
            s += (double)v * v;
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * (kSumBlocks + 1) + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

struct Work {  // fragment matrices of one matrix of the batch; the next one's follow at the strides
    u32x4_t *x, *xt[2], *a, *q;
    int64_t bx, ba;    // strides between matrices, in u32x4_t
    int64_t Sp, Lp;    // padded sides, multiples of the tile
};

// 32 x 32 blocks of X_0 into both fragment matrices, zeros in the padding.
template <class T>
__global__ __launch_bounds__(kThreads) void ns_pack(Mat in, const T *g, double *part, double eps, Work w) {
    __shared__ float tile[4][32][33];
    __shared__ double red[4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int64_t batch = blockIdx.y, nb = w.Lp / 32, blocks = nb * (w.Sp / 32);
    static_assert(kSumBlocks < kThreads, "one partial sum a thread");
    double *sums = part + batch * (kSumBlocks + 1);
    double ss = t < kSumBlocks ? sums[t] : 0.;  // joined in the same order by every workgroup
#pragma unroll
    for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if (lane == 0) red[wave] = ss;
    __syncthreads();
    ss = (red[0] + red[1]) + (red[2] + red[3]);
    const double inv = inverse_norm(ss, eps);
    const int k0 = first_power(ss, inv);
    if (blockIdx.x == 0 && t == 0) sums[kSumBlocks] = (double)k0;
    const T *src = g + batch * in.sb;
    const int64_t blk = (int64_t)blockIdx.x * 4 + wave;
    const int64_t r0 = blk / nb * 32, c0 = blk % nb * 32;
    const bool flip = in.sr == 1;
    if (blk < blocks) {
#pragma unroll 4
        for (int i = lane; i < 1024; i += 64) {
            const int r = flip ? i & 31 : i >> 5, c = flip ? i >> 5 : i & 31;
            float v = 0.f;
            if (r0 + r < in.S && c0 + c < in.L)
                v = (float)ldexp((double)(float)src[(r0 + r) * in.sr + (c0 + c) * in.sc] * inv, k0) * (float)(1 << kScale);
            tile[wave][r][c] = v;
        }
    }
    __syncthreads();
    if (blk >= blocks) return;
    const int row = lane & 31, h = lane >> 5;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] = tile[wave][row][k * 16 + h * 8 + e];
            b[e] = tile[wave][k * 16 + h * 8 + e][row];
        }
        Frag2 f;
        split8(a, f);
        u32x4_t *x = w.x + batch * w.bx + ((r0 / 32 * (w.Lp / 16) + c0 / 16 + k) * 2) * 64 + lane;
        x[0] = __builtin_bit_cast(u32x4_t, f.p[0]);
        x[64] = __builtin_bit_cast(u32x4_t, f.p[1]);
        split8(b, f);
        u32x4_t *xt = w.xt[0] + batch * w.bx + ((c0 / 32 * (w.Sp / 16) + r0 / 16 + k) * 2) * 64 + lane;
        xt[0] = __builtin_bit_cast(u32x4_t, f.p[0]);
        xt[64] = __builtin_bit_cast(u32x4_t, f.p[1]);
    }
}

// The three products of a step (and the last one, into the caller's matrix).
enum Mode { kGram, kPoly, kUpdate, kLast };

struct Prod {
    const u32x4_t *p, *q;     // fragment matrices: rows of the result, columns of the result
    int64_t bp, bq;         // batch strides
    int64_t KS;             // 16-column steps of both
    int64_t tiles, tm;      // tiles, and those along the rows (kUpdate, kLast)
    u32x4_t *d0, *d1;         // result as rows = its columns (straight) and rows = its rows (turned)
    int64_t KS0, KS1, b0, b1;
    const u32x4_t *add;       // what is added, with d0's layout
    int64_t badd;
    float f_add, f_mul;     // result = f_add add + f_mul product
    const double *power;    // first powers, kSumBlocks + 1 apart
    int32_t step;
    Growth growth;
    int64_t splits, per;    // of the contraction, in 16-column steps (256-high tiles)
    float4 *part;
};

// The factors of a step's sums, with the powers of two that X and A are held times.
struct Factors {
    float add, mul;
    int k;  // the result's power (kLast)
};
// (its first power is read at a kernel's start, so that no load stands between the products and their results)
template <int MODE>
__device__ __forceinline__ int power_at(const Prod &a, int64_t batch) {
    return MODE == kGram ? 0 : __builtin_amdgcn_readfirstlane((int)a.power[batch * (kSumBlocks + 1)]);
}
template <int MODE>
__device__ __forceinline__ Factors factors_of(const Prod &a, int k0) {
    if constexpr (MODE == kGram) return {0.f, 1.f, 0};
    const int k = power_of(k0, a.step, a.growth);
    if constexpr (MODE == kPoly) return {ldexpf(a.f_add, -2 * k), ldexpf(a.f_mul, -4 * k), 0};
    const int next = power_of(k0, a.step + 1, a.growth);
    return {ldexpf(a.f_add, next - k), ldexpf(a.f_mul, next - k), next};
}

// One 32 x 32 block at (m0, n0): scaled, added to, written both ways.  `turn` is a wave's 32 x 33 floats.
template <int MODE, class T>
__device__ __forceinline__ void emit(const Prod &a, const Mat &out, T *y, int64_t batch, int64_t m0, int64_t n0,
                                     bool mirror, const Factors &f, const f32x16_t &acc, float (*turn)[33], int lane) {
    constexpr float down = 1.f / (1 << kScale);
    float v[16];
    if constexpr (MODE == kGram) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = acc[i] * down;
    } else {
        get_block(a.add + batch * a.badd, n0 / 32, a.KS0, m0, v, lane);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = fmaf(f.add, v[i], f.mul * (acc[i] * down));
    }
    if constexpr (MODE == kLast) {
        T *dst = y + batch * out.sb;
        const int64_t c = n0 + (lane & 31);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t r = m0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
            if (r < out.S && c < out.L) dst[r * out.sr + c * out.sc] = (T)ldexpf(v[i] * down, -f.k);
        }
        return;
    }
    put_block(a.d0 + batch * a.b0, n0 / 32, a.KS0, m0, v, lane);
    if (!mirror) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) turn[8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)][lane & 31] = v[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = turn[lane & 31][k * 16 + 8 * (lane >> 5) + e];
        Frag2 fr;
        split8(r, fr);
        u32x4_t *d = a.d1 + batch * a.b1 + ((m0 / 32 * a.KS1 + n0 / 16 + k) * 2) * 64 + lane;
        d[0] = __builtin_bit_cast(u32x4_t, fr.p[0]);
        d[64] = __builtin_bit_cast(u32x4_t, fr.p[1]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The tile of a workgroup: each XCD (blockIdx % 8) takes a run of consecutive tiles, so that tiles which
// share operand rows share an L2.  False for the surplus workgroups of the last run.
// A tile is R times as high as wide.
__device__ __forceinline__ int64_t tile_id() {
    return (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
}
template <int MODE, int R>
__device__ __forceinline__ bool tile_of(const Prod &a, int64_t &m, int64_t &n) {
    const int64_t id = tile_id();
    if (id >= a.tiles) return false;
    if constexpr (MODE == kGram || MODE == kPoly) {  // tiles that reach the diagonal or below, row by row
        auto before = [](int64_t row) { return R * row * (row + 1) / 2; };
        m = (int64_t)((sqrtf(8.f / R * (float)id + 1.f) - 1.f) * 0.5f);
        while (before(m) > id) --m;
        while (before(m + 1) <= id) ++m;
        n = id - before(m);
    } else {  // column by column
        m = id % a.tm;
        n = id / a.tm;
    }
    return true;
}

// Few tiles: BT x BT blocks a workgroup, the contraction dealt out to its NW waves, which load fragments
// straight from memory (four steps in flight) and join their sums in LDS in wave order.  A long
// contraction is dealt out to workgroups first (ns_join_blocks adds theirs).
template <int MODE, class T, int BT, int NW>
__global__ __launch_bounds__(NW * 64) void ns_prod_split(Prod a, Mat out, T *y) {
    __shared__ float part[NW][BT * BT][16][64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int64_t batch = blockIdx.y / a.splits, split = blockIdx.y % a.splits;
    const int64_t k0 = split * a.per, k1 = k0 + a.per < a.KS ? k0 + a.per : a.KS;
    int64_t tm, tn;
    if (!tile_of<MODE, 1>(a, tm, tn)) return;
    const int k_first = power_at<MODE>(a, batch);
    const u32x4_t *p = a.p + batch * a.bp, *q = a.q + batch * a.bq;
    f32x16_t acc[BT][BT];
#pragma unroll
    for (int i = 0; i < BT * BT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i / BT][i % BT][r] = 0.f;
    auto multiply = [&](int64_t k, auto steps) {
        constexpr int N = decltype(steps)::value;
        Frag2 fp[N][BT], fq[N][BT];
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
            for (int i = 0; i < BT; ++i) {
                load2(p, (tm * BT + i) * a.KS + k + s * NW, lane, fp[s][i]);
                load2(q, (tn * BT + i) * a.KS + k + s * NW, lane, fq[s][i]);
            }
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
            for (int i = 0; i < BT; ++i)
                mfma_row<SplitF32, BT>(fp[s][i], [&](int n) -> const Frag2 & { return fq[s][n]; }, acc[i]);
    };
    int64_t k = k0 + wave;
    for (; k + 3 * NW < k1; k += 4 * NW) multiply(k, std::integral_constant<int, 4>());
    for (; k < k1; k += NW) multiply(k, std::integral_constant<int, 1>());
#pragma unroll
    for (int i = 0; i < BT * BT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) part[wave][i][r][lane] = acc[i / BT][i % BT][r];
    __syncthreads();
    f32x16_t s;
    if (wave < BT * BT) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = part[0][wave][r][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) s[r] += part[w][wave][r][lane];
        }
    }
    __syncthreads();
    if (wave >= BT * BT) return;
    if (a.splits > 1) {
        float4 *d = a.part + (((batch * a.splits + split) * a.tiles + tile_id()) * BT * BT + wave) * 256 + lane;
#pragma unroll
        for (int g = 0; g < 4; ++g) d[g * 64] = make_float4(s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]);
        return;
    }
    const bool mirror = MODE == kUpdate || tm != tn;
    emit<MODE, T>(a, out, y, batch, (tm * BT + wave / BT) * 32, (tn * BT + wave % BT) * 32, mirror,
                  factors_of<MODE>(a, k_first), s,
                  reinterpret_cast<float (*)[33]>(&part[wave * (BT == 1 ? 2 : 1)][0][0][0]), lane);
}

// The workgroups' partial sums in split order, a wave a block.
__device__ __forceinline__ f32x16_t join_block(const Prod &a, int64_t batch, int64_t block, int64_t blocks, int lane) {
    f32x16_t s;
    for (int64_t k = 0; k < a.splits; ++k) {
        const float4 *d = a.part + (((batch * a.splits + k) * a.tiles + tile_id()) * blocks + block) * 256 + lane;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v = d[g * 64];
            s[4 * g] = k ? s[4 * g] + v.x : v.x;
            s[4 * g + 1] = k ? s[4 * g + 1] + v.y : v.y;
            s[4 * g + 2] = k ? s[4 * g + 2] + v.z : v.z;
            s[4 * g + 3] = k ? s[4 * g + 3] + v.w : v.w;
        }
    }
    return s;
}

template <int MODE, class T, int BT>
__global__ __launch_bounds__(BT * BT * 64) void ns_join_blocks(Prod a, Mat out, T *y) {
    __shared__ float turn[BT * BT][32][33];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int64_t tm, tn;
    if (!tile_of<MODE, 1>(a, tm, tn)) return;
    const int k_first = power_at<MODE>(a, blockIdx.y);
    emit<MODE, T>(a, out, y, blockIdx.y, (tm * BT + wave / BT) * 32, (tn * BT + wave % BT) * 32,
                  MODE == kUpdate || tm != tn, factors_of<MODE>(a, k_first), join_block(a, blockIdx.y, wave, BT * BT, lane), turn[wave], lane);
}

// Many tiles: 256 x 128 a workgroup, four waves of 128 x 64 (one a SIMD, half the register file in
// sums), two 16-column steps at a time.  The rows' operand goes through double-buffered LDS (one
// barrier a stage), the columns' straight to registers.  A wave's 24 MFMAs a step need 12 KB of
// operands: 43 bytes a clock and CU from LDS and 21 into it, 43 from the vector cache, of 128 and 64.
// With fewer tiles than CUs the contraction is split as well, into partial sums that ns_join adds.
// The update of 2048 x 4096 takes 114 us, 900 TFLOP/s of 16-bit products; the library's fp16 product of
// 8192^3 reaches 1555 here.
template <int MODE, class T>
__global__ __launch_bounds__(kThreads, 1) void ns_prod256(Prod a, Mat out, T *y) {
    constexpr int ST = 8 * 2 * 2 * 64;  // 16-byte groups of a stage: 8 row blocks, 2 steps, 2 planes
    __shared__ u32x4_t lds[2][ST];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wm = wave >> 1, wn = wave & 1;
    const int64_t batch = blockIdx.y / a.splits, split = blockIdx.y % a.splits;
    int64_t tm, tn;
    if (!tile_of<MODE, 2>(a, tm, tn)) return;
    const int k_first = power_at<MODE>(a, batch);
    const int64_t k0 = split * a.per, k1 = k0 + a.per < a.KS ? k0 + a.per : a.KS;
    // thread t stages 16 bytes of each row block: 256 threads are the block's 2 steps of 2 planes
    const u32x4_t *p = a.p + batch * a.bp + tm * 8 * a.KS * 128 + t;
    const u32x4_t *q = a.q + batch * a.bq;
    auto fetch = [&](int64_t k, u32x4_t (&sp)[8]) {
        k = k < k1 ? k : k1 - 2;
#pragma unroll
        for (int i = 0; i < 8; ++i) sp[i] = p[(i * a.KS + k) * 128];
    };
    auto stage = [&](int buf, const u32x4_t (&sp)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[buf][i * 256 + t] = sp[i];
    };
    auto columns = [&](int64_t k, Frag2 (&f)[2][2]) {
        k = k < k1 ? k : k1 - 2;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) load2(q, (tn * 4 + wn * 2 + i) * a.KS + k + s, lane, f[s][i]);
    };
    f32x16_t acc[4][2];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i >> 1][i & 1][r] = 0.f;
    // A stage's loads are given three stages to arrive (the columns' to their registers, the rows' two
    // to registers and one in LDS).  Past the end the last stage is loaded again: a load under a condition
    // would make the compiler wait for all loads at each use.
    u32x4_t s0[8], s1[8];
    Frag2 f0[2][2], f1[2][2], f2[2][2], f3[2][2];
    fetch(k0, s0);
    fetch(k0 + 2, s1);
    columns(k0, f0);
    columns(k0 + 2, f1);
    columns(k0 + 4, f2);
    stage(0, s0);
    fetch(k0 + 4, s0);
    __syncthreads();
    // One wave a SIMD: its own MFMAs have to cover its LDS traffic.  While a step multiplies, the next step's
    // fragments are read and (in the first step) the next stage written, a few instructions between
    // MFMAs; the barrier stands between the two steps.
    Frag2 fp0[4], fp1[4];
    auto rows = [&](int buf, int s, Frag2 (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load2(lds[buf], (wm * 4 + i) * 2 + s, lane, f[i]);
    };
    auto multiply = [&](const Frag2 (&f)[4], const Frag2 (&g)[2]) {
#pragma unroll
        for (int part = 0; part < 3; ++part)  // lo hi, hi lo, hi hi: eight sums apart
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[i][n] = mfma32(f[i].p[part == 0], g[n].p[part == 1], acc[i][n]);
    };
    rows(0, 0, fp0);
    auto step = [&](int64_t k, int buf, u32x4_t (&sp)[8], Frag2 (&now)[2][2], Frag2 (&ahead)[2][2]) {
        rows(buf, 1, fp1);
        stage(buf ^ 1, sp);
        fetch(k + 6, sp);
        columns(k + 6, ahead);
        multiply(fp0, now[0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 2, 0);  // loads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __syncthreads();
        rows(buf ^ 1, 0, fp0);
        multiply(fp1, now[1]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x008, 3, 1);
        }
    };
    for (int64_t k = k0; k < k1; k += 8) {  // KS and per are multiples of 8
        step(k, 0, s1, f0, f3);
        step(k + 2, 1, s0, f1, f0);
        step(k + 4, 0, s1, f2, f1);
        step(k + 6, 1, s0, f3, f2);
    }
    if (a.splits > 1) {
        float4 *d = a.part + (((batch * a.splits + split) * a.tiles + tile_id()) * 4 + wave) * 8 * 256 + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                d[(i * 4 + g) * 64] = make_float4(acc[i >> 1][i & 1][4 * g], acc[i >> 1][i & 1][4 * g + 1],
                                                  acc[i >> 1][i & 1][4 * g + 2], acc[i >> 1][i & 1][4 * g + 3]);
        return;
    }
    const bool mirror = MODE == kUpdate || tn < 2 * tm;  // a square's own tiles hold both its triangles
    float(*turn)[33] = reinterpret_cast<float(*)[33]>(reinterpret_cast<float *>(&lds[0][0]) + wave * 32 * 33);
    const Factors f = factors_of<MODE>(a, k_first);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        emit<MODE, T>(a, out, y, batch, (tm * 8 + wm * 4 + (i >> 1)) * 32, (tn * 4 + wn * 2 + (i & 1)) * 32, mirror, f,
                      acc[i >> 1][i & 1], turn, lane);
}

template <int MODE, class T>
__global__ __launch_bounds__(kThreads) void ns_join(Prod a, Mat out, T *y) {
    __shared__ float turn[4][32][33];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wm = wave >> 1, wn = wave & 1;
    int64_t tm, tn;
    if (!tile_of<MODE, 2>(a, tm, tn)) return;
    const int k_first = power_at<MODE>(a, blockIdx.y);
    const int i = blockIdx.z;  // one block of each wave's eight
    emit<MODE, T>(a, out, y, blockIdx.y, (tm * 8 + wm * 4 + (i >> 1)) * 32, (tn * 4 + wn * 2 + (i & 1)) * 32,
                  MODE == kUpdate || tn < 2 * tm, factors_of<MODE>(a, k_first), join_block(a, blockIdx.y, wave * 8 + i, 32, lane), turn[wave], lane);
}

// ------------------------------------------------------------------ host side

struct Plan {
    bool small;
    int tile;            // rows of a tile: 256 (128 wide), 64 or 32 (square)
    int64_t Sp, Lp, xsz, asz, splits_gram, splits_poly, part, bytes;
};

inline int64_t up_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
inline int64_t tri_tiles(const Plan &p) {  // tiles of a symmetric product that reach the diagonal or below
    const int64_t n = p.Sp / p.tile;
    return p.tile == 256 ? n * (n + 1) : n * (n + 1) / 2;
}

inline Plan plan_of(int64_t batch, int64_t S, int64_t L) {
    Plan p{};
    p.small = S <= 64 && L <= 256;
    if (p.small) return p;
    // the largest tiles once the update has enough of them for a good part of the chip and they are
    // not mostly padding, 64-wide ones once there are 256
    auto tiles = [&](int64_t h, int64_t w) { return ((S + h - 1) / h) * ((L + w - 1) / w) * batch; };
    const bool filled = 4 * up_to(S, 256) * up_to(L, 128) <= 5 * S * L;
    p.tile = filled && tiles(256, 128) >= 96 ? 256 : tiles(64, 64) >= 256 ? 64 : 32;
    p.Sp = up_to(S, p.tile);
    p.Lp = up_to(L, p.tile == 256 ? 128 : p.tile);
    p.xsz = p.Sp * p.Lp / 4;  // 16-byte groups: 4 bytes an element
    p.asz = p.Sp * p.Sp / 4;
    p.splits_gram = p.splits_poly = 1;
    if (p.tile < 256) {
        // long rows (X^T X of an embedding table): 2048 columns a workgroup at least, at most one a CU
        p.splits_gram = std::max<int64_t>(1, std::min<int64_t>(256 / (tri_tiles(p) * batch), p.Lp / 2048));
        p.part = p.splits_gram > 1 ? batch * p.splits_gram * tri_tiles(p) * p.tile * p.tile / 4 : 0;
    } else {
        // one workgroup a CU: as many splits as keep to 256 of them, 512 columns each at least
        auto splits = [&](int64_t K) {
            return std::max<int64_t>(1, std::min<int64_t>(256 / (tri_tiles(p) * batch), K / 512));
        };
        p.splits_gram = splits(p.Lp);
        p.splits_poly = splits(p.Sp);
        const int64_t most = std::max(p.splits_gram, p.splits_poly);
        p.part = most > 1 ? batch * most * tri_tiles(p) * 256 * 128 / 4 : 0;
    }
    p.bytes = batch * (3 * p.xsz + 2 * p.asz) * 16 + p.part * 16 + batch * (kSumBlocks + 1) * 8;
    return p;
}

template <class T>
int run(const char *fn, const Plan &p, int64_t batch, Mat in, Mat out, const void *g, void *y, int32_t steps, float ca,
        float cb, float cc, double eps, Growth growth, void *ws, hipStream_t st) {
    const T *src = static_cast<const T *>(g);
    T *dst = static_cast<T *>(y);
    if (p.small) {
        const dim3 gr((unsigned)batch), b(kThreads);
        if (in.L <= 64) hipLaunchKernelGGL((ns_small<T, 1>), gr, b, 0, st, in, out, src, dst, steps, ca, cb, cc, eps, growth);
        else if (in.L <= 128) hipLaunchKernelGGL((ns_small<T, 2>), gr, b, 0, st, in, out, src, dst, steps, ca, cb, cc, eps, growth);
        else hipLaunchKernelGGL((ns_small<T, 4>), gr, b, 0, st, in, out, src, dst, steps, ca, cb, cc, eps, growth);
        return launch_status(fn);
    }
    Work w{};
    u32x4_t *c = static_cast<u32x4_t *>(ws);
    w.x = c, c += batch * p.xsz;
    w.xt[0] = c, c += batch * p.xsz;
    w.xt[1] = c, c += batch * p.xsz;
    w.a = c, c += batch * p.asz;
    w.q = c, c += batch * p.asz;
    float4 *partial = reinterpret_cast<float4 *>(c);
    c += p.part;
    double *part = reinterpret_cast<double *>(c);
    w.bx = p.xsz, w.ba = p.asz, w.Sp = p.Sp, w.Lp = p.Lp;
    const unsigned nb = (unsigned)batch;
    hipLaunchKernelGGL((ns_sumsq<T>), dim3(kSumBlocks, nb), dim3(kThreads), 0, st, in, src, part);
    const int64_t blocks = (p.Sp / 32) * (p.Lp / 32);
    hipLaunchKernelGGL((ns_pack<T>), dim3((unsigned)((blocks + 3) / 4), nb), dim3(kThreads), 0, st, in, src, part, eps, w);
    const int64_t ts = p.Sp / p.tile, tl = p.Lp / (p.tile == 256 ? 128 : p.tile);
    const int64_t tri = tri_tiles(p), all = ts * tl;
    const int64_t ks = p.Sp / 16, kl = p.Lp / 16;
    const double *power = part + kSumBlocks;
    auto go = [&](auto mode, Prod a, int64_t splits) {
        constexpr int M = decltype(mode)::value;
        const unsigned n = (unsigned)((a.tiles + 7) / 8 * 8);
        a.per = up_to((a.KS + splits - 1) / splits, 8);
        a.splits = (a.KS + a.per - 1) / a.per;
        a.part = partial;
        if (p.tile == 256) {
            hipLaunchKernelGGL((ns_prod256<M, T>), dim3(n, nb * (unsigned)a.splits), dim3(kThreads), 0, st, a, out, dst);
            if (a.splits > 1)
                hipLaunchKernelGGL((ns_join<M, T>), dim3(n, nb, 8), dim3(kThreads), 0, st, a, out, dst);
        } else if (p.tile == 64) {
            hipLaunchKernelGGL((ns_prod_split<M, T, 2, 4>), dim3(n, nb * (unsigned)a.splits), dim3(256), 0, st, a, out, dst);
            if (a.splits > 1) hipLaunchKernelGGL((ns_join_blocks<M, T, 2>), dim3(n, nb), dim3(256), 0, st, a, out, dst);
        } else {
            hipLaunchKernelGGL((ns_prod_split<M, T, 1, 8>), dim3(n, nb * (unsigned)a.splits), dim3(512), 0, st, a, out, dst);
            if (a.splits > 1) hipLaunchKernelGGL((ns_join_blocks<M, T, 1>), dim3(n, nb), dim3(64), 0, st, a, out, dst);
        }
    };
    for (int32_t s = 0; s < steps; ++s) {
        u32x4_t *cur = w.xt[s & 1], *nxt = w.xt[(s + 1) & 1];
        go(std::integral_constant<int, kGram>(),
           Prod{w.x, w.x, w.bx, w.bx, kl, tri, 0, w.a, w.a, ks, ks, w.ba, w.ba, nullptr, 0, 0.f, 1.f, power, s, growth, 1, 0, nullptr},
           p.splits_gram);
        go(std::integral_constant<int, kPoly>(),
           Prod{w.a, w.a, w.ba, w.ba, ks, tri, 0, w.q, w.q, ks, ks, w.ba, w.ba, w.a, w.ba, cb, cc, power, s, growth, 1, 0, nullptr},
           p.splits_poly);
        const Prod u{w.q, cur, w.ba, w.bx, ks, all, ts, nxt, w.x, ks, kl, w.bx, w.bx, cur, w.bx, ca, 1.f, power, s, growth, 1, 0, nullptr};
        if (s + 1 < steps) go(std::integral_constant<int, kUpdate>(), u, 1);
        else go(std::integral_constant<int, kLast>(), u, 1);
    }
    return launch_status(fn);
}

// The fixed scale holds X up to 4 and Q up to 16: follow the interval [0, hi] of singular values through the
// steps, each image's bound from the ends and the critical points of the odd quintic.
inline bool coefficients_fit(int32_t steps, double a, double b, double c) {
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    double hi = 1.;
    for (int32_t s = 0; s < steps; ++s) {
        double x = 0., q = 0.;
        auto at = [&](double l) {  // l = sigma^2
            if (l < 0. || l > hi * hi) return;
            q = std::max(q, std::fabs(b * l + c * l * l));
            x = std::max(x, std::sqrt(l) * std::fabs(a + b * l + c * l * l));
        };
        at(hi * hi);
        if (c != 0.) {
            at(-b / (2. * c));  // of b l + c l^2
            const double d = 9. * b * b - 20. * a * c;  // a + 3 b l + 5 c l^2 = 0
            if (d >= 0.) {
                at((-3. * b + std::sqrt(d)) / (10. * c));
                at((-3. * b - std::sqrt(d)) / (10. * c));
            }
        } else if (b != 0.) {
            at(-a / (3. * b));
        }
        if (!(x <= 4.) || !(q <= 16.)) return false;
        hi = x * (1. + 1e-5);  // roundings
    }
    return true;
}

// ------------------------------------------------------------------ around the products

constexpr int kSlotBlocks = 64;  // workgroups a slot, striding over it

struct Slots {
    igr_muon_slot s[IGR_MUON_MAX_SLOTS];
};

// Elementwise: a launch reads and writes each weight's arrays once.  The dense layers of a recommender are bound by the
// launch (six of 64 x 64: 8 us); one of 2048 x 4096 takes 40 us (3.4 TB/s), its apply 44 (2.3 TB/s), four bytes a
// lane on at most 256 workgroups.
__global__ __launch_bounds__(kThreads) void muon_direction(Slots a, float mu, int32_t nesterov) {
    const igr_muon_slot s = a.s[blockIdx.y];
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < s.n; i += (int64_t)gridDim.x * kThreads) {
        const float g = s.grad[i], m = fmaf(mu, s.momentum[i], g);
        s.momentum[i] = m;
        s.direction[i] = nesterov ? fmaf(mu, m, g) : m;
    }
}

__global__ __launch_bounds__(kThreads) void muon_apply(Slots a, float keep, float step) {
    const igr_muon_slot s = a.s[blockIdx.y];
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < s.n; i += (int64_t)gridDim.x * kThreads)
        s.param[i] = fmaf(-step, s.direction[i], keep * s.param[i]);
}

inline int take_slots(const char *fn, int32_t n_slots, const igr_muon_slot *slots, bool direction, Slots &a,
                      unsigned &blocks) {
    if (n_slots < 0 || n_slots > IGR_MUON_MAX_SLOTS) return arg_error(fn, "0 <= n_slots <= IGR_MUON_MAX_SLOTS");
    if (n_slots > 0 && !slots) return arg_error(fn, "NULL slots");
    int64_t most = 1;
    for (int k = 0; k < n_slots; ++k) {
        const igr_muon_slot &s = slots[k];
        if (s.n <= 0) return arg_error(fn, "slot size must be positive");
        if (!s.direction || (direction ? !s.grad || !s.momentum : !s.param)) return arg_error(fn, "NULL pointer in a slot");
        a.s[k] = s;
        most = std::max(most, (s.n + kThreads - 1) / kThreads);
    }
    blocks = (unsigned)std::min<int64_t>(most, n_slots > 4 ? kSlotBlocks : 4 * kSlotBlocks);
    return IGR_OK;
}

}  // namespace
}  // namespace igr

using namespace igr;

extern "C" int igr_muon_direction_f32(int32_t n_slots, const igr_muon_slot *slots, double mu, int32_t nesterov,
                                      void *stream) {
    return guarded("igr_muon_direction_f32", [&]() -> int {
        const char *fn = "igr_muon_direction_f32";
        Slots a;
        unsigned blocks = 0;
        if (int rc = take_slots(fn, n_slots, slots, true, a, blocks)) return rc;
        if (n_slots == 0) return IGR_OK;
        hipLaunchKernelGGL(muon_direction, dim3(blocks, (unsigned)n_slots), dim3(kThreads), 0,
                           reinterpret_cast<hipStream_t>(stream), a, (float)mu, nesterov);
        return launch_status(fn);
    });
}

extern "C" int igr_muon_apply_f32(int32_t n_slots, const igr_muon_slot *slots, double lr, double weight_decay,
                                  double scale, void *stream) {
    return guarded("igr_muon_apply_f32", [&]() -> int {
        const char *fn = "igr_muon_apply_f32";
        Slots a;
        unsigned blocks = 0;
        if (int rc = take_slots(fn, n_slots, slots, false, a, blocks)) return rc;
        if (n_slots == 0) return IGR_OK;
        hipLaunchKernelGGL(muon_apply, dim3(blocks, (unsigned)n_slots), dim3(kThreads), 0,
                           reinterpret_cast<hipStream_t>(stream), a, (float)(1. - lr * weight_decay), (float)(lr * scale));
        return launch_status(fn);
    });
}

extern "C" int64_t igr_newton_schulz_workspace_size(int64_t batch, int64_t rows, int64_t cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    return plan_of(batch, std::min(rows, cols), std::max(rows, cols)).bytes;
}

extern "C" int igr_newton_schulz(int32_t dtype, int64_t batch, int64_t rows, int64_t cols, const void *g, int64_t ldg,
                                 int64_t stride_g, int32_t steps, double a, double b, double c, double eps, void *out,
                                 void *workspace, int64_t ws_bytes, void *stream) {
    return guarded("igr_newton_schulz", [&]() -> int {
        const char *fn = "igr_newton_schulz";
        if (dtype < kF32 || dtype > kF16) return arg_error(fn, "unknown dtype");
        if (batch < 0 || rows < 0 || cols < 0) return arg_error(fn, "negative size");
        if (ldg < cols || (batch > 1 && stride_g < 0)) return arg_error(fn, "leading dimension too small");
        if (steps < 1 || steps > 100) return arg_error(fn, "steps outside 1..100");
        if (!(eps >= 0.) || !std::isfinite(eps)) return arg_error(fn, "eps must be finite and not negative");
        if (!coefficients_fit(steps, a, b, c))
            return arg_error(fn, "the coefficients drive singular values out of the range that is held");
        if (batch == 0 || rows == 0 || cols == 0) return IGR_OK;
        if (batch > 65535 || rows > (1 << 24) || cols > (1 << 24) || std::min(rows, cols) > (1 << 15))
            return arg_error(fn, "too large: at most 65535 matrices, sides of 2^24, the shorter 2^15");
        const int64_t S = std::min(rows, cols), L = std::max(rows, cols);
        const Plan p = plan_of(batch, S, L);
        if (!p.small && (p.Sp / 32 * (p.Lp / 32) / 4 > INT32_MAX || batch * std::max(p.splits_gram, p.splits_poly) > 65535))
            return arg_error(fn, "too many tiles");
        if (!g || !out) return arg_error(fn, "null pointer");
        if (p.bytes > 0 && (!workspace || ws_bytes < p.bytes || !aligned16(workspace)))
            return arg_error(fn, "workspace too small or not 16-byte aligned");
        const bool flip = rows > cols;
        const Mat in{S, L, flip ? 1 : ldg, flip ? ldg : 1, stride_g};
        const Mat to{S, L, flip ? 1 : cols, flip ? cols : 1, rows * cols};
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        const float fa = (float)a, fb = (float)b, fc = (float)c;
        const Growth growth{std::fabs(a), std::fabs(b), std::fabs(c)};
        if (dtype == kF32) return run<float>(fn, p, batch, in, to, g, out, steps, fa, fb, fc, eps, growth, workspace, st);
        if (dtype == kBF16) return run<__bf16>(fn, p, batch, in, to, g, out, steps, fa, fb, fc, eps, growth, workspace, st);
        return run<_Float16>(fn, p, batch, in, to, g, out, steps, fa, fb, fc, eps, growth, workspace, st);
    });
}
