// int8.hip - serving from 8-bit tables (gfx950 matrix cores): the row quantiser and the product of
// two quantised tables.
//
//   quantise:  a_r = max_k |x_rk|,  q_rk = rint(x_rk / a_r * 127),  s_r = a_r / 127
//   product:   y_mn = (sum_k a_mk b_nk) sa_m sb_n       sums exact in 32-bit integers
//
// The quantiser reads a table once and writes a quarter (a half) of it: bound by memory (10^6 x 64
// floats: 71 us, 4.5 TB/s; rows that are not whole 16-byte groups go by single elements: 66 floats 185 us, 100 bf16
// 213 us).  The
// product of a catalogue ranking has K = 32..256 and a result of 4 M N bytes, which is nearly all of its
// traffic: bound by the stores.  A single user's row is bound by reading the item table once
// (10^6 x 64: 17 us, 4.2 TB/s; 20,000 x 2048: 20 us, 2.0 TB/s, each wave walking all of K).
// Only wide products (K in the hundreds and above) are bound by the matrix cores.
//
// A 32x32x32 MFMA takes 16 consecutive bytes of a row from each lane, which is how the tables
// lie in memory, so narrow products load their operands straight into registers; wide
// ones stage 128 rows x 64 bytes of each table in LDS, in lane order, for four waves.
#include <algorithm>
#include <type_traits>

#include "half_split.h"

namespace igr {
namespace {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
typedef int32_t i32x16_t __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;

// ------------------------------------------------------------------ quantiser

// G lanes share a row, each holding R groups of VE consecutive elements (VE = 1: any alignment).
// Rows longer than G R VE are read a second time.
template <class T, int VE, int R>
__global__ __launch_bounds__(kThreads) void quantize_rows(int64_t n, int32_t k, int32_t g, const T *__restrict__ x,
                                                          int64_t ldx, int8_t *__restrict__ q, int64_t ldq,
                                                          float *__restrict__ scale) {
    const int lane = threadIdx.x & (g - 1);
    const int64_t row = (flat_group() * kThreads + threadIdx.x) / g;
    if (row >= n) return;  // whole groups leave together
    const T *xr = x + row * ldx;
    struct alignas(sizeof(T) * VE) Vec {
        T e[VE];
    };
    Vec v[R];
    uint32_t bits = 0;  // of the largest magnitude: NaN above infinity above the finite
    auto take = [&](const Vec &w) {
#pragma unroll
        for (int i = 0; i < VE; ++i)
            bits = max(bits, __builtin_bit_cast(uint32_t, (float)w.e[i]) & 0x7fffffffu);
    };
    const int step = g * VE;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = r * step + lane * VE;
        if (c < k) {
            v[r] = *reinterpret_cast<const Vec *>(xr + c);
            take(v[r]);
        }
    }
    for (int c = R * step + lane * VE; c < k; c += step) take(*reinterpret_cast<const Vec *>(xr + c));
    for (int o = g / 2; o; o >>= 1) bits = max(bits, (uint32_t)__shfl_xor((int)bits, o, 64));
    const bool finite = bits < 0x7f800000u;
    const float amax = __builtin_bit_cast(float, bits);
    if (lane == 0) scale[row] = finite ? amax / 127.f : __builtin_nanf("");
    const bool live = finite && bits != 0;
    const float by = live ? amax : 1.f;
    auto put = [&](const Vec &w, int c) {
        struct alignas(VE) Out {
            int8_t e[VE];
        } o;
#pragma unroll
        for (int i = 0; i < VE; ++i) o.e[i] = live ? (int8_t)rintf((float)w.e[i] / by * 127.f) : (int8_t)0;
        *reinterpret_cast<Out *>(q + row * ldq + c) = o;
    };
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = r * step + lane * VE;
        if (c < k) put(v[r], c);
    }
    for (int c = R * step + lane * VE; c < k; c += step) put(*reinterpret_cast<const Vec *>(xr + c), c);
    for (int64_t c = k + lane; c < ldq; c += g) q[row * ldq + c] = 0;  // the row's padding
}

template <class T>
int launch_quantize(int64_t n, int32_t k, const void *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale,
                    hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = k % V == 0 && ldx % V == 0 && ldq % V == 0 && aligned16(x) &&
                     reinterpret_cast<uintptr_t>(q) % V == 0;
    const int ve = vec ? V : 1;
    int g = 1;  // lanes a row: enough for four groups each
    while (g < 64 && g * ve * 4 < k) g *= 2;
    while (g < 64 && vec && g * ve < k && g < 16) g *= 2;  // and 16-lane rows where they are that long
    const int64_t grid = (n * g + kThreads - 1) / kThreads;
    if (grid > INT32_MAX) return arg_error("igr_quantize_rows", "too many rows");
    const T *xt = static_cast<const T *>(x);
    const dim3 gr = flat_grid(grid), b(kThreads);
    if (vec) {
        if (g * ve * 2 >= k) hipLaunchKernelGGL((quantize_rows<T, V, 2>), gr, b, 0, st, n, k, g, xt, ldx, q, ldq, scale);
        else hipLaunchKernelGGL((quantize_rows<T, V, 8>), gr, b, 0, st, n, k, g, xt, ldx, q, ldq, scale);
    } else {
        hipLaunchKernelGGL((quantize_rows<T, 1, 8>), gr, b, 0, st, n, k, g, xt, ldx, q, ldq, scale);
    }
    return launch_status("igr_quantize_rows");
}

// ------------------------------------------------------------------ product

struct MulArgs {
    int64_t M, N, ldc;
    int64_t lda, ldb;
    int32_t K;
    const int8_t *a, *b;
    const float *sa, *sb;
    void *c;
    int64_t tm, tn;  // tiles
};

// 16 bytes of a row from column k on, zeros past its end; any alignment.  The last group is
// taken from the row's last 16 bytes, so that nothing past the row is read.
__device__ __forceinline__ i32x4_t row_chunk(const int8_t *row, int k, int K) {
    i32x4_t v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else if (k < K) {
        if (K >= 16) {
            unsigned __int128 w;
            __builtin_memcpy(&w, row + K - 16, 16);
            w >>= 8 * (16 - (K - k));
            __builtin_memcpy(&v, &w, 16);
        } else {
            unsigned __int128 w = 0;
            for (int i = K - 1; i >= k; --i) w = w << 8 | (uint8_t)row[i];
            __builtin_memcpy(&v, &w, 16);
        }
    }
    return v;
}

// Result tile of MB x NB blocks of 32 x 32: lane l holds column l % 32, register i row
// 8 (i/4) + 4 (l/32) + i%4.  A store writes 32 consecutive columns of two rows.  m0 and n0 are the
// same in all lanes.
template <class T, int MB, int NB>
__device__ __forceinline__ void store_tile(const MulArgs &g, int64_t m0, int64_t n0, const i32x16_t (&acc)[MB][NB],
                                           int lane) {
    const int col = lane & 31, h = lane >> 5;
    float sb[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int64_t n = n0 + j * 32 + col;
        sb[j] = g.sb[n < g.N ? n : g.N - 1];
    }
    T *c = static_cast<T *>(g.c) + m0 * g.ldc + n0;
    if (m0 + MB * 32 <= g.M && n0 + NB * 32 <= g.N && g.ldc < (1 << 26)) {
        // whole tile: rows by a uniform base, the lane's part of the address once, in 32 bits
        const uint32_t at = (uint32_t)(4 * h * g.ldc + col);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float sa[4];
                __builtin_memcpy(sa, g.sa + m0 + i * 32 + q * 8 + h * 4, 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    T *row = c + (i * 32 + q * 8 + r) * g.ldc;
#pragma unroll
                    for (int j = 0; j < NB; ++j) row[at + j * 32] = (T)((float)acc[i][j][q * 4 + r] * sa[r] * sb[j]);
                }
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int dm = i * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
            if (m0 + dm >= g.M) continue;
            const float sa = g.sa[m0 + dm];
#pragma unroll
            for (int j = 0; j < NB; ++j)
                if (n0 + j * 32 + col < g.N) c[dm * g.ldc + j * 32 + col] = (T)((float)acc[i][j][r] * sa * sb[j]);
        }
}

// The tile of a workgroup.  Each XCD (blockIdx % 8) takes a run of consecutive tiles along the rows of the
// result, so that the cache lines which neighbouring tiles share are completed in one L2 before they
// go out (6550 x 40,981 floats: 220 us, 4.8 TB/s; with the tiles dealt
// out in turn the stores took half as long again).
__device__ __forceinline__ bool tile_of(const MulArgs &g, int64_t &tm, int64_t &tn) {
    const int64_t id = (int64_t)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    tm = id / g.tn;
    tn = id % g.tn;
    return id < g.tm * g.tn;
}

// Narrow products and few rows: operands straight from memory.  WM x (4 / WM) waves of MB x NB blocks.
template <class T, int MB, int NB, int WM>
__global__ __launch_bounds__(kThreads) void mul_direct(MulArgs g) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t tm, tn;
    if (!tile_of(g, tm, tn)) return;
    const int64_t m0 = (tm * WM + wave % WM) * MB * 32, n0 = (tn * (4 / WM) + wave / WM) * NB * 32;
    if (m0 >= g.M || n0 >= g.N) return;
    const int8_t *pa[MB], *pb[NB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {  // rows past the end: the last one again, not stored
        const int64_t m = m0 + i * 32 + (lane & 31);
        pa[i] = g.a + (m < g.M ? m : g.M - 1) * g.lda;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int64_t n = n0 + j * 32 + (lane & 31);
        pb[j] = g.b + (n < g.N ? n : g.N - 1) * g.ldb;
    }
    i32x16_t acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int h16 = (lane >> 5) * 16;
    auto multiply = [&](int k, auto whole) {
        i32x4_t fa[MB], fb[NB];
        auto chunk = [&](const int8_t *row) {
            i32x4_t v;
            if constexpr (decltype(whole)::value) __builtin_memcpy(&v, row + k + h16, 16);
            else v = row_chunk(row, k + h16, g.K);
            return v;
        };
#pragma unroll
        for (int i = 0; i < MB; ++i) fa[i] = chunk(pa[i]);
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[j] = chunk(pb[j]);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
    };
    int k = 0;
    for (; k + 64 <= g.K; k += 64) {
        multiply(k, std::true_type());
        multiply(k + 32, std::true_type());
    }
    for (; k + 32 <= g.K; k += 32) multiply(k, std::true_type());
    if (k < g.K) multiply(k, std::false_type());
    store_tile<T, MB, NB>(g, m0, n0, acc, lane);
}

// Wide products: 128 x 128 results a workgroup (four waves of 64 x 64), 64 bytes of K a step,
// double-buffered in LDS in fragment order (one barrier a step).  32 KB of LDS leave room for four
// workgroups on a CU: 1999 x 12,345 x 1000 to bf16 takes 80 us, 107 with steps of 128 bytes and two
// workgroups.  4096^3 reaches 1160 TOP/s; LDS, which moves 170 bytes for each clock of the full MFMA
// rate and can 128, bounds it.
constexpr int kBK = 64, kTile = 128;
template <class T>
__global__ __launch_bounds__(kThreads, 4) void mul_tiled(MulArgs g) {
    __shared__ i32x4_t lds[2][2][kTile * kBK / 16];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    int64_t tm, tn;
    if (!tile_of(g, tm, tn)) return;
    const int64_t m0 = tm * kTile, n0 = tn * kTile;
    constexpr int NCH = kTile * kBK / 16 / kThreads;  // 16-byte groups a thread stages of each table
    // group i of thread t: row t / G + i 256 / G, bytes 16 (t % G); its place: fragment (row / 32, byte / 32)
    constexpr int G = kBK / 16, RS = kThreads / G;
    const int c = t % G, r = t / G;
    const int8_t *pa[NCH], *pb[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int64_t m = m0 + r + RS * i, n = n0 + r + RS * i;
        pa[i] = g.a + (m < g.M ? m : g.M - 1) * g.lda;
        pb[i] = g.b + (n < g.N ? n : g.N - 1) * g.ldb;
    }
    auto place = [&](int i) {
        const int row = r + RS * i;
        return ((row >> 5) * (kBK / 32) + (c >> 1)) * 64 + (c & 1) * 32 + (row & 31);
    };
    i32x4_t sa[NCH], sb[NCH];
    auto fetch = [&](int k) {
        if (k + kBK <= g.K) {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                __builtin_memcpy(&sa[i], pa[i] + k + 16 * c, 16);
                __builtin_memcpy(&sb[i], pb[i] + k + 16 * c, 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                sa[i] = row_chunk(pa[i], k + 16 * c, g.K);
                sb[i] = row_chunk(pb[i], k + 16 * c, g.K);
            }
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            lds[buf][0][place(i)] = sa[i];
            lds[buf][1][place(i)] = sb[i];
        }
    };
    i32x16_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0;
    const int wm = wave & 1, wn = wave >> 1;
    fetch(0);
    stage(0);
    __syncthreads();
    int buf = 0;
    for (int k = 0; k < g.K; k += kBK, buf ^= 1) {
        const bool more = k + kBK < g.K;
        if (more) fetch(k + kBK);
#pragma unroll
        for (int s = 0; s < kBK / 32; ++s) {
            i32x4_t fa[2], fb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                fa[i] = lds[buf][0][((wm * 2 + i) * (kBK / 32) + s) * 64 + lane];
                fb[i] = lds[buf][1][((wn * 2 + i) * (kBK / 32) + s) * 64 + lane];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
        if (more) stage(buf ^ 1);
        __syncthreads();
    }
    store_tile<T, 2, 2>(g, m0 + wm * 64, n0 + wn * 64, acc, lane);
}

template <class T>
int launch_mul(const char *fn, MulArgs g, hipStream_t st) {
    auto go = [&](auto kernel, int64_t bm, int64_t bn) -> int {
        g.tm = (g.M + bm - 1) / bm;
        g.tn = (g.N + bn - 1) / bn;
        const int64_t n = (g.tm * g.tn + 7) / 8 * 8;
        if (n > kMaxGroups) return arg_error(fn, "too many result tiles");
        hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(kThreads), 0, st, g);
        return launch_status(fn);
    };
    if (g.M <= 32) return go(mul_direct<T, 1, 2, 1>, 32, 256);
    if (g.K <= 256) return go(mul_direct<T, 2, 2, 2>, 128, 128);
    return go(mul_tiled<T>, kTile, kTile);
}

}  // namespace
}  // namespace igr

using namespace igr;

extern "C" int igr_quantize_rows(int32_t dtype, int64_t n, int32_t k, const void *x, int64_t ldx, int8_t *q,
                                 int64_t ldq, float *scale, void *stream) {
    return guarded("igr_quantize_rows", [&]() -> int {
        const char *fn = "igr_quantize_rows";
        if (dtype < kF32 || dtype > kF16) return arg_error(fn, "unknown dtype");
        if (n < 0 || k <= 0) return arg_error(fn, "sizes must be positive");
        if (k > (1 << 30)) return arg_error(fn, "k above 2^30");
        if (ldx < k || ldq < k) return arg_error(fn, "leading dimension too small");
        if (n == 0) return IGR_OK;
        if (!x || !q || !scale) return arg_error(fn, "null pointer");
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        if (dtype == kF32) return launch_quantize<float>(n, k, x, ldx, q, ldq, scale, st);
        if (dtype == kBF16) return launch_quantize<__bf16>(n, k, x, ldx, q, ldq, scale, st);
        return launch_quantize<_Float16>(n, k, x, ldx, q, ldq, scale, st);
    });
}

extern "C" int igr_gemm_int8(int64_t m, int64_t n, int32_t k, const int8_t *a, int64_t lda, const float *a_scale,
                             const int8_t *b, int64_t ldb, const float *b_scale, int32_t out_dtype, void *c,
                             int64_t ldc, void *stream) {
    return guarded("igr_gemm_int8", [&]() -> int {
        const char *fn = "igr_gemm_int8";
        if (out_dtype < kF32 || out_dtype > kF16) return arg_error(fn, "unknown output dtype");
        if (m < 0 || n < 0 || k <= 0) return arg_error(fn, "sizes must be positive");
        if (k > 131071) return arg_error(fn, "k above 131071: sums of 8-bit products could pass 32 bits");
        if (lda < k || ldb < k || ldc < n) return arg_error(fn, "leading dimension too small");
        if (m == 0 || n == 0) return IGR_OK;
        if (!a || !b || !a_scale || !b_scale || !c) return arg_error(fn, "null pointer");
        MulArgs g{m, n, ldc, lda, ldb, k, a, b, a_scale, b_scale, c, 0, 0};
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        if (out_dtype == kF32) return launch_mul<float>(fn, g, st);
        if (out_dtype == kBF16) return launch_mul<__bf16>(fn, g, st);
        return launch_mul<_Float16>(fn, g, st);
    });
}
