// softmax_loss.hip - softmax cross entropy over a whole item catalogue, and its gradients,
// without ever holding the logits (gfx950 matrix cores).
//
//   s_bv   = scale <x_b, w_v>                       b < B batch rows, v < V items, width d <= 256
//   loss_b = log sum_v exp(s_bv) - s_b,t(b)         0 for rows whose target is ignore_index
//   dx_b   = c_b (o_b - r_b w_t(b)),  o_b = sum_{v != t} p_bv w_v,  p_bv = exp(s_bv - lse_b)
//   dw_v   = sum_b c_b g_bv x_b,  g_bv = p_bv, at the target -r_b;   c_b = scale d(total)/d(loss_b)
//   r_b    = sum_{v != t} p_bv = 1 - p_bt, summed without the target: a row that is sure of it keeps
//            its digits (1 - p would lose them), in the loss (log(1 + r/p)) as in the gradients
//
// o_b and r_b do not depend on the incoming gradient, so the forward pass computes them along with
// the running maximum and sum (each tile of logits is used for both and dropped); the backward
// recomputes the logits once, for dw.  That is 8 B V d flops in all, where the logits
// kept would need 6 and B V floats.
//
// Layout.  Both tables are first packed into 16-bit matrix fragments (half_split.h), per block
// of 32 rows: an S part (contraction over the width: lane l holds row l % 32, eight
// consecutive columns) and a T part (contraction over the rows: lane l holds column l % 32
// and eight rows, in exactly the order in which a 32x32 MFMA leaves its results in a lane).
// So the weights p of one product are, in the registers they were made in, the operand of the next,
// and a tile is copied to LDS and read back as it lies, 16 bytes a lane, without conflicts.
//
// Forward: a workgroup of four waves holds 32 NB batch rows a wave in registers and streams a range of
// item blocks; few batch rows split the catalogue over many workgroups, whose (max, sum, o) are
// joined in split order.  Backward: the same with the roles exchanged, item rows
// in registers and batch blocks streamed; no atomics on memory, the same bits on every run.
//
// Bound by the matrix cores and, beside them, the softmax's own arithmetic (an exponential, a
// subtraction and two conversions a weight).  B = 2048, d = 64, fp32: one million items take 1.44 to 1.54 ms
// forward and 1.32 to 1.39 backward (from card to card), 1.0 to 1.2 PFLOP/s of fp16 products.  On operands
// that are not constant MFMAs alone sustain 1.56 here (2.3 on constants: the clock falls with what they
// switch), a large library product 1.55.  40,981 items take 82 and 93 us; at d = 256 (one wave a SIMD) 0.35
// and 0.31 ms with the small kernels.
//
// fp32 in fewer bits than fp32's: operands are pairs of halves (2^-23, the rows' own powers of two).  Of half
// types the argument of an exponent in the backward, which log-sum, coefficient and power of two go into
// together, is one fp32 of up to 40, so that a row's weights in dw share an error of up to 2^-20.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "half_split.h"

namespace igr {
namespace {

constexpr int kRB = 32;       // rows of a packed block
constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int64_t kWantGroups = 512;  // two workgroups on each of 256 CUs

inline int pad_width(int32_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }
__host__ __device__ inline int64_t blocks_of(int64_t rows) { return (rows + kRB - 1) / kRB; }
// 16-bit values of one packed block: S part and T part of NS planes
template <class P>
__host__ __device__ constexpr int block_halves(int dp) { return 2 * P::NS * kRB * dp; }
inline int64_t block_bytes(int32_t dtype, int dp) { return (dtype == kF32 ? 2 : 1) * 2ll * kRB * dp * 2; }
inline int64_t align256(int64_t n) { return (n + 255) & ~255ll; }

// A packed table: its blocks, then fp32's exponents, then (of the batch, for the backward) what fp32 left of the rows'
// log-sums.  A row's entries are held times 2^(14 - its exponent).  A block whose rows are within 2^kNarrow of
// each other has one exponent for all of them (its largest row's), and the kernels their short path; the digits
// of a row 2^8 below it still reach 2^-31 of its largest entry.  In the others each row has its own, however
// large its neighbours are (an item masked by an entry of -1e9 or the type's lowest value).
struct Packed {
    const u32x4_t *blocks;
    const int32_t *exps;      // per block: its largest row's, plus kWide where rows have their own
    const int8_t *row_exps;   // per row, padded to whole blocks
    const int16_t *lse_rest;  // per row, in units of rest_unit(lse2)
};
constexpr int kNarrow = 8, kWide = 1024, kZeros = -101;  // kZeros: a block of zeros
inline Packed packed_view(const void *p, int64_t rows, int32_t dtype, int dp) {
    const char *c = static_cast<const char *>(p) + blocks_of(rows) * block_bytes(dtype, dp);
    return Packed{static_cast<const u32x4_t *>(p), reinterpret_cast<const int32_t *>(c),
                  reinterpret_cast<const int8_t *>(c + blocks_of(rows) * sizeof(int32_t)),
                  reinterpret_cast<const int16_t *>(c + blocks_of(rows) * (sizeof(int32_t) + kRB))};
}
// lse2, a maximum and the log of a sum (below 32) in one fp32, is off by half its step or that log at most:
// 2^-15 of it.
__device__ __forceinline__ float rest_unit(float lse2) {
    const int step = (int)((__builtin_bit_cast(uint32_t, lse2) >> 23) & 255u) - 127 - 24;  // of half a step
    return ldexpf(1.f, min(step, 5) - 15);
}
__host__ __device__ inline int largest_exp(int e) { return e >= kWide / 2 ? e - kWide : e; }
__host__ __device__ inline bool is_wide(int e) { return e >= kWide / 2; }
// f(i, exponent of register i's row) for the 16 rows that a lane of half h holds of block k's product.  Read where
// they are used (volatile: kept from there to there they cost the short path its registers).
template <class F>
__device__ __forceinline__ void each_exp(const int8_t *row_exps, int64_t k, int h, F &&f) {
    const volatile int32_t *p = reinterpret_cast<const volatile int32_t *>(row_exps + k * kRB) + h;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int32_t v = p[2 * g];
#pragma unroll
        for (int i = 0; i < 4; ++i) f(4 * g + i, (int)(int8_t)(v >> (8 * i)));
    }
}

struct PackArgs {
    int64_t rows, ld;
    const void *src;
    u32x4_t *blocks;
    int32_t *exps;
    int8_t *row_exps;
    const int64_t *target;  // rows whose target is `ignore` are packed as zeros; NULL: none
    int64_t ignore;
};

// One block of 32 rows per workgroup; bound by its traffic (a table row is read once and written
// twice, as S and T fragments).
template <class P, int DP>
__global__ __launch_bounds__(kThreads) void pack_rows(PackArgs a0, PackArgs a1, int64_t n0, int32_t d, int32_t vec) {
    __shared__ float tile[kRB][DP + 1];
    __shared__ uint32_t rmax[kRB];  // bits of the rows' largest finite magnitudes
    const int64_t id = flat_group(), blk = id < n0 ? id : id - n0;
    const PackArgs a = id < n0 ? a0 : a1;
    if (blk * kRB >= a.rows) return;
    const typename P::elem *src = static_cast<const typename P::elem *>(a.src);
    const int64_t r0 = blk * kRB;
    const int t = threadIdx.x;
    constexpr int VE = 16 / sizeof(typename P::elem);
    if constexpr (P::kScaled) {
        if (t < kRB) rmax[t] = 0;
        __syncthreads();
    }
    // row r's magnitudes, G neighbouring lanes of it at a time
    auto note = [&](int r, float amax, auto lanes) {
        constexpr int G = decltype(lanes)::value < 64 ? decltype(lanes)::value : 64;
        if constexpr (P::kScaled) {
#pragma unroll
            for (int o = G / 2; o; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
            // in LDS; a maximum does not depend on the order
            if (t % G == 0) atomicMax(&rmax[r], __builtin_bit_cast(uint32_t, amax));
        }
    };
    auto finite = [](float v) { return fabsf(v) <= 3.402823466e38f ? fabsf(v) : 0.f; };  // finite entries set the scale
    if (vec) {  // rows of whole 16-byte groups
        for (int i = t; i < kRB * DP / VE; i += kThreads) {
            const int r = i / (DP / VE), c = (i % (DP / VE)) * VE;
            const int64_t gr = r0 + r;
            u32x4_t raw = u32x4_t{0, 0, 0, 0};
            if (gr < a.rows && c < d && !(a.target && a.target[gr] == a.ignore))
                raw = *reinterpret_cast<const u32x4_t *>(src + gr * a.ld + c);
            typename P::elem e[VE];
            __builtin_memcpy(e, &raw, 16);
            float amax = 0.f;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                tile[r][c + j] = (float)e[j];
                amax = fmaxf(amax, finite((float)e[j]));
            }
            note(r, amax, std::integral_constant<int, DP / VE>());
        }
    } else {
        for (int i = t; i < kRB * DP; i += kThreads) {
            const int r = i / DP, c = i % DP;
            const int64_t gr = r0 + r;
            float v = 0.f;
            if (gr < a.rows && c < d && !(a.target && a.target[gr] == a.ignore)) v = (float)src[gr * a.ld + c];
            tile[r][c] = v;
            note(r, finite(v), std::integral_constant<int, DP>());
        }
    }
    __syncthreads();
    const int lane = t & 63, col = lane & 31, h = lane >> 5;
    int e = 0;              // the exponent of row `col`
    float s = 1.f;          // and its scale
    bool wide = false;
    if constexpr (P::kScaled) {
        const float amax = __builtin_bit_cast(float, rmax[col]);
        e = block_exponent(amax);
        int most = e, least = amax > 0.f ? e : 127;  // rows of zeros are as narrow as any
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            most = max(most, __shfl_xor(most, o, 64));
            least = min(least, __shfl_xor(least, o, 64));
        }
        wide = __builtin_amdgcn_readfirstlane(most - least) > kNarrow;
        if (!wide || amax == 0.f) e = most;
        s = pow2f(P::kOff - e);
        if (t < kRB) a.row_exps[r0 + t] = (int8_t)e;
        if (t == 0) a.exps[blk] = least == 127 && most == -100 ? kZeros : most + (wide ? kWide : 0);
    }
    u32x4_t *out = a.blocks + blk * (block_halves<P>(DP) / 8);
    constexpr int KS = DP / 16, DB = DP / 32;
    for (int f = t >> 6; f < 2 * KS; f += kThreads / 64) {
        float v[8];
        if (f < KS) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = tile[col][f * 16 + h * 8 + i] * s;
        } else {
            const int g = f - KS, db = g >> 1, st = g & 1;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = 16 * st + 8 * (i >> 2) + 4 * h + (i & 3);
                v[i] = tile[r][db * 32 + col] * (wide ? __shfl(s, r, 64) : s);
            }
        }
        Frags<P> fr;
        split8(v, fr);
#pragma unroll
        for (int n = 0; n < P::NS; ++n) out[(f * P::NS + n) * 64 + lane] = __builtin_bit_cast(u32x4_t, fr.p[n]);
    }
    static_assert(DB * 2 == KS, "T part has as many fragments as the S part");
}

template <class P>
__device__ __forceinline__ void load_frags(const u32x4_t *base, int f, int lane, Frags<P> &fr) {
#pragma unroll
    for (int n = 0; n < P::NS; ++n)
        fr.p[n] = __builtin_bit_cast(typename P::frag, base[(f * P::NS + n) * 64 + lane]);
}

// acc[n] += a streamed block's rows times the NB blocks of rows held in registers, over the width.  Four
// steps' fragments are read from LDS before the first of their MFMAs: read one by one right before its
// use, as the compiler orders them, each waits for LDS (1500 x 50,021 x 200 bf16, the kernel with weights
// rounded once: 156 us, like this 148; at d = 64 the other workgroup covers most of it).
template <class P, int KS, int NB, class B>
__device__ __forceinline__ void logits(const u32x4_t *lds, int lane, const B &held, f32x16_t (&acc)[NB]) {
    constexpr int G = KS < 4 ? KS : 4;
#pragma unroll
    for (int s0 = 0; s0 < KS; s0 += G) {
        Frags<P> f[G];
#pragma unroll
        for (int s = 0; s < G; ++s) load_frags<P>(lds, s0 + s, lane, f[s]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < G; ++s)
            mfma_row<P, NB>(f[s], [&](int n) -> const Frags<P> & { return held(n, s0 + s); }, acc);
    }
}

// A tile's weights as operands of the product with the table's rows.  fp32's are pairs of halves already;
// half types' become pairs too, what the first rounding left as the second operand: rounded once, a weight
// is off by half a step (2^-8 of it for bf16), and a sum of few large weights by as much.  1500 x 50,021 x
// 200 in bf16: rounded once, the items' gradient, whose target's term often is nearly all there is, is off by
// 2.8e-3 of its norm, as pairs by 1.7e-3, the result's own rounding; x's gradient differs from one of 32-bit
// weights by 2.6e-4 and 9e-5 of its norm.  The second product takes the forward's kernel from 148 to 187 us.
template <class P, int NR>
__device__ __forceinline__ void split_weights(float (&p)[16], Frags<P> (&w)[2], Frags<P> (&rest)[NR]) {
    float (&pl)[8] = reinterpret_cast<float (&)[8]>(p[0]);
    float (&ph)[8] = reinterpret_cast<float (&)[8]>(p[8]);
    split8(pl, w[0]);
    split8(ph, w[1]);
    if constexpr (P::NS == 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] -= (float)w[i >> 3].p[0][i & 7];
        split8(pl, rest[0]);
        split8(ph, rest[1]);
    }
}

// Logits (log2) beyond kFar take a path of their own: exp2(acc c - m), one fused operation, is off by the rounding of m
// to fp32, which there is no small one (for a split of items that are all masked by -1e15 it is 2^25, and the
// power infinite).
constexpr float kFar = 512.f;
// a b rounded to fp32, not to be fused with a difference: less a maximum that was rounded likewise it is 0 at most.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

struct FwdArgs {
    int64_t B, V, nbt, splits, per;  // batch tiles, catalogue splits, item blocks per split
    Packed x, w;
    const int64_t *target;
    float scale2;  // scale log2(e)
    float *pm, *pz, *pt, *po;  // partials: [splits][B] max (log2), sum without the target, its logit; [splits][B][DP]
    int32_t *pd;               // [splits][B] exponent of po
};

// WITH_O = false: the loss alone (no product with the T part, which is then not copied either).
// Two workgroups a CU wherever the registers do: all but o of fp32 rows of 256.
template <class P, int DP, int NB, bool WITH_O>
__global__ __launch_bounds__(kThreads, (DP * P::NS <= 256 || !WITH_O ? 2 : 1)) void softmax_fwd(FwdArgs a) {
    constexpr int KS = DP / 16, DB = DP / 32;
    constexpr int TILE = block_halves<P>(DP) / 8 / (WITH_O ? 1 : 2);  // u32x4_t of a streamed block
    constexpr int BLK = block_halves<P>(DP) / 8;
    __shared__ u32x4_t lds0[TILE], lds1[TILE];
    __shared__ int32_t most_s, least_s;
    // workgroups of one split sit on one XCD (blockIdx % 8), next to each other in time: the
    // split's item blocks come from that XCD's L2 for all batch tiles but the first
    const int64_t id = blockIdx.x, xcd = id & 7, j = id >> 3;
    const int64_t split = (j / a.nbt) * 8 + xcd, bt = j % a.nbt;
    if (split >= a.splits) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 31, h = lane >> 5;
    const int64_t nblk = blocks_of(a.V);
    const int64_t k0 = split * a.per, k1 = k0 + a.per < nblk ? k0 + a.per : nblk;
    const int64_t nxb = blocks_of(a.B);

    // The exponents of the split's blocks.  Where they are within 2^kNarrow of each other, as a trained table's are,
    // the weights are made for the largest, C; else for what weighs most so far, row by row of the batch
    // (a large item that weighs nothing must not push the others' weights out of the halves' range).  With an
    // item in 1000 masked by -1e9, 2048 x a million x 64 takes 3.0 ms forward instead of 1.55.
    int C = 0;
    bool even = true;
    if constexpr (P::kScaled) {
        if (t == 0) most_s = -127, least_s = 127;
        __syncthreads();
        int most = -127, least = 127;
        for (int64_t k = k0 + t; k < k1; k += kThreads) {
            const int e = a.w.exps[k];
            most = max(most, largest_exp(e));
            if (e != kZeros) least = min(least, is_wide(e) ? -1000 : e);
        }
        const int64_t xb = bt * 4 * NB + t;  // and no batch row of the workgroup has its own
        if (t < 4 * NB && xb < nxb && is_wide(a.x.exps[xb])) least = -1000;
        atomicMax(&most_s, most);  // in LDS; these do not depend on the order
        atomicMin(&least_s, least);
        __syncthreads();
        C = __builtin_amdgcn_readfirstlane(most_s);
        even = C - __builtin_amdgcn_readfirstlane(least_s) <= kNarrow;
    }

    // EVEN: one exponent a block; else every row has its own.  The two share neither variables nor, for the differing
    // asm lines, loads: with one loop for both, or shared loads before two, the first reloaded spilled
    // registers in each step (2048 x a million x 64: 2390 and 1882 us, like this 1546).
    auto body = [&](auto kind) __attribute__((always_inline)) {
        constexpr bool EVEN = decltype(kind)::value;
        if constexpr (EVEN) asm volatile("; one exponent a block");
        else asm volatile("; one exponent a row");
        // this wave's batch blocks
        Frags<P> xf[NB][KS];
        // top: the largest log2 of a weight (relative to m) times its row's power of two so far; far: some |m| is
        // beyond kFar
        float c_x[NB], m[NB], top[NB], z[NB], tl[NB];
        int tgt[NB];
        bool live[NB], far[NB];
        f32x16_t o[WITH_O ? DB : 1][NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int64_t xb = (bt * 4 + wave) * NB + n;
            live[n] = xb < nxb;
            const int64_t xs = live[n] ? xb : 0;
#pragma unroll
            for (int k = 0; k < KS; ++k) load_frags<P>(a.x.blocks + xs * BLK, k, lane, xf[n][k]);
            if constexpr (!P::kScaled) c_x[n] = a.scale2;
            else c_x[n] = a.scale2 * pow2f((EVEN ? largest_exp(a.x.exps[xs]) : a.x.row_exps[xs * kRB + col]) - P::kOff);
            m[n] = top[n] = -INFINITY;
            far[n] = false;
            z[n] = 0.f;
            tl[n] = 0.f;
            const int64_t b = xs * kRB + col;
            const int64_t tt = live[n] && b < a.B ? a.target[b] : -1;
            tgt[n] = tt >= 0 && tt < a.V ? (int)tt : -1;
#pragma unroll
            for (int q = 0; q < (WITH_O ? DB : 1); ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[q][n][i] = 0.f;
        }

        // w: the block in LDS that is used; next: the buffer that the following block is copied to meanwhile.
        // (Two arrays by name, and the loop in pairs: so the compiler sees that reading one need not wait for
        // the copy into the other.)
        // o is held times 2^(14 - C or down) and its rows' 2^14: the largest product's weight is 2^14 in the halves' range
        auto down_of = [](float top) { return top > -INFINITY ? (int)ceilf(top) : 0; };
        int ew_next = P::kScaled ? a.w.exps[k0] : 0;  // loaded a block ahead, before that block's copy is begun
        auto step = [&](int64_t k, const u32x4_t *__restrict__ w, u32x4_t *__restrict__ next) __attribute__((always_inline)) {
            const int ew = P::kScaled ? largest_exp(__builtin_amdgcn_readfirstlane(ew_next)) : 0;
            if (k + 1 < k1) {
                if (P::kScaled) ew_next = a.w.exps[k + 1];
                copy_to_lds<TILE>(a.w.blocks + (k + 1) * BLK, next, t);
            }
            const float c_w = P::kScaled ? pow2f(ew - P::kOff) : 1.f;
            f32x16_t acc[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
            logits<P, KS, NB>(w, lane, [&](int n, int s) -> const Frags<P> & { return xf[n][s]; }, acc);
            if constexpr (!EVEN)
                each_exp(a.w.row_exps, k, h, [&](int i, int e) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) acc[n][i] = ldexpf(acc[n][i], e - ew);
                });
            const int v0 = (int)(k * kRB);
            const int nv = a.V - k * kRB < kRB ? (int)(a.V - k * kRB) : kRB;  // items of this block
            Frags<P> pf[NB][2];
            Frags<P> rest[NB][P::NS == 1 ? 2 : 1];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                // lane: batch row `col` of block n; register i: item 8 (i/4) + 4 h + i%4
                // (c of two tables of zeros would round to 0, and 0 times infinity is none)
                const float c = fmaxf(c_x[n] * c_w, 1.17549435e-38f);
                if (__any((unsigned)(tgt[n] - v0) < 32u)) {  // some row's target is here: its logit apart from the others
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (tgt[n] - v0 == 8 * (i >> 2) + 4 * h + (i & 3)) {
                            tl[n] = acc[n][i] * c;
                            acc[n][i] = -INFINITY;
                        }
                }
                if (nv < kRB) {  // the catalogue's last block: its padding takes no part
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (8 * (i >> 2) + 4 * h + (i & 3) >= nv) acc[n][i] = -INFINITY;
                }
                float mx = acc[n][0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, acc[n][i]);
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
                const float mn = fmaxf(m[n], mx), base = mn == -INFINITY ? 0.f : mn;  // (none yet but the target)
                float mt = -INFINITY;  // of the block's weights times their rows' powers of two the largest log2
                if constexpr (!EVEN) {
                    each_exp(a.w.row_exps, k, h, [&](int i, int e) {
                        mt = fmaxf(mt, rounded_product(acc[n][i], c) - base + (float)e);
                    });
                    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
                }
                if (__any(mx > m[n] || (!EVEN && mt > top[n]))) {  // rare after the first blocks
                    const float less = m[n] == mn ? 0.f : m[n] - mn;  // (both may be -infinity)
                    const float f = __builtin_amdgcn_exp2f(less);
                    z[n] *= f;
                    float fo = f;
                    if constexpr (!EVEN) {
                        const float tn = fmaxf(top[n] + less, mt);
                        fo = __builtin_amdgcn_exp2f(less + (float)(down_of(top[n]) - down_of(tn)));
                        top[n] = tn;
                    }
                    m[n] = mn;
                    far[n] = __any(fabsf(base) > kFar);
                    if constexpr (WITH_O) {
#pragma unroll
                        for (int q = 0; q < DB; ++q)
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[q][n][i] *= fo;
                    }
                }
                // weights p 2^sh: up to 2^14 in the halves' range, less where the block's rows are
                // smaller than the split's largest.  -60 keeps the sum exact; a block that far
                // below adds nothing to o either way.
                // (without o the same powers, for the same sums bit for bit)
                const int sh = EVEN ? 14 + (P::kScaled ? max(ew - C, -60) : 0) : 0;
                float p[16];
                if (!EVEN || far[n]) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        p[i] = ldexpf(__builtin_amdgcn_exp2f(rounded_product(acc[n][i], c) - base), sh);
                } else {
                    const float off = base - (float)sh;
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(acc[n][i], c, -off));
                }
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    s0 += p[i];
                    s1 += p[i + 1];
                }
                z[n] = fmaf(s0 + s1, pow2f(-sh), z[n]);
                if constexpr (WITH_O) {
                    if constexpr (!EVEN) {  // each weight by its own row's power, up to 2^14 again
                        const int up = 14 - down_of(top[n]);
                        each_exp(a.w.row_exps, k, h, [&](int i, int e) { p[i] = ldexpf(p[i], e + up); });
                    }
                    split_weights<P>(p, pf[n], rest[n]);
                }
            }
            if constexpr (WITH_O) {
#pragma unroll
                for (int f = 0; f < 2 * DB; ++f) {
                    Frags<P> wf;
                    load_frags<P>(w, KS + f, lane, wf);
                    f32x16_t (&of)[NB] = o[f >> 1];
                    mfma_row<P, NB>(wf, [&](int n) -> const Frags<P> & { return pf[n][f & 1]; }, of);
                    if constexpr (P::NS == 1) mfma_row<P, NB>(wf, [&](int n) -> const Frags<P> & { return rest[n][f & 1]; }, of);
                }
            }
            copies_done();
            __syncthreads();
        };
        copy_to_lds<TILE>(a.w.blocks + k0 * BLK, lds0, t);
        copies_done();
        __syncthreads();
        for (int64_t k = k0; k < k1; k += 2) {
            step(k, lds0, lds1);
            if (k + 1 < k1) step(k + 1, lds1, lds0);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int64_t b = ((bt * 4 + wave) * NB + n) * kRB + col;
            // the two halves of a row: same maximum, sums of different items, one target logit
            const float zz = z[n] + __shfl_xor(z[n], 32, 64);
            const float ot = __shfl_xor(tl[n], 32, 64);
            const bool mine = (tgt[n] >> 2 & 1) == h;  // items 8q + 4h + 0..3 are this half's
            if (!live[n] || b >= a.B) continue;
            if (h == 0) {
                a.pm[split * a.B + b] = m[n];
                a.pz[split * a.B + b] = zz;
                a.pt[split * a.B + b] = mine ? tl[n] : ot;
                if (WITH_O) a.pd[split * a.B + b] = EVEN ? C : down_of(top[n]);
            }
            if constexpr (WITH_O) {
                float *dst = a.po + (split * a.B + b) * DP;
#pragma unroll
                for (int q = 0; q < DB; ++q)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        *reinterpret_cast<float4 *>(dst + q * 32 + g * 8 + h * 4) =
                            make_float4(o[q][n][4 * g], o[q][n][4 * g + 1], o[q][n][4 * g + 2], o[q][n][4 * g + 3]);
            }
        }
    };
    if (even) body(std::true_type());
    if constexpr (P::kScaled)
        if (!even) body(std::false_type());
}

struct JoinArgs {
    int64_t B, V, splits, per;
    int32_t d, ooff;  // ooff: po carries 2^(ooff - pd)
    const float *pm, *pz, *pt, *po;
    const int32_t *pd;
    const int64_t *target;
    int64_t ignore;
    float *loss, *lse2, *rest, *o;  // rest: r; o: [B, DP] or NULL
    int16_t *lse_rest;
};

// One batch row per workgroup: the splits' (max, sum, o) joined in split order, a quarter of them
// per wave.  Reads the partials once.
template <int DP>
__global__ __launch_bounds__(kThreads) void softmax_join(JoinArgs a) {
    __shared__ float part[4][DP];
    __shared__ float wm[4], wz[4];
    const int64_t b = flat_group();
    if (b >= a.B) return;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int64_t tg = a.target[b];
    if (tg == a.ignore) {
        if (t == 0) {
            a.loss[b] = 0.f;
            a.lse2[b] = 0.f;
            a.lse_rest[b] = 0;
            a.rest[b] = 0.f;
        }
        if (a.o)
            for (int c = t; c < DP; c += kThreads) a.o[b * DP + c] = 0.f;
        return;
    }
    const bool named = tg >= 0 && tg < a.V;
    const float st = named ? a.pt[(tg / kRB / a.per) * a.B + b] : -INFINITY;
    float m = st;
    for (int64_t s = t; s < a.splits; s += kThreads) m = fmaxf(m, a.pm[s * a.B + b]);
#pragma unroll
    for (int q = 32; q; q >>= 1) m = fmaxf(m, __shfl_xor(m, q, 64));
    if (lane == 0) wm[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    float z = 0.f;
    for (int64_t s = t; s < a.splits; s += kThreads)
        z += a.pz[s * a.B + b] * __builtin_amdgcn_exp2f(a.pm[s * a.B + b] - m);
#pragma unroll
    for (int q = 32; q; q >>= 1) z += __shfl_xor(z, q, 64);
    if (lane == 0) wz[wave] = z;
    __syncthreads();
    const float others = (wz[0] + wz[1]) + (wz[2] + wz[3]);
    z = others;
    float loss = NAN;  // a target that names no item
    if (named) {
        const float zt = __builtin_amdgcn_exp2f(st - m);
        z += zt;
        // terms >= 0 either way, no cancellation
        loss = st - m > -1.f ? log1pf(others / zt) : kLn2 * (m - st) + logf(z);
    }
    if (t == 0) {
        a.loss[b] = loss;
        const float l = log2f(z), lse = m + l;
        a.lse2[b] = lse;
        a.lse_rest[b] = (int16_t)fminf(fmaxf(rintf(((m - lse) + l) / rest_unit(lse)), -32767.f), 32767.f);
        a.rest[b] = others / z;
    }
    if (!a.o) return;
    const int64_t q0 = a.splits * wave / 4, q1 = a.splits * (wave + 1) / 4;
    constexpr int NC = (DP + 63) / 64;
    float acc[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = 0.f;
#pragma unroll 4
    for (int64_t s = q0; s < q1; ++s) {
        const float f = ldexpf(__builtin_amdgcn_exp2f(a.pm[s * a.B + b] - m), a.pd[s * a.B + b] - a.ooff);
        // (of items that are all masked po may be infinite: 0 in its place, by its bits, for a load under a condition
        // takes the kernel from 11 to 16 us)
        const uint32_t bits = f == 0.f ? 0u : ~0u;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (c * 64 + lane < DP) {
                const float v = a.po[(s * a.B + b) * DP + c * 64 + lane];
                acc[c] = fmaf(__builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & bits), f, acc[c]);
            }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
        if (c * 64 + lane < DP) part[wave][c * 64 + lane] = acc[c];
    __syncthreads();
    for (int c = t; c < DP; c += kThreads)
        a.o[b * DP + c] = ((part[0][c] + part[1][c]) + (part[2][c] + part[3][c])) / z;
}

// The loss's sum or mean over the rows that are not ignored, and their number.
constexpr int kReduceThreads = 1024;
__global__ __launch_bounds__(kReduceThreads) void softmax_reduce(int64_t B, const float *loss, const int64_t *target,
                                                                 int64_t ignore, int32_t mean, float *total,
                                                                 float *count) {
    __shared__ double ss[kReduceThreads / 64];
    __shared__ int64_t sn[kReduceThreads / 64];
    const int t = threadIdx.x;
    double s = 0.;
    int64_t n = 0;
    for (int64_t b = t; b < B; b += kReduceThreads) {
        s += loss[b];
        n += target[b] != ignore;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        s += __shfl_xor(s, o, 64);
        n += __shfl_xor((long long)n, o, 64);
    }
    if ((t & 63) == 0) {
        ss[t >> 6] = s;
        sn[t >> 6] = n;
    }
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kReduceThreads / 64; ++w) {
            s += ss[w];
            n += sn[w];
        }
        *total = (float)(mean ? s / (double)(n > 0 ? n : 1) : s);
        *count = (float)n;
    }
}

// What the streamed batch blocks of the backward carry besides their fragments, per row: lse2 and what stands
// beside it to make exp2(acc c - lse + beside) = |c_b| p 2^(14 + e - C), the same power of c_b r_b for the
// target's own term (with c_b's sign, zero or not), the target.  off is the two in one fp32, off by half the
// step of up to 40, 2^-20, for all of a row's weights: the half types take it, whose results round further
// (1500 x 50,021 x 200 in bf16: 140 us backward, 166 from the two), fp32 does not (2048 x a million x 64: dw
// off by 9.7e-7 of its norm, 7.7e-7 to 8.5e-7 from the two; 1.35 and 1.36 ms).
struct RowInfo {
    float *lse, *beside, *hot, *off;
    int32_t *tgt;
    int32_t *flags; // per block: kMinus, some c_b < 0; kFarRows, some |lse2| > kFar
    int32_t *cmax;  // C: the largest e + floor(log2 |c_b|)
    int32_t *part;  // kScanGroups partial maxima
};
constexpr int kMinus = 1, kFarRows = 2;
constexpr int kScanGroups = 256;         // one partial maximum a thread of softmax_coef
constexpr int64_t kScanInline = 8192;   // terms that every workgroup of softmax_coef goes through itself

struct CoefArgs {
    int64_t B, V;
    int32_t d, per_row, mean;
    const float *grad, *count, *lse2, *rest, *o;
    const int64_t *target;
    int64_t ignore;
    float scale;
    Packed x;
    RowInfo info;
    int64_t n_info;    // workgroups that fill the row info (0: dw is not wanted)
    int32_t scanned;   // info.part is filled
    const void *items; // for dx
    int64_t ld_items;
    void *dx;
};

__device__ __forceinline__ float row_coef(const CoefArgs &a, int64_t b, int64_t tg) {
    if (tg == a.ignore) return 0.f;
    if (tg < 0 || tg >= a.V) return NAN;
    const float g = (a.per_row ? a.grad[b] : a.grad[0]) * a.scale;
    return a.mean ? g / fmaxf(*a.count, 1.f) : g;
}

// A thread's share of C, terms first, first + stride, ...
template <bool SCALED>
__device__ __forceinline__ int scan_exponents(const CoefArgs &a, int64_t first, int64_t stride) {
    int most = -250;
    if (a.per_row) {
        for (int64_t b = first; b < a.B; b += stride) {
            const float c = fabsf(row_coef(a, b, a.target[b]));
            if (c > 0.f) most = max(most, block_exponent(c) + (SCALED ? a.x.row_exps[b] : 0));
        }
    } else {  // one coefficient; blocks of nothing but ignored rows are packed as zeros and do not count
        const float c = a.grad[0] * a.scale / (a.mean ? fmaxf(*a.count, 1.f) : 1.f);
        const int e = block_exponent(fabsf(c));
        if (!SCALED) return e;
        for (int64_t k = first; k < blocks_of(a.B); k += stride) most = max(most, e + largest_exp(a.x.exps[k]));
    }
    return most;
}
inline int64_t scan_terms(int64_t b, bool per_row, bool scaled) { return per_row ? b : scaled ? blocks_of(b) : 1; }

// C's partial maxima, for batches whose terms are too many for every workgroup of softmax_coef to go through: that
// grows with the square of the batch.  A backward with a gradient for each row (V = 1024, d = 64, fp32) takes
// 62 us at 8192 rows without this launch; at 16,384 rows 89 us without and 64 with it, at 65,536 237 and 111.
template <bool SCALED>
__global__ __launch_bounds__(kThreads) void softmax_scan(CoefArgs a) {
    __shared__ int32_t wm[kThreads / 64];
    const int t = threadIdx.x;
    int most = scan_exponents<SCALED>(a, (int64_t)blockIdx.x * kThreads + t, (int64_t)kScanGroups * kThreads);
#pragma unroll
    for (int o = 32; o; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    if ((t & 63) == 0) wm[t >> 6] = most;
    __syncthreads();
    if (t == 0) a.info.part[blockIdx.x] = max(max(wm[0], wm[1]), max(wm[2], wm[3]));
}

// Workgroups below n_info: the row info of 256 rows.  The others: dx of four rows, one a wave.
template <class T, int DP, bool SCALED>
__global__ __launch_bounds__(kThreads) void softmax_coef(CoefArgs a) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int64_t id = flat_group();
    if (id >= a.n_info) {
        const int64_t b = (id - a.n_info) * 4 + wave;
        if (b >= a.B || !a.dx) return;
        const int64_t tg = a.target[b];
        const float c = row_coef(a, b, tg);
        const bool ok = tg != a.ignore;
        const float r = a.rest[b];
        const T *w = static_cast<const T *>(a.items) + (tg >= 0 && tg < a.V ? tg : 0) * a.ld_items;
        T *dx = static_cast<T *>(a.dx) + b * a.d;
        for (int q = lane; q < a.d; q += 64) dx[q] = ok ? (T)(c * fmaf(-r, (float)w[q], a.o[b * DP + q])) : (T)0.f;
        return;
    }
    __shared__ int32_t cm;
    if (t == 0) cm = -250;
    __syncthreads();
    static_assert(kScanGroups == kThreads, "one partial maximum a thread");
    const int c_all = a.scanned ? a.info.part[t] : scan_exponents<SCALED>(a, t, kThreads);
    atomicMax(&cm, c_all);  // in LDS; a maximum does not depend on the order
    __syncthreads();
    const int C = cm;
    const int64_t b = id * kThreads + t;
    if (b >= blocks_of(a.B) * kRB) return;
    float lse = 0.f, beside = -INFINITY, hot = 0.f;
    int tgt = -1;
    bool minus = false, far = false;
    if (b < a.B) {
        const int64_t tg = a.target[b];
        const float c = row_coef(a, b, tg);
        const int e = SCALED ? a.x.row_exps[b] : 0;
        if (c != 0.f) {
            lse = a.lse2[b];
            beside = log2f(fabsf(c)) + (float)(14 + e - C) - (float)a.x.lse_rest[b] * rest_unit(lse);
            far = fabsf(lse) > kFar;
            hot = ldexpf(c * a.rest[b], 14 + e - C);
            minus = c < 0.f;
            tgt = tg >= 0 && tg < a.V ? (int)tg : -1;
        }
    }
    a.info.off[b] = lse - beside;
    a.info.hot[b] = hot;
    a.info.tgt[b] = tgt;
    a.info.lse[b] = lse;
    a.info.beside[b] = beside;
    const uint64_t neg = __ballot(minus), wide = __ballot(far);
    if ((lane & 31) == 0)
        a.info.flags[b / kRB] = ((uint32_t)(neg >> lane) ? kMinus : 0) | ((uint32_t)(wide >> lane) ? kFarRows : 0);
    if (b == 0) *a.info.cmax = C;
}

struct BwdArgs {
    int64_t B, V, splits, per;  // batch splits, batch blocks per split
    int32_t d, vec;
    Packed x, w;
    RowInfo info;
    float scale2;
    void *dw;
    float *part;  // [splits][V][DP] when splits > 1
};

template <class T>
__device__ __forceinline__ void store4(T *dst, int c, int d, bool vec, float a, float b, float e, float f) {
    if (vec) {  // d and the leading dimension are multiples of 4
        if (c < d) {
            T v[4] = {(T)a, (T)b, (T)e, (T)f};
            __builtin_memcpy(__builtin_assume_aligned(dst + c, 4 * sizeof(T)), v, sizeof v);
        }
        return;
    }
    if (c < d) dst[c] = (T)a;
    if (c + 1 < d) dst[c + 1] = (T)b;
    if (c + 2 < d) dst[c + 2] = (T)e;
    if (c + 3 < d) dst[c + 3] = (T)f;
}

// (As for the forward, two workgroups a CU but for fp32 rows of 256.)
// dw of 32 NB items a wave: logits recomputed tile by tile, weights times batch rows accumulated.
template <class P, int DP, int NB>
__global__ __launch_bounds__(kThreads, (DP * P::NS <= 256 ? 2 : 1)) void softmax_bwd(BwdArgs a) {
    constexpr int KS = DP / 16, DB = DP / 32;
    constexpr int BLK = block_halves<P>(DP) / 8;
    __shared__ u32x4_t lds0[BLK], lds1[BLK];
    constexpr int kInfo = P::NS == 1 ? 5 : 4;
    // lse, beside, hot, target (, off) of the streamed block
    __shared__ __align__(16) float info0[kInfo][kRB], info1[kInfo][kRB];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, col = lane & 31, h = lane >> 5;
    const int64_t nvb = blocks_of(a.V), nxb = blocks_of(a.B);
    const int64_t split = blockIdx.y;
    const int64_t k0 = split * a.per, k1 = k0 + a.per < nxb ? k0 + a.per : nxb;

    Frags<P> wf[NB][KS];
    float c_w[NB];
    int v0[NB];
    bool live[NB];
    f32x16_t o[DB][NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int64_t vb = ((int64_t)blockIdx.x * 4 + wave) * NB + n;
        live[n] = vb < nvb;
        const int64_t vs = live[n] ? vb : 0;
        v0[n] = (int)(vs * kRB);
#pragma unroll
        for (int k = 0; k < KS; ++k) load_frags<P>(a.w.blocks + vs * BLK, k, lane, wf[n][k]);
        c_w[n] = a.scale2 * (P::kScaled ? pow2f(a.w.row_exps[vs * kRB + col] - P::kOff) : 1.f);
#pragma unroll
        for (int q = 0; q < DB; ++q)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[q][n][i] = 0.f;
    }

    // As in the forward: x and info in use, the next ones filled meanwhile, two arrays by name.
    auto fetch_info = [&](int64_t k) {
        float v = 0.f;
        if (t < kRB) v = a.info.lse[k * kRB + t];
        else if (t < 2 * kRB) v = a.info.beside[k * kRB + t - kRB];
        else if (t < 3 * kRB) v = a.info.hot[k * kRB + t - 2 * kRB];
        else if (t < 4 * kRB) v = __builtin_bit_cast(float, a.info.tgt[k * kRB + t - 3 * kRB]);
        else if (kInfo == 5 && t < 5 * kRB) v = a.info.off[k * kRB + t - 4 * kRB];
        return v;
    };
    int e_next = P::kScaled ? a.x.exps[k0] : 0, flags_next = a.info.flags[k0];
    auto step = [&](int64_t k, const u32x4_t *__restrict__ x, u32x4_t *__restrict__ next, const float (*info)[kRB],
                    float (*info_next)[kRB]) {
        const int e_k = P::kScaled ? __builtin_amdgcn_readfirstlane(e_next) : 0;
        const int e_x = largest_exp(e_k);
        const float c_x = P::kScaled ? pow2f(e_x - P::kOff) : 1.f;
        const int flags = __builtin_amdgcn_readfirstlane(flags_next);
        const bool neg = flags & kMinus;
        float si = 0.f;
        if (k + 1 < k1) {
            if (P::kScaled) e_next = a.x.exps[k + 1];
            flags_next = a.info.flags[k + 1];
            si = fetch_info(k + 1);
            copy_to_lds<BLK>(a.x.blocks + (k + 1) * BLK, next, t);
        }
        f32x16_t acc[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[n][i] = 0.f;
        logits<P, KS, NB>(x, lane, [&](int n, int s) -> const Frags<P> & { return wf[n][s]; }, acc);
        // lane: item v0 + col; register i: batch row 8 (i/4) + 4 h + i%4 of the block
        if (P::kScaled && is_wide(e_k))
            each_exp(a.x.row_exps, k, h, [&](int i, int e) {
#pragma unroll
                for (int n = 0; n < NB; ++n) acc[n][i] = ldexpf(acc[n][i], e - e_x);
            });
        const int tcol = __builtin_bit_cast(int, info[3][col]);
        Frags<P> pf[NB][2];
        Frags<P> rest[NB][P::NS == 1 ? 2 : 1];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const float c = c_w[n] * c_x;
            float p[16];
            auto weights = [&](auto exponent, int first) {  // exponent(logit / c, the row's lse or off, its beside)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 l = *reinterpret_cast<const float4 *>(&info[first][8 * g + 4 * h]);
                    const float4 b = *reinterpret_cast<const float4 *>(&info[1][8 * g + 4 * h]);
                    p[4 * g] = __builtin_amdgcn_exp2f(exponent(acc[n][4 * g], l.x, b.x));
                    p[4 * g + 1] = __builtin_amdgcn_exp2f(exponent(acc[n][4 * g + 1], l.y, b.y));
                    p[4 * g + 2] = __builtin_amdgcn_exp2f(exponent(acc[n][4 * g + 2], l.z, b.z));
                    p[4 * g + 3] = __builtin_amdgcn_exp2f(exponent(acc[n][4 * g + 3], l.w, b.w));
                }
            };
            // (far: equal logits as in the forward, one less the other is 0)
            if (flags & kFarRows)
                weights([&](float s, float lse, float b) { return rounded_product(s, c) - lse + b; }, 0);
            else if constexpr (kInfo == 5) weights([&](float s, float off, float) { return fmaf(s, c, -off); }, 4);
            else weights([&](float s, float lse, float b) { return fmaf(s, c, -lse) + b; }, 0);
            if (neg) {  // a negative c_b: only where the caller's gradients are
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = copysignf(p[i], info[2][8 * (i >> 2) + 4 * h + (i & 3)]);
            }
            if (__any((unsigned)(tcol - v0[n]) < 32u)) {  // some row's target is one of these items
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 8 * (i >> 2) + 4 * h + (i & 3);
                    if (__builtin_bit_cast(int, info[3][r]) == v0[n] + col) p[i] = -info[2][r];
                }
            }
            split_weights<P>(p, pf[n], rest[n]);
        }
#pragma unroll
        for (int f = 0; f < 2 * DB; ++f) {
            Frags<P> xf;
            load_frags<P>(x, KS + f, lane, xf);
            f32x16_t (&of)[NB] = o[f >> 1];
            mfma_row<P, NB>(xf, [&](int n) -> const Frags<P> & { return pf[n][f & 1]; }, of);
            if constexpr (P::NS == 1) mfma_row<P, NB>(xf, [&](int n) -> const Frags<P> & { return rest[n][f & 1]; }, of);
        }
        if (k + 1 < k1 && t < kInfo * kRB) info_next[t / kRB][t % kRB] = si;
        copies_done();
        __syncthreads();
    };
    copy_to_lds<BLK>(a.x.blocks + k0 * BLK, lds0, t);
    if (t < kInfo * kRB) info0[t / kRB][t % kRB] = fetch_info(k0);
    copies_done();
    __syncthreads();
    for (int64_t k = k0; k < k1; k += 2) {
        step(k, lds0, lds1, info0, info1);
        if (k + 1 < k1) step(k + 1, lds1, lds0, info1, info0);
    }
    const float f = a.splits > 1 ? 1.f : ldexpf(1.f, *a.info.cmax - 14 - P::kOff);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int64_t v = (int64_t)v0[n] + col;
        if (!live[n] || v >= a.V) continue;
#pragma unroll
        for (int q = 0; q < DB; ++q)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = q * 32 + g * 8 + h * 4;
                const float w0 = o[q][n][4 * g] * f, w1 = o[q][n][4 * g + 1] * f, w2 = o[q][n][4 * g + 2] * f,
                            w3 = o[q][n][4 * g + 3] * f;
                if (a.splits > 1)
                    *reinterpret_cast<float4 *>(a.part + (split * a.V + v) * DP + c) = make_float4(w0, w1, w2, w3);
                else
                    store4(static_cast<typename P::elem *>(a.dw) + v * a.d, c, a.d, a.vec, w0, w1, w2, w3);
            }
    }
}

// dw from the batch splits' partials, in split order.
template <class T, int DP>
__global__ __launch_bounds__(kThreads) void softmax_bwd_join(int64_t V, int32_t d, int64_t splits, int32_t off,
                                                             const int32_t *cmax, const float *part, int32_t vec,
                                                             T *dw) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t v = i / (DP / 4);
    const int c = (int)(i % (DP / 4)) * 4;
    if (v >= V || c >= d) return;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int64_t k = 0; k < splits; ++k)
        s = f4_add(s, *reinterpret_cast<const float4 *>(part + (k * V + v) * DP + c));
    s = f4_scale(ldexpf(1.f, *cmax - off), s);
    store4(dw + v * d, c, d, vec, s.x, s.y, s.z, s.w);
}

// ------------------------------------------------------------------ host side

struct FwdPlan {
    int nb;
    int64_t nbt, splits, per;
};
// Two blocks of batch rows a wave where they fit the registers of two workgroups on a CU and there
// are that many rows: a streamed block then serves twice the rows.  (Workgroups are counted over the whole chip, but
// the kernel deals whole splits to the XCDs: few splits of a large batch leave XCDs idle.  65,536 rows
// against 40,981 items of d = 64 are two splits, 7.1 ms forward beside 2.3 backward.)
inline FwdPlan fwd_plan(int64_t B, int64_t V, int dp) {
    FwdPlan p;
    p.nb = dp <= 64 && B > 4 * kRB ? 2 : 1;
    p.nbt = (blocks_of(B) + 4 * p.nb - 1) / (4 * p.nb);
    const int64_t nblk = blocks_of(V);
    p.per = std::max<int64_t>(1, (nblk * p.nbt + kWantGroups - 1) / kWantGroups);
    p.splits = (nblk + p.per - 1) / p.per;
    return p;
}
inline FwdPlan bwd_plan(int64_t B, int64_t V, int dp) {
    FwdPlan p;
    p.nb = dp <= 64 && blocks_of(V) >= 8 * kWantGroups ? 2 : 1;
    p.nbt = (blocks_of(V) + 4 * p.nb - 1) / (4 * p.nb);
    const int64_t nblk = blocks_of(B);
    p.per = std::max<int64_t>(1, (nblk * p.nbt + kWantGroups - 1) / kWantGroups);
    p.splits = (nblk + p.per - 1) / p.per;
    return p;
}

inline int check_shape(const char *fn, int32_t dtype, int64_t b, int64_t v, int32_t d) {
    if (dtype < kF32 || dtype > kF16) return arg_error(fn, "unknown dtype");
    if (b < 0 || v <= 0 || d <= 0) return arg_error(fn, "sizes must be positive");
    if (d > 256) {
        set_error(std::string(fn) + ": width above 256");
        return IGR_ERR_UNSUPPORTED;
    }
    if (v > INT32_MAX - 64 || b > INT32_MAX - 64) return arg_error(fn, "more than 2^31 - 65 rows");
    return IGR_OK;
}

struct Carve {  // a workspace cut into 256-byte aligned pieces
    char *p;
    int64_t used = 0;
    template <class T>
    T *take(int64_t n) {
        T *r = reinterpret_cast<T *>(p + used);
        used += align256(n * (int64_t)sizeof(T));
        return r;
    }
};

template <class F>
int by_type_width(int32_t dtype, int dp, F &&f) {
    auto w = [&](auto pol) {
        switch (dp) {
            case 32: return f(pol, std::integral_constant<int, 32>());
            case 64: return f(pol, std::integral_constant<int, 64>());
            case 128: return f(pol, std::integral_constant<int, 128>());
            default: return f(pol, std::integral_constant<int, 256>());
        }
    };
    return dtype == kF32 ? w(SplitF32()) : dtype == kBF16 ? w(PlainBF16()) : w(PlainF16());
}

FwdArgs fwd_args(Carve &c, int64_t b, int64_t v, int dp, bool with_o) {
    const FwdPlan p = fwd_plan(b, v, dp);
    FwdArgs a{};
    a.B = b, a.V = v, a.nbt = p.nbt, a.splits = p.splits, a.per = p.per;
    a.pm = c.take<float>(p.splits * b);
    a.pz = c.take<float>(p.splits * b);
    a.pt = c.take<float>(p.splits * b);
    a.pd = with_o ? c.take<int32_t>(p.splits * b) : nullptr;
    a.po = with_o ? c.take<float>(p.splits * b * dp) : nullptr;
    return a;
}

BwdArgs bwd_args(Carve &c, int64_t b, int64_t v, int dp) {
    const FwdPlan p = bwd_plan(b, v, dp);
    BwdArgs a{};
    a.B = b, a.V = v, a.splits = p.splits, a.per = p.per;
    const int64_t rows = blocks_of(b) * kRB;
    a.info.hot = c.take<float>(rows);
    a.info.tgt = c.take<int32_t>(rows);
    a.info.flags = c.take<int32_t>(rows / kRB);
    a.info.lse = c.take<float>(rows);
    a.info.off = c.take<float>(rows);
    a.info.beside = c.take<float>(rows);
    a.info.cmax = c.take<int32_t>(1);
    a.info.part = c.take<int32_t>(kScanGroups);
    a.part = p.splits > 1 ? c.take<float>(p.splits * v * dp) : nullptr;
    return a;
}

}  // namespace
}  // namespace igr

using namespace igr;

extern "C" int64_t igr_softmax_loss_pack_size(int64_t rows, int32_t d, int32_t dtype) {
    if (rows <= 0 || d <= 0 || d > 256 || dtype < kF32 || dtype > kF16) return 0;
    return align256(blocks_of(rows) * (block_bytes(dtype, pad_width(d)) + (int64_t)sizeof(int32_t) + 3 * kRB));
}

extern "C" int64_t igr_softmax_loss_workspace_size(int64_t b, int64_t v, int32_t d, int32_t backward, int32_t with_o) {
    if (b <= 0 || v <= 0 || d <= 0 || d > 256) return 0;
    Carve c{nullptr};
    if (backward) bwd_args(c, b, v, pad_width(d));
    else fwd_args(c, b, v, pad_width(d), with_o != 0);
    return c.used;
}

extern "C" int igr_softmax_loss_fwd(int32_t dtype, int64_t b, int64_t v, int32_t d, const void *x, int64_t ldx,
                                    const void *items, int64_t ld_items, const int64_t *target, int64_t ignore_index,
                                    float scale, int32_t mean, void *x_pack, void *item_pack, float *loss, float *lse2,
                                    float *total, float *count, float *o, void *workspace, int64_t ws_bytes, void *stream) {
    return guarded("igr_softmax_loss_fwd", [&]() -> int {
        const char *fn = "igr_softmax_loss_fwd";
        if (int rc = check_shape(fn, dtype, b, v, d)) return rc;
        if (ldx < d || ld_items < d) return arg_error(fn, "leading dimension too small");
        if (!(scale > 0.f) || !std::isfinite(scale)) return arg_error(fn, "scale must be positive and finite");
        if (b > 0 && (!items || !x_pack || !item_pack || !loss || !lse2 || !x || !target)) return arg_error(fn, "null pointer");
        if (!total != !count) return arg_error(fn, "total and count go together");
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        if (b > 0) {
            const int dp = pad_width(d);
            Carve c{static_cast<char *>(workspace)};
            FwdArgs a = fwd_args(c, b, v, dp, o != nullptr);
            if (!workspace || ws_bytes < c.used || !aligned16(workspace) || !aligned16(x_pack) || !aligned16(item_pack))
                return arg_error(fn, "workspace or pack too small or not 16-byte aligned");
            a.x = packed_view(x_pack, b, dtype, dp);
            a.w = packed_view(item_pack, v, dtype, dp);
            a.target = target;
            a.scale2 = scale * kLog2e;
            const int64_t nx = blocks_of(b), nw = blocks_of(v), eb = dtype_bytes(dtype);
            const bool vec = d * eb % 16 == 0 && ldx * eb % 16 == 0 && ld_items * eb % 16 == 0 && aligned16(x) &&
                             aligned16(items);
            PackArgs px{b, ldx, x, const_cast<u32x4_t *>(a.x.blocks), const_cast<int32_t *>(a.x.exps),
                        const_cast<int8_t *>(a.x.row_exps), target, ignore_index};
            PackArgs pw{v, ld_items, items, const_cast<u32x4_t *>(a.w.blocks), const_cast<int32_t *>(a.w.exps),
                        const_cast<int8_t *>(a.w.row_exps), nullptr, 0};
            const FwdPlan plan = fwd_plan(b, v, dp);
            const int64_t grid = (a.splits + 7) / 8 * 8 * a.nbt;
            if (grid > kMaxGroups) return arg_error(fn, "too many batch rows for one launch");
            const int rc = by_type_width(dtype, dp, [&](auto pol, auto width) -> int {
                using P = decltype(pol);
                constexpr int DP = decltype(width)::value;
                hipLaunchKernelGGL((pack_rows<P, DP>), flat_grid(nx + nw), dim3(kThreads), 0, st, px, pw, nx, d,
                                   (int32_t)vec);
                const dim3 g((unsigned)grid);
                if constexpr (DP <= 64) {
                    if (plan.nb == 2) {
                        if (o) hipLaunchKernelGGL((softmax_fwd<P, DP, 2, true>), g, dim3(kThreads), 0, st, a);
                        else hipLaunchKernelGGL((softmax_fwd<P, DP, 2, false>), g, dim3(kThreads), 0, st, a);
                    }
                }
                if (plan.nb == 1) {
                    if (o) hipLaunchKernelGGL((softmax_fwd<P, DP, 1, true>), g, dim3(kThreads), 0, st, a);
                    else hipLaunchKernelGGL((softmax_fwd<P, DP, 1, false>), g, dim3(kThreads), 0, st, a);
                }
                JoinArgs j{b, v, a.splits, a.per, d, 14 + P::kOff, a.pm, a.pz, a.pt, a.po, a.pd, target, ignore_index,
                           loss, lse2, lse2 + b, o,
                           const_cast<int16_t *>(a.x.lse_rest)};
                hipLaunchKernelGGL((softmax_join<DP>), flat_grid(b), dim3(kThreads), 0, st, j);
                return IGR_OK;
            });
            if (rc) return rc;
        }
        if (total)
            hipLaunchKernelGGL(softmax_reduce, dim3(1), dim3(kReduceThreads), 0, st, b, loss, target, ignore_index, mean, total,
                               count);
        return launch_status(fn);
    });
}

extern "C" int igr_softmax_loss_bwd(int32_t dtype, int64_t b, int64_t v, int32_t d, const void *items,
                                    int64_t ld_items, const int64_t *target, int64_t ignore_index, float scale,
                                    int32_t mean, int32_t per_row, const float *grad, const void *x_pack,
                                    const void *item_pack, const float *lse2, const float *count, const float *o, void *dx,
                                    void *dw, void *workspace, int64_t ws_bytes, void *stream) {
    return guarded("igr_softmax_loss_bwd", [&]() -> int {
        const char *fn = "igr_softmax_loss_bwd";
        if (int rc = check_shape(fn, dtype, b, v, d)) return rc;
        if (ld_items < d) return arg_error(fn, "leading dimension too small");
        if (!(scale > 0.f) || !std::isfinite(scale)) return arg_error(fn, "scale must be positive and finite");
        if (b == 0 || (!dx && !dw)) return IGR_OK;
        if (!target || !grad || !lse2 || (mean && !count) || (dx && (!o || !items)) || (dw && (!x_pack || !item_pack)))
            return arg_error(fn, "null pointer");
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        const int dp = pad_width(d);
        Carve c{static_cast<char *>(workspace)};
        BwdArgs a = bwd_args(c, b, v, dp);
        if (!workspace || ws_bytes < c.used || !aligned16(workspace) || !aligned16(x_pack) || !aligned16(item_pack))
            return arg_error(fn, "workspace or pack too small or not 16-byte aligned");
        a.x = packed_view(x_pack, b, dtype, dp);
        a.w = packed_view(item_pack, v, dtype, dp);
        a.d = d;
        a.vec = d % 4 == 0 && aligned16(dw);
        a.scale2 = scale * kLog2e;
        a.dw = dw;
        const FwdPlan plan = bwd_plan(b, v, dp);
        const bool scan = dw && scan_terms(b, per_row != 0, dtype == kF32) > kScanInline;
        CoefArgs ca{b, v, d, per_row, mean, grad, count, lse2, lse2 + b, o, target, ignore_index, scale, a.x, a.info,
                    dw ? (blocks_of(b) * kRB + kThreads - 1) / kThreads : 0, (int32_t)scan, items, ld_items, dx};
        const int64_t cg = ca.n_info + (dx ? (b + 3) / 4 : 0);
        if (plan.splits > 65535 || plan.nbt > kMaxGroups) return arg_error(fn, "too many workgroups");
        const int rc = by_type_width(dtype, dp, [&](auto pol, auto width) -> int {
            using P = decltype(pol);
            using T = typename P::elem;
            constexpr int DP = decltype(width)::value;
            if (scan) hipLaunchKernelGGL((softmax_scan<P::kScaled>), dim3(kScanGroups), dim3(kThreads), 0, st, ca);
            hipLaunchKernelGGL((softmax_coef<T, DP, P::kScaled>), flat_grid(cg), dim3(kThreads), 0, st, ca);
            if (!dw) return IGR_OK;
            const dim3 g((unsigned)plan.nbt, (unsigned)plan.splits);
            if constexpr (DP <= 64) {
                if (plan.nb == 2) hipLaunchKernelGGL((softmax_bwd<P, DP, 2>), g, dim3(kThreads), 0, st, a);
            }
            if (plan.nb == 1) hipLaunchKernelGGL((softmax_bwd<P, DP, 1>), g, dim3(kThreads), 0, st, a);
            if (plan.splits > 1)
                hipLaunchKernelGGL((softmax_bwd_join<T, DP>), dim3((unsigned)((v * (DP / 4) + kThreads - 1) / kThreads)),
                                   dim3(kThreads), 0, st, v, d, plan.splits, 14 + P::kOff, a.info.cmax, a.part,
                                   (int32_t)a.vec, static_cast<T *>(dw));
            return IGR_OK;
        });
        if (rc) return rc;
        return launch_status(fn);
    });
}
