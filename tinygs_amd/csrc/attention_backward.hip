// The gradients of attention.hip from its out and lse: p = exp(s - lse),
// delta = sum of do o over a head, dv = p^T do, ds = p (do v^T - delta),
// dq = scale ds k, dk = scale ds^T q.
//
// Two kernels, each with what it sums in registers and the other side in tiles
// through LDS: dq has rows in the lanes, s^T = k q^T and dp^T = v do^T, and adds
// k^T ds^T; dk and dv have states in the lanes, s = q k^T and dp = do v^T, and
// add do^T p and q^T ds. Weights and their gradients are operands as they stand
// in both. The scores are formed twice (seven products in place of five); in
// one kernel, either sum would have to leave it in as many parts as there are
// blocks of the other side. 2 x 8192 rows of 8 heads of 128 halves, 2 shared, at 4096
// states, 2500 of them in one: 1076 us, of which dq 342, dk 385, dv 320 and their
// joins 21. Matrix cores are busy 48, 44 and 34% of the time, vector instructions 38, 40
// and 30%, LDS 24, 30 and 22%: two waves a SIMD overlap little, and wait half of theirs.
//
// Halves: p is held times 2^13 (down to 2^-27 it keeps the bits of a half; scores of
// 2^25 and their lse, rounded to floats, leave it below 8), and ds times a power of
// two that brings the largest it can be, |do| |v| + |delta|, to 2^14: of a row's and
// all states' in dq, of a state's and all rows' of its element and head in dk, so that
// small ones keep their bits, and no element's or head's gradients depend on another's.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "row_chunks.h"

namespace tgs {

namespace {

constexpr int kWaves = 4;

template <class T>
constexpr float kBoost = 0.0f;   // of p, in powers of two
template <>
constexpr float kBoost<_Float16> = 13.0f;

struct Grid {
    int64_t first;    // number of the launch's first workgroup
    int64_t blocks;   // of rows (of states), for each pair: a batch element and a head of the states
    int64_t rows;     // of a pair: queries x shared heads
    int64_t units;    // dk, dv: tiles of rows, of all shared heads
    int shared;
    int splits;
    int64_t part;     // tiles of a split
    float c;          // scale log2(e)
    float* delta;     // [row][head]
    float* norms;     // halves: of each 64 states' values
    float* largest;   // halves: [pair][lifts][2], the largest |do| and |delta| of parts of a pair's rows
    int64_t lifts;
    float* sums;      // the splits' parts
};

// The exponent of the power of two that lifts gradients of weights up to `largest` to 2^14; 0 where that says nothing.
template <class T>
__device__ __forceinline__ int lift_of(float largest) {
    if constexpr (kBoost<T> == 0.0f) return 0;
    return largest > 0.0f && largest < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(largest) : 0;
}

// The largest of n numbers, for all lanes of a wave.
__device__ __forceinline__ float largest_of(const float* p, int64_t n) {
    float v = 0.0f;
#pragma unroll 4
    for (int64_t k = threadIdx.x & 63; k < n; k += 64) v = fmaxf(v, p[k]);
    for (int k = 32; k > 0; k >>= 1) v = fmaxf(v, __shfl_xor(v, k, 64));
    return v;
}

// Halves: of each 64 states' values, the largest norm of a row.
template <class T>
__global__ void __launch_bounds__(256) norms_kernel(Attention a, float* norms) {
    static_assert(kChunk<T> == 8, "");
    const int64_t blocks = (a.states + 63) / 64, n = a.batch * a.kv_heads * blocks;
    const int lane = threadIdx.x & 63;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        const int64_t pair = i / blocks, j = (i - pair * blocks) * 64 + lane, e = pair / a.kv_heads;
        const int kv = (int)(pair - e * a.kv_heads);
        float v = 0.0f;
        if (j < a.states && (!a.mask || a.mask[e * a.mask_stride + j])) {
            const T* p = (const T*)a.v.p + (e * a.states + j) * a.v.stride + (int64_t)kv * a.head;
#pragma unroll 8
            for (int c = 0; c < (a.head + 7) / 8; ++c) {
                float x[8];
                load_chunk<T>(p, c, a.head, x);
#pragma unroll
                for (int k = 0; k < 8; ++k) v = fmaf(x[k], x[k], v);
            }
        }
        for (int k = 32; k > 0; k >>= 1) v = fmaxf(v, __shfl_xor(v, k, 64));
        if (lane == 0) norms[i] = sqrtf(v);
    }
}

// The largest of each of two numbers over the workgroup's threads.
__device__ __forceinline__ void workgroup_largest(float& x, float& y) {
    __shared__ float s[2][kWaves];
    for (int k = 32; k > 0; k >>= 1) {
        x = fmaxf(x, __shfl_xor(x, k, 64));
        y = fmaxf(y, __shfl_xor(y, k, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        s[0][threadIdx.x >> 6] = x;
        s[1][threadIdx.x >> 6] = y;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        x = fmaxf(x, s[0][k]);
        y = fmaxf(y, s[1][k]);
    }
}

// A workgroup's largest |do|^2 and |delta| to place n of its pair, as |do| and |delta|.
__device__ __forceinline__ void leave_largest(const Grid& g, int64_t pair, int64_t n, float most, float most_delta) {
    workgroup_largest(most, most_delta);
    if (threadIdx.x != 0) return;
    float* const to = g.largest + 2 * (pair * g.lifts + n);
    to[0] = sqrtf(most);
    to[1] = most_delta;
}
// The largest of those of a pair's rows, for all threads of the workgroup.
__device__ __forceinline__ void find_largest(const Grid& g, int64_t pair, float& most, float& most_delta) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2* const from = (const f32x2*)(g.largest + 2 * pair * g.lifts);
    most = most_delta = 0.0f;
#pragma unroll 4
    for (int64_t k = threadIdx.x; k < g.lifts; k += 64 * kWaves) {
        const f32x2 x = from[k];
        most = fmaxf(most, x[0]);
        most_delta = fmaxf(most_delta, x[1]);
    }
    workgroup_largest(most, most_delta);
}

// Whether weights and their gradients are operands in two parts, the second what the first was rounded by: 16-bit heads
// up to 32, in every kernel, so that the precision does not depend on the number of rows. Over few columns the sums cancel
// more than they average the roundings: in one part, heads of 16 are off by 1.6 times what rounding the gradients
// themselves leaves, heads of 2 by 2.6, of 32 by 1.47; in two parts by no more than 1.01. 2 x 2e5 rows of 4 heads of 32
// halves at 200 states, 2 shared, take 505 us so and 409 in one part; 1e6 of 4 bfloat16 at 256 states in one pass 968 and
// 595. Wider heads are held in one part, off by 1.37 to 1.47 times: in two, 2 x 8192 rows of 8 heads of 128 halves at 4096
// states would take 1315 us, 1080 in one, and 1e6 x 4 x 64 bfloat16 at 256 1750 (in two kernels: both parts of the
// weights do not fit beside the tiles in LDS) and 950.
template <class T, int D>
constexpr bool kTwoParts = sizeof(T) == 2 && D == 32;

// lse in the exponent's unit; +infinity where there is no state: all weights are 0.
template <class T>
__device__ __forceinline__ float lse_exponent(float lse) {
    return lse == -INFINITY ? INFINITY : lse * kLog2E;
}

// delta where dq is not asked for, with the same bits: a workgroup for g.part times 128 rows of a pair.
template <class T, int D>
__global__ void __launch_bounds__(64 * kWaves) delta_kernel(AttentionBackward b, Grid g) {
    using S = Square<T>;
    constexpr int kSteps = D / S::kDepth;
    const Attention& a = b.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t number = g.first + blockIdx.x, pair = number / g.blocks, block = number % g.blocks;
    const int64_t e = pair / a.kv_heads;
    const int kv = (int)(pair % a.kv_heads);
    float most = 0.0f, most_delta = 0.0f;
    const int64_t last = min((block + 1) * g.part * kWaves, (g.rows + 31) / 32);
    for (int64_t i = block * g.part * kWaves + wave; i < last; i += kWaves) {
        LaneRows<1> rows;
        rows.begin(e * a.queries, i * 32, g.rows, kv * g.shared, g.shared, lane);
        typename S::Frag go[1][kSteps], o[1][kSteps];
        rows.template load<T, kSteps>(b.grad_out, a.head, lane, go);
        rows.template load<T, kSteps>(a.out, a.head, lane, o);
        f32x16 dots = S::product(o[0][0], go[0][0]);
#pragma unroll
        for (int s = 1; s < kSteps; ++s) S::multiply(o[0][s], go[0][s], dots);
        float dot = 0.0f, square = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) dot = square_row(r, lane) == (lane & 31) ? dots[r] : dot;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int k = 0; k < 16 / (int)sizeof(T); ++k) square = fmaf((float)go[0][s][k], (float)go[0][s][k], square);
        float other = dot;
        swap32(dot, other);
        dot += other;
        other = square;
        swap32(square, other);
        most = fmaxf(most, square + other);
        most_delta = fmaxf(most_delta, fabsf(dot));
        if (rows.exists[0] && lane < 32) g.delta[rows.row(0) * a.heads + rows.head[0]] = dot;
    }
    if constexpr (kBoost<T> != 0.0f) leave_largest(g, pair, block, most, most_delta);
}

template <class T, int D, int QB, int KT, bool SPLIT>
__global__ void __launch_bounds__(64 * kWaves, D <= 64 || sizeof(T) == 2 ? 2 : 1) grad_q_kernel(AttentionBackward b, Grid g) {
    using S = Square<T>;
    using Tile = RowTile<T, D, KT, kWaves>;
    constexpr int kSteps = D / S::kDepth, kParts = 32 / S::kDepth, kSubs = KT / 32, kCols = D / 32;
    __shared__ __align__(1024) unsigned char lds[2][2][Tile::kBytes];
    const Attention& a = b.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t number = g.first + xcd_contiguous_index(blockIdx.x, gridDim.x);
    const int split = SPLIT ? (int)(number % g.splits) : 0;
    const int64_t block = (SPLIT ? number / g.splits : number) % g.blocks;
    const int64_t pair = (SPLIT ? number / g.splits : number) / g.blocks;
    const int64_t e = pair / a.kv_heads;
    const int kv = (int)(pair % a.kv_heads), d = a.head;

    LaneRows<QB> rows;
    typename S::Frag q[QB][kSteps], go[QB][kSteps];
    float lse[QB], delta[QB], by[QB];   // by: of the sums
    rows.begin(e * a.queries, (block * kWaves + wave) * QB * 32, g.rows, kv * g.shared, g.shared, lane);
    {
        typename S::Frag o[QB][kSteps];
        rows.template load<T, kSteps>(b.grad_out, d, lane, go);
        rows.template load<T, kSteps>(a.out, d, lane, o);
        rows.template load<T, kSteps>(a.q, d, lane, q);
        float norm = 0.0f, most = 0.0f, most_delta = 0.0f;
        if constexpr (kBoost<T> != 0.0f) {
            const int64_t blocks = (a.states + 63) / 64;
            norm = largest_of(g.norms + pair * blocks, blocks);
        }
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            // by the product that forms dp: where a row has one state, dp - delta is nothing
            f32x16 dots = S::product(o[n][0], go[n][0]);
#pragma unroll
            for (int s = 1; s < kSteps; ++s) S::multiply(o[n][s], go[n][s], dots);
            float dot = 0.0f, square = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) dot = square_row(r, lane) == (lane & 31) ? dots[r] : dot;
            if constexpr (kBoost<T> != 0.0f) {
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int k = 0; k < 16 / (int)sizeof(T); ++k) square = fmaf((float)go[n][s][k], (float)go[n][s][k], square);
            }
            float other = dot;   // one of the halves has it, the other 0
            swap32(dot, other);
            delta[n] = dot + other;
            other = square;
            swap32(square, other);
            square += other;
            most = fmaxf(most, square);
            most_delta = fmaxf(most_delta, fabsf(delta[n]));
            const int lift = lift_of<T>(fmaf(sqrtf(square), norm, fabsf(delta[n])));
            by[n] = __builtin_ldexpf(a.scale, -lift);
            lse[n] = INFINITY;
            if (rows.exists[n]) {
                lse[n] = lse_exponent<T>(a.lse[rows.row(n) * a.lse_row_step + rows.head[n] * a.lse_head_step]) - (float)lift;
                if (lane < 32 && split == 0) g.delta[rows.row(n) * a.heads + rows.head[n]] = delta[n];
            }
        }
        if constexpr (kBoost<T> != 0.0f)
            if (split == 0) leave_largest(g, pair, block, most, most_delta);
    }

    Tile tk, tv;
    const int64_t k_pitch = a.k.stride * (int64_t)sizeof(T), v_pitch = a.v.stride * (int64_t)sizeof(T);
    tk.begin(k_pitch, d, wave, lane);
    tv.begin(v_pitch, d, wave, lane);
    const unsigned char* k0 = (const unsigned char*)a.k.p + e * a.states * k_pitch + (int64_t)kv * d * sizeof(T);
    const unsigned char* v0 = (const unsigned char*)a.v.p + e * a.states * v_pitch + (int64_t)kv * d * sizeof(T);
    const int64_t k_end = (a.states - 1) * k_pitch + d * (int64_t)sizeof(T);
    const int64_t v_end = (a.states - 1) * v_pitch + d * (int64_t)sizeof(T);
    const uint8_t* mask = a.mask ? a.mask + e * a.mask_stride : nullptr;
    const int64_t t1 = min((split + 1) * g.part, (a.states + KT - 1) / KT);
    int64_t t = split * g.part - 1;
    const auto state_exists = [&](int64_t tile) {
        const int64_t j = tile * KT + lane;
        return lane < KT && j < a.states && (!mask || mask[j]);
    };
    bool next = state_exists(t + 1);
    uint64_t exist = 0;
    const auto load = [&](int buffer) {   // as the forward's
        do {
            if (++t >= t1) return false;
            exist = ballot(next);
            next = state_exists(t + 1);
        } while (exist == 0);
        tk.load(lds[buffer][0], k0 + t * KT * k_pitch, k_end - t * KT * k_pitch, exist, d, wave, lane);
        tv.load(lds[buffer][1], v0 + t * KT * v_pitch, v_end - t * KT * v_pitch, exist, d, wave, lane);
        return true;
    };

    f32x16 sums[QB][kCols];
#pragma unroll
    for (int n = 0; n < QB; ++n)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[n][c][r] = 0.0f;
    int buffer = 0;
    bool more = load(0);
    while (more) {
        const uint64_t bits = exist;
        wait_for_stage<1>(0);
        more = load(buffer ^ 1);
        const unsigned char* const at = lds[buffer][0];
        buffer ^= 1;
#pragma unroll 1
        for (int u = 0; u < kSubs; ++u) {
            const unsigned char *lk = at + 32 * u * Tile::kRowBytes, *lv = lk + Tile::kBytes;
            f32x16 s[QB], dp[QB];
#pragma unroll
            for (int p = 0; p < kSteps; ++p) {
                const auto f = Tile::along(lk, p, lane), w = Tile::along(lv, p, lane);
#pragma unroll
                for (int n = 0; n < QB; ++n) {
                    if (p == 0) {
                        s[n] = S::product(f, q[n][0]);
                        dp[n] = S::product(w, go[n][0]);
                    } else {
                        S::multiply(f, q[n][p], s[n]);
                        S::multiply(w, go[n][p], dp[n]);
                    }
                }
            }
            if (__builtin_expect((uint32_t)(bits >> (32 * u)) != ~0u, 0)) {
                const uint32_t w = (uint32_t)(bits >> (32 * u)) >> (4 * (lane >> 5));
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int n = 0; n < QB; ++n)
                        s[n][r] = w & (1u << ((r & 3) + 8 * (r >> 2))) ? s[n][r] : -INFINITY;
            }
#pragma unroll
            for (int n = 0; n < QB; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    dp[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], g.c, -lse[n])) * (dp[n][r] - delta[n]);
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                typename S::Frag w[QB];
#pragma unroll
                for (int n = 0; n < QB; ++n) w[n] = S::rounded(dp[n], p);
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const auto f = Tile::across(lk, p * S::kDepth, 32 * c, lane);
#pragma unroll
                    for (int n = 0; n < QB; ++n) {
                        S::multiply(f, w[n], sums[n][c]);
                        if constexpr (kTwoParts<T, D>) S::multiply(f, S::template rest<true>(dp[n], p, w[n]), sums[n][c]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < QB; ++n) {
        if (!rows.exists[n]) continue;
        const int64_t place = ((int64_t)split * a.q.rows + rows.row(n)) * a.heads + rows.head[n];
        T* to = SPLIT ? nullptr : (T*)b.grad_q.p + rows.row(n) * b.grad_q.stride + (int64_t)rows.head[n] * d;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                float v[8];
                square_rows(sums[n][c], p, v);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] *= by[n];
                const int c0 = 32 * c + 16 * p + 8 * (lane >> 5);
                if constexpr (SPLIT) store_eight<float>(g.sums + place * D, c0, D, v);
                else store_eight<T>(to, c0, d, v);
            }
    }
}

// Tiles of QT rows of one of the shared heads at a time; a wave has 32 states.
// Both sums of wide heads would leave room for one wave a SIMD: they are formed by
// a launch each, the scores in both (five products in place of four; 128 columns,
// 2 x 8192 rows x 8 heads at 4096 shared states: 705 us the two, 1018 in one launch).
enum { kGradK = 1, kGradV = 2 };
template <class T, int D>
constexpr bool kApart = sizeof(T) == 2 && D > 64;

template <class T, int D, int QT, bool SPLIT, int WHAT>
__global__ void __launch_bounds__(64 * kWaves, (D <= 64 || kApart<T, D> ? 2 : 1)) grad_kv_kernel(AttentionBackward b, Grid g) {
    using S = Square<T>;
    using Tile = RowTile<T, D, QT, kWaves>;
    constexpr int kSteps = D / S::kDepth, kParts = 32 / S::kDepth, kSubs = QT / 32, kCols = D / 32;
    __shared__ __align__(1024) unsigned char lds[2][2][Tile::kBytes];
    __shared__ __align__(16) float row_lse[2][QT], row_delta[2][QT];
    const Attention& a = b.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t number = g.first + xcd_contiguous_index(blockIdx.x, gridDim.x);
    // blocks of states that read the same rows are neighbours
    const int64_t block = number % g.blocks, split = number / g.blocks % g.splits, pair = number / g.blocks / g.splits;
    const int64_t e = pair / a.kv_heads;
    const int kv = (int)(pair % a.kv_heads), d = a.head;

    const int64_t j = (block * kWaves + wave) * 32 + (lane & 31);   // the lane's state
    const bool inside = j < a.states;
    const bool exists = inside && (!a.mask || a.mask[e * a.mask_stride + j]);
    const int64_t state = e * a.states + j;
    typename S::Frag k[1][kSteps], v[1][kSteps];
    LaneRows<1> states;
    states.begin(e * a.states, (block * kWaves + wave) * 32, a.states, kv, 1, lane);
    states.exists[0] = exists;
    states.template load<T, kSteps>(a.k, d, lane, k);
    states.template load<T, kSteps>(a.v, d, lane, v);
    int lift = 0;
    if constexpr (kBoost<T> != 0.0f && (WHAT & kGradK)) {
        float most, most_delta, square = 0.0f;
        find_largest(g, pair, most, most_delta);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int c = 0; c < 8; ++c) square = fmaf((float)v[0][s][c], (float)v[0][s][c], square);
        float other = square;
        swap32(square, other);
        lift = lift_of<T>(fmaf(most, sqrtf(square + other), most_delta));
    }
    const float lifted = __builtin_ldexpf(1.0f, lift - (int)kBoost<T>);   // p is held lifted by kBoost

    Tile tq, to;
    const int64_t q_pitch = a.q.stride * (int64_t)sizeof(T), o_pitch = b.grad_out.stride * (int64_t)sizeof(T);
    tq.begin(q_pitch, d, wave, lane);
    to.begin(o_pitch, d, wave, lane);
    const unsigned char* q0 = (const unsigned char*)a.q.p + e * a.queries * q_pitch + (int64_t)kv * g.shared * d * sizeof(T);
    const unsigned char* o0 =
        (const unsigned char*)b.grad_out.p + e * a.queries * o_pitch + (int64_t)kv * g.shared * d * sizeof(T);
    const int64_t per_head = max(g.units / g.shared, (int64_t)1);   // no queries: no tile of them either
    // a workgroup whose states all do not exist only writes zeros
    const int64_t t1 = __syncthreads_or(exists) ? min((split + 1) * g.part, g.units) : 0;
    // a wave whose states do not exist only loads: 2e5 rows of 4 heads of 64 floats at one state 551 us, 679 without
    const int subs = ballot(exists) ? kSubs : 0;
    int64_t t = split * g.part - 1;
    int h = (int)((t + 1) / per_head);         // of the next tile, among the shared heads
    int64_t in = (t + 1) - h * per_head - 1;   // the tile's number in its head
    float value = 0.0f;                        // of the thread's row: lse, or delta, on its way to LDS
    const int of = threadIdx.x % QT;
    const auto load = [&](int buffer) {
        if (++t >= t1) return false;
        if (++in == per_head) {
            in = 0;
            ++h;
        }
        const int64_t r0 = in * QT, left = a.queries - r0;
        const int64_t at = (int64_t)h * d * (int64_t)sizeof(T);
        const int64_t width = d * (int64_t)sizeof(T);
        // rows past the last: its q, an lse of +infinity and zeros for do, so that nothing of theirs is but 0 or what
        // its own is
        tq.template load_first<true, false>(lds[buffer][0], q0 + at + r0 * q_pitch, (left - 1) * q_pitch + width, left,
                                            q_pitch, d, wave, lane);
        to.template load_first<false, false>(lds[buffer][1], o0 + at + r0 * o_pitch, (left - 1) * o_pitch + width, left,
                                             o_pitch, d, wave, lane);
        const int64_t row = e * a.queries + r0 + of;
        const int head = kv * g.shared + h;
        if (threadIdx.x < QT)
            value = of < left ? lse_exponent<T>(a.lse[row * a.lse_row_step + head * a.lse_head_step]) - kBoost<T> : INFINITY;
        else if (threadIdx.x < 2 * QT)
            value = of < left ? g.delta[row * a.heads + head] : 0.0f;
        return true;
    };

    f32x16 gk[kCols], gv[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) gk[c][r] = gv[c][r] = 0.0f;
    int buffer = 0;
    bool more = load(0);
    while (more) {
        if (threadIdx.x < QT) row_lse[buffer][of] = value;
        else if (threadIdx.x < 2 * QT) row_delta[buffer][of] = value;
        wait_for_stage<1>(0);
        more = load(buffer ^ 1);
        const unsigned char* const from = lds[buffer][0];
        const float *le = row_lse[buffer], *de = row_delta[buffer];
        buffer ^= 1;
#pragma unroll 1
        for (int u = 0; u < subs; ++u) {
            const unsigned char *lq = from + 32 * u * Tile::kRowBytes, *lo = lq + Tile::kBytes;
            f32x16 s = S::product(Tile::along(lq, 0, lane), k[0][0]), dp;
            if constexpr (WHAT & kGradK) dp = S::product(Tile::along(lo, 0, lane), v[0][0]);
#pragma unroll
            for (int p = 1; p < kSteps; ++p) {
                S::multiply(Tile::along(lq, p, lane), k[0][p], s);
                if constexpr (WHAT & kGradK) S::multiply(Tile::along(lo, p, lane), v[0][p], dp);
            }
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += 4) {
                const int at = 32 * u + square_row(r0, lane);
                const f32x4 l4 = *(const f32x4*)(le + at), d4 = *(const f32x4*)(de + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[r0 + r] = __builtin_amdgcn_exp2f(fmaf(s[r0 + r], g.c, -l4[r]));
                    if constexpr (WHAT & kGradK) {
                        const float x = dp[r0 + r] - d4[r];
                        dp[r0 + r] = s[r0 + r] * (kBoost<T> != 0.0f ? x * lifted : x);
                    }
                }
            }
#pragma unroll
            for (int p = 0; p < kParts; ++p) {
                typename S::Frag w, x;
                if constexpr (WHAT & kGradV) w = S::rounded(s, p);
                if constexpr (WHAT & kGradK) x = S::rounded(dp, p);
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    if constexpr (kTwoParts<T, D>) {
                        const auto fo = Tile::across(lo, p * S::kDepth, 0, lane), fq = Tile::across(lq, p * S::kDepth, 0, lane);
                        S::multiply(fo, w, gv[0]);
                        S::multiply(fq, x, gk[0]);
                        S::multiply(fo, S::template rest<false>(s, p, w), gv[0]);
                        S::multiply(fq, S::template rest<true>(dp, p, x), gk[0]);
                        continue;
                    }
                    if constexpr (WHAT & kGradV) S::multiply(Tile::across(lo, p * S::kDepth, 32 * c, lane), w, gv[c]);
                    if constexpr (WHAT & kGradK) S::multiply(Tile::across(lq, p * S::kDepth, 32 * c, lane), x, gk[c]);
                }
            }
        }
    }
    if (!inside) return;
    // a state that does not exist gets zeros, whatever the rows hold
    const float by_k = __builtin_ldexpf(a.scale, -lift), by_v = __builtin_ldexpf(1.0f, -(int)kBoost<T>);
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            float x[8], y[8];
            square_rows(gk[c], p, x);
            square_rows(gv[c], p, y);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                x[n] = exists ? x[n] * by_k : 0.0f;
                y[n] = exists ? y[n] * by_v : 0.0f;
            }
            const int c0 = 32 * c + 16 * p + 8 * (lane >> 5);
            if constexpr (SPLIT) {
                const int64_t n = a.k.rows * a.kv_heads, at = state * a.kv_heads + kv;
                if constexpr (WHAT & kGradK) store_eight<float>(g.sums + ((2 * split) * n + at) * D, c0, D, x);
                if constexpr (WHAT & kGradV) store_eight<float>(g.sums + ((2 * split + 1) * n + at) * D, c0, D, y);
            } else {
                if ((WHAT & kGradK) && b.grad_k.p)
                    store_eight<T>((T*)b.grad_k.p + state * b.grad_k.stride + (int64_t)kv * d, c0, d, x);
                if ((WHAT & kGradV) && b.grad_v.p)
                    store_eight<T>((T*)b.grad_v.p + state * b.grad_v.stride + (int64_t)kv * d, c0, d, y);
            }
        }
}

// ---- up to 256 states of heads up to 64: all three gradients in one pass over
// the rows. A workgroup's waves hold 32 states each, with the sums of dk and dv;
// tiles of 64 rows go by. What a tile's ds is to dq needs all states: it goes to LDS
// as [state][row], and in the next step, behind that tile's barrier, the waves share the
// product k^T ds^T among them, 16 columns by 16 rows at a time, with k^T in registers.
// 1e6 rows of 4 heads of 64 bfloat16 at 256 states 930 to 995 us by card (1356 in two
// kernels), 0.7 PFLOP/s: matrix cores busy 32% of the time, vector instructions 39%,
// LDS 38%. The two waves that a SIMD has registers for do not fill one another's waits,
// which are half of their time: of 1004 us on one card 930 were left without its loads, 800
// without dq, 884 without the exponentials.
constexpr int kOnceWaves = 8, kOnceStates = 32 * kOnceWaves, kOnceRows = 64;

template <class T, int D>
__global__ void __launch_bounds__(64 * kOnceWaves, 2) once_kernel(AttentionBackward b, Grid g) {
    using S = Square<T>;
    constexpr int kTileLoads = kOnceRows * D * (int)sizeof(T) / 1024;
    constexpr int kLoaders = kTileLoads < kOnceWaves ? kTileLoads : kOnceWaves;
    using Tile = RowTile<T, D, kOnceRows, kLoaders>;
    using Weights = RowTile<T, kOnceRows, kOnceStates, kOnceWaves>;   // ds: a row a state
    constexpr int kSteps = D / 16, kCols = D / 32;
    constexpr int kAcross = D / 16, kDown = 4 * kAcross / kOnceWaves;   // 16 x 16 squares of dq across; a wave's
    constexpr int kChunks = D / 8;                                      // of a row's head
    constexpr int kWeightParts = kTwoParts<T, D> ? 2 : 1;
    __shared__ __align__(1024) unsigned char lds[2][2][Tile::kBytes], weights[2][kWeightParts][Weights::kBytes];
    __shared__ __align__(16) float row_lse[2][kOnceRows], row_delta[2][kOnceRows];
    const Attention& a = b.a;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t number = xcd_contiguous_index(blockIdx.x, gridDim.x);
    const int64_t split = number % g.splits, pair = number / g.splits;
    const int64_t e = pair / a.kv_heads;
    const int kv = (int)(pair % a.kv_heads), d = a.head;

    const int64_t j = wave * 32 + (lane & 31);   // the lane's state
    const bool inside = j < a.states;
    const bool exists = inside && (!a.mask || a.mask[e * a.mask_stride + j]);
    const int64_t state = e * a.states + j;
    typename S::Frag k[1][kSteps], v[1][kSteps];
    LaneRows<1> states;
    states.begin(e * a.states, wave * 32, a.states, kv, 1, lane);
    states.exists[0] = exists;
    states.template load<T, kSteps>(a.k, d, lane, k);
    states.template load<T, kSteps>(a.v, d, lane, v);

    // k^T of the wave's 16 columns, all states, through LDS
    const int across = wave % kAcross, down = wave / kAcross * kDown;
    typename S::Frag kt[kOnceStates / 32];
    {
        using Keys = RowTile<T, D, kOnceStates, kOnceWaves>;
        static_assert(Keys::kBytes <= (int)sizeof(weights), "");
        unsigned char* const at = weights[0][0];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {   // the lane's row, as it would be loaded
            const int r = (int)j, c = (2 * s + (lane >> 5)) ^ Keys::turn(r);
            *(typename S::Frag*)(at + r * Keys::kRowBytes + (c << 4)) = k[0][s];
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < kOnceStates / 32; ++s) kt[s] = Keys::across16(at, 32 * s, 16 * across, lane);
        __syncthreads();
    }

    Tile tq, to;
    const int64_t q_pitch = a.q.stride * (int64_t)sizeof(T), o_pitch = b.grad_out.stride * (int64_t)sizeof(T);
    tq.begin(q_pitch, d, wave, lane);
    to.begin(o_pitch, d, wave, lane);
    const int64_t first_row = e * a.queries;
    const int64_t per_head = g.units / g.shared;
    const int64_t t0 = split * g.part, t1 = min(t0 + g.part, g.units);
    int64_t t = t0 - 1;
    int h = (int)(t0 / per_head);         // of the next tile, among the shared heads
    int64_t in = t0 - h * per_head - 1;   // the tile's number in its head
    float lse = 0.0f;                     // of the thread's row, on its way to LDS
    bool lse_there = false;
    typename S::Frag o = {}, go = {};     // the thread's chunks of a row, for delta
    const int of = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks;
    const auto load = [&](int buffer) {
        if (++t >= t1) return false;
        if (++in == per_head) {
            in = 0;
            ++h;
        }
        const int64_t r0 = in * kOnceRows, left = a.queries - r0;
        const int head = kv * g.shared + h;
        const int64_t at = (int64_t)head * d * (int64_t)sizeof(T), width = d * (int64_t)sizeof(T);
        if (wave < kLoaders) {   // rows past the last: as in grad_kv_kernel
            const unsigned char* const from_q = (const unsigned char*)a.q.p + at + (first_row + r0) * q_pitch;
            const unsigned char* const from_o = (const unsigned char*)b.grad_out.p + at + (first_row + r0) * o_pitch;
            tq.template load_first<true, true>(lds[buffer][0], from_q, (left - 1) * q_pitch + width, left, q_pitch, d, wave,
                                               lane);
            to.template load_first<false, true>(lds[buffer][1], from_o, (left - 1) * o_pitch + width, left, o_pitch, d, wave,
                                                lane);
        }
        // without branches, which would wait for the loads where they meet
        const int64_t x_pitch = a.out.stride * (int64_t)sizeof(T);
        const auto outs = resource_of((const unsigned char*)a.out.p + at + (first_row + r0) * x_pitch,
                                      (left - 1) * x_pitch + width);
        const auto grads = resource_of((const unsigned char*)b.grad_out.p + at + (first_row + r0) * o_pitch,
                                       (left - 1) * o_pitch + width);
        const bool there = of < kOnceRows && of < left && chunk * 8 < d;
        o = __builtin_bit_cast(typename S::Frag, __builtin_amdgcn_raw_buffer_load_b128(
            outs, there ? (int)(uint32_t)(of * x_pitch + chunk * 16) : (int)kPastEnd, 0, 0));
        go = __builtin_bit_cast(typename S::Frag, __builtin_amdgcn_raw_buffer_load_b128(
            grads, there ? (int)(uint32_t)(of * o_pitch + chunk * 16) : (int)kPastEnd, 0, 0));
        const int64_t row = threadIdx.x % kOnceRows;
        lse = a.lse[(first_row + r0 + min(row, left - 1)) * a.lse_row_step + head * a.lse_head_step];
        lse_there = row < left;
        return true;
    };
    // dq of the tile whose ds stands in `from`: rows r0 .. of the head
    const auto add_rows = [&](const unsigned char (*from)[Weights::kBytes], int head, int64_t r0, bool there) {
        const int64_t left = there ? a.queries - r0 : 0;
#pragma unroll
        for (int n = 0; n < kDown; ++n) {
            f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < kOnceStates / 32; ++s)
#pragma unroll
                for (int part = 0; part < kWeightParts; ++part)
                    x = multiply(kt[s], Weights::across16(from[part], 32 * s, 16 * (down + n), lane), x);
            const int row = 16 * (down + n) + (lane & 15), c0 = 16 * across + 4 * (lane >> 4);
            if (row < left && c0 < d) {   // d is a multiple of 8
                typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
                Four y;
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = (T)(x[c] * a.scale);
                *(Four*)((T*)b.grad_q.p + (first_row + r0 + row) * b.grad_q.stride + (int64_t)head * d + c0) = y;
            }
        }
    };

    f32x16 gk[kCols], gv[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) gk[c][r] = gv[c][r] = 0.0f;
    const uint32_t keep = exists ? ~0u : 0u;
    int buffer = 0, last_head = 0;
    int64_t last_row = 0;
    bool more = load(0), begun = false;
    while (more) {
        float delta = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) delta = fmaf((float)go[c], (float)o[c], delta);
        float parts[1] = {delta};
        int none = 0;
        group_sum<kChunks>(parts, nullptr, none);
        if (of < kOnceRows && chunk == 0) row_delta[buffer][of] = parts[0];
        if (threadIdx.x < kOnceRows) row_lse[buffer][threadIdx.x] = lse_there ? lse_exponent<T>(lse) : INFINITY;
        const int head = kv * g.shared + h;
        const int64_t r0 = in * kOnceRows;
        wait_for_stage<1>(0);   // the tile is there, and the last one's ds; their buffers are free
        more = load(buffer ^ 1);
        // the two waves of a SIMD in opposite order: one's products beside the other's exponentials
        if (wave < kOnceWaves / 2) add_rows(weights[buffer ^ 1], last_head, last_row, begun);
        unsigned char* const to_weights = weights[buffer][0] + (int)j * Weights::kRowBytes;
#pragma unroll
        for (int u = 0; u < kOnceRows / 32; ++u) {
            const unsigned char *lq = lds[buffer][0] + 32 * u * Tile::kRowBytes, *lo = lq + Tile::kBytes;
            f32x16 s = S::product(Tile::along(lq, 0, lane), k[0][0]), dp = S::product(Tile::along(lo, 0, lane), v[0][0]);
#pragma unroll
            for (int p = 1; p < kSteps; ++p) {
                S::multiply(Tile::along(lq, p, lane), k[0][p], s);
                S::multiply(Tile::along(lo, p, lane), v[0][p], dp);
            }
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += 4) {
                const int at = 32 * u + square_row(r0, lane);
                const f32x4 l4 = *(const f32x4*)(row_lse[buffer] + at), d4 = *(const f32x4*)(row_delta[buffer] + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[r0 + r] = __builtin_amdgcn_exp2f(fmaf(s[r0 + r], g.c, -l4[r]));
                    dp[r0 + r] = s[r0 + r] * (dp[r0 + r] - d4[r]);
                }
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const auto w = S::rounded(s, p), x = S::rounded(dp, p);
                const auto leave = [&](const typename S::Frag& f, unsigned char* to) {
                    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                    const u32x4 bits = __builtin_bit_cast(u32x4, f) & keep;   // zeros for a state that does not exist
#pragma unroll
                    for (int n = 0; n < 2; ++n) {   // rows 32 u + 16 p + 8 n + 4 (lane / 32) .. + 3
                        const int c = (4 * u + 2 * p + n) ^ Weights::turn((int)j);
                        *(u32x2*)(to + (c << 4) + 8 * (lane >> 5)) = u32x2{bits[2 * n], bits[2 * n + 1]};
                    }
                };
                leave(x, to_weights);
                if constexpr (kTwoParts<T, D>) {
                    const auto fo = Tile::across(lo, p * 16, 0, lane), fq = Tile::across(lq, p * 16, 0, lane);
                    const auto rest = S::template rest<true>(dp, p, x);
                    leave(rest, to_weights + Weights::kBytes);
                    S::multiply(fo, w, gv[0]);
                    S::multiply(fq, x, gk[0]);
                    S::multiply(fo, S::template rest<false>(s, p, w), gv[0]);
                    S::multiply(fq, rest, gk[0]);
                } else {
#pragma unroll
                    for (int c = 0; c < kCols; ++c) {
                        S::multiply(Tile::across(lo, p * 16, 32 * c, lane), w, gv[c]);
                        S::multiply(Tile::across(lq, p * 16, 32 * c, lane), x, gk[c]);
                    }
                }
            }
        }
        if (wave >= kOnceWaves / 2) add_rows(weights[buffer ^ 1], last_head, last_row, begun);
        begun = true;
        last_head = head;
        last_row = r0;
        buffer ^= 1;
    }
    __syncthreads();
    add_rows(weights[buffer ^ 1], last_head, last_row, begun);
    if (!inside) return;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            float x[8], y[8];
            square_rows(gk[c], p, x);
            square_rows(gv[c], p, y);
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                x[n] = exists ? x[n] * a.scale : 0.0f;
                y[n] = exists ? y[n] : 0.0f;
            }
            const int c0 = 32 * c + 16 * p + 8 * (lane >> 5);
            const int64_t n = a.k.rows * a.kv_heads, at = state * a.kv_heads + kv;
            store_eight<float>(g.sums + ((2 * split) * n + at) * D, c0, D, x);
            store_eight<float>(g.sums + ((2 * split + 1) * n + at) * D, c0, D, y);
        }
}

// Sums of the splits' parts, in their order: set `n` x D floats, `step` sets apart.
template <class T, int D>
__global__ void __launch_bounds__(256) join_kernel(const float* sums, int splits, int64_t step, Mat to, int heads, int d) {
    const int64_t n = to.rows * heads * d;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i / d, row = at / heads;
        const int c = (int)(i - at * d), h = (int)(at - row * heads);
        float v = 0.0f;
#pragma unroll 8
        for (int k = 0; k < splits; ++k) v += sums[(k * step + at) * D + c];
        ((T*)to.p)[row * to.stride + (int64_t)h * d + c] = (T)v;
    }
}

// The splits of `tiles` for about `target` workgroups where there are half as many
// or fewer, no shorter than `least` tiles.
void split_tiles(int64_t whole, int64_t tiles, int64_t target, int64_t least, int& splits, int64_t& part) {
    int64_t n = 1;
    if (whole > 0 && 2 * whole <= target && tiles >= 2 * least) n = std::min(target / whole, tiles / least);
    part = tiles > 0 ? (tiles + n - 1) / n : 1;
    splits = tiles > 0 ? (int)((tiles + part - 1) / part) : 1;
}
// dq, as the forward: 100 rows of 4 heads of 64 at 4096 states, all three gradients,
// 24 us in 64 parts and 40 in 128, 16000 of one at 272 47 whole and 65 in parts.
// dk and dv: two workgroups a compute unit (2 x 8192 rows of 8 heads of 128 at 4096
// states 1255 us, 3060 in half as many), 64 rows a part of floats (3000 rows of 2 heads
// of 64 at 33 states 41 us, 53 with 128) and 128 of halves (132 rows of 2 heads of 16
// at 448 states 24 us, 30 with 64).
constexpr int64_t kRowTarget = 256, kRowLeast = 4, kStateTarget = 512, kStateLeast = 64;

// Whether the one-pass kernel takes it: states and heads that it holds, more states than one wave's, and as many rows as
// pay for its start and its sums' join. 1e6 rows of 4 heads at 256 states, in one pass and in two kernels: of 8 913 us and
// 1153, of 16 952 and 1227, of 32 968 and 1279, of 64 950 and 1356. Its eight waves go over all rows whatever states they
// have, which two parts of the weights make dear: of heads up to 32, up to 128 states of many rows are left to two
// kernels (5e5 x 4 x 32 at 33 states 494 us in one pass and 397, 2e5 x 4 x 32 at 64 190 and 171; few launches are
// better for few rows: 70000 x 1 x 32 at 100 50 and 69, 2e4 x 4 x 8 at 40 37 and 40).
bool at_once(const AttentionBackward& b) {
    const Attention& a = b.a;
    const int64_t tiles = (a.queries + kOnceRows - 1) / kOnceRows * (a.heads / a.kv_heads) * a.batch * a.kv_heads;
    return a.dtype == TGS_DTYPE_BFLOAT16 && b.grad_q.p && (b.grad_k.p || b.grad_v.p) && a.head <= 64 &&
           a.head % 8 == 0 && a.states > 32 && a.states <= kOnceStates && a.batch * a.kv_heads <= 1 << 21 &&
           tiles >= 1024 && (a.head > 32 || a.states > 128 || tiles < 4096);
}

// Rows of a tile of dk's and dv's: 64 but for wide floats (2e5 rows of 4 heads of 64 floats at 256 states 1539 us,
// 1555 with 32; 5e5 of 2 heads of 32 at 33 474 and 509).
constexpr int row_tile_of(int size, int64_t width) { return size == 2 || width <= 64 ? 64 : 32; }

struct Plan {
    bool once;
    int qb;
    Grid q, kv, delta;         // delta: its kernel's, where dq is not asked for
    int64_t q_workgroups, kv_workgroups, delta_workgroups;
    size_t delta_bytes, norms_bytes, largest_bytes, bytes;
};

Plan plan_of(const AttentionBackward& b) {
    const Attention& a = b.a;
    Plan p{};
    const bool halves = a.dtype != TGS_DTYPE_FLOAT32;
    const int64_t width = (a.head + 31) / 32 * 32;
    const int size = halves ? 2 : 4, state_tile = halves ? 64 : 32, row_tile = row_tile_of(size, width);
    p.q.shared = p.kv.shared = p.delta.shared = a.heads / a.kv_heads;
    p.q.rows = p.kv.rows = p.delta.rows = a.queries * p.q.shared;
    p.q.c = p.kv.c = exponent_of(a.scale);
    p.once = at_once(b);
    if (p.once) {
        const int64_t pairs = a.batch * a.kv_heads;
        p.kv.units = (a.queries + kOnceRows - 1) / kOnceRows * p.kv.shared;
        const int64_t splits = pairs < 256 ? 256 / pairs : 1;
        p.kv.part = (p.kv.units + splits - 1) / splits;
        p.kv.splits = (int)((p.kv.units + p.kv.part - 1) / p.kv.part);
        p.kv_workgroups = pairs * p.kv.splits;
        p.bytes = sizeof(float) * 2 * (size_t)(p.kv.splits * a.k.rows * a.kv_heads * width);
        return p;
    }
    p.qb = halves && width <= 64 && p.q.rows > 32 * kWaves ? 2 : 1;
    p.q.blocks = (p.q.rows + 32 * kWaves * p.qb - 1) / (32 * kWaves * p.qb);
    int64_t whole = a.batch * a.kv_heads * p.q.blocks;
    split_tiles(whole, (a.states + state_tile - 1) / state_tile, kRowTarget, kRowLeast, p.q.splits, p.q.part);
    p.q_workgroups = whole * p.q.splits;
    p.kv.blocks = (a.states + 32 * kWaves - 1) / (32 * kWaves);
    p.kv.units = (a.queries + row_tile - 1) / row_tile * p.kv.shared;
    whole = a.batch * a.kv_heads * p.kv.blocks;
    split_tiles(whole, p.kv.units, kStateTarget, (halves ? 2 : 1) * kStateLeast / row_tile, p.kv.splits, p.kv.part);
    p.kv_workgroups = whole * p.kv.splits;
    p.delta_bytes = (sizeof(float) * (size_t)(a.q.rows * a.heads) + 255) / 256 * 256;
    size_t sums = 0;
    if (b.grad_q.p && p.q.splits > 1) sums = sizeof(float) * (size_t)(p.q.splits * a.q.rows * a.heads * width);
    if ((b.grad_k.p || b.grad_v.p) && p.kv.splits > 1)
        sums = std::max(sums, sizeof(float) * 2 * (size_t)(p.kv.splits * a.k.rows * a.kv_heads * width));
    // the delta kernel: up to 4096 workgroups, one a pair at least
    const int64_t pairs = a.batch * a.kv_heads, row_blocks = (p.delta.rows + 32 * kWaves - 1) / (32 * kWaves);
    const int64_t most = std::max<int64_t>(4096 / pairs, 1);
    p.delta.part = row_blocks > 0 ? (row_blocks + most - 1) / most : 1;
    p.delta.blocks = (row_blocks + p.delta.part - 1) / p.delta.part;
    p.delta_workgroups = pairs * p.delta.blocks;
    if (a.dtype == TGS_DTYPE_FLOAT16) {
        p.q.lifts = p.delta.lifts = p.kv.lifts = b.grad_q.p ? p.q.blocks : p.delta.blocks;
        p.norms_bytes = (sizeof(float) * (size_t)(pairs * ((a.states + 63) / 64)) + 255) / 256 * 256;
        p.largest_bytes = (sizeof(float) * 2 * (size_t)(pairs * p.kv.lifts) + 255) / 256 * 256;
    }
    p.bytes = p.delta_bytes + p.norms_bytes + p.largest_bytes + sums;
    return p;
}

// f(workgroups) for launches below 2^32 threads; grid.first says where each starts.
template <class F>
void in_launches(Grid& grid, int64_t workgroups, F f) {
    constexpr int64_t kMost = ((int64_t)1 << 32) / (64 * kWaves) / 2;
    for (grid.first = 0; grid.first < workgroups; grid.first += kMost)
        f((unsigned)(workgroups - grid.first < kMost ? workgroups - grid.first : kMost));
}

unsigned join_blocks(int64_t elements) {
    const int64_t n = (elements + 255) / 256;
    return (unsigned)(n < 8192 ? n : 8192);
}

}  // namespace

size_t attention_backward_workspace(const AttentionBackward& b) { return plan_of(b).bytes; }

int launch_attention_backward(const AttentionBackward& b, void* workspace, hipStream_t s) {
    const Attention& a = b.a;
    Plan p = plan_of(b);
    p.q.delta = p.kv.delta = p.delta.delta = (float*)workspace;
    unsigned char* at = (unsigned char*)workspace + p.delta_bytes;
    p.q.norms = p.kv.norms = (float*)at;
    p.q.largest = p.kv.largest = p.delta.largest = (float*)(at += p.norms_bytes);
    p.q.sums = p.kv.sums = (float*)(at += p.largest_bytes);
    const bool states = (b.grad_k.p || b.grad_v.p) && a.k.rows > 0;
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        by_head_width(a.head, [&](auto width) {
            constexpr int D = decltype(width)::value, kTile = sizeof(T) == 2 ? 64 : 32;
            constexpr int kRowTile = row_tile_of(sizeof(T), D);
            const auto join = [&] {
                const int64_t n = a.k.rows * a.kv_heads;
                const unsigned blocks = join_blocks(n * a.head);
                if (b.grad_k.p)
                    join_kernel<T, D><<<blocks, 256, 0, s>>>(p.kv.sums, p.kv.splits, 2 * n, b.grad_k, a.kv_heads, a.head);
                if (b.grad_v.p)
                    join_kernel<T, D><<<blocks, 256, 0, s>>>(p.kv.sums + n * D, p.kv.splits, 2 * n, b.grad_v, a.kv_heads,
                                                             a.head);
            };
            if (p.once) {
                if constexpr (D <= 64 && std::is_same_v<T, __bf16>) {
                    once_kernel<T, D><<<(unsigned)p.kv_workgroups, 64 * kOnceWaves, 0, s>>>(b, p.kv);
                    join();
                }
                return;
            }
            if (b.grad_q.p && a.q.rows) {
                if (p.norms_bytes) {
                    const int64_t n = (a.batch * a.kv_heads * ((a.states + 63) / 64) + 3) / 4;
                    if constexpr (sizeof(T) == 2) norms_kernel<T><<<(unsigned)std::min<int64_t>(n, 4096), 256, 0, s>>>(a, p.q.norms);
                }
                const auto launch = [&](auto qb) {
                    constexpr int QB = decltype(qb)::value;
                    in_launches(p.q, p.q_workgroups, [&](unsigned n) {
                        if (p.q.splits > 1) grad_q_kernel<T, D, QB, kTile, true><<<n, 64 * kWaves, 0, s>>>(b, p.q);
                        else grad_q_kernel<T, D, QB, kTile, false><<<n, 64 * kWaves, 0, s>>>(b, p.q);
                    });
                };
                if constexpr (sizeof(T) == 2 && D <= 64) {
                    if (p.qb == 2) launch(Constant<2>{});
                    else launch(Constant<1>{});
                } else {
                    launch(Constant<1>{});
                }
                if (p.q.splits > 1)
                    join_kernel<T, D><<<join_blocks(a.q.rows * a.heads * a.head), 256, 0, s>>>(
                        p.q.sums, p.q.splits, a.q.rows * a.heads, b.grad_q, a.heads, a.head);
            } else if (a.q.rows && states) {
                in_launches(p.delta, p.delta_workgroups,
                            [&](unsigned n) { delta_kernel<T, D><<<n, 64 * kWaves, 0, s>>>(b, p.delta); });
            }
            if (!states) return;
            const auto launch = [&](auto what) {
                constexpr int W = decltype(what)::value;
                in_launches(p.kv, p.kv_workgroups, [&](unsigned n) {
                    if (p.kv.splits > 1) grad_kv_kernel<T, D, kRowTile, true, W><<<n, 64 * kWaves, 0, s>>>(b, p.kv);
                    else grad_kv_kernel<T, D, kRowTile, false, W><<<n, 64 * kWaves, 0, s>>>(b, p.kv);
                });
            };
            if constexpr (kApart<T, D>) {
                if (b.grad_k.p) launch(Constant<kGradK>{});
                if (b.grad_v.p) launch(Constant<kGradV>{});
            } else {
                launch(Constant<kGradK | kGradV>{});
            }
            if (p.kv.splits > 1) join();
        });
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
