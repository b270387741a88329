// Attention of a network's rows to an encoder's states: for each row and head
// s = scale q k^T over the states that exist, out = softmax(s) v, lse = log sum exp s.
//
// One pass over the states: a wave holds 32 or 64 rows' queries, and their sums out^T = v^T p^T, in registers; tiles of
// states go through LDS, loaded one ahead. The scores are formed as
// s^T = k q^T: a lane then has one row's scores, so that maxima and sums need one
// exchange between the halves of the wave, and the weights p^T are the second
// product's operand as they stand. The maximum m is that of a row's first 32
// states: later scores may pass it by what the weights' type holds, and the sum of
// the weights tells if they did (halves: the sum of weights times v, which an infinite
// weight leaves infinite or NaN). Then the wave looks for the maxima of all states and
// adds them once more where a row's is too far above. A running maximum takes a tenth
// more of the vector instructions, and a scaling of the sums on the way, even one that is never reached,
// made the compiler copy them all at every step.
//
// 16-bit weights are rounded to the values' type ahead of the second product; their
// sum is not. An output is off by up to 1.4 times what its own rounding leaves. In two
// parts (attention_backward.hip, kTwoParts) nothing would be added to that, at a
// quarter more time (1e6 x 4 x 64 bfloat16 at 256 states 511 us and 388 in one part,
// 2 x 8192 x 8 x 128 halves at 4096 333 and 274), and an infinite value would meet a
// second part of either sign, or 0: NaN, where its average is infinite.
//
// 2 x 8192 rows of 8 heads of 128 halves, 2 shared, at 4096 states: 252 to 285 us by
// card, 0.77 PFLOP/s; wide heads with 32 rows a wave, two waves a SIMD (one wave of 64
// rows 361). Matrix cores busy 37% of the time, vector instructions 41%, LDS 19%: the two
// waves overlap little, and wait for LDS and the tiles' barriers 39% of theirs.
//
// Heads that share the states' are rows side by side, so that a tile is loaded
// once for all of them. Where there are few rows, workgroups take parts of the
// states and their sums are joined by a second kernel.
#include <math.h>

#include <type_traits>

#include "attention.h"
#include "row_chunks.h"

namespace tgs {

namespace {

constexpr float kLn2 = 0.69314718055994531f;

// The sum of a lane's weights up to which floats and bfloat16 stay relative to the first states' maximum: sums of
// their products with values below 2^95 are finite then, of 256 parts of the states as well.
constexpr float kMostSum = 0x1p24f;

// A half keeps its bits down to 2^-14 of what is held as 1, and is off by at most 2^-25 of that below: with 4096 such
// states by 2^-13 of the values. For more states halves' weights are held times 2^L, with L = log2(states) - 12
// rounded up, at most 12, so that the bound stays up to 2^24 states; what later scores may be above the first ones (16
// - L powers of two) shrinks by as much.
inline int lift_of(int64_t states) {
    int lift = 0;
    while (lift < 12 && states > (int64_t)4096 << lift) ++lift;
    return lift;
}

struct Grid {
    int64_t first;       // number of the launch's first workgroup
    int64_t blocks;      // of rows, for each batch element and head of the states
    int64_t rows;        // queries x shared heads
    int shared;
    int splits;          // of the states
    int tiles;           // of a split
    int64_t part;        // held states: blocks of a wave's rows for each workgroup
    float c;             // scale log2(e)
    float lift;          // halves: L / c, what the maximum is held below its value by
    float* sums;         // of a split's parts: [splits][all rows][D], then m and l
    float* tops;
};

// A wave's 32 or 64 rows on their way over the states.
template <class T, int D, int QB>
struct WaveRows {
    using S = Square<T>;
    static constexpr bool kHalves = std::is_same_v<T, _Float16>;
    static constexpr int kSteps = D / S::kDepth;    // of the scores' product
    static constexpr int kParts = 32 / S::kDepth;   // of a square's rows as an operand
    static constexpr int kCols = D / 32;
    LaneRows<QB> at;
    typename S::Frag q[QB][kSteps];
    f32x16 out[QB][kCols];   // sums of weights times v
    float top[QB], sum[QB];  // the maximum that the weights are relative to; of the weights
    float high[QB];          // the maximum of all states, where it is looked for
    bool low[QB];            // the maximum may have to be raised

    // Rows from number i0 on of batch element b and head kv of the states.
    __device__ __forceinline__ void begin(const Attention& a, const Grid& g, int64_t b, int kv, int64_t i0, int lane) {
        at.begin(b * a.queries, i0, g.rows, kv * g.shared, g.shared, lane);
        at.template load<T, kSteps>(a.q, a.head, lane, q);
#pragma unroll
        for (int n = 0; n < QB; ++n) top[n] = -INFINITY;
    }

    // Before a pass over the states.
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            sum[n] = 0.0f;
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) out[n][c][r] = 0.0f;
        }
    }

    // Scores of the 32 states whose keys start at lk; `bits`: which of them exist.
    template <class Tile>
    __device__ __forceinline__ void score(const unsigned char* lk, uint32_t bits, f32x16 (&s)[QB], int lane) {
        typename S::Frag k[kSteps];
#pragma unroll
        for (int p = 0; p < kSteps; ++p) k[p] = Tile::along(lk, p, lane);
#pragma unroll
        for (int n = 0; n < QB; ++n) s[n] = S::product(k[0], q[n][0]);
#pragma unroll
        for (int p = 1; p < kSteps; ++p)
#pragma unroll
            for (int n = 0; n < QB; ++n) S::multiply(k[p], q[n][p], s[n]);
        if (__builtin_expect(bits != ~0u, 0)) {
            const uint32_t w = bits >> (4 * (lane >> 5));
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int n = 0; n < QB; ++n) s[n][r] = w & (1u << ((r & 3) + 8 * (r >> 2))) ? s[n][r] : -INFINITY;
        }
    }

    // Raises maxima to those of the scores. A NaN goes into the weights instead.
    static __device__ __forceinline__ void raise(const f32x16 (&s)[QB], float (&to)[QB]) {
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            float m = s[n][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) m = fmaxf(m, s[n][r]);
            float other = m;
            swap32(m, other);
            to[n] = fmaxf(fmaxf(m, other), to[n]);
        }
    }

    // Adds 32 states, whose rows start at lk and lv. `first`: the maxima are theirs.
    template <class Tile>
    __device__ __forceinline__ void add(const unsigned char* lk, const unsigned char* lv, uint32_t bits, bool first,
                                        const Grid& g, int lane) {
        const float c = g.c;
        f32x16 s[QB];
        typename S::Frag v[kParts][kCols];
        score<Tile>(lk, bits, s, lane);
        // the second product's operands are read while the weights are formed
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int k = 0; k < kCols; ++k) v[p][k] = Tile::across(lv, p * S::kDepth, 32 * k, lane);
        if (first) {
            raise(s, top);
            if constexpr (kHalves)
#pragma unroll
                for (int n = 0; n < QB; ++n) top[n] -= g.lift;
        }
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            const float less = -(top[n] == -INFINITY ? 0.0f : top[n]) * c;
            float part = 0.0f;   // of the sum: one rounding of the whole for sixteen weights
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                // floats: in two roundings, so that the largest score's weight is 1
                s[n][r] = __builtin_amdgcn_exp2f(sizeof(T) == 4 ? s[n][r] * c + less : fmaf(s[n][r], c, less));
                part = r ? part + s[n][r] : s[n][r];
            }
            sum[n] += part;
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p)
#pragma unroll
            for (int n = 0; n < QB; ++n) {
                const auto w = S::rounded(s[n], p);
#pragma unroll
                for (int k = 0; k < kCols; ++k) S::multiply(v[p][k], w, out[n][k]);
            }
    }

    // Whether the maxima of the first states may not do for some row: scores passed it
    // by more than the weights' range, or its first scores were all -infinity.
    __device__ __forceinline__ bool passed() {
        bool any = false;
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            float a, b;
            if constexpr (kHalves) a = b = out[n][0][0] * 0.0f;   // NaN: a weight was infinite, or a value is not finite
            else a = b = sum[n];
            swap32(a, b);
            low[n] = (kHalves ? !(a == 0.0f && b == 0.0f) : a > kMostSum || b > kMostSum) || top[n] == -INFINITY;
            high[n] = -INFINITY;
            any |= low[n];
        }
        return ballot(any) != 0;
    }

    // With the maxima of all states in `high`: raises those that do not do; whether there are any. The other rows keep
    // theirs, and so their results do not depend on it.
    __device__ __forceinline__ bool settle(const Grid& g) {
        bool any = false;
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            bool raised = low[n] && high[n] > top[n];
            if constexpr (kHalves) {
                const float w = __builtin_amdgcn_exp2f(fmaf(high[n], g.c, -top[n] * g.c));   // as in add
                raised = raised && (top[n] == -INFINITY || (float)(T)w == INFINITY);
            }
            if (raised) top[n] = high[n] - (kHalves ? g.lift : 0.0f);
            any |= raised;
        }
        return ballot(any) != 0;
    }

    // The sums of the lane's half of the states become those of all.
    __device__ __forceinline__ void join() {
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            float other = sum[n];
            swap32(sum[n], other);
            sum[n] += other;
        }
    }

    __device__ __forceinline__ void store(const Attention& a, int lane) {
        join();
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            if (!at.exists[n]) continue;
            const float inv = sum[n] == 0.0f ? 0.0f : 1.0f / sum[n];
            T* to = (T*)a.out.p + at.row(n) * a.out.stride + (int64_t)at.head[n] * a.head;
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float v[8];
                    square_rows(out[n][c], p, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= inv;
                    store_eight<T>(to, 32 * c + 16 * p + 8 * (lane >> 5), a.head, v);
                }
            if (a.lse && lane < 32)
                a.lse[at.row(n) * a.lse_row_step + at.head[n] * a.lse_head_step] =
                    sum[n] == 0.0f ? -INFINITY : fmaf(top[n], a.scale, logf(sum[n]));
        }
    }

    __device__ __forceinline__ void store_part(const Attention& a, const Grid& g, int split, int lane) {
        join();
#pragma unroll
        for (int n = 0; n < QB; ++n) {
            if (!at.exists[n]) continue;
            const int64_t place = ((int64_t)split * a.q.rows + at.row(n)) * a.heads + at.head[n];
            if (lane < 32) {
                g.tops[2 * place] = top[n];
                g.tops[2 * place + 1] = sum[n];
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    float v[8];
                    square_rows(out[n][c], p, v);
                    store_eight<float>(g.sums + place * D, 32 * c + 16 * p + 8 * (lane >> 5), D, v);
                }
        }
    }
};

template <class T, int D, int QB, int WAVES, int KT, bool SPLIT>
__global__ void __launch_bounds__(64 * WAVES, (D <= 64 || sizeof(T) == 2 ? 2 : 1)) attention_kernel(Attention a, Grid g) {
    using Tile = RowTile<T, D, KT, WAVES>;
    __shared__ __align__(1024) unsigned char lds[2][2][Tile::kBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t number = g.first + xcd_contiguous_index(blockIdx.x, gridDim.x);
    const int split = SPLIT ? (int)(number % g.splits) : 0;
    const int64_t block = (SPLIT ? number / g.splits : number) % g.blocks;
    const int64_t pair = (SPLIT ? number / g.splits : number) / g.blocks;
    const int64_t b = pair / a.kv_heads;
    const int kv = (int)(pair % a.kv_heads), d = a.head;

    Tile tk, tv;
    const int64_t k_pitch = a.k.stride * (int64_t)sizeof(T), v_pitch = a.v.stride * (int64_t)sizeof(T);
    tk.begin(k_pitch, d, wave, lane);
    tv.begin(v_pitch, d, wave, lane);
    // bytes of each that belong to this element's head, from its first row on
    const unsigned char* k0 = (const unsigned char*)a.k.p + b * a.states * k_pitch + (int64_t)kv * d * sizeof(T);
    const unsigned char* v0 = (const unsigned char*)a.v.p + b * a.states * v_pitch + (int64_t)kv * d * sizeof(T);
    const int64_t k_end = (a.states - 1) * k_pitch + d * (int64_t)sizeof(T);
    const int64_t v_end = (a.states - 1) * v_pitch + d * (int64_t)sizeof(T);
    const uint8_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
    const int64_t t1 = min((int64_t)(split + 1) * g.tiles, (a.states + KT - 1) / KT);
    int64_t t = (int64_t)split * g.tiles - 1;   // the last tile whose loads were started
    const auto state_exists = [&](int64_t tile) {
        const int64_t j = tile * KT + lane;
        return lane < KT && j < a.states && (!mask || mask[j]);
    };
    bool next = state_exists(t + 1);
    uint64_t exist = 0;   // of that tile's states
    const auto load = [&](int buffer) {   // the next tile that has states; false: none
        do {
            if (++t >= t1) return false;
            exist = ballot(next);
            next = state_exists(t + 1);
        } while (exist == 0);
        tk.load(lds[buffer][0], k0 + t * KT * k_pitch, k_end - t * KT * k_pitch, exist, d, wave, lane);
        tv.load(lds[buffer][1], v0 + t * KT * v_pitch, v_end - t * KT * v_pitch, exist, d, wave, lane);
        return true;
    };
    WaveRows<T, D, QB> rows;
    bool more = load(0);
    rows.begin(a, g, b, kv, (block * WAVES + wave) * QB * 32, lane);
    const auto each = [&](auto f) {   // f(keys, values, which exist) of 32 states at a time
        int buffer = 0;
        while (more) {
            const uint64_t bits = exist;
            wait_for_stage<1>(0);   // the tile is there, and every wave is done with the other buffer
            more = load(buffer ^ 1);
            const unsigned char *lk = lds[buffer][0], *lv = lds[buffer][1];
            buffer ^= 1;
#pragma unroll 1
            for (int u = 0; u < KT; u += 32) f(lk + u * Tile::kRowBytes, lv + u * Tile::kRowBytes, (uint32_t)(bits >> u));
        }
    };
    const auto restart = [&] {
        t = (int64_t)split * g.tiles - 1;
        next = state_exists(t + 1);
        more = load(0);
    };
    bool first = true;
    const auto add = [&](const unsigned char* lk, const unsigned char* lv, uint32_t bits) {
        rows.template add<Tile>(lk, lv, bits, first && bits != 0, g, lane);
        first = first && bits == 0;
    };
    rows.clear();
    each(add);
    // the tiles are loaded for all waves: any of them takes the others along
    if (__builtin_expect(__syncthreads_or(rows.passed()), 0)) {
        restart();
        each([&](const unsigned char* lk, const unsigned char*, uint32_t bits) {
            f32x16 s[QB];
            rows.template score<Tile>(lk, bits, s, lane);
            rows.raise(s, rows.high);
        });
        if (__syncthreads_or(rows.settle(g))) {
            restart();
            rows.clear();
            first = false;
            each(add);
        }
    }
    if constexpr (SPLIT) rows.store_part(a, g, split, lane);
    else rows.store(a, lane);
}

// All states of a head in LDS, loaded once; the waves go over rows by themselves,
// without a barrier, while others of the SIMD compute: four of them where a wave's
// square of rows needs 128 registers. 1e6 rows of 4 heads of 64 bfloat16 at 256
// states 388 us (0.68 PFLOP/s; 470 with tiles through LDS): 38% of the time the
// matrix cores are busy, 77% the vector units, half of whose time are the
// exponentials.
constexpr int held_waves(int size, int width) { return width <= (size == 2 ? 64 : 32) ? 16 : 8; }
template <class T, int D>
constexpr int kHeldWaves = held_waves((int)sizeof(T), D);
constexpr int kHeldBytes = 64 * 1024;   // of the keys, and as many of the values

template <class T, int D>
__global__ void __launch_bounds__((64 * kHeldWaves<T, D>)) held_kernel(Attention a, Grid g) {
    constexpr int kTileLoads = D * (int)sizeof(T) * 64 / 1024;
    constexpr int kLoaders = kTileLoads % kHeldWaves<T, D> == 0 ? kHeldWaves<T, D> : kTileLoads % 8 == 0 ? 8 : 4;
    using Tile = RowTile<T, D, 64, kLoaders>;
    constexpr int kTiles = kHeldBytes / Tile::kBytes;
    __shared__ __align__(1024) unsigned char lk[kHeldBytes], lv[kHeldBytes];
    __shared__ uint32_t exist[2 * kTiles];   // of each 32 states
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t number = xcd_contiguous_index(blockIdx.x, gridDim.x);
    const int64_t part = number % g.blocks, pair = number / g.blocks;
    const int64_t b = pair / a.kv_heads;
    const int kv = (int)(pair % a.kv_heads), d = a.head;
    const int tiles = (int)((a.states + 63) / 64);
    {
        Tile tk, tv;
        const int64_t k_pitch = a.k.stride * (int64_t)sizeof(T), v_pitch = a.v.stride * (int64_t)sizeof(T);
        tk.begin(k_pitch, d, wave, lane);
        tv.begin(v_pitch, d, wave, lane);
        const unsigned char* k0 = (const unsigned char*)a.k.p + b * a.states * k_pitch + (int64_t)kv * d * sizeof(T);
        const unsigned char* v0 = (const unsigned char*)a.v.p + b * a.states * v_pitch + (int64_t)kv * d * sizeof(T);
        const int64_t k_end = (a.states - 1) * k_pitch + d * (int64_t)sizeof(T);
        const int64_t v_end = (a.states - 1) * v_pitch + d * (int64_t)sizeof(T);
        for (int t = 0; t < tiles; ++t) {
            const int j = t * 64 + lane;
            const uint64_t bits = ballot(j < a.states && (!a.mask || a.mask[b * a.mask_stride + j]));
            if (threadIdx.x < 2) exist[2 * t + threadIdx.x] = (uint32_t)(bits >> (32 * threadIdx.x));
            if (wave >= kLoaders) continue;
            tk.load(lk + t * Tile::kBytes, k0 + t * 64 * k_pitch, k_end - t * 64 * k_pitch, bits, d, wave, lane);
            tv.load(lv + t * Tile::kBytes, v0 + t * 64 * v_pitch, v_end - t * 64 * v_pitch, bits, d, wave, lane);
        }
        wait_for_stage<1>(0);
    }
    const int squares = (int)((a.states + 31) / 32);
    const auto next = [&](int u, uint32_t& bits) {   // the next 32 states after the u-th of which any exists
        do {
            if (++u == squares) break;
            bits = (uint32_t)__builtin_amdgcn_readfirstlane((int)exist[u]);
        } while (bits == 0);
        return u;
    };
    const int64_t wave_blocks = (g.rows + 31) / 32;
    const int64_t last = min((part + 1) * g.part, wave_blocks);
    for (int64_t i = part * g.part + wave; i < last; i += kHeldWaves<T, D>) {
        WaveRows<T, D, 1> rows;
        rows.begin(a, g, b, kv, i * 32, lane);
        for (bool again = false;; again = true) {
            rows.clear();
            uint32_t bits = 0;
            const int u0 = next(-1, bits);
            for (int u = u0; u < squares; u = next(u, bits))
                rows.template add<Tile>(lk + u * 32 * Tile::kRowBytes, lv + u * 32 * Tile::kRowBytes, bits,
                                        u == u0 && !again, g, lane);
            if (__builtin_expect(again || !rows.passed(), 1)) break;
            for (int u = next(-1, bits); u < squares; u = next(u, bits)) {
                f32x16 s[1];
                rows.template score<Tile>(lk + u * 32 * Tile::kRowBytes, bits, s, lane);
                rows.raise(s, rows.high);
            }
            if (!rows.settle(g)) break;
        }
        rows.store(a, lane);
    }
}

// One to four rows (heads that share the states' included) at a few hundred states:
// one workgroup for each batch element and head of the states, eight lanes a state,
// plain multiply-adds, and one launch, where the matrix cores' kernel would have
// most of its rows empty and its parts joined by a second launch (1 row of 4 heads
// of 64 at 256 states, the call: 13.3 us so). Keys and values are on their way
// together; the scores meet in LDS.
constexpr int kFewThreads = 1024, kFewAtOnce = kFewThreads / 8, kFewTurns = 4, kFewStates = kFewAtOnce * kFewTurns;
constexpr int kFewRows = 4;
constexpr float kFewUnit = 1.0f / kFewStates;

template <class T, int PIECES, int R>
__global__ void __launch_bounds__(kFewThreads) few_kernel(Attention a, Grid g) {
    constexpr int V = kChunk<T>, kWavesFew = kFewThreads / 64, kWidth = 8 * PIECES * V;
    __shared__ float weights[R][kFewStates], parts[kWavesFew][R][kWidth];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = threadIdx.x & 7, d = a.head;
    const int64_t b = blockIdx.x / a.kv_heads;
    const int kv = (int)(blockIdx.x % a.kv_heads), states = (int)a.states;
    float q[R][PIECES][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = min(r, (int)g.rows - 1);
        const T* p = (const T*)a.q.p + (b * a.queries + i / g.shared) * a.q.stride + (int64_t)(kv * g.shared + i % g.shared) * d;
#pragma unroll
        for (int n = 0; n < PIECES; ++n) load_chunk<T>(p, l + 8 * n, d, q[r][n]);
    }
    float v[kFewTurns][PIECES][V];
    int there = 0;   // which of them exist
#pragma unroll
    for (int t = 0; t < kFewTurns; ++t) {
        const int j = t * kFewAtOnce + (int)threadIdx.x / 8;
        const int64_t at = b * a.states + min(j, states - 1);   // the loads need no branch
        const bool exists = j < states && (!a.mask || a.mask[b * a.mask_stride + j]);
        there |= (int)exists << t;
        float k[PIECES][V], s[R];
#pragma unroll
        for (int n = 0; n < PIECES; ++n) {
            load_chunk<T>((const T*)a.k.p + at * a.k.stride + (int64_t)kv * d, l + 8 * n, d, k[n]);
            load_chunk<T>((const T*)a.v.p + at * a.v.stride + (int64_t)kv * d, l + 8 * n, d, v[t][n]);
        }
        int none = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = 0.0f;
#pragma unroll
            for (int n = 0; n < PIECES; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) s[r] = fmaf(q[r][n][e], k[n][e], s[r]);
        }
        group_sum<8>(s, nullptr, none);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (l == 0) weights[r][j] = exists ? s[r] * g.c : -INFINITY;
    }
    __syncthreads();
    float top[R], sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {   // each wave by itself
        top[r] = -INFINITY;
        sum[r] = 0.0f;
        for (int j = lane; j < kFewStates; j += 64) top[r] = fmaxf(top[r], weights[r][j]);
        for (int k = 32; k > 0; k >>= 1) top[r] = fmaxf(top[r], __shfl_xor(top[r], k, 64));
        const float from = top[r] == -INFINITY ? 0.0f : top[r];
        for (int j = lane; j < kFewStates; j += 64) sum[r] += __builtin_amdgcn_exp2f(weights[r][j] - from);
        for (int k = 32; k > 0; k >>= 1) sum[r] += __shfl_xor(sum[r], k, 64);
        float out[PIECES][V] = {};
#pragma unroll
        for (int t = 0; t < kFewTurns; ++t) {
            if (!(there >> t & 1)) continue;   // what does not exist may hold anything
            // weights of 1 and less times a power of two: the sums stay below the largest value
            const float w = kFewUnit * __builtin_amdgcn_exp2f(weights[r][t * kFewAtOnce + (int)threadIdx.x / 8] - from);
#pragma unroll
            for (int n = 0; n < PIECES; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) out[n][e] = fmaf(w, v[t][n][e], out[n][e]);
        }
#pragma unroll
        for (int n = 0; n < PIECES; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float x = out[n][e], y;
                x = dpp_add<0x128>(x);   // eight lanes on
                y = x;
                swap16(x, y);
                y = x += y;
                swap32(x, y);
                x += y;
                if (lane < 8) parts[wave][r][(l + 8 * n) * V + e] = x;
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (int)g.rows * kWidth; i += kFewThreads) {
        const int r = i / kWidth, c = i % kWidth;
        if (c >= d) continue;
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kWavesFew; ++w) x += parts[w][r][c];
        float of = 0.0f, most = 0.0f;
#pragma unroll
        for (int k = 0; k < R; ++k) {
            of = k == r ? sum[k] : of;
            most = k == r ? top[k] : most;
        }
        const int64_t row = b * a.queries + r / g.shared;
        const int head = kv * g.shared + r % g.shared;
        ((T*)a.out.p)[row * a.out.stride + (int64_t)head * d + c] = (T)(of == 0.0f ? 0.0f : x * (1.0f / kFewUnit / of));
        // the maximum is in the exponent's unit, of a scale that is never 0
        if (a.lse && c == 0)
            a.lse[row * a.lse_row_step + head * a.lse_head_step] =
                of == 0.0f ? -INFINITY : fmaf(most, kLn2, logf(of));
    }
}

// Joins the splits' sums: a wave for each row and head.
template <class T, int D>
__global__ void __launch_bounds__(256) join_kernel(Attention a, Grid g) {
    const int lane = threadIdx.x & 63;
    const int64_t n = a.q.rows * a.heads;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int64_t)gridDim.x * 4) {
        float top = -INFINITY;
#pragma unroll 8
        for (int k = 0; k < g.splits; ++k) top = fmaxf(top, g.tops[2 * (k * n + i)]);
        const float less = -(top == -INFINITY ? 0.0f : top) * g.c;
        float sum = 0.0f, v[(D + 63) / 64] = {};
#pragma unroll 8
        for (int k = 0; k < g.splits; ++k) {
            const int64_t at = k * n + i;
            const float w = __builtin_amdgcn_exp2f(g.tops[2 * at] * g.c + less);   // 1 for the largest
            sum = fmaf(w, g.tops[2 * at + 1], sum);
#pragma unroll
            for (int c = 0; c < (D + 63) / 64; ++c)
                if (64 * c + lane < D) v[c] = fmaf(w, g.sums[at * D + 64 * c + lane], v[c]);
        }
        const int64_t r = i / a.heads;
        const int h = (int)(i % a.heads);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* to = (T*)a.out.p + r * a.out.stride + (int64_t)h * a.head;
#pragma unroll
        for (int c = 0; c < (D + 63) / 64; ++c)
            if (64 * c + lane < a.head) to[64 * c + lane] = (T)(v[c] * inv);
        if (a.lse && lane == 0)
            a.lse[r * a.lse_row_step + h * a.lse_head_step] =
                sum == 0.0f ? -INFINITY : fmaf(top, a.scale, logf(sum));
    }
}

struct Plan {
    int qb;
    bool held, few;
    Grid grid;
    int64_t workgroups;
    size_t bytes;
};

constexpr int kWaves = 4;
constexpr int64_t kMostPairs = 1 << 21;   // of 1024 threads: a launch below 2^32

Plan plan_of(const Attention& a) {
    Plan p{};
    const bool halves = a.dtype != TGS_DTYPE_FLOAT32;
    const int64_t width = (a.head + 31) / 32 * 32, pairs = a.batch * a.kv_heads;
    p.grid.shared = a.heads / a.kv_heads;
    p.grid.rows = a.queries * p.grid.shared;
    p.grid.c = exponent_of(a.scale);
    p.grid.lift = a.dtype == TGS_DTYPE_FLOAT16 ? fminf((float)lift_of(a.states) / p.grid.c, 0x1p126f) : 0.0f;
    p.grid.splits = 1;
    const int64_t wave_blocks = (p.grid.rows + 31) / 32;
    // where the states fit and every wave has rows; floats of wide heads need too many registers for its eight waves
    p.held = a.states > 0 && (a.states + 63) / 64 * 64 * width * (halves ? 2 : 4) <= kHeldBytes && (halves || width <= 64) &&
             wave_blocks * pairs >= 256 * held_waves(halves ? 2 : 4, (int)width) && pairs <= kMostPairs;
    if (p.held) {
        const int64_t parts = pairs < 256 ? 256 / pairs : 1;
        p.grid.part = (wave_blocks + parts - 1) / parts;
        p.grid.blocks = (wave_blocks + p.grid.part - 1) / p.grid.part;
        p.workgroups = p.grid.blocks * pairs;
        return p;
    }
    // several rows of heads above 128 bytes are no faster so (4 rows of 128 halves at 300 states 17.9 us and 17.0, of
    // 128 floats at 500 25.3 and 16.4; of 64 halves at 100 13.7 and 16.2)
    p.few = (p.grid.rows == 1 || (p.grid.rows <= kFewRows && a.head * (halves ? 2 : 4) <= 128)) && a.states >= 1 &&
            a.states <= kFewStates && pairs <= kMostPairs;
    if (p.few) {
        p.workgroups = pairs;
        return p;
    }
    const int kt = halves ? 64 : 32;
    // two squares of rows a wave where their workgroups still fill the card twice: 2000 rows of 4 heads of 64 at 2000
    // states 34.2 us with two and 25.9 with one, 16384 of 8 at 4096 193 and 225
    p.qb = halves && width <= 64 && pairs * ((p.grid.rows + 64 * kWaves - 1) / (64 * kWaves)) >= 512 ? 2 : 1;
    p.grid.blocks = (p.grid.rows + 32 * kWaves * p.qb - 1) / (32 * kWaves * p.qb);
    const int64_t whole = pairs * p.grid.blocks, tiles = (a.states + kt - 1) / kt;
    int64_t splits = 1;
    // parts of the states for half a card of workgroups or less, once each workgroup has eight tiles: 16000 rows of a
    // head of 64 at 272 states 14.7 us whole and 27.5 in four parts, 100 rows of 4 at 4096 41 and 18 (in 64)
    if (whole < 128 && tiles >= 8) {
        splits = 256 / whole < tiles ? 256 / whole : tiles;
        p.grid.tiles = (int)((tiles + splits - 1) / splits);
        splits = (tiles + p.grid.tiles - 1) / p.grid.tiles;
    }
    if (splits == 1) p.grid.tiles = (int)(tiles < 0x7fffffff ? tiles : 0x7fffffff);
    p.grid.splits = (int)splits;
    p.workgroups = whole * splits;
    if (splits > 1) p.bytes = sizeof(float) * (size_t)(splits * a.q.rows * a.heads * (width + 2));
    return p;
}

}  // namespace

size_t attention_workspace(const Attention& a) { return plan_of(a).bytes; }

int launch_attention(const Attention& a, void* workspace, hipStream_t s) {
    Plan p = plan_of(a);
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        by_head_width(a.head, [&](auto width) {
            constexpr int D = decltype(width)::value, KT = sizeof(T) == 2 ? 64 : 32;
            if (p.held) {
                if constexpr (sizeof(T) == 2 || D <= 64)
                    held_kernel<T, D>
                        <<<(unsigned)p.workgroups, 64 * kHeldWaves<T, D>, 0, s>>>(a, p.grid);
                return;
            }
            if (p.few) {
                constexpr int kPieces = (D + 8 * kChunk<T> - 1) / (8 * kChunk<T>);
                if (p.grid.rows == 1) few_kernel<T, kPieces, 1><<<(unsigned)p.workgroups, kFewThreads, 0, s>>>(a, p.grid);
                else few_kernel<T, 1, kFewRows><<<(unsigned)p.workgroups, kFewThreads, 0, s>>>(a, p.grid);
                return;
            }
            p.grid.sums = (float*)workspace;
            p.grid.tops = p.grid.sums + (p.grid.splits > 1 ? p.grid.splits * a.q.rows * a.heads * D : 0);
            // a launch of 2^32 threads or more loses what is above
            constexpr int64_t kMost = ((int64_t)1 << 32) / (64 * kWaves) / 2;
            for (p.grid.first = 0; p.grid.first < p.workgroups; p.grid.first += kMost) {
                const int64_t left = p.workgroups - p.grid.first;
                const unsigned n = (unsigned)(left < kMost ? left : kMost);
                const auto launch = [&](auto qb, auto split) {
                    attention_kernel<T, D, decltype(qb)::value, kWaves, KT, decltype(split)::value != 0>
                        <<<n, 64 * kWaves, 0, s>>>(a, p.grid);
                };
                const auto by_split = [&](auto qb) {
                    if (p.grid.splits > 1) launch(qb, Constant<1>{});
                    else launch(qb, Constant<0>{});
                };
                if constexpr (sizeof(T) == 2 && D <= 64) {
                    if (p.qb == 2) by_split(Constant<2>{});
                    else by_split(Constant<1>{});
                } else {
                    by_split(Constant<1>{});
                }
            }
            if (p.grid.splits > 1) {
                const int64_t n = (a.q.rows * a.heads + 3) / 4;
                join_kernel<T, D><<<(unsigned)(n < 65536 ? n : 65536), 256, 0, s>>>(a, p.grid);
            }
        });
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
