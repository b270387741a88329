// Muon's update of a network's matrices (K. Jordan and others, "Muon: an
// optimizer for hidden layers in neural networks", 2024: the coefficients and
// the factor for tall matrices; the momentum is averaged here): momentum, the
// Newton-Schulz steps on the normalised update, the weights. Every phase is one
// launch over all matrices.
//
// X is kept with its shorter side as rows (the transpose of a tall matrix), so
// that X X^T is the smaller of the two Gram matrices. X, the Gram matrix G and
// the polynomial P = b G + c G^2 are held as two halves each, hi + lo with
// lo = half(v - hi), of the value times 2^12: 22 bits of every element down to
// 2^-14 of one and 2^-37 absolutely below, where lo is subnormal, in the range of
// halves (|X|, |G| < 2, |P| < 3: the singular values of X stay below 1.3). A
// product is then three of halves, hi hi + hi lo + lo hi with float sums (lo lo
// is 2^-22 of it), at the matrix cores' half rate: the update is off by 1e-6 to
// 2e-6 of itself, as the same formula in float products is. Halves alone (11
// bits) would leave the update's small singular directions, which the steps lift
// up to 485 times, wrong by several percent.
// A row holds 32 hi and then their 32 lo in turn, so that a step of 32 of k is
// one cache line of it.
//
// Four of 1024 x 4096: Gram 97 us, square 33, update 130, which is 0.61, 0.45 and
// 0.80 PFLOP/s of halves where large products reach 1.4. Gram's and the square's
// 144 tiles are on 256 compute units; otherwise the tiles' turns of loads, LDS
// reads and matrix instructions bound them. A small network's launches (256 x
// 256: 7 to 9 us) are bound by their chains of waits. The element passes move 12
// bytes an element in 39 to 51 us (17 M elements, 4 to 5.2 TB/s).
//
// G and P are symmetric: only the tiles on and below the diagonal are made, and
// each is stored a second time transposed, through LDS.
#include <math.h>

#include "mfma_tile.h"

namespace tgs {

namespace {

constexpr float kScale = 4096.0f;
constexpr int kPatch = 64;   // edge of the element passes' patches

// Halves between a row's end and the next row: rows of a power of two would all
// start on the same few channels of the cache.
constexpr int kRowPad = 64;
// A patch's threads: sixteen on a row, four columns each, over four rows apart by kPatchDown.
constexpr int kPatchThreads = 256;
constexpr int kPatchWaves = kPatchThreads / 64;
constexpr int kPatchDown = kPatchThreads / 16, kPatchTurns = kPatch / kPatchDown;

// The matrix that number `n` of a launch's work belongs to: the last whose
// first number is not above it. `firsts` are the matrices' first numbers; a
// wave looks at 64 of them at a time.
__device__ __forceinline__ int part_of(const uint32_t* firsts, int count, uint32_t n) {
    const int lane = threadIdx.x & 63;
    int part = -1;
    for (int k = 0; k < count; k += 64) {
        const uint64_t below = ballot(k + lane < count && firsts[min(k + lane, count - 1)] <= n);
        part += __popcll(below);
        if (below != ~0ull) break;
    }
    return __builtin_amdgcn_readfirstlane(part);
}

// Where column c of a row is: its hi, and 32 elements on its lo.
__device__ __forceinline__ int64_t column(int64_t c) { return (c >> 5) * 64 + (c & 31); }

__device__ __forceinline__ double workgroup_sum(double v) {
    __shared__ double s[kPatchWaves];
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int k = 1; k < kPatchWaves; ++k) v += s[k];
    return v;
}

__device__ __forceinline__ float update_of(float g, float m, const MuonStep& p) {
    return p.nesterov ? fmaf(p.momentum, m, g) : m;
}

template <class T>
struct Loose4 {   // four elements of a row, at any element's address
    typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
template <class T>
__device__ __forceinline__ f32x4 load4(const T* p, int n) {
    if (n >= 4) return __builtin_convertvector(*(const typename Loose4<T>::type*)p, f32x4);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) v[e] = (float)p[e];
    return v;
}
template <class T>
__device__ __forceinline__ void store4(T* p, int n, f32x4 v) {
    if (n >= 4) {
        *(typename Loose4<T>::type*)p = __builtin_convertvector(v, typename Loose4<T>::type);
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = (T)v[e];
}

// Where a thread's fours of a patch are: rows r, r + kPatchDown, ..., columns
// c .. c + 3, of which n exist in a matrix of `cols`.
struct PatchPlace {
    int q, l;
    int64_t r0, c0, r, c;
    int n;
    __device__ PatchPlace(uint32_t number, int64_t cols)
        : q(threadIdx.x >> 4), l(threadIdx.x & 15) {
        const uint32_t across = (uint32_t)((cols + kPatch - 1) / kPatch);
        r0 = (int64_t)(number / across) * kPatch;
        c0 = (int64_t)(number % across) * kPatch;
        r = r0 + q;
        c = c0 + 4 * l;
        n = (int)min(max(cols - c, (int64_t)0), (int64_t)4);
    }
};

// The thread's gradients and momenta, all on their way at once.
template <class G>
__device__ __forceinline__ void load_patch(const MuonPart& a, const PatchPlace& at, f32x4 (&g)[kPatchTurns],
                                           f32x4 (&m)[kPatchTurns]) {
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {
        const int64_t r = at.r + k * kPatchDown;
        const int n = r < a.w.rows ? at.n : 0;
        g[k] = load4((const G*)a.g.p + r * a.g.stride + at.c, n);
        m[k] = load4((const float*)a.m.p + r * a.m.stride + at.c, n);
    }
}

// M <- mu M + (1 - mu) s G, and the patch's sum of squares of U.
template <class G>
__global__ void __launch_bounds__(kPatchThreads) momentum_kernel(const MuonPart* parts, const uint32_t* firsts, int count,
                                                                 MuonStep p, double* sums) {
    const MuonPart& a = parts[part_of(firsts, count, blockIdx.x)];
    const PatchPlace at(blockIdx.x - a.first[kMuonPatches], a.w.cols);
    f32x4 g[kPatchTurns], m[kPatchTurns];
    load_patch<G>(a, at, g, m);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {
        const int64_t r = at.r + k * kPatchDown;
#pragma unroll
        for (int e = 0; e < 4; ++e) {   // those that do not exist are zeros
            const float s = g[k][e] * p.grad_scale;
            m[k][e] = fmaf(p.momentum, m[k][e], s);
            const double u = (double)update_of(s, m[k][e], p);
            if (r < a.w.rows && e < at.n) sum += u * u;
        }
        store4((float*)a.m.p + r * a.m.stride + at.c, r < a.w.rows ? at.n : 0, m[k]);
    }
    sum = workgroup_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// Four columns from c, a multiple of four, of a row of split values.
__device__ __forceinline__ void store_split(_Float16* row, int64_t c, f32x4 v) {
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    const half4 hi = __builtin_convertvector(v, half4);
    *(half4*)(row + column(c)) = hi;
    *(half4*)(row + column(c) + 32) = __builtin_convertvector(v - __builtin_convertvector(hi, f32x4), half4);
}
__device__ __forceinline__ f32x4 load_split(const _Float16* row, int64_t c) {
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    return __builtin_convertvector(*(const half4*)(row + column(c)), f32x4) +
           __builtin_convertvector(*(const half4*)(row + column(c) + 32), f32x4);
}

// X = U / max(|U|, epsilon), scaled and split; a tall matrix through LDS into
// its transpose. Columns up to a multiple of 32 are zeros.
template <class G>
__global__ void __launch_bounds__(kPatchThreads) normalise_kernel(const MuonPart* parts, const uint32_t* firsts, int count,
                                                                  MuonStep p, const double* sums) {
    const MuonPart& a = parts[part_of(firsts, count, blockIdx.x)];
    const PatchPlace at(blockIdx.x - a.first[kMuonPatches], a.w.cols);
    f32x4 g[kPatchTurns], m[kPatchTurns];
    load_patch<G>(a, at, g, m);
    const int64_t patches = (a.w.cols + kPatch - 1) / kPatch * ((a.w.rows + kPatch - 1) / kPatch);
    double sum = 0.0;
#pragma unroll 4
    for (int64_t k = threadIdx.x; k < patches; k += kPatchThreads) sum += sums[a.first[kMuonPatches] + k];
    const double norm = sqrt(workgroup_sum(sum));
    const double inv = (double)kScale / (norm < (double)p.epsilon ? (double)p.epsilon : norm);   // NaN stays
    _Float16* const x = a.x[0];
    __shared__ float t[kPatch][kPatch + 1];
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {
        const int q = at.q + k * kPatchDown;
        const int64_t r = at.r0 + q;
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = r < a.w.rows && e < at.n
                       ? (float)((double)update_of(g[k][e] * p.grad_scale, m[k][e], p) * inv) : 0.0f;
        if (a.tall) {
#pragma unroll
            for (int e = 0; e < 4; ++e) t[q][4 * at.l + e] = v[e];
        } else if (r < a.side && 2 * at.c < a.x_cols) {
            store_split(x + r * a.x_stride, at.c, v);
        }
    }
    if (!a.tall) return;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {
        const int q = at.q + k * kPatchDown;
        const int64_t r = at.c0 + q, c = at.r0 + 4 * at.l;   // of X
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = t[4 * at.l + e][q];
        if (r < a.side && 2 * c < a.x_cols) store_split(x + r * a.x_stride, c, v);
    }
}

// W <- keep W - lr shape X, and the copy.
template <class C>
__global__ void __launch_bounds__(kPatchThreads) apply_kernel(const MuonPart* parts, const uint32_t* firsts, int count,
                                                              MuonStep p) {
    const MuonPart& a = parts[part_of(firsts, count, blockIdx.x)];
    const PatchPlace at(blockIdx.x - a.first[kMuonPatches], a.w.cols);
    const _Float16* const x = a.x[p.iterations & 1];
    const float step = p.lr * a.shape * (1.0f / kScale);
    __shared__ float t[kPatch][kPatch + 1];
    f32x4 w[kPatchTurns], v[kPatchTurns];
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {
        const int64_t r = at.r + k * kPatchDown;
        w[k] = load4((const float*)a.w.p + r * a.w.stride + at.c, r < a.w.rows ? at.n : 0);
    }
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {   // X's rows are the patch's columns if it is tall
        const int64_t r = (a.tall ? at.c0 : at.r0) + at.q + k * kPatchDown, c = (a.tall ? at.r0 : at.c0) + 4 * at.l;
        v[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (r < a.side && 2 * c < a.x_cols) v[k] = load_split(x + r * a.x_stride, c);
    }
    if (a.tall) {
#pragma unroll
        for (int k = 0; k < kPatchTurns; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) t[4 * at.l + e][at.q + k * kPatchDown] = v[k][e];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kPatchTurns; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] = t[at.q + k * kPatchDown][4 * at.l + e];
    }
#pragma unroll
    for (int k = 0; k < kPatchTurns; ++k) {
        const int64_t r = at.r + k * kPatchDown;
        const int n = r < a.w.rows ? at.n : 0;
        f32x4 u;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = fmaf(-step, v[k][e], p.keep * w[k][e]);
        store4((float*)a.w.p + r * a.w.stride + at.c, n, u);
        if (a.c.p) store4((C*)a.c.p + r * a.c.stride + at.c, n, u);
    }
}

// ---- the products

// A tile of the three-product sum, in steps of 32 of k, two of them a stage of
// the ring and a barrier. K-contiguous operands are matrices of twice the
// columns, whose steps of 128 bytes are a row's 32 hi and 32 lo; the
// R-contiguous X has tiles of twice the rows and steps of 32 k.
template <int WI, int WJ, int TI, int TJ, int STAGES, bool A_RC>
struct SplitTile {
    static constexpr int kWavesI = WI, kWavesJ = WJ;
    static constexpr int kWaves = WI * WJ, kThreads = 64 * kWaves;
    static constexpr int BI = WI * TI * 16, BJ = WJ * TJ * 16;
    using T = _Float16;
    using A = TileSide<T, A_RC ? 2 * BI : BI, kWaves, A_RC, A_RC ? 64 : 128>;
    using B = TileSide<T, BJ, kWaves, false, 128>;
    static constexpr int kStep = A::kBytes + B::kBytes, kStage = 2 * kStep, kLds = STAGES * kStage;
    static constexpr int kLoads = 2 * (A::kLoads + B::kLoads);   // a wave and stage

    static __device__ __forceinline__ void run(unsigned char* lds, const TileOperand& a, const TileOperand& b, int64_t i0,
                                               int64_t j0, int steps, f32x4 (&acc)[TI][TJ]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wi = wave / WJ, wj = wave % WJ;
        A sa;
        B sb;
        sa.begin(a, A_RC ? 2 * i0 : i0, 0, wave, lane);
        sb.begin(b, j0, 0, wave, lane);
#pragma unroll
        for (int u = 0; u < TI; ++u)
#pragma unroll
            for (int v = 0; v < TJ; ++v) acc[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const int stages = (steps + 1) / 2;
        int left = steps;   // of the steps from the next load on; none: zeros
        unsigned char* fill = lds;
        const auto load = [&] {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                sa.load(fill + q * kStep, (int64_t)left * A::kDepth, wave, lane);
                sb.load(fill + q * kStep + A::kBytes, (int64_t)left * B::kDepth, wave, lane);
                --left;
            }
            fill = fill + kStage < lds + kLds ? fill + kStage : lds;
        };
#pragma unroll
        for (int n = 0; n < STAGES; ++n)
            if (n < stages) load();
        const unsigned char* from = lds;
        typename Frag<T>::type fa[2][2][TI], fb[2][2][TJ];   // of the stage's first and second step; hi, lo
        const auto read = [&](int q) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int v = 0; v < TJ; ++v)
                    fb[q][h][v] = B::fragment(from + q * kStep + A::kBytes, (wj * TJ + v) * 16, h, lane);
#pragma unroll
                for (int u = 0; u < TI; ++u) {
                    const int r = (wi * TI + u) * 16;
                    fa[q][h][u] = A_RC ? A::fragment(from + q * kStep, (r & ~31) * 2 + 32 * h + (r & 16), 0, lane)
                                       : A::fragment(from + q * kStep, r, h, lane);
                }
            }
        };
        const auto multiply_all = [&](int q) {
#pragma unroll
            for (int h = 0; h < 3; ++h)   // hi hi, hi lo, lo hi: the squares in turn, no sum waits for its last
#pragma unroll
                for (int u = 0; u < TI; ++u)
#pragma unroll
                    for (int v = 0; v < TJ; ++v)
                        acc[u][v] = multiply(fa[q][h == 2][u], fb[q][h == 1][v], acc[u][v]);
        };
        wait_for_stage<kLoads>(min(stages - 1, STAGES - 1));
        read(0);
        for (int t = 0; t + 1 < stages; ++t) {   // as Tile's
            read(1);
            multiply_all(0);
            wait_for_stage<kLoads>(min(stages - 2 - t, STAGES - 2));
            if (t + STAGES < stages) load();
            from = from + kStage < lds + kLds ? from + kStage : lds;
            read(0);
            multiply_all(1);
        }
        read(1);
        multiply_all(0);
        multiply_all(1);
    }
};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Gram: G = X X^T. Square: P = b G + c G G. Update: X' = a X + P X. The stored
// matrices are zero up to a multiple of 32 columns, which the products keep:
// they run over whole strides.
template <int PHASE, int WI, int WJ, int TI, int TJ, int STAGES>
__global__ void __launch_bounds__(64 * WI * WJ) product_kernel(const MuonPart* parts, const uint32_t* firsts, int count,
                                                               uint32_t total, int turn) {
    constexpr bool kUpdate = PHASE == kMuonUpdate;
    using P = SplitTile<WI, WJ, TI, TJ, STAGES, kUpdate>;
    __shared__ __align__(1024) unsigned char lds[P::kLds];
    // an XCD's workgroups take neighbouring tiles of each matrix; the larger matrices come first
    const int part = part_of(firsts, count, blockIdx.x);
    const MuonPart& a = parts[part];
    const uint32_t first = firsts[part], tiles = (part + 1 < count ? firsts[part + 1] : total) - first;
    const uint32_t local = xcd_contiguous_index(blockIdx.x - first, tiles);
    const _Float16* x = a.x[turn];
    const int64_t out_stride = kUpdate ? a.x_stride : a.g_stride, out_cols = kUpdate ? a.x_cols : a.g_cols;
    uint32_t ti, tj;
    if constexpr (kUpdate) {
        tile_of(local, (uint32_t)((out_cols / 2 + P::BI - 1) / P::BI), (uint32_t)((a.side + P::BJ - 1) / P::BJ), ti, tj);
    } else {   // row ti of the triangle starts at ti (ti + 1) / 2
        static_assert(P::BI == P::BJ, "the mirrored tile has the same shape");
        ti = (uint32_t)((sqrtf(8.0f * (float)local + 1.0f) - 1.0f) * 0.5f);
        while ((uint64_t)ti * (ti + 1) / 2 > local) --ti;
        while ((uint64_t)(ti + 1) * (ti + 2) / 2 <= local) ++ti;
        tj = local - (uint32_t)((uint64_t)ti * (ti + 1) / 2);
    }
    const int64_t i0 = (int64_t)ti * P::BI, j0 = (int64_t)tj * P::BJ;
    f32x4 acc[TI][TJ];
    const TileOperand tx{x, a.side, a.x_cols, a.x_stride};
    const _Float16* from = nullptr;   // added to the products, and to where
    _Float16* to;
    if constexpr (PHASE == kMuonGram) {
        P::run(lds, tx, tx, i0, j0, (int)(a.x_cols / 64), acc);
        to = a.gram;
    } else if constexpr (PHASE == kMuonSquare) {
        const TileOperand tg{a.gram, a.side, a.g_cols, a.g_stride};
        P::run(lds, tg, tg, i0, j0, (int)(a.g_cols / 64), acc);
        from = a.gram;
        to = a.poly;
    } else {
        // k runs over P's columns, X's rows: those past the side are zeros in P and not there in X
        const TileOperand tp{a.poly, a.side, a.g_cols, a.g_stride};
        P::run(lds, tx, tp, i0, j0, (int)(a.g_cols / 64), acc);
        from = x;
        to = a.x[turn ^ 1];
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = wave / WJ, wj = wave % WJ;
    constexpr float kProducts = (PHASE == kMuonSquare ? kNewtonSchulzC : 1.0f) / kScale;
    constexpr float kAdded = PHASE == kMuonSquare ? kNewtonSchulzB : kNewtonSchulzA;
    const bool mirrored = !kUpdate && ti != tj;
    constexpr int kMirrorPitch = P::BJ + 8;   // halves; 16-byte rows, neighbouring ones on other banks
    static_assert(kUpdate || 2 * P::BI * kMirrorPitch * 2 <= P::kLds, "the stages hold the mirrored tile");
    _Float16* const mirror = (_Float16*)lds;   // [hi, lo][i][j]
    if (mirrored) lds_barrier();               // the stages are read
#pragma unroll
    for (int u = 0; u < TI; u += 2) {
        const int il = (wi * TI + u) * 16 + neighbours_at(lane);
        const int64_t i = i0 + il;
#pragma unroll
        for (int t = 0; t < TJ; ++t) {
            const int jl = (wj * TJ + t) * 16 + (lane & 15);
            const int64_t j = j0 + jl;
            float v[8];
            neighbours(acc[u][t], acc[u + 1][t], v);
            const bool exists = 2 * i < out_cols && j < a.side;
            const int64_t at = j * out_stride + column(i);
            f16x8 hi = {}, lo = {};
            if (PHASE != kMuonGram && exists) {
                hi = *(const f16x8*)(from + at);
                lo = *(const f16x8*)(from + at + 32);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float y = v[e] * kProducts;
                if (PHASE != kMuonGram) y = fmaf(kAdded, (float)hi[e] + (float)lo[e], y);
                _Float16 h, l;
                split(y, h, l);
                hi[e] = h;
                lo[e] = l;
            }
            if (exists) {
                *(f16x8*)(to + at) = hi;
                *(f16x8*)(to + at + 32) = lo;
            }
            if (mirrored) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    mirror[(il + e) * kMirrorPitch + jl] = hi[e];
                    mirror[(P::BI + il + e) * kMirrorPitch + jl] = lo[e];
                }
            }
        }
    }
    if (!mirrored) return;
    lds_barrier();
    // rows i of the mirrored tile, 8 of j at a time; j is inside the matrix (tj < ti)
    for (int q = threadIdx.x; q < 2 * P::BI * (P::BJ / 8); q += 64 * WI * WJ) {
        const int c = q % (P::BJ / 8), r = q / (P::BJ / 8), il = r % P::BI, h = r / P::BI;
        if (i0 + il < a.side)
            *(f16x8*)(to + (i0 + il) * out_stride + column(j0 + 8 * c) + 32 * h) =
                *(const f16x8*)(mirror + (h * P::BI + il) * kMirrorPitch + 8 * c);
    }
}

__global__ void __launch_bounds__(256) zero_kernel(Mat m) {
    const int64_t n = m.rows * m.cols;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256)
        ((float*)m.p)[q / m.cols * m.stride + q % m.cols] = 0.0f;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles of 128 x 128 where they occupy half of the card, else of 64 x 64: a
// small network's matrices are too few large tiles. Whole steps, large and
// small: four of 1024 x 4096 1299 and 1571 us, four of 1024 x 1024 (144 and 256
// tiles) 497 and 571, two of them (72 and 128) 452 and 327, eight of 256 x 256
// 212 and 143.
uint32_t count_tiles(const MuonPart* parts, int count, bool large, int phase, MuonPart* set) {
    int64_t n = 0;
    const int64_t edge = large ? 128 : 64;
    for (int i = 0; i < count; ++i) {
        const MuonPart& a = parts[i];
        if (set) set[i].first[phase] = (uint32_t)n;
        const int64_t down = ceil_div(a.side, edge);
        n += phase == kMuonUpdate ? ceil_div(a.x_cols / 2, edge) * down : down * (down + 1) / 2;
    }
    return n < 0x7fffffff ? (uint32_t)n : 0x7fffffffu;
}

}  // namespace

MuonPlan plan_muon(MuonPart* parts, int count) {
    MuonPlan plan{};
    int64_t at = 0, patches = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    for (int i = 0; i < count; ++i) {
        MuonPart& a = parts[i];
        a.tall = a.w.rows > a.w.cols;
        a.side = a.tall ? a.w.cols : a.w.rows;
        a.length = a.tall ? a.w.rows : a.w.cols;
        a.x_cols = ceil_div(a.length, 32) * 64;
        a.g_cols = ceil_div(a.side, 32) * 64;
        a.x_stride = a.x_cols + kRowPad;
        a.g_stride = a.g_cols + kRowPad;
        a.shape = a.tall ? sqrtf((float)a.w.rows / (float)a.w.cols) : 1.0f;
        a.first[kMuonPatches] = (uint32_t)patches;
        patches += ceil_div(a.w.rows, kPatch) * ceil_div(a.w.cols, kPatch);
        for (int k = 0; k < 2; ++k) a.x[k] = (_Float16*)take(2 * a.side * a.x_stride);
        a.gram = (_Float16*)take(2 * a.side * a.g_stride);
        a.poly = (_Float16*)take(2 * a.side * a.g_stride);
    }
    plan.patches = (uint32_t)patches;
    plan.large[0] = count_tiles(parts, count, true, kMuonGram, nullptr) >= 128;
    plan.large[1] = count_tiles(parts, count, true, kMuonUpdate, nullptr) >= 128;
    plan.tiles[0] = count_tiles(parts, count, plan.large[0], kMuonGram, parts);
    plan.tiles[1] = count_tiles(parts, count, plan.large[1], kMuonUpdate, parts);
    plan.sums_at = take(8 * patches);
    plan.parts_at = take((int64_t)sizeof(MuonPart) * count);
    plan.firsts_at = take((int64_t)sizeof(uint32_t) * 3 * count);
    plan.bytes = at;
    // a launch of 2^32 threads or more loses what is above without an error
    const auto holds = [](int64_t workgroups, int64_t threads) { return workgroups * threads < ((int64_t)1 << 32); };
    plan.fits = holds(patches, kPatchThreads) && holds(plan.tiles[0], plan.large[0] ? 512 : 256) &&
                holds(plan.tiles[1], plan.large[1] ? 512 : 256);
    return plan;
}

void place_muon(MuonPart* parts, int count, unsigned char* workspace) {
    for (int i = 0; i < count; ++i) {
        MuonPart& a = parts[i];
        for (int k = 0; k < 2; ++k) a.x[k] = (_Float16*)(workspace + (int64_t)a.x[k]);
        a.gram = (_Float16*)(workspace + (int64_t)a.gram);
        a.poly = (_Float16*)(workspace + (int64_t)a.poly);
    }
}

template <int PHASE>
static void launch_product(const MuonPlan& plan, const MuonPart* parts, const uint32_t* firsts, int count, int turn,
                           hipStream_t s) {
    const int w = PHASE == kMuonUpdate;
    const uint32_t* f = firsts + (w ? kMuonUpdate : kMuonGram) * count;
    if (plan.large[w])
        product_kernel<PHASE, 2, 4, 4, 2, 2><<<plan.tiles[w], 512, 0, s>>>(parts, f, count, plan.tiles[w], turn);
    else
        product_kernel<PHASE, 2, 2, 2, 2, 2><<<plan.tiles[w], 256, 0, s>>>(parts, f, count, plan.tiles[w], turn);
}

int launch_muon_step(const MuonPlan& plan, int count, const MuonStep& p, unsigned char* workspace, hipStream_t s) {
    const MuonPart* parts = (const MuonPart*)(workspace + plan.parts_at);
    const uint32_t* firsts = (const uint32_t*)(workspace + plan.firsts_at);
    double* sums = (double*)(workspace + plan.sums_at);
    by_dtype(p.grad_dtype, [&](auto t) {
        momentum_kernel<decltype(t)><<<plan.patches, kPatchThreads, 0, s>>>(parts, firsts, count, p, sums);
        normalise_kernel<decltype(t)><<<plan.patches, kPatchThreads, 0, s>>>(parts, firsts, count, p, sums);
    });
    for (int k = 0; k < p.iterations; ++k) {
        launch_product<kMuonGram>(plan, parts, firsts, count, k & 1, s);
        launch_product<kMuonSquare>(plan, parts, firsts, count, k & 1, s);
        launch_product<kMuonUpdate>(plan, parts, firsts, count, k & 1, s);
    }
    by_dtype(p.copy_dtype, [&](auto t) {
        apply_kernel<decltype(t)><<<plan.patches, kPatchThreads, 0, s>>>(parts, firsts, count, p);
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_zero_matrix(const Mat& m, hipStream_t s) {
    zero_kernel<<<256, 256, 0, s>>>(m);
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
