// Muon's update of a network's matrices: momentum, the Newton-Schulz steps on
// the normalised update, the weights. Every phase is one launch over all
// matrices.
//
// X is kept with its shorter side as rows (the transpose of a tall matrix), so
// that X X^T is the smaller of the two Gram matrices. X, the Gram matrix G and
// the polynomial P = b G + c G^2 are held as two halves each, hi + lo with
// lo = half(v - hi), of the value times 2^12: 22 bits of every element down to
// 2^-25 of one, in the range of halves (|X|, |G| < 2, |P| < 3: the singular
// values of X stay below 1.3). A product is then three of halves, hi hi + hi lo
// + lo hi with float sums (lo lo is 2^-22 of it), at the matrix cores' half
// rate: 5.4 times the float products' (1.42 and 0.153 PFLOP/s measured), over
// three. Halves alone (11 bits) would leave the update's small singular
// directions, which the steps lift up to 485 times, wrong by several percent.
#include <math.h>

#include "mfma_tile.h"

namespace tgs {

namespace {

constexpr float kScale = 4096.0f;
constexpr int kPatch = 64;   // edge of the element passes' patches

// The matrix that number `n` of a launch's work belongs to: the last whose
// first number is not above it.
__device__ __forceinline__ int part_of(const MuonPart* parts, int count, int phase, uint32_t n) {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (parts[mid].first[phase] <= n) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float update_of(float g, float m, const MuonStep& p) {
    return p.nesterov ? fmaf(p.momentum, m, g) : m;
}

// M <- mu M + (1 - mu) s G, and the patch's sum of squares of U.
template <class G>
__global__ void __launch_bounds__(256) momentum_kernel(const MuonPart* parts, int count, MuonStep p, double* sums) {
    const MuonPart& a = parts[part_of(parts, count, kMuonPatches, blockIdx.x)];
    const uint32_t n = blockIdx.x - a.first[kMuonPatches];
    const int64_t across = (a.w.cols + kPatch - 1) / kPatch;
    const int64_t r0 = n / across * kPatch, c0 = n % across * kPatch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum = 0.0;
#pragma unroll 4
    for (int k = wave; k < kPatch; k += 4) {
        const int64_t r = r0 + k, c = c0 + lane;
        if (r >= a.w.rows || c >= a.w.cols) continue;
        const float g = (float)((const G*)a.g.p)[r * a.g.stride + c] * p.grad_scale;
        float* at = (float*)a.m.p + r * a.m.stride + c;
        const float m = fmaf(p.momentum, *at, g);
        *at = m;
        const double u = (double)update_of(g, m, p);
        sum += u * u;
    }
    __shared__ double s[256];
    s[threadIdx.x] = sum;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) s[threadIdx.x] += s[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) sums[blockIdx.x] = s[0];
}

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// X = U / max(|U|, epsilon), scaled and split; a tall matrix through LDS into
// its transpose. Columns up to the stride are zeros.
template <class G>
__global__ void __launch_bounds__(256) normalise_kernel(const MuonPart* parts, int count, MuonStep p,
                                                        const double* sums) {
    const MuonPart& a = parts[part_of(parts, count, kMuonPatches, blockIdx.x)];
    const uint32_t n = blockIdx.x - a.first[kMuonPatches];
    const int64_t across = (a.w.cols + kPatch - 1) / kPatch, down = (a.w.rows + kPatch - 1) / kPatch;
    __shared__ double s[256];
    double sum = 0.0;
    for (int64_t k = threadIdx.x; k < across * down; k += 256) sum += sums[a.first[kMuonPatches] + k];
    s[threadIdx.x] = sum;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) s[threadIdx.x] += s[threadIdx.x + k];
        __syncthreads();
    }
    const double norm = sqrt(s[0]);
    const double inv = (double)kScale / (norm < (double)p.epsilon ? (double)p.epsilon : norm);   // NaN stays
    const int64_t r0 = n / across * kPatch, c0 = n % across * kPatch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __shared__ float t[kPatch][kPatch + 1];
#pragma unroll 4
    for (int k = wave; k < kPatch; k += 4) {
        const int64_t r = r0 + k, c = c0 + lane;
        float v = 0.0f;
        if (r < a.w.rows && c < a.w.cols) {
            const float g = (float)((const G*)a.g.p)[r * a.g.stride + c] * p.grad_scale;
            v = (float)((double)update_of(g, ((const float*)a.m.p)[r * a.m.stride + c], p) * inv);
        }
        if (a.tall) t[k][lane] = v;
        else if (r < a.side && c < a.x_stride) split(v, a.x[0][r * a.x_stride + c], a.x[0][a.x_plane + r * a.x_stride + c]);
    }
    if (!a.tall) return;
    __syncthreads();
#pragma unroll 4
    for (int k = wave; k < kPatch; k += 4) {
        const int64_t r = c0 + k, c = r0 + lane;   // of X
        if (r < a.side && c < a.x_stride)
            split(t[lane][k], a.x[0][r * a.x_stride + c], a.x[0][a.x_plane + r * a.x_stride + c]);
    }
}

// W <- keep W - lr shape X, and the copy.
template <class C>
__global__ void __launch_bounds__(256) apply_kernel(const MuonPart* parts, int count, MuonStep p) {
    const MuonPart& a = parts[part_of(parts, count, kMuonPatches, blockIdx.x)];
    const uint32_t n = blockIdx.x - a.first[kMuonPatches];
    const int64_t across = (a.w.cols + kPatch - 1) / kPatch;
    const int64_t r0 = n / across * kPatch, c0 = n % across * kPatch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const _Float16* x = a.x[p.iterations & 1];
    const float step = p.lr * a.shape * (1.0f / kScale);
    __shared__ float t[kPatch][kPatch + 1];
    if (a.tall) {
#pragma unroll 4
        for (int k = wave; k < kPatch; k += 4) {
            const int64_t r = c0 + k, c = r0 + lane;
            if (r < a.side && c < a.length)
                t[lane][k] = (float)x[r * a.x_stride + c] + (float)x[a.x_plane + r * a.x_stride + c];
        }
        __syncthreads();
    }
#pragma unroll 4
    for (int k = wave; k < kPatch; k += 4) {
        const int64_t r = r0 + k, c = c0 + lane;
        if (r >= a.w.rows || c >= a.w.cols) continue;
        const float v = a.tall ? t[k][lane]
                               : (float)x[r * a.x_stride + c] + (float)x[a.x_plane + r * a.x_stride + c];
        float* w = (float*)a.w.p + r * a.w.stride + c;
        const float u = fmaf(-step, v, p.keep * *w);
        *w = u;
        if (a.c.p) ((C*)a.c.p)[r * a.c.stride + c] = (C)u;
    }
}

// ---- the products

// A tile of the three-product sum. Steps of 64 bytes of k: four planes of
// 128 rows twice are 64 KB, two workgroups a compute unit.
template <int WI, int WJ, int TI, int TJ, bool A_RC>
struct SplitTile {
    static constexpr int kWavesI = WI, kWavesJ = WJ;
    static constexpr int kWaves = WI * WJ, kThreads = 64 * kWaves;
    static constexpr int BI = WI * TI * 16, BJ = WJ * TJ * 16;
    using T = _Float16;
    using A = TileSide<T, BI, kWaves, A_RC, 64>;
    using B = TileSide<T, BJ, kWaves, false, 64>;
    static constexpr int kStage = 2 * (A::kBytes + B::kBytes);

    static __device__ __forceinline__ void run(unsigned char* lds, TileOperand a, int64_t a_plane, TileOperand b,
                                               int64_t b_plane, int64_t i0, int64_t j0, int64_t k_size,
                                               f32x4 (&acc)[TI][TJ]) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wi = wave / WJ, wj = wave % WJ;
        A sa[2];
        B sb[2];
        for (int h = 0; h < 2; ++h) {
            sa[h].begin({(const T*)a.p + h * a_plane, a.rows, a.cols, a.stride}, i0, 0, wave, lane);
            sb[h].begin({(const T*)b.p + h * b_plane, b.rows, b.cols, b.stride}, j0, 0, wave, lane);
        }
#pragma unroll
        for (int u = 0; u < TI; ++u)
#pragma unroll
            for (int v = 0; v < TJ; ++v) acc[u][v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const auto load = [&](unsigned char* to, int64_t left) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sa[h].load(to + h * A::kBytes, left, wave, lane);
                sb[h].load(to + 2 * A::kBytes + h * B::kBytes, left, wave, lane);
            }
        };
        const int steps = (int)((k_size + A::kDepth - 1) / A::kDepth);
        load(lds, k_size);
        for (int t = 0; t < steps; ++t) {
            const unsigned char* now = lds + (t & 1) * kStage;
            wait_all_and_barrier();
            if (t + 1 < steps) load(lds + ((t + 1) & 1) * kStage, k_size - (int64_t)(t + 1) * A::kDepth);
            typename Frag<T>::type fa[2][TI], fb[2][TJ];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int v = 0; v < TJ; ++v)
                    fb[h][v] = B::fragment(now + 2 * A::kBytes + h * B::kBytes, (wj * TJ + v) * 16, 0, lane);
#pragma unroll
                for (int u = 0; u < TI; ++u) fa[h][u] = A::fragment(now + h * A::kBytes, (wi * TI + u) * 16, 0, lane);
            }
#pragma unroll
            for (int q = 0; q < 3; ++q)   // hi hi, hi lo, lo hi: the squares in turn, no sum waits for its last
#pragma unroll
                for (int u = 0; u < TI; ++u)
#pragma unroll
                    for (int v = 0; v < TJ; ++v) acc[u][v] = multiply(fa[q == 2][u], fb[q == 1][v], acc[u][v]);
        }
    }
};

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Gram: G = X X^T. Square: P = b G + c G G. Update: X' = a X + P X. Rows of
// the stored matrices are 16-byte aligned and zero up to their stride, which
// the products keep: they run over whole strides.
template <int PHASE, int WI, int WJ, int TI, int TJ>
__global__ void __launch_bounds__(64 * WI * WJ) product_kernel(const MuonPart* parts, int count, uint32_t total, int turn) {
    constexpr bool kUpdate = PHASE == kMuonUpdate;
    using P = SplitTile<WI, WJ, TI, TJ, kUpdate>;
    __shared__ __align__(1024) unsigned char lds[2 * P::kStage];
    const uint32_t n = xcd_contiguous_index(blockIdx.x, total);
    const MuonPart& a = parts[part_of(parts, count, kUpdate ? kMuonUpdate : kMuonGram, n)];
    const uint32_t local = n - a.first[kUpdate ? kMuonUpdate : kMuonGram];
    const _Float16* x = a.x[turn];
    const int64_t out_stride = kUpdate ? a.x_stride : a.g_stride;
    const uint32_t ni = (uint32_t)((out_stride + P::BI - 1) / P::BI), nj = (uint32_t)((a.side + P::BJ - 1) / P::BJ);
    uint32_t ti, tj;
    tile_of(local, ni, nj, ti, tj);
    const int64_t i0 = (int64_t)ti * P::BI, j0 = (int64_t)tj * P::BJ;
    f32x4 acc[TI][TJ];
    const TileOperand tx{x, a.side, a.x_stride, a.x_stride};
    const _Float16* from;   // added to the products, and to where
    _Float16* to;
    int64_t plane;
    if constexpr (PHASE == kMuonGram) {
        P::run(lds, tx, a.x_plane, tx, a.x_plane, i0, j0, a.x_stride, acc);
        from = nullptr;
        to = a.gram;
        plane = a.g_plane;
    } else if constexpr (PHASE == kMuonSquare) {
        const TileOperand tg{a.gram, a.side, a.g_stride, a.g_stride};
        P::run(lds, tg, a.g_plane, tg, a.g_plane, i0, j0, a.g_stride, acc);
        from = a.gram;
        to = a.poly;
        plane = a.g_plane;
    } else {
        // k runs over P's columns, X's rows: those past the side are zeros in P and not there in X
        const TileOperand tp{a.poly, a.side, a.g_stride, a.g_stride};
        P::run(lds, tx, a.x_plane, tp, a.g_plane, i0, j0, a.g_stride, acc);
        from = x;
        to = a.x[turn ^ 1];
        plane = a.x_plane;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = wave / WJ, wj = wave % WJ;
    constexpr float kProducts = (PHASE == kMuonSquare ? kNewtonSchulzC : 1.0f) / kScale;
    constexpr float kAdded = PHASE == kMuonSquare ? kNewtonSchulzB : kNewtonSchulzA;
#pragma unroll
    for (int u = 0; u < TI; u += 2) {
        const int64_t i = i0 + (wi * TI + u) * 16 + neighbours_at(lane);
#pragma unroll
        for (int t = 0; t < TJ; ++t) {
            const int64_t j = j0 + (wj * TJ + t) * 16 + (lane & 15);
            float v[8];
            neighbours(acc[u][t], acc[u + 1][t], v);
            if (i >= out_stride || j >= a.side) continue;
            const int64_t at = j * out_stride + i;
            f16x8 hi, lo;
            if (PHASE != kMuonGram) {
                hi = *(const f16x8*)(from + at);
                lo = *(const f16x8*)(from + plane + at);
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
            *(f16x8*)(to + at) = hi;
            *(f16x8*)(to + plane + at) = lo;
        }
    }
}

__global__ void __launch_bounds__(256) zero_kernel(Mat m) {
    const int64_t n = m.rows * m.cols;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256)
        ((float*)m.p)[q / m.cols * m.stride + q % m.cols] = 0.0f;
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tiles of 128 x 128 where they fill the card, else of 64 x 64: a small
// network's matrices are too few large tiles.
uint32_t count_tiles(const MuonPart* parts, int count, int edge, int phase, MuonPart* set) {
    int64_t n = 0;
    for (int i = 0; i < count; ++i) {
        const MuonPart& a = parts[i];
        if (set) set[i].first[phase] = (uint32_t)n;
        n += ceil_div(phase == kMuonUpdate ? a.x_stride : a.g_stride, edge) * ceil_div(a.side, edge);
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
        a.x_stride = ceil_div(a.length, 8) * 8;
        a.g_stride = ceil_div(a.side, 8) * 8;
        a.x_plane = a.side * a.x_stride;
        a.g_plane = a.side * a.g_stride;
        a.shape = a.tall ? sqrtf((float)a.w.rows / (float)a.w.cols) : 1.0f;
        a.first[kMuonPatches] = (uint32_t)patches;
        patches += ceil_div(a.w.rows, kPatch) * ceil_div(a.w.cols, kPatch);
        for (int k = 0; k < 2; ++k) a.x[k] = (_Float16*)take(4 * a.x_plane);
        a.gram = (_Float16*)take(4 * a.g_plane);
        a.poly = (_Float16*)take(4 * a.g_plane);
    }
    plan.patches = (uint32_t)patches;
    plan.large[0] = count_tiles(parts, count, 128, kMuonGram, nullptr) >= 256;
    plan.large[1] = count_tiles(parts, count, 128, kMuonUpdate, nullptr) >= 256;
    plan.tiles[0] = count_tiles(parts, count, plan.large[0] ? 128 : 64, kMuonGram, parts);
    plan.tiles[1] = count_tiles(parts, count, plan.large[1] ? 128 : 64, kMuonUpdate, parts);
    plan.sums_at = take(8 * patches);
    plan.parts_at = take((int64_t)sizeof(MuonPart) * count);
    plan.bytes = at;
    plan.fits = patches < 0x7fffffff && plan.tiles[0] < 0x7fffffffu && plan.tiles[1] < 0x7fffffffu;
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
static void launch_product(const MuonPlan& plan, const MuonPart* parts, int count, int turn, hipStream_t s) {
    const int w = PHASE == kMuonUpdate;
    if (plan.large[w]) product_kernel<PHASE, 2, 2, 4, 4><<<plan.tiles[w], 256, 0, s>>>(parts, count, plan.tiles[w], turn);
    else product_kernel<PHASE, 2, 2, 2, 2><<<plan.tiles[w], 256, 0, s>>>(parts, count, plan.tiles[w], turn);
}

int launch_muon_step(const MuonPlan& plan, int count, const MuonStep& p, unsigned char* workspace, hipStream_t s) {
    const MuonPart* parts = (const MuonPart*)(workspace + plan.parts_at);
    double* sums = (double*)(workspace + plan.sums_at);
    by_dtype(p.grad_dtype, [&](auto t) {
        momentum_kernel<decltype(t)><<<plan.patches, 256, 0, s>>>(parts, count, p, sums);
        normalise_kernel<decltype(t)><<<plan.patches, 256, 0, s>>>(parts, count, p, sums);
    });
    for (int k = 0; k < p.iterations; ++k) {
        launch_product<kMuonGram>(plan, parts, count, k & 1, s);
        launch_product<kMuonSquare>(plan, parts, count, k & 1, s);
        launch_product<kMuonUpdate>(plan, parts, count, k & 1, s);
    }
    by_dtype(p.copy_dtype, [&](auto t) { apply_kernel<decltype(t)><<<plan.patches, 256, 0, s>>>(parts, count, p); });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_zero_matrix(const Mat& m, hipStream_t s) {
    zero_kernel<<<256, 256, 0, s>>>(m);
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
