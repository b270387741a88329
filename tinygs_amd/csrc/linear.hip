// Linear layers: z = x w^T + bias, y = act(z) + residual, and their gradients
// dx = dz w, dw = dz^T x, db = the column sums of dz, dz = dy act'(z).
//
// The three products are tiles of mfma_tile.h with the contiguous axis of the
// output as i. Forward: A = w, B = x, both K-contiguous, bias, activation and
// residual on the sums. dx: A = w R-contiguous, B = dz. dw: A = x, B = dz, both
// R-contiguous; its long axis (the rows) is split over workgroups whose float
// sums a second kernel joins in order. An activation's dz is written once, by
// the pass that also sums its columns, and read by both products.
#include <algorithm>

#include "mfma_tile.h"

namespace tgs {

namespace {

template <class T>
struct Packed {   // 8 elements of a row, at any element's address
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

template <class T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    if (n >= 8) {
        const auto u = *(const typename Packed<T>::type*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)u[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? (float)p[e] : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if (n >= 8) {
        typename Packed<T>::type u;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = (T)v[e];
        *(typename Packed<T>::type*)p = u;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = (T)v[e];
    }
}

// A lane's outputs are runs of 8 (i .. i + 7, j), n of which exist (0: none, or
// j is past the end). For every column of TJ runs of one i: before(i, n) and
// ahead(t, i, j, n) for each t, which start their loads, then
// f(t, i, j, n, v) with the values.
template <class Shape, int TI, int TJ, class Before, class Ahead, class F>
__device__ __forceinline__ void for_outputs(const f32x4 (&acc)[TI][TJ], int64_t i0, int64_t j0, int64_t ni, int64_t nj,
                                            Before before, Ahead ahead, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = wave / Shape::kWavesJ, wj = wave % Shape::kWavesJ;
#pragma unroll
    for (int u = 0; u < TI; u += 2) {
        const int64_t i = i0 + (wi * TI + u) * 16 + neighbours_at(lane);
        const int n = (int)min(max(ni - i, (int64_t)0), (int64_t)8);
        before(i, n);
#pragma unroll
        for (int t = 0; t < TJ; ++t) {
            const int64_t j = j0 + (wj * TJ + t) * 16 + (lane & 15);
            ahead(t, i, j, j < nj ? n : 0);
        }
#pragma unroll
        for (int t = 0; t < TJ; ++t) {
            const int64_t j = j0 + (wj * TJ + t) * 16 + (lane & 15);
            float v[8];
            neighbours(acc[u][t], acc[u + 1][t], v);
            if (n > 0 && j < nj) f(t, i, j, n, v);
        }
    }
}
template <class Shape, int TI, int TJ, class F>
__device__ __forceinline__ void for_outputs(const f32x4 (&acc)[TI][TJ], int64_t i0, int64_t j0, int64_t ni, int64_t nj,
                                            F f) {
    for_outputs<Shape>(acc, i0, j0, ni, nj, [](int64_t, int) {}, [](int, int64_t, int64_t, int) {},
                       [&](int, int64_t i, int64_t j, int n, float(&v)[8]) { f(i, j, n, v); });
}

// Tile shapes, as waves and squares of 16 a wave on each axis. A ring of two
// stages of 128 bytes of k, which is a whole cache line of each row of a
// K-contiguous operand (four stages of half a line fetched every line twice: 75
// against 66 us for 16384 x 2048 -> 1024 halves; without such an operand 81
// against 75 us).
template <int WI_, int WJ_, int TI_, int TJ_>
struct Shape {
    static constexpr int kWavesI = WI_, kWavesJ = WJ_, kSquaresI = TI_, kSquaresJ = TJ_;
    static constexpr int kI = WI_ * TI_ * 16, kJ = WJ_ * TJ_ * 16, kThreads = 64 * WI_ * WJ_;
    template <class T, bool A_RC, bool B_RC>
    using Product = Tile<T, WI_, WJ_, TI_, TJ_, A_RC, B_RC, 128, 2>;
    // workgroups that a compute unit's LDS holds
    static constexpr int kResident = 160 * 1024 / (256 * (kI + kJ));
};
using Large = Shape<2, 4, 8, 4>;    // 256 x 256, 8 waves, 128 KB of LDS: one workgroup a compute unit
using Middle = Shape<2, 2, 4, 4>;   // 128 x 128, 4 waves, 64 KB
using Narrow = Shape<1, 4, 4, 4>;   // 64 x 256, 4 waves, 80 KB: few columns
using Small = Shape<2, 2, 2, 2>;    // 64 x 64, 4 waves, 32 KB: few tiles

// Large tiles read each operand least often, from as many tiles as compute
// units on; with fewer, smaller tiles fill the card. Without bias, whole calls, the
// shape taken first: 16384 x 1024 -> 2048 halves 80 us (860 TFLOP/s) in Large, 99
// in Middle, 134 in Small; 8192 x 1024 -> 1024 (128 large tiles) 27 in Middle, 35
// in Large, 34 in Small; 2000 x 1024 -> 1024 11.2 in Small and in Middle; floats
// 345, 393, 518; 96, 150, 132. Of few columns, in Narrow and in Small: floats
// 100000 x 600 -> 64 62 and 73 us, but 200000 x 84 -> 59 40 and 30; halves 1e6 x
// 600 -> 64 315 and 341, 200000 x 600 -> 64 61 and 50, 65536 x 84 -> 59 12.3 and
// 8.7. So Narrow is for `deep` products: of floats with k of 256 and more, where
// its fewer reads of A are worth its longer tiles, and for the sums over rows.
template <class T>
bool is_deep(int64_t k) { return sizeof(T) == 4 && k >= 256; }
template <class F>
void by_shape(int64_t ni, int64_t nj, int64_t splits_most, bool deep, F f) {
    const auto tiles = [&](int64_t bi, int64_t bj) { return ((ni + bi - 1) / bi) * ((nj + bj - 1) / bj) * splits_most; };
    if (ni > 128 && nj > 128 && tiles(256, 256) >= 256) f(Large{});
    else if (ni > 64 && nj > 64 && tiles(128, 128) >= 256) f(Middle{});
    else if (deep && ni <= 64 && nj > 64 && tiles(64, 256) >= 256) f(Narrow{});
    else f(Small{});
}

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Few tiles and a long k (an ordinary batch of rows through wide layers): k is
// split over workgroups, in whole stages of 128 bytes and at least four of
// them, until 256 small tiles are at work, and a second kernel joins the sums.
// Whole calls, without and with the split: 512 x 4096 -> 512 halves 35.3 and
// 15.3 us, floats 104 and 33.5; 64 x 4096 -> 256 halves 24.5 and 12.0, floats
// 102 and 17.8. The join is a launch more, so a short k stays whole: 512 x 512
// -> 512 halves (8 stages) 7.3 and 9.4 us, 1024 -> 512 (16) 8.7 and 9.7,
// 2048 x 2048 -> 256 (32) 14.2 and 13.2; floats, whose stage is six products
// long, 16.2 and 11.4 at 512 x 512 -> 512 (16).
struct KSplits {
    int64_t splits = 1, depth = 0;
};
KSplits split_k(int64_t ni, int64_t nj, int64_t k, int size) {
    const int64_t stage = 128 / size, stages = ceil_div(k, stage), tiles = ceil_div(ni, 64) * ceil_div(nj, 64);
    KSplits s;
    int64_t want = tiles > 0 ? 256 / tiles : 1;
    if (want > stages / 4) want = stages / 4;
    if (want < 2 || stages < (size == 4 ? 16 : 32)) {
        s.depth = k;
        return s;
    }
    s.depth = ceil_div(stages, want) * stage;
    s.splits = ceil_div(k, s.depth);
    return s;
}

template <class T, int ACT, class S>
__device__ __forceinline__ void forward_outputs(const LinearForward& a, const f32x4 (&acc)[S::kSquaresI][S::kSquaresJ],
                                                int64_t i0, int64_t j0) {
    // bias and residual are on their way before the first of their runs needs them
    float bias[8];
    typename Packed<T>::type residual[S::kSquaresJ];
    for_outputs<S>(
        acc, i0, j0, a.y.cols, a.y.rows,
        [&](int64_t i, int n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[e] = 0.0f;
            if (a.bias && n > 0) load8(a.bias + i, n, bias);
        },
        [&](int t, int64_t i, int64_t j, int n) {
            if (a.residual.p && n == 8)
                residual[t] = *(const typename Packed<T>::type*)((const T*)a.residual.p + j * a.residual.stride + i);
        },
        [&](int t, int64_t i, int64_t j, int n, float(&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += bias[e];
            if (a.preact.p) store8((T*)a.preact.p + j * a.preact.stride + i, n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = activate<ACT>(v[e]);
            if (a.residual.p) {
                if (n == 8) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += (float)residual[t][e];
                } else {
                    float r[8];
                    load8((const T*)a.residual.p + j * a.residual.stride + i, n, r);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += r[e];
                }
            }
            store8((T*)a.y.p + j * a.y.stride + i, n, v);
        });
}

// Float sums of a tile to their place in split `split` of rows x cols.
template <class S, int TI, int TJ>
__device__ __forceinline__ void store_sums(const f32x4 (&acc)[TI][TJ], int64_t i0, int64_t j0, float* partial, int64_t split,
                                           int64_t rows, int64_t cols) {
    float* out = partial + split * rows * cols;
    for_outputs<S>(acc, i0, j0, cols, rows,
                   [&](int64_t i, int64_t j, int n, float(&v)[8]) { store8(out + j * cols + i, n, v); });
}

// Rows of a launch at most. A launch of 2^32 threads or more loses what is above
// without an error: 256 threads for 64 rows reached that at 2^30 rows.
constexpr int64_t kLaunchRows = (int64_t)1 << 27;

// The call's rows from `first` on, as many as one launch takes.
template <class T>
LinearForward rows_of(LinearForward a, int64_t first) {
    for (Mat* m : {&a.x, &a.residual, &a.preact, &a.y}) {
        if (!m->p) continue;
        m->p = (T*)m->p + first * m->stride;
        m->rows = std::min(m->rows - first, kLaunchRows);
    }
    return a;
}

// With `partial`, the float sums over the k of split blockIdx.y.
template <class T, class S>
__global__ void __launch_bounds__(S::kThreads) forward_kernel(LinearForward a, float* partial, int64_t depth, uint32_t ni,
                                                              uint32_t nj) {
    using P = typename S::template Product<T, false, false>;
    __shared__ __align__(1024) unsigned char lds[P::kLds];
    uint32_t ti, tj;
    tile_of(xcd_contiguous_index(blockIdx.x, ni * nj), ni, nj, ti, tj);
    const int64_t i0 = (int64_t)ti * S::kI, j0 = (int64_t)tj * S::kJ;
    const int64_t k0 = (int64_t)blockIdx.y * depth, k1 = min(k0 + depth, a.x.cols);
    f32x4 acc[S::kSquaresI][S::kSquaresJ];
    P::run(lds, {a.w.p, a.w.rows, a.w.cols, a.w.stride}, {a.x.p, a.x.rows, a.x.cols, a.x.stride}, i0, j0, k0, k1, acc);
    if (partial) store_sums<S>(acc, i0, j0, partial, blockIdx.y, a.y.rows, a.y.cols);
    else if (a.activation == kActGelu) forward_outputs<T, kActGelu, S>(a, acc, i0, j0);
    else if (a.activation == kActSilu) forward_outputs<T, kActSilu, S>(a, acc, i0, j0);
    else if (a.activation == kActRelu) forward_outputs<T, kActRelu, S>(a, acc, i0, j0);
    else forward_outputs<T, kActNone, S>(a, acc, i0, j0);
}

// The splits' sums joined in order, and the forward's epilogue on them: eight
// outputs of a row a thread.
template <class T, int ACT>
__global__ void __launch_bounds__(256) join_rows_kernel(LinearForward a, const float* partial, int splits) {
    const int64_t across = (a.y.cols + 7) / 8, q = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= across * a.y.rows) return;
    const int64_t j = q / across, i = q % across * 8, all = a.y.rows * a.y.cols;
    const int n = (int)min(a.y.cols - i, (int64_t)8);
    float v[8], u[8];
    load8(partial + j * a.y.cols + i, n, v);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
        load8(partial + k * all + j * a.y.cols + i, n, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
    if (a.bias) {
        load8(a.bias + i, n, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
    if (a.preact.p) store8((T*)a.preact.p + j * a.preact.stride + i, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = activate<ACT>(v[e]);
    if (a.residual.p) {
        load8((const T*)a.residual.p + j * a.residual.stride + i, n, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
    store8((T*)a.y.p + j * a.y.stride + i, n, v);
}

// grad_x = dz w; with `partial`, the float sums over the out of split blockIdx.y.
template <class T, class S>
__global__ void __launch_bounds__(S::kThreads) grad_x_kernel(Mat dz, Mat w, Mat gx, float* partial, int64_t depth,
                                                             uint32_t ni, uint32_t nj) {
    using P = typename S::template Product<T, true, false>;
    __shared__ __align__(1024) unsigned char lds[P::kLds];
    uint32_t ti, tj;
    tile_of(xcd_contiguous_index(blockIdx.x, ni * nj), ni, nj, ti, tj);
    const int64_t i0 = (int64_t)ti * S::kI, j0 = (int64_t)tj * S::kJ;
    const int64_t k0 = (int64_t)blockIdx.y * depth, k1 = min(k0 + depth, w.rows);
    f32x4 acc[S::kSquaresI][S::kSquaresJ];
    P::run(lds, {w.p, w.rows, w.cols, w.stride}, {dz.p, dz.rows, dz.cols, dz.stride}, i0, j0, k0, k1, acc);
    if (partial) {
        store_sums<S>(acc, i0, j0, partial, blockIdx.y, gx.rows, gx.cols);
        return;
    }
    for_outputs<S>(acc, i0, j0, gx.cols, gx.rows, [&](int64_t i, int64_t j, int n, float (&v)[8]) {
        store8((T*)gx.p + j * gx.stride + i, n, v);
    });
}

// grad_w = dz^T x over the rows of split blockIdx.y: to grad_w, or its float
// sums to partial + blockIdx.y * (out * in).
template <class T, class S>
__global__ void __launch_bounds__(S::kThreads) grad_w_kernel(Mat dz, Mat x, Mat gw, float* partial, int64_t split_rows,
                                                             uint32_t ni, uint32_t nj) {
    using P = typename S::template Product<T, true, true>;
    __shared__ __align__(1024) unsigned char lds[P::kLds];
    uint32_t ti, tj;
    tile_of(xcd_contiguous_index(blockIdx.x, ni * nj), ni, nj, ti, tj);
    const int64_t i0 = (int64_t)ti * S::kI, j0 = (int64_t)tj * S::kJ;
    const int64_t k0 = (int64_t)blockIdx.y * split_rows, k1 = min(k0 + split_rows, x.rows);
    f32x4 acc[S::kSquaresI][S::kSquaresJ];
    P::run(lds, {x.p, x.rows, x.cols, x.stride}, {dz.p, dz.rows, dz.cols, dz.stride}, i0, j0, k0, k1, acc);
    float* out = partial ? partial + (int64_t)blockIdx.y * gw.rows * gw.cols : nullptr;
    for_outputs<S>(acc, i0, j0, gw.cols, gw.rows, [&](int64_t i, int64_t j, int n, float (&v)[8]) {
        if (out) store8(out + j * gw.cols + i, n, v);
        else store8((T*)gw.p + j * gw.stride + i, n, v);
    });
}

// The splits' float sums joined in a fixed order: 256 neighbouring ones a
// workgroup, four a lane; each of its sixteen waves takes every sixteenth
// split, with four loads in flight. A split holds out's elements and, after
// them, those of `bias` (either may be left out); `width` is the distance
// between splits.
template <class T>
__global__ void __launch_bounds__(1024) join_kernel(const float* partial, int splits, int64_t width, Mat out, float* bias,
                                                    int64_t biases) {
    constexpr int kParts = 16;
    __shared__ f32x4 s[kParts][64];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    const int64_t n = out.rows * out.cols, end = n + biases, q = ((int64_t)blockIdx.x * 64 + lane) * 4;
    typedef float loose4 __attribute__((ext_vector_type(4), aligned(4)));
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (q + 4 <= end) {
        int k = part;
        for (; k + 3 * kParts < splits; k += 4 * kParts) {
            f32x4 u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = *(const loose4*)(partial + (k + kParts * e) * width + q);
#pragma unroll
            for (int e = 0; e < 4; ++e) v += u[e];
        }
        for (; k < splits; k += kParts) v += *(const loose4*)(partial + k * width + q);
    } else {
        for (int k = part; k < splits; k += kParts)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (q + e < end) v[e] += partial[k * width + q + e];
    }
    s[part][lane] = v;
    __syncthreads();
    if (part != 0) return;
    for (int k = 1; k < kParts; ++k) v += s[k][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (q + e < n) {
            if (out.p) ((T*)out.p)[(q + e) / out.cols * out.stride + (q + e) % out.cols] = (T)v[e];
        } else if (q + e < end) {
            bias[q + e - n] = v[e];
        }
    }
}

// Few splits are read by a thread for eight outputs, many are shared by the
// waves of a workgroup. 8 splits of 2048 x 1024 halves: 11.3 us by threads, 25.4
// by waves; whole backwards with 64000 x 300 -> 300 halves' many splits: 137 us by
// threads, 121 by waves.
constexpr int64_t kFewSplits = 16;
template <class T>
void join(const float* partial, int64_t splits, const Mat& out, hipStream_t s) {
    if (splits <= kFewSplits) {
        LinearForward a{};
        a.y = out;
        join_rows_kernel<T, kActNone>
            <<<(unsigned)ceil_div(ceil_div(out.cols, 8) * out.rows, 256), 256, 0, s>>>(a, partial, (int)splits);
    } else {
        join_kernel<T><<<(unsigned)ceil_div(out.rows * out.cols, 256), 1024, 0, s>>>(partial, (int)splits,
                                                                                    out.rows * out.cols, out, nullptr, 0);
    }
}

// dz = dy act'(z) rounded to T (when dz.p), and the workgroup's column sums of
// the float dz at sums + blockIdx.x * cols (when sums). Rounded because the two
// products take operands of T: dz as two halves, high and low, would make both
// twice as long (16384 x 1024 -> 2048: 140 us of 188 once more). It costs the
// gradients 0.0024 of themselves for bfloat16 where a float dz has 0.0017,
// float16 0.00029 and 0.00021; the results' own rounding is most of either.
// A thread keeps 8 columns; `across` (a power of two) threads share a row, the
// others of the 256 take further rows. Bound by its bytes: 16384 x 2048 halves,
// 201 MB, 40 us (5.0 TB/s).
template <class T, int ACT>
__global__ void __launch_bounds__(256) slope_kernel(Mat gy, Mat z, Mat dz, float* sums, int across) {
    const int lane = threadIdx.x & (across - 1), group = threadIdx.x / across, groups = 256 / across;
    const int64_t c = ((int64_t)blockIdx.y * across + lane) * 8;
    const int n = (int)(gy.cols - c < 8 ? gy.cols - c : 8);
    float sum[8] = {};
    if (n > 0)
        for (int64_t r = (int64_t)blockIdx.x * groups + group; r < gy.rows; r += (int64_t)gridDim.x * groups) {
            float v[8];
            load8((const T*)gy.p + r * gy.stride + c, n, v);
            if constexpr (ACT != kActNone) {
                float u[8];
                load8((const T*)z.p + r * z.stride + c, n, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= activate_slope<ACT>(u[e]);
                if (dz.p) store8((T*)dz.p + r * dz.stride + c, n, v);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[e];
        }
    if (!sums) return;
    __shared__ float s[256][9];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[threadIdx.x][e] = sum[e];
    __syncthreads();
    for (int q = threadIdx.x; q < across * 8; q += 256) {
        const int64_t k = (int64_t)blockIdx.y * across * 8 + q;
        float v = 0.0f;
        for (int w = 0; w < groups; ++w) v += s[w * across + q / 8][q % 8];
        if (k < gy.cols) sums[(int64_t)blockIdx.x * gy.cols + k] = v;
    }
}

// ---- the backward's plan: what it keeps in the workspace
struct BackwardPlan {
    bool narrow = false;         // one pass over the rows (linear_narrow.hip)
    bool dz = false;             // an activation's dz is written
    int64_t dz_stride = 0;
    int across = 1;              // threads on a row of the slope pass
    int64_t slope_x = 0, slope_y = 0;   // its grid; 0: no pass
    int64_t splits = 1, split_rows = 0;   // of grad_w's rows
    KSplits gx;                  // of grad_x's out
    size_t dz_bytes = 0, sums_bytes = 0, partial_bytes = 0;
};

// Rows a split of grad_w is worth at least: its float sums are written and read again.
constexpr int64_t kSplitRows = 1024;

BackwardPlan plan_backward(const LinearBackward& a) {
    BackwardPlan p;
    const int64_t rows = a.grad_y.rows, out = a.grad_y.cols, in = a.x.cols;
    if (linear_backward_is_narrow(a)) {
        p.narrow = true;
        p.splits = narrow_backward_splits(a);
        p.partial_bytes = sizeof(float) * (size_t)(p.splits * (in * out + out));
        return p;
    }
    p.dz = a.activation != kActNone && (a.grad_x.p || a.grad_w.p) && rows > 0;
    if (a.grad_x.p && rows > 0) {
        p.gx = split_k(in, rows, out, a.dtype == TGS_DTYPE_FLOAT32 ? 4 : 2);
        if (p.gx.splits > 1) p.partial_bytes = sizeof(float) * (size_t)(p.gx.splits * rows * in);
    }
    if (p.dz || a.grad_bias) {
        while (p.across < 256 && p.across * 8 < out) p.across *= 2;
        p.slope_y = ceil_div(out, (int64_t)p.across * 8);
        const int64_t by_rows = ceil_div(rows, 256 / p.across);
        const int64_t most = ceil_div(1024, p.slope_y);
        p.slope_x = by_rows < most ? by_rows : most;
        if (a.grad_bias) p.sums_bytes = sizeof(float) * (size_t)(p.slope_x * out + 64);
    }
    if (p.dz) {
        p.dz_stride = ceil_div(out, 8) * 8;
        p.dz_bytes = (size_t)(rows * p.dz_stride) * (a.dtype == TGS_DTYPE_FLOAT32 ? 4 : 2);
    }
    if (a.grad_w.p) {
        const int64_t most = ceil_div(rows, kSplitRows) > 1 ? ceil_div(rows, kSplitRows) : 1;
        by_shape(in, out, most, true, [&](auto shape) {
            using S = decltype(shape);
            const int64_t tiles = ceil_div(in, S::kI) * ceil_div(out, S::kJ);
            // as many workgroups as fit the card at once (LDS: one to five a compute unit)
            const int64_t want = ceil_div(256 * S::kResident, tiles);
            p.splits = want < most ? want : most;
        });
        p.split_rows = ceil_div(ceil_div(rows, p.splits), 64) * 64;
        if (p.split_rows < 64) p.split_rows = 64;
        p.splits = ceil_div(rows, p.split_rows);
        if (p.splits < 1) p.splits = 1;
        // the two products' sums take turns in one place
        if (p.splits > 1) p.partial_bytes = std::max(p.partial_bytes, sizeof(float) * (size_t)(p.splits * in * out));
    }
    const auto round = [](size_t n) { return (n + 255) / 256 * 256; };
    p.dz_bytes = round(p.dz_bytes);
    p.sums_bytes = round(p.sums_bytes);
    p.partial_bytes = round(p.partial_bytes);
    return p;
}

template <class T>
void backward(const LinearBackward& a, unsigned char* workspace, hipStream_t s) {
    const BackwardPlan p = plan_backward(a);
    const int64_t rows = a.grad_y.rows, out = a.grad_y.cols, in = a.x.cols;
    if (p.narrow) {
        float* split = (float*)workspace;
        launch_narrow_backward(a, split, s);
        const Mat gw{a.grad_w.p, out, in, a.grad_w.p ? a.grad_w.stride : in};
        const int64_t biases = a.grad_bias ? out : 0;
        if (gw.p)
            join_kernel<T><<<(unsigned)ceil_div(in * out + biases, 256), 1024, 0, s>>>(split, (int)p.splits, in * out + out,
                                                                                      gw, a.grad_bias, biases);
        else if (biases)
            join_kernel<T><<<(unsigned)ceil_div(out, 256), 1024, 0, s>>>(split + in * out, (int)p.splits, in * out + out,
                                                                        Mat{nullptr, 0, 1, 1}, a.grad_bias, biases);
        return;
    }
    Mat dz = a.grad_y;
    float* sums = (float*)(workspace + p.dz_bytes);
    float* partial = (float*)(workspace + p.dz_bytes + p.sums_bytes);
    if (p.dz) dz = Mat{workspace, rows, out, p.dz_stride};
    if (p.slope_x)
        by_activation(a.activation, [&](auto act) {
            slope_kernel<T, decltype(act)::value><<<dim3((unsigned)p.slope_x, (unsigned)p.slope_y), 256, 0, s>>>(
                a.grad_y, a.preact, p.dz ? dz : Mat{}, a.grad_bias ? sums : nullptr, p.across);
        });
    if (a.grad_bias)
        launch_column_sums(sums, (int)p.slope_x, out, out, a.grad_bias, nullptr, s);
    if (a.grad_x.p && rows)
        by_shape(in, rows, 1, is_deep<T>(out), [&](auto shape) {
            using S = decltype(shape);
            const uint32_t ni = (uint32_t)ceil_div(in, S::kI), nj = (uint32_t)ceil_div(rows, S::kJ);
            grad_x_kernel<T, S><<<dim3(ni * nj, (unsigned)p.gx.splits), S::kThreads, 0, s>>>(
                dz, a.w, a.grad_x, p.gx.splits > 1 ? partial : nullptr, p.gx.depth, ni, nj);
        });
    if (a.grad_x.p && rows && p.gx.splits > 1)
        join<T>(partial, p.gx.splits, a.grad_x, s);
    if (a.grad_w.p) {
        const int64_t most = ceil_div(rows, kSplitRows) > 1 ? ceil_div(rows, kSplitRows) : 1;
        by_shape(in, out, most, true, [&](auto shape) {
            using S = decltype(shape);
            const uint32_t ni = (uint32_t)ceil_div(in, S::kI), nj = (uint32_t)ceil_div(out, S::kJ);
            grad_w_kernel<T, S><<<dim3(ni * nj, (unsigned)p.splits), S::kThreads, 0, s>>>(
                dz, a.x, a.grad_w, p.splits > 1 ? partial : nullptr, p.split_rows, ni, nj);
        });
        if (p.splits > 1) join<T>(partial, p.splits, a.grad_w, s);
    }
}

}  // namespace

size_t linear_backward_workspace(const LinearBackward& a) {
    const BackwardPlan p = plan_backward(a);
    return p.dz_bytes + p.sums_bytes + p.partial_bytes;
}

size_t linear_forward_workspace(const LinearForward& a) {
    if (linear_forward_is_few(a) || linear_forward_by_rows(a)) return 0;
    const KSplits k = split_k(a.y.cols, a.y.rows, a.x.cols, a.dtype == TGS_DTYPE_FLOAT32 ? 4 : 2);
    return k.splits > 1 ? sizeof(float) * (size_t)(k.splits * a.y.rows * a.y.cols) : 0;
}

int launch_linear_forward(const LinearForward& a, void* workspace, hipStream_t s) {
    if (linear_forward_is_few(a)) {
        launch_linear_few(a, s);
    } else if (linear_forward_by_rows(a)) {
        launch_linear_rows(a, s);
    } else {
        by_dtype(a.dtype, [&](auto t) {
            using T = decltype(t);
            const KSplits k = split_k(a.y.cols, a.y.rows, a.x.cols, (int)sizeof(T));
            float* partial = k.splits > 1 ? (float*)workspace : nullptr;
            by_shape(a.y.cols, a.y.rows, 1, is_deep<T>(a.x.cols), [&](auto shape) {
                using S = decltype(shape);
                for (int64_t first = 0; first < a.y.rows; first += kLaunchRows) {
                    const LinearForward part = rows_of<T>(a, first);
                    const uint32_t ni = (uint32_t)ceil_div(a.y.cols, S::kI), nj = (uint32_t)ceil_div(part.y.rows, S::kJ);
                    forward_kernel<T, S>
                        <<<dim3(ni * nj, (unsigned)k.splits), S::kThreads, 0, s>>>(part, partial, k.depth, ni, nj);
                }
            });
            if (partial)
                by_activation(a.activation, [&](auto act) {
                    join_rows_kernel<T, decltype(act)::value>
                        <<<(unsigned)ceil_div(ceil_div(a.y.cols, 8) * a.y.rows, 256), 256, 0, s>>>(a, partial, (int)k.splits);
                });
        });
    }
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_linear_backward(const LinearBackward& a, void* workspace, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) { backward<decltype(t)>(a, (unsigned char*)workspace, s); });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
