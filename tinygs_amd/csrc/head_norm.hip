// Norms of queries and keys over each head, with the turning of their pairs by
// their positions, and the gradients:
//   h = x r, r = 1 / sqrt(mean(x^2) + eps), u = h gamma, y = u turned;
//   with g = dy turned back: dgamma = sum g h, dx = r (g gamma - h mean(g gamma h)).
//
// Bound by the bytes: x is read once and y written once (backward x and dy, and
// dx), so a head stays in the registers of the LANES lanes that share it, a
// chunk of 16 bytes each. A lane takes the same columns of every head of a row:
// its pairs' angles, the same for all heads, are formed once a row.
//
// An angle is a sum of up to four products in 64 bits, reduced to half a turn
// there: at a position of 1e4 and ten radians a unit, 32 bits would leave an
// error of 0.004. Its sine and cosine are then of a float within half a turn.
#include <type_traits>

#include "row_chunks.h"

namespace tgs {

namespace {

constexpr int kThreads = 256;
constexpr int kAxes = 4;
constexpr int kHeads = 4;   // of a row whose loads are on their way together

// Sines and cosines of a lane's pairs: a row's angles. Pairs that are not turned have 0 and 1.
template <int PAIRS>
struct Turn {
    float f[PAIRS][kAxes];   // frequencies, 0 where there are none
    float sine[PAIRS], cosine[PAIRS];

    __device__ __forceinline__ void begin(const HeadNorm& a, int lane) {
        const int axes = (int)a.frequencies.cols;
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
            const int64_t pair = lane * PAIRS + p;
            sine[p] = 0.0f;
            cosine[p] = 1.0f;
#pragma unroll
            for (int k = 0; k < kAxes; ++k)
                f[p][k] = a.positions.p && k < axes && pair < a.frequencies.rows
                              ? ((const float*)a.frequencies.p)[pair * a.frequencies.stride + k] : 0.0f;
        }
    }

    __device__ __forceinline__ void row(const HeadNorm& a, int64_t r, int lane) {
        if (!a.positions.p) return;
        const float* at = (const float*)a.positions.p + r * a.positions.stride;
        double x[kAxes];
#pragma unroll
        for (int k = 0; k < kAxes; ++k) x[k] = k < (int)a.positions.cols ? (double)at[k] : 0.0;
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
            double t = x[0] * (double)f[p][0];
#pragma unroll
            for (int k = 1; k < kAxes; ++k) t = fma(x[k], (double)f[p][k], t);
            t *= 0.15915494309189535;   // in turns
            t -= rint(t);
            float s, c;
            sincospif(2.0f * (float)t, &s, &c);
            const bool turned = lane * PAIRS + p < a.frequencies.rows;   // an infinite position leaves the others alone
            sine[p] = turned ? s : 0.0f;
            cosine[p] = turned ? c : 1.0f;
        }
    }

    // By the angles (SIGN 1) or back (-1).
    template <int SIGN>
    __device__ __forceinline__ void apply(float* v) const {
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
            const float x = v[2 * p], y = v[2 * p + 1], s = SIGN > 0 ? sine[p] : -sine[p];
            v[2 * p] = fmaf(x, cosine[p], -(y * s));
            v[2 * p + 1] = fmaf(x, s, y * cosine[p]);
        }
    }
};

// A lane's chunk of a head as it lies in memory; zeros past the head. WHOLE: heads of
// whole chunks. Their loads have no branch, which would wait for each where its
// paths meet: lanes without a chunk read another one's.
template <class T, bool WHOLE>
__device__ __forceinline__ typename ChunkOf<T>::type load_raw(const T* head, int lane, int d) {
    constexpr int V = kChunk<T>;
    using Raw = typename ChunkOf<T>::type;
    if constexpr (WHOLE) return *(const Raw*)(head + min(lane, d / V - 1) * V);
    Raw u = {};
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (lane * V + i < d) u[i] = head[lane * V + i];
    return u;
}
template <class T, bool WHOLE>
__device__ __forceinline__ void unpack(const typename ChunkOf<T>::type& u, int lane, int d, float* v) {
#pragma unroll
    for (int i = 0; i < kChunk<T>; ++i) v[i] = !WHOLE || lane * kChunk<T> < d ? (float)u[i] : 0.0f;
}

// The power of two by which a head's elements and epsilon are multiplied where the squares' sum leaves the range of
// floats or its bits: elements above 2^60, and below 2^-40 where epsilon is below 2^-80. 1 else. Halves hold neither.
template <class T>
constexpr bool kLifted = !std::is_same_v<T, _Float16>;
__device__ __forceinline__ float lift_of(float sum, float eps) {
    return !(sum <= 0x1p120f) ? 0x1p-70f : sum < 0x1p-80f && eps < 0x1p-80f ? 0x1p100f : 1.0f;
}
// 1 / sqrt(mean(x^2) + epsilon) of such heads, whose elements are multiplied; the others' as they are.
template <int LANES, int V>
__device__ __forceinline__ float lifted_rstd(float (&v)[V], float by, float eps, float inv) {
    float sum[1] = {0.0f};
    int none = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        v[i] *= by;
        sum[0] = fmaf(v[i], v[i], sum[0]);
    }
    group_sum<LANES>(sum, nullptr, none);
    return 1.0f / sqrtf(fmaf(sum[0], inv, eps * by * by));
}

template <class T, int LANES, bool WHOLE>
__global__ void __launch_bounds__(kThreads) forward_kernel(HeadNorm a) {
    constexpr int V = kChunk<T>, kRows = kThreads / LANES;
    const int lane = threadIdx.x % LANES, d = a.head;
    int none = 0;
    float gamma[V];
    load_vector<V>(a.gamma, lane, d, 1.0f, gamma);
    Turn<V / 2> turn;
    turn.begin(a, lane);
    const float inv = 1.0f / (float)d;
    for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES; r < a.x.rows; r += (int64_t)gridDim.x * kRows) {
        const T* x = (const T*)a.x.p + r * a.x.stride;
        T* y = (T*)a.y.p + r * a.y.stride;
        for (int h0 = 0; h0 < a.heads; h0 += kHeads) {
            typename ChunkOf<T>::type raw[kHeads];
#pragma unroll
            for (int k = 0; k < kHeads; ++k)
                raw[k] = load_raw<T, WHOLE>(x + (int64_t)min(h0 + k, a.heads - 1) * d, lane, d);
            if (h0 == 0) turn.row(a, r, lane);   // beside the first loads
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                if (h0 + k >= a.heads) break;
                float v[V], sum[1] = {0.0f};
                unpack<T, WHOLE>(raw[k], lane, d, v);
#pragma unroll
                for (int i = 0; i < V; ++i) sum[0] = fmaf(v[i], v[i], sum[0]);
                group_sum<LANES>(sum, nullptr, none);
                float rstd = 1.0f / sqrtf(fmaf(sum[0], inv, a.eps));
                if constexpr (kLifted<T>) {
                    const float by = lift_of(sum[0], a.eps);
                    if (__builtin_expect(__ballot(by != 1.0f) != 0, 0)) rstd = lifted_rstd<LANES>(v, by, a.eps, inv);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = v[i] * rstd * gamma[i];
                turn.template apply<1>(v);
                store_chunk<T>(y + (int64_t)(h0 + k) * d, lane, d, v);
            }
        }
    }
}

// Column sums: a workgroup's, over its rows and all heads, to row blockIdx.x of `partial`.
template <class T, int LANES, bool WHOLE, bool SUMS>
__global__ void __launch_bounds__(kThreads) backward_kernel(HeadNorm a, float* partial) {
    constexpr int V = kChunk<T>, kRows = kThreads / LANES;
    const int lane = threadIdx.x % LANES, d = a.head;
    int none = 0;
    float gamma[V], grad_gamma[V];
    load_vector<V>(a.gamma, lane, d, 1.0f, gamma);
#pragma unroll
    for (int i = 0; i < V; ++i) grad_gamma[i] = 0.0f;
    Turn<V / 2> turn;
    turn.begin(a, lane);
    const float inv = 1.0f / (float)d;
    for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES; r < a.x.rows; r += (int64_t)gridDim.x * kRows) {
        const T* x = (const T*)a.x.p + r * a.x.stride;
        const T* gy = (const T*)a.grad_y.p + r * a.grad_y.stride;
        T* gx = a.y.p ? (T*)a.y.p + r * a.y.stride : nullptr;
        for (int h0 = 0; h0 < a.heads; h0 += kHeads) {
            typename ChunkOf<T>::type rx[kHeads], rg[kHeads];
            bool lifted[kHeads] = {};
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const int64_t at = (int64_t)min(h0 + k, a.heads - 1) * d;
                rx[k] = load_raw<T, WHOLE>(x + at, lane, d);
                rg[k] = load_raw<T, WHOLE>(gy + at, lane, d);
            }
            if (h0 == 0) turn.row(a, r, lane);
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                if (h0 + k >= a.heads) break;
                float v[V], g[V], sum[2] = {0.0f, 0.0f};
                unpack<T, WHOLE>(rx[k], lane, d, v);
                unpack<T, WHOLE>(rg[k], lane, d, g);
                turn.template apply<-1>(g);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sum[0] = fmaf(v[i], v[i], sum[0]);
                    sum[1] = fmaf(g[i] * gamma[i], v[i], sum[1]);
                }
                group_sum<LANES>(sum, nullptr, none);
                float rstd = 1.0f / sqrtf(fmaf(sum[0], inv, a.eps));
                if constexpr (kLifted<T>) {   // such a head waits: it adds nothing here
                    lifted[k] = lift_of(sum[0], a.eps) != 1.0f;
                    rstd = lifted[k] ? 0.0f : rstd;
                }
                const float c = sum[1] * rstd * inv;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float h = v[i] * rstd;
                    if (SUMS) grad_gamma[i] = fmaf(g[i], h, grad_gamma[i]);
                    v[i] = rstd * fmaf(-h, c, g[i] * gamma[i]);
                }
                if (gx && !(kLifted<T> && lifted[k])) store_chunk<T>(gx + (int64_t)(h0 + k) * d, lane, d, v);
            }
            if constexpr (!kLifted<T>) continue;
            if (__builtin_expect(__ballot(lifted[0] || lifted[1] || lifted[2] || lifted[3]) == 0, 1)) continue;
#pragma unroll 1
            for (int k = 0; k < kHeads; ++k) {   // one branch for the heads, and theirs alone once more
                if (!(k == 0 ? lifted[0] : k == 1 ? lifted[1] : k == 2 ? lifted[2] : lifted[3])) continue;
                const int64_t at = (int64_t)(h0 + k) * d;
                float v[V], g[V], sum[1] = {0.0f}, dot[1] = {0.0f};
                unpack<T, WHOLE>(load_raw<T, WHOLE>(x + at, lane, d), lane, d, v);
                unpack<T, WHOLE>(load_raw<T, WHOLE>(gy + at, lane, d), lane, d, g);
                turn.template apply<-1>(g);
#pragma unroll
                for (int i = 0; i < V; ++i) sum[0] = fmaf(v[i], v[i], sum[0]);
                group_sum<LANES>(sum, nullptr, none);
                const float by = lift_of(sum[0], a.eps), rstd = lifted_rstd<LANES>(v, by, a.eps, inv);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    v[i] *= rstd;
                    dot[0] = fmaf(g[i] * gamma[i], v[i], dot[0]);
                    if (SUMS) grad_gamma[i] = fmaf(g[i], v[i], grad_gamma[i]);
                }
                group_sum<LANES>(dot, nullptr, none);
                const float c = dot[0] * inv;
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = rstd * fmaf(-v[i], c, g[i] * gamma[i]) * by;
                if (gx) store_chunk<T>(gx + at, lane, d, v);
            }
        }
    }
    if constexpr (SUMS) {
        __shared__ float s[kThreads * V];
#pragma unroll
        for (int i = 0; i < V; ++i) s[threadIdx.x * V + i] = grad_gamma[i];
        __syncthreads();
        for (int c = threadIdx.x; c < d; c += kThreads) {
            float v = s[c];
            for (int k = 1; k < kRows; ++k) v += s[k * LANES * V + c];
            partial[(int64_t)blockIdx.x * d + c] = v;
        }
    }
}

// f<lanes, whether heads are whole chunks> with the least power of two of lanes whose chunks hold a head.
template <class T, class F>
void by_head(int head, F with) {
    constexpr int V = kChunk<T>;
    const auto f = [&](auto lanes) {
        if (head % V == 0) with(lanes, Constant<1>{});
        else with(lanes, Constant<0>{});
    };
    if (head <= V) f(Constant<1>{});
    else if (head <= 2 * V) f(Constant<2>{});
    else if (head <= 4 * V) f(Constant<4>{});
    else if (head <= 8 * V) f(Constant<8>{});
    else if (head <= 16 * V) f(Constant<16>{});
    else if (head <= 32 * V) f(Constant<32>{});
    else f(Constant<64>{});
}

// Workgroups for rows of `lanes` lanes each: no more than `most`.
unsigned blocks_of(int64_t rows, int lanes, int64_t most) {
    const int64_t want = (rows * lanes + kThreads - 1) / kThreads;
    return (unsigned)(want < most ? want : most);
}
constexpr int64_t kSumBlocks = 1024;   // each leaves a row of column sums

}  // namespace

size_t head_norm_backward_workspace(const HeadNorm& a) {
    return a.grad_gamma ? sizeof(float) * kSumBlocks * (size_t)a.head : 0;
}

int launch_head_norm(const HeadNorm& a, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        by_head<T>(a.head, [&](auto lanes, auto whole) {
            constexpr int kLanes = decltype(lanes)::value;
            constexpr bool kWhole = decltype(whole)::value != 0;
            forward_kernel<T, kLanes, kWhole><<<blocks_of(a.x.rows, kLanes, 2048), kThreads, 0, s>>>(a);
        });
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_head_norm_backward(const HeadNorm& a, void* workspace, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        by_head<T>(a.head, [&](auto lanes, auto whole) {
            constexpr int kLanes = decltype(lanes)::value;
            constexpr bool kWhole = decltype(whole)::value != 0;
            if (!a.grad_gamma) {
                const unsigned blocks = blocks_of(a.x.rows, kLanes, 2048);
                if (blocks && a.y.p) backward_kernel<T, kLanes, kWhole, false><<<blocks, kThreads, 0, s>>>(a, nullptr);
                return;
            }
            const unsigned blocks = blocks_of(a.x.rows, kLanes, kSumBlocks);
            if (blocks) backward_kernel<T, kLanes, kWhole, true><<<blocks, kThreads, 0, s>>>(a, (float*)workspace);
            launch_column_sums((const float*)workspace, (int)blocks, a.head, a.head, a.grad_gamma, nullptr, s);
        });
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
