// The norm of many gradients together, and clipping:
//   norm = scale sqrt(sum of squares), g <- g f, f = scale min(1, max_norm / (norm + eps)).
//
// Two launches over all tensors: the first leaves a sum of squares for each
// workgroup, the second joins them (every workgroup by itself, in one order) and
// multiplies; in place and with f = 1 it writes nothing. Bound by the bytes.
// Squares are of doubles: those of floats above 2^64 or below 2^-75 leave the
// range of floats. A double multiply-add an element is a tenth of the time that
// the element's load takes.
//
// The elements of all tensors are cut into chunks of kChunkElements, which the
// workgroups take in turn, so that a launch is the same size for a few small
// tensors and for many.
#include "row_chunks.h"

namespace tgs {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kChunkElements = 8192;
constexpr int64_t kMost = 1024;   // workgroups, and sums that each of the second launch joins

// The part that chunk n belongs to: the last whose first chunk is not above
// it. Parts without elements have no chunk: their first is that of the next.
__device__ __forceinline__ int part_of(const uint32_t* firsts, int count, uint32_t n) {
    const int lane = threadIdx.x & 63;
    int part = -1;
    for (int k = 0; k < count; k += 64) {
        const uint64_t below = __ballot(k + lane < count && firsts[min(k + lane, count - 1)] <= n);
        part += __popcll(below);
        if (below != ~0ull) break;
    }
    return __builtin_amdgcn_readfirstlane(part);
}

__device__ __forceinline__ double workgroup_sum(double v) {
    __shared__ double s[kThreads / 64];
    for (int d = 32; d > 0; d >>= 1) v += __shfl_down(v, d, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int k = 1; k < kThreads / 64; ++k) v += s[k];
    __syncthreads();
    return v;
}

// Elements [first, last) of a part: f(where it goes, Constant<how many>, values),
// in chunks of 16 bytes where its rows follow each other without gaps.
template <class T, class F>
__device__ __forceinline__ void each(const ClipPart& a, int64_t first, int64_t last, F f) {
    constexpr int V = kChunk<T>, kAhead = 4, kWhole = (int)(kChunkElements / (kThreads * V));
    const T* g = (const T*)a.g;
    const bool packed = a.stride == a.cols && a.c_stride == a.cols;
    if (packed && last - first == kChunkElements) {   // all loads on their way, without branches between them
        typename ChunkOf<T>::type raw[kWhole];
        const int64_t k = first + threadIdx.x * V;
#pragma unroll
        for (int q = 0; q < kWhole; ++q) raw[q] = *(const typename ChunkOf<T>::type*)(g + k + q * kThreads * V);
#pragma unroll
        for (int q = 0; q < kWhole; ++q) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (float)raw[q][i];
            f(k + q * kThreads * V, Constant<V>{}, v);
        }
        return;
    }
    if (packed) {
        for (int64_t k = first + threadIdx.x * V; k < last; k += kThreads * V * kAhead) {
            float v[kAhead][V];
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int64_t at = k + (int64_t)q * kThreads * V;
                if (at < last) load_chunk<T>(g + at, 0, (int)min(last - at, (int64_t)V), v[q]);
            }
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                const int64_t at = k + (int64_t)q * kThreads * V;
                if (at + V <= last) f(at, Constant<V>{}, v[q]);
                else
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (at + i < last) f(at + i, Constant<1>{}, v[q] + i);
            }
        }
        return;
    }
    const int64_t row = first / a.cols;
    const uint32_t col = (uint32_t)(first - row * a.cols), cols = (uint32_t)a.cols;
    for (uint32_t k = threadIdx.x; k < (uint32_t)(last - first); k += kThreads) {
        const uint32_t down = (col + k) / cols, across = (col + k) - down * cols;
        const float v = (float)g[(row + down) * a.stride + across];
        f((row + down) * a.c_stride + across, Constant<1>{}, &v);
    }
}

template <class C, int N>
struct Some {
    typedef C type __attribute__((ext_vector_type(N), aligned(sizeof(C))));
};

__global__ void __launch_bounds__(kThreads) squares_kernel(const ClipPart* parts, const uint32_t* firsts, int count,
                                                           uint32_t chunks, double* sums) {
    double sum = 0.0;
    for (uint32_t n = blockIdx.x; n < chunks; n += gridDim.x) {
        const int part = part_of(firsts, count, n);
        const ClipPart a = parts[part];
        const int64_t first = (int64_t)(n - firsts[part]) * kChunkElements, last = min(first + kChunkElements, a.count);
        const auto add = [&](int64_t, auto some, const float* v) {
#pragma unroll
            for (int i = 0; i < decltype(some)::value; ++i) sum = fma((double)v[i], (double)v[i], sum);
        };
        if (a.dtype == TGS_DTYPE_FLOAT32) each<float>(a, first, last, add);
        else if (a.dtype == TGS_DTYPE_FLOAT16) each<_Float16>(a, first, last, add);
        else each<__bf16>(a, first, last, add);
    }
    sum = workgroup_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

template <class T>
__device__ __forceinline__ void scale_chunk(const ClipPart& a, int64_t first, int64_t last, float factor) {
    const auto write = [&](auto c) {
        using C = decltype(c);
        each<T>(a, first, last, [&](int64_t at, auto some, const float* v) {
            constexpr int N = decltype(some)::value;
            typename Some<C, N>::type u;
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] = (C)(v[i] * factor);
            *(typename Some<C, N>::type*)((C*)a.c + at) = u;
        });
    };
    if (a.c_dtype == TGS_DTYPE_FLOAT32) write(float{});
    else if (a.c_dtype == TGS_DTYPE_FLOAT16) write(_Float16{});
    else write(__bf16{});
}

__global__ void __launch_bounds__(kThreads) scale_kernel(const ClipPart* parts, const uint32_t* firsts, int count,
                                                         uint32_t chunks, int sums_count, const double* sums, ClipRun p) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < sums_count; k += kThreads) sum += sums[k];
    const double norm = p.scale * sqrt(workgroup_sum(sum));
    if (p.norm && blockIdx.x == 0 && threadIdx.x == 0) *p.norm = (float)norm;
    const double within = p.max_norm / (norm + p.epsilon);
    const float factor = (float)(p.scale * (isinf(p.max_norm) ? 1.0 : within > 1.0 ? 1.0 : within));   // NaN stays
    if (factor == 1.0f && !p.apart) return;
    for (uint32_t n = blockIdx.x; n < chunks; n += gridDim.x) {
        const int part = part_of(firsts, count, n);
        const ClipPart a = parts[part];
        const int64_t first = (int64_t)(n - firsts[part]) * kChunkElements, last = min(first + kChunkElements, a.count);
        if (a.dtype == TGS_DTYPE_FLOAT32) scale_chunk<float>(a, first, last, factor);
        else if (a.dtype == TGS_DTYPE_FLOAT16) scale_chunk<_Float16>(a, first, last, factor);
        else scale_chunk<__bf16>(a, first, last, factor);
    }
}

}  // namespace

ClipPlan plan_clip(const ClipPart* parts, int count, uint32_t* firsts) {
    ClipPlan plan{};
    int64_t chunks = 0;
    for (int i = 0; i < count; ++i) {
        if (firsts) firsts[i] = (uint32_t)chunks;
        chunks += (parts[i].count + kChunkElements - 1) / kChunkElements;
    }
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    plan.chunks = chunks < 0x7fffffff ? (uint32_t)chunks : 0x7fffffffu;   // which the entry refuses
    plan.workgroups = (uint32_t)(chunks < kMost ? (chunks ? chunks : 1) : kMost);
    plan.sums_at = take(sizeof(double) * kMost);
    plan.parts_at = take((int64_t)sizeof(ClipPart) * count);
    plan.firsts_at = take((int64_t)sizeof(uint32_t) * count);
    plan.bytes = at;
    return plan;
}

int launch_clip(const ClipPlan& plan, int count, const ClipRun& p, unsigned char* workspace, hipStream_t s) {
    const ClipPart* parts = (const ClipPart*)(workspace + plan.parts_at);
    const uint32_t* firsts = (const uint32_t*)(workspace + plan.firsts_at);
    double* sums = (double*)(workspace + plan.sums_at);
    squares_kernel<<<plan.workgroups, kThreads, 0, s>>>(parts, firsts, count, plan.chunks, sums);
    scale_kernel<<<plan.workgroups, kThreads, 0, s>>>(parts, firsts, count, plan.chunks, (int)plan.workgroups, sums, p);
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
