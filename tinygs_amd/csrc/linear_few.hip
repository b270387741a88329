// y = act(x w^T + bias) + residual for a few rows (a query, a picked set of
// Gaussians), bound by the bytes of w and by latency.
//
// A workgroup makes 16 columns of up to 16 rows. Its eight waves share k: each
// takes every eighth step of 32, reads the fragments of w and x straight from
// memory, four steps in flight, and the eight sums are joined through LDS in
// order. w passes no LDS, and all of k is on its way at once up to 1024. One row of 4096
// x 4096 halves takes 7.9 us a call (34 MB, 4.2 TB/s), of 256 x 256 a kernel of
// 4.3 us, its launch and one round of loads.
#include "narrow_rows.h"

namespace tgs {

namespace {

constexpr int kWaves = 8;
constexpr int kAhead = 4;

template <class T, int ACT>
__device__ __forceinline__ void few_outputs(const LinearForward& a, f32x4 v, int64_t row, int64_t column) {
    const int n = (int)min(a.y.cols - column, (int64_t)4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e >= n) break;
        float z = v[e] + (a.bias ? a.bias[column + e] : 0.0f);
        if (a.preact.p) ((T*)a.preact.p)[row * a.preact.stride + column + e] = (T)z;
        z = activate<ACT>(z);
        if (a.residual.p) z += (float)((const T*)a.residual.p)[row * a.residual.stride + column + e];
        ((T*)a.y.p)[row * a.y.stride + column + e] = (T)z;
    }
}

template <class T>
__global__ void __launch_bounds__(64 * kWaves) few_kernel(LinearForward a) {
    using C = Chunk<T>;
    constexpr int V = C::V, kChunks = 8 / V;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int in = (int)a.x.cols, steps = (in + 31) / 32;
    const int64_t n0 = (int64_t)blockIdx.x * 16, r0 = (int64_t)blockIdx.y * 16;
    const bool ragged = in % V != 0;   // the last step then has partial chunks

    struct Side {
        const T* base;
        __amdgpu_buffer_rsrc_t buffer;
        uint32_t offset;
        int64_t stride;
        bool exists;
    };
    const auto side = [&](const Mat& m, int64_t first) {
        const int64_t held = min(m.rows - first, (int64_t)16), pitch = m.stride * (int64_t)sizeof(T);
        Side s;
        s.base = (const T*)m.p + first * m.stride;
        s.buffer = resource_of(s.base, (held - 1) * pitch + in * (int64_t)sizeof(T));
        s.offset = (uint32_t)(lane & 15) * (uint32_t)pitch;
        s.stride = m.stride;
        s.exists = (lane & 15) < held;
        return s;
    };
    const Side w = side(a.w, n0), x = side(a.x, r0);
    typedef typename C::type chunk;
    const auto load = [&](const Side& s, int step, chunk(&to)[kChunks]) {
#pragma unroll
        for (int h = 0; h < kChunks; ++h) {
            const int k = 32 * step + 8 * (lane >> 4) + V * h;
            if (ragged && step == steps - 1) {
                const int left = s.exists ? min(max(in - k, 0), V) : 0;
                to[h] = C::gather(s.base + (left > 0 ? (lane & 15) * s.stride + k : 0), left);
            } else {
                to[h] = __builtin_bit_cast(chunk, __builtin_amdgcn_raw_buffer_load_b128(
                                                      s.buffer, (int)((k < in ? s.offset : kNowhere) + (uint32_t)k * (uint32_t)sizeof(T)), 0, 0));
            }
        }
    };
    const auto fragment = [&](const chunk(&v)[kChunks]) {
        if constexpr (sizeof(T) == 4) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = v[e / 4][e % 4];
            return split3(f);
        } else {
            return __builtin_bit_cast(typename Frag<T>::type, v[0]);
        }
    };
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = wave; s < steps; s += kWaves * kAhead) {
        chunk cw[kAhead][kChunks], cx[kAhead][kChunks];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {   // steps past the last are zeros
            load(w, s + q * kWaves, cw[q]);
            load(x, s + q * kWaves, cx[q]);
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) acc = multiply(fragment(cw[q]), fragment(cx[q]), acc);
    }
    if constexpr (sizeof(T) == 4) {   // k as this wave's steps hold it
        f32x4 one[1][1] = {{acc}};
        const int own = steps > wave ? (steps - wave - 1) / kWaves + 1 : 0;
        const auto element = [&](const Side& s, int row, int64_t k) {
            const int64_t at = 32 * (wave + kWaves * (k >> 5)) + (k & 31);
            return s.exists && at < in ? s.base[row * s.stride + at] : 0.0f;
        };
        form_again(
            one, 0, 32 * own, [&](int, int row, int64_t k) { return element(w, row, k); },
            [&](int, int row, int64_t k) { return element(x, row, k); }, [](int, int, int) { return true; });
        acc = one[0][0];
    }
    __shared__ f32x4 sums[kWaves][64];
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int q = 1; q < kWaves; ++q) acc += sums[q][lane];
    const int64_t row = r0 + (lane & 15), column = n0 + 4 * (lane >> 4);
    if (row >= a.y.rows || column >= a.y.cols) return;
    if (a.activation == kActGelu) few_outputs<T, kActGelu>(a, acc, row, column);
    else if (a.activation == kActSilu) few_outputs<T, kActSilu>(a, acc, row, column);
    else if (a.activation == kActRelu) few_outputs<T, kActRelu>(a, acc, row, column);
    else few_outputs<T, kActNone>(a, acc, row, column);
}

}  // namespace

// Against tiles with k split, SiLU, whole calls: 1 x 4096 -> 4096 halves 7.9 and
// 13.3 us, floats 20.0 and 33.2; 16 rows 10.8 and 14.4, 22.9 and 33.3. More rows
// read w a second time: 32 x 4096 -> 4096 17.9 and 15.1, floats 37.8 and 33.6,
// but 32 x 1024 -> 1024, all on its way at once, 6.8 and 8.6, floats 7.4 and 10.9.
bool linear_forward_is_few(const LinearForward& a) { return a.y.rows <= (a.x.cols <= 1024 ? 32 : 16); }

void launch_linear_few(const LinearForward& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.y.cols + 15) / 16), (unsigned)((a.y.rows + 15) / 16));
    by_dtype(a.dtype, [&](auto t) { few_kernel<decltype(t)><<<grid, 64 * kWaves, 0, s>>>(a); });
}

}  // namespace tgs
