// Layer norm over the rows of a matrix, and its gradients:
//   y = (x - mean) rstd gamma + beta;  with h = (x - mean) rstd, g = dy gamma:
//   dx = rstd (g - avg(g) - h avg(g h)) + residual's, dgamma = sum dy h, dbeta = sum dy.
//
// All of it is bound by the bytes: forward reads x once and writes y,
// backward reads x, dy (and the residual's gradient) once and writes dx. So a
// row stays in the registers of the LANES threads that share it (4 to 64
// lanes of a wave, or a workgroup of 256 or 1024), in PIECES chunks of 16
// bytes each, between its statistics and its output; a group walks over rows
// with gamma and beta (and backward the column sums) in registers. The
// variance is a second pass over the registers, from differences to the mean.
// Rows need no alignment: 16-byte loads and stores work from any element, and
// a row's last, partial chunk moves element by element. 1e6 x 256 halves: forward
// 1.02 GB in 218 us (4.7 TB/s), backward with the residual's gradient 2.05 GB in
// 370 us (5.5 TB/s).
#include "row_chunks.h"

namespace tgs {

namespace {

constexpr int threads_of(int lanes) { return lanes > 256 ? lanes : 256; }

template <class T, int LANES, int PIECES>
__global__ void __launch_bounds__(threads_of(LANES)) forward_kernel(LayerNormForward a) {
    constexpr int V = kChunk<T>, kGroups = threads_of(LANES) / LANES;
    __shared__ float s[2 * (LANES > 64 ? LANES / 64 : 1)];
    int turn = 0;
    const int lane = threadIdx.x % LANES, n = (int)a.x.cols;
    const float inv = 1.0f / (float)n;
    float gamma[PIECES][V], beta[PIECES][V];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        load_vector<V>(a.gamma, lane + p * LANES, n, 1.0f, gamma[p]);
        load_vector<V>(a.beta, lane + p * LANES, n, 0.0f, beta[p]);
    }
    for (int64_t r = (int64_t)blockIdx.x * kGroups + threadIdx.x / LANES; r < a.x.rows;
         r += (int64_t)gridDim.x * kGroups) {
        const T* x = (const T*)a.x.p + r * a.x.stride;
        T* y = (T*)a.y.p + r * a.y.stride;
        float v[PIECES][V], sum[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            load_chunk<T>(x, lane + p * LANES, n, v[p]);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0] += v[p][i];
        }
        group_sum<LANES>(sum, s, turn);
        const float mean = sum[0] / (float)n;   // exact for a row of one value
        sum[0] = 0.0f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[p][i] = (lane + p * LANES) * V + i < n ? v[p][i] - mean : 0.0f;
                sum[0] = fmaf(v[p][i], v[p][i], sum[0]);
            }
        group_sum<LANES>(sum, s, turn);
        const float rstd = 1.0f / sqrtf(sum[0] * inv + a.eps);
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[p][i] = fmaf(v[p][i] * rstd, gamma[p][i], beta[p][i]);
            store_chunk<T>(y, lane + p * LANES, n, v[p]);
        }
        if (lane == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// grad_x, and the workgroup's column sums of dy h and dy at
// partial + blockIdx.x * 2 n (nothing is summed without SUMS).
template <class T, int LANES, int PIECES, bool SUMS>
__global__ void __launch_bounds__(threads_of(LANES)) backward_kernel(LayerNormBackward a, float* partial) {
    constexpr int V = kChunk<T>, kGroups = threads_of(LANES) / LANES;
    __shared__ float s[4 * (LANES > 64 ? LANES / 64 : 1)];
    int turn = 0;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, n = (int)a.x.cols;
    const float inv = 1.0f / (float)n;
    float gamma[PIECES][V], sg[PIECES][V] = {}, sb[PIECES][V] = {};
#pragma unroll
    for (int p = 0; p < PIECES; ++p) load_vector<V>(a.gamma, lane + p * LANES, n, 1.0f, gamma[p]);
    for (int64_t r = (int64_t)blockIdx.x * kGroups + group; r < a.x.rows; r += (int64_t)gridDim.x * kGroups) {
        const T* x = (const T*)a.x.p + r * a.x.stride;
        const T* gy = (const T*)a.grad_y.p + r * a.grad_y.stride;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float h[PIECES][V], g[PIECES][V], res[PIECES][V], sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            load_chunk<T>(x, lane + p * LANES, n, h[p]);
            load_chunk<T>(gy, lane + p * LANES, n, g[p]);
        }
        if (a.residual.p) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
                load_chunk<T>((const T*)a.residual.p + r * a.residual.stride, lane + p * LANES, n, res[p]);
        }
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < V; ++i) {   // past the row g = 0, so h there adds nothing
                h[p][i] = (h[p][i] - mean) * rstd;
                if constexpr (SUMS) {
                    sg[p][i] = fmaf(g[p][i], h[p][i], sg[p][i]);
                    sb[p][i] += g[p][i];
                }
                g[p][i] *= gamma[p][i];
                sum[0] += g[p][i];
                sum[1] = fmaf(g[p][i], h[p][i], sum[1]);
            }
        if (!a.grad_x.p) continue;
        group_sum<LANES>(sum, s, turn);
        const float c1 = sum[0] * inv, c2 = sum[1] * inv;
        T* gx = (T*)a.grad_x.p + r * a.grad_x.stride;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = rstd * fmaf(-h[p][i], c2, g[p][i] - c1);
                g[p][i] = a.residual.p ? d + res[p][i] : d;
            }
            store_chunk<T>(gx, lane + p * LANES, n, g[p]);
        }
    }
    if constexpr (SUMS) {
        float* out = partial + (int64_t)blockIdx.x * 2 * n;
        if constexpr (kGroups == 1) {
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int k = (lane + p * LANES) * V + i;
                    if (k < n) {
                        out[k] = sg[p][i];
                        out[n + k] = sb[p][i];
                    }
                }
        } else {
            // the groups' sums in LDS, joined in the order of the groups
            __shared__ float t[kGroups][LANES * V];
#pragma unroll
            for (int q = 0; q < 2 * PIECES; ++q) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V; ++i) t[group][lane * V + i] = q & 1 ? sb[q / 2][i] : sg[q / 2][i];
                __syncthreads();
                for (int c = threadIdx.x; c < LANES * V; c += threads_of(LANES)) {
                    const int k = (q / 2) * LANES * V + c;
                    float v = t[0][c];
                    for (int w = 1; w < kGroups; ++w) v += t[w][c];
                    if (k < n) out[(q & 1) * n + k] = v;
                }
            }
        }
    }
}

// The sums of `blocks` rows of n (and, for `second`, n more) columns: 32
// columns a workgroup, 32 threads a column, each over every 32nd row with eight
// loads in flight, joined in order. 1024 rows of 256 columns take 4 us; with
// one load in flight at a time they took 33.
__global__ void __launch_bounds__(1024) column_sums_kernel(const float* partial, int blocks, int64_t n, int64_t width,
                                                           float* first, float* second) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t k = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (k < width) {
        int b = part;
        for (; b + 7 * 32 < blocks; b += 8 * 32) {
            float u[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) u[q] = partial[(int64_t)(b + 32 * q) * width + k];
#pragma unroll
            for (int q = 0; q < 8; ++q) v += u[q];
        }
        for (; b < blocks; b += 32) v += partial[(int64_t)b * width + k];
    }
    s[part][lane] = v;
    __syncthreads();
    if (part != 0 || k >= width) return;
    for (int q = 1; q < 32; ++q) v += s[q][lane];
    if (k < n) {
        if (first) first[k] = v;
    } else if (second) {
        second[k - n] = v;
    }
}

// Calls f with the lanes and pieces that hold a row of n elements. A wave
// takes up to 256 chunks (4 KB): more than one row a wave below 64. Workgroups
// per row above: 256 threads up to 16 KB, 1024 up to 32 KB (with four chunks a
// thread there the backward's sums no longer fit its registers).
template <class T, class F>
bool by_width(int64_t n, F f) {
    const int64_t chunks = (n + kChunk<T> - 1) / kChunk<T>;
    if (chunks <= 4) f(Constant<4>{}, Constant<1>{});
    else if (chunks <= 8) f(Constant<8>{}, Constant<1>{});
    else if (chunks <= 16) f(Constant<16>{}, Constant<1>{});
    else if (chunks <= 32) f(Constant<32>{}, Constant<1>{});
    else if (chunks <= 64) f(Constant<64>{}, Constant<1>{});
    else if (chunks <= 128) f(Constant<64>{}, Constant<2>{});
    else if (chunks <= 256) f(Constant<64>{}, Constant<4>{});
    else if (chunks <= 1024) f(Constant<256>{}, Constant<4>{});
    else if (chunks <= 2048) f(Constant<1024>{}, Constant<2>{});
    else return false;
    return true;
}

// ---- rows over 32 KB: the row is read again from memory for each pass, one
// workgroup a row; the column sums run one workgroup a column, whose threads take
// an element of each row, so that a cache line is asked for by 32 or 64 of them.
// 1000 x 20000 halves: forward 40 us, backward 225, where their 80 and 120 MB take
// 16 and 24; kept simple, for widths past any network's that this package makes.
// A launch of 2^32 threads or more loses what is above without an error:
// workgroups take further rows.
constexpr int kWide = 1024;

template <class T>
__global__ void __launch_bounds__(kWide) wide_forward_kernel(LayerNormForward a) {
    __shared__ float s[2 * kWide / 64];
    int turn = 0;
    const int64_t n = a.x.cols;
    for (int64_t r = blockIdx.x; r < a.x.rows; r += gridDim.x) {
        const T* x = (const T*)a.x.p + r * a.x.stride;
        T* y = (T*)a.y.p + r * a.y.stride;
        float v[1] = {0.0f};
        for (int64_t k = threadIdx.x; k < n; k += kWide) v[0] += (float)x[k];
        group_sum<kWide>(v, s, turn);
        const float mean = v[0] / (float)n;
        v[0] = 0.0f;
        for (int64_t k = threadIdx.x; k < n; k += kWide) {
            const float d = (float)x[k] - mean;
            v[0] = fmaf(d, d, v[0]);
        }
        group_sum<kWide>(v, s, turn);
        const float rstd = 1.0f / sqrtf(v[0] / (float)n + a.eps);
        for (int64_t k = threadIdx.x; k < n; k += kWide) {
            const float h = ((float)x[k] - mean) * rstd;
            y[k] = (T)fmaf(h, a.gamma ? a.gamma[k] : 1.0f, a.beta ? a.beta[k] : 0.0f);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kWide) wide_backward_kernel(LayerNormBackward a) {
    __shared__ float s[4 * kWide / 64];
    int turn = 0;
    const int64_t n = a.x.cols;
    for (int64_t r = blockIdx.x; r < a.x.rows; r += gridDim.x) {
        const T* x = (const T*)a.x.p + r * a.x.stride;
        const T* gy = (const T*)a.grad_y.p + r * a.grad_y.stride;
        const T* res = a.residual.p ? (const T*)a.residual.p + r * a.residual.stride : nullptr;
        T* gx = (T*)a.grad_x.p + r * a.grad_x.stride;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float v[2] = {0.0f, 0.0f};
        for (int64_t k = threadIdx.x; k < n; k += kWide) {
            const float h = ((float)x[k] - mean) * rstd, g = (float)gy[k] * (a.gamma ? a.gamma[k] : 1.0f);
            v[0] += g;
            v[1] = fmaf(g, h, v[1]);
        }
        group_sum<kWide>(v, s, turn);
        const float c1 = v[0] / (float)n, c2 = v[1] / (float)n;
        for (int64_t k = threadIdx.x; k < n; k += kWide) {
            const float h = ((float)x[k] - mean) * rstd, g = (float)gy[k] * (a.gamma ? a.gamma[k] : 1.0f);
            const float d = rstd * fmaf(-h, c2, g - c1);
            gx[k] = (T)(res ? d + (float)res[k] : d);
        }
    }
}

template <class T>
__global__ void __launch_bounds__(256) wide_columns_kernel(LayerNormBackward a) {
    __shared__ float s[4 * 256 / 64];
    int turn = 0;
    const int64_t k = blockIdx.x;
    float v[2] = {0.0f, 0.0f};
    for (int64_t r = threadIdx.x; r < a.x.rows; r += 256) {
        const float g = (float)((const T*)a.grad_y.p)[r * a.grad_y.stride + k];
        v[0] += g;
        v[1] = fmaf(g, ((float)((const T*)a.x.p)[r * a.x.stride + k] - a.mean[r]) * a.rstd[r], v[1]);
    }
    group_sum<256>(v, s, turn);
    if (threadIdx.x == 0) {
        if (a.grad_gamma) a.grad_gamma[k] = v[1];
        if (a.grad_beta) a.grad_beta[k] = v[0];
    }
}

// Workgroups of a backward with column sums: each writes 8 n bytes of sums, so
// no more than fill the card four times over, and at least two rows a group
// (6007 x 323 floats: the kernel 8.9 us and the sums 5.6 with two, 12.1 and 3.8
// with eight).
int backward_blocks(int64_t rows, int groups) {
    const int64_t want = (rows + 2 * groups - 1) / (2 * groups);
    return (int)(want < 1024 ? want : 1024);
}

}  // namespace

void launch_column_sums(const float* partial, int blocks, int64_t n, int64_t width, float* first, float* second,
                        hipStream_t s) {
    column_sums_kernel<<<(unsigned)((width + 31) / 32), 1024, 0, s>>>(partial, blocks, n, width, first, second);
}

// Workgroups for rows over 32 KB (also for tests).
int64_t layer_norm_wide_blocks(int64_t rows) { return rows < 65536 ? rows : 65536; }

size_t layer_norm_backward_workspace(const LayerNormBackward& a) {
    if (!a.grad_gamma && !a.grad_beta) return 0;
    size_t bytes = 0;
    by_dtype(a.dtype, [&](auto t) {
        by_width<decltype(t)>(a.x.cols, [&](auto lanes, auto) {
            constexpr int kLanes = decltype(lanes)::value;
            bytes = sizeof(float) * 2 * (size_t)a.x.cols *
                    (size_t)backward_blocks(a.x.rows, threads_of(kLanes) / kLanes);
        });
    });
    return bytes;
}

int launch_layer_norm_forward(const LayerNormForward& a, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        const bool held = by_width<T>(a.x.cols, [&](auto lanes, auto pieces) {
            constexpr int kLanes = decltype(lanes)::value, kThreads = threads_of(kLanes);
            const int64_t want = (a.x.rows * kLanes + kThreads - 1) / kThreads;
            const unsigned blocks = (unsigned)(want < 2048 ? want : 2048);
            forward_kernel<T, kLanes, decltype(pieces)::value><<<blocks, kThreads, 0, s>>>(a);
        });
        if (!held) wide_forward_kernel<T><<<(unsigned)layer_norm_wide_blocks(a.x.rows), kWide, 0, s>>>(a);
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_layer_norm_backward(const LayerNormBackward& a, void* workspace, hipStream_t s) {
    const bool sums = a.grad_gamma || a.grad_beta;
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        const bool held = by_width<T>(a.x.cols, [&](auto lanes, auto pieces) {
            constexpr int kLanes = decltype(lanes)::value, kThreads = threads_of(kLanes);
            constexpr int kPieces = decltype(pieces)::value;
            if (!sums) {
                const int64_t want = (a.x.rows * kLanes + kThreads - 1) / kThreads;
                const unsigned blocks = (unsigned)(want < 2048 ? want : 2048);
                if (blocks && a.grad_x.p)
                    backward_kernel<T, kLanes, kPieces, false><<<blocks, kThreads, 0, s>>>(a, nullptr);
                return;
            }
            const int blocks = backward_blocks(a.x.rows, kThreads / kLanes);
            if (blocks)
                backward_kernel<T, kLanes, kPieces, true><<<blocks, kThreads, 0, s>>>(a, (float*)workspace);
            launch_column_sums((const float*)workspace, blocks, a.x.cols, 2 * a.x.cols, a.grad_gamma, a.grad_beta, s);
        });
        if (held) return;
        // grad_x may take grad_y's place: its column sums come first
        if (sums) wide_columns_kernel<T><<<(unsigned)a.x.cols, 256, 0, s>>>(a);
        if (a.grad_x.p && a.x.rows) wide_backward_kernel<T><<<(unsigned)layer_norm_wide_blocks(a.x.rows), kWide, 0, s>>>(a);
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
