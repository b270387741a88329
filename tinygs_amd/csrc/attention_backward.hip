// The gradients of attention.hip from its out and lse: p = exp(s - lse),
// delta = sum of do o over a head, dv = p^T do, ds = p (do v^T - delta),
// dq = scale ds k, dk = scale ds^T q.
#include <math.h>

#include "network.h"

namespace tgs {

namespace {

constexpr int kMaxHead = 128;

template <class T>
__device__ __forceinline__ const T* at(const Mat& m, int64_t r, int c) {
    return (const T*)m.p + r * m.stride + c;
}

// delta[row, head]
template <class T>
__global__ void __launch_bounds__(256) delta_kernel(AttentionBackward b, float* delta) {
    const Attention& a = b.a;
    const int64_t n = a.q.rows * a.heads;
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < n; k += (int64_t)gridDim.x * 256) {
        const int64_t r = k / a.heads;
        const int h = (int)(k % a.heads);
        const T *x = at<T>(b.grad_out, r, h * a.head), *y = at<T>(a.out, r, h * a.head);
        float v = 0.0f;
        for (int c = 0; c < a.head; ++c) v = fmaf((float)x[c], (float)y[c], v);
        delta[k] = v;
    }
}

// One wave a row and head, as the forward's.
template <class T>
__global__ void __launch_bounds__(64) grad_q_kernel(AttentionBackward b, const float* delta) {
    __shared__ float q[kMaxHead], go[kMaxHead], ds[64];
    const Attention& a = b.a;
    const int lane = threadIdx.x, d = a.head, h = blockIdx.y, g = h / (a.heads / a.kv_heads);
    for (int64_t r = blockIdx.x; r < a.q.rows; r += gridDim.x) {
        const int64_t e = r / a.queries;
        const uint8_t* mask = a.mask ? a.mask + e * a.mask_stride : nullptr;
        for (int c = lane; c < d; c += 64) {
            q[c] = (float)*at<T>(a.q, r, h * d + c);
            go[c] = (float)*at<T>(b.grad_out, r, h * d + c);
        }
        __syncthreads();
        const float lse = a.lse[r * a.lse_row_step + h * a.lse_head_step], del = delta[r * a.heads + h];
        float o[2] = {0.0f, 0.0f};
        for (int64_t j0 = 0; j0 < a.states; j0 += 64) {
            const int64_t j = j0 + lane;
            float v = 0.0f;
            if (j < a.states && (!mask || mask[j]) && lse != -INFINITY) {
                const T *k = at<T>(a.k, e * a.states + j, g * d), *w = at<T>(a.v, e * a.states + j, g * d);
                float s = 0.0f, dp = 0.0f;
                for (int c = 0; c < d; ++c) {
                    s = fmaf(q[c], (float)k[c], s);
                    dp = fmaf(go[c], (float)w[c], dp);
                }
                v = expf(s * a.scale - lse) * (dp - del) * a.scale;
            }
            ds[lane] = v;
            __syncthreads();
            for (int n = 0; n < 2; ++n) {
                const int c = lane + 64 * n;
                if (c < d)
                    for (int k = 0; k < 64 && j0 + k < a.states; ++k)
                        if (!mask || mask[j0 + k]) o[n] = fmaf(ds[k], (float)*at<T>(a.k, e * a.states + j0 + k, g * d + c), o[n]);
            }
            __syncthreads();
        }
        for (int n = 0; n < 2; ++n)
            if (lane + 64 * n < d) ((T*)b.grad_q.p)[r * b.grad_q.stride + h * d + lane + 64 * n] = (T)o[n];
    }
}

// One wave a state and head of the states: a lane takes a row of 64, then a column or two.
template <class T>
__global__ void __launch_bounds__(64) grad_kv_kernel(AttentionBackward b, const float* delta) {
    __shared__ float k[kMaxHead], v[kMaxHead], ps[64], ds[64];
    const Attention& a = b.a;
    const int lane = threadIdx.x, d = a.head, g = blockIdx.y, shared = a.heads / a.kv_heads;
    for (int64_t j = blockIdx.x; j < a.k.rows; j += gridDim.x) {
        const int64_t e = j / a.states;
        const bool exists = !a.mask || a.mask[e * a.mask_stride + j % a.states];
        for (int c = lane; c < d; c += 64) {
            k[c] = (float)*at<T>(a.k, j, g * d + c);
            v[c] = (float)*at<T>(a.v, j, g * d + c);
        }
        __syncthreads();
        float gk[2] = {0.0f, 0.0f}, gv[2] = {0.0f, 0.0f};
        for (int h = g * shared; exists && h < (g + 1) * shared; ++h)
            for (int64_t r0 = e * a.queries; r0 < (e + 1) * a.queries; r0 += 64) {
                const int64_t r = r0 + lane;
                float p = 0.0f, x = 0.0f;
                if (r < (e + 1) * a.queries && a.lse[r * a.lse_row_step + h * a.lse_head_step] != -INFINITY) {
                    const T *q = at<T>(a.q, r, h * d), *go = at<T>(b.grad_out, r, h * d);
                    float s = 0.0f, dp = 0.0f;
                    for (int c = 0; c < d; ++c) {
                        s = fmaf(k[c], (float)q[c], s);
                        dp = fmaf(v[c], (float)go[c], dp);
                    }
                    p = expf(s * a.scale - a.lse[r * a.lse_row_step + h * a.lse_head_step]);
                    x = p * (dp - delta[r * a.heads + h]) * a.scale;
                }
                ps[lane] = p;
                ds[lane] = x;
                __syncthreads();
                for (int n = 0; n < 2; ++n) {
                    const int c = lane + 64 * n;
                    if (c < d)
                        for (int i = 0; i < 64 && r0 + i < (e + 1) * a.queries; ++i) {
                            gv[n] = fmaf(ps[i], (float)*at<T>(b.grad_out, r0 + i, h * d + c), gv[n]);
                            gk[n] = fmaf(ds[i], (float)*at<T>(a.q, r0 + i, h * d + c), gk[n]);
                        }
                }
                __syncthreads();
            }
        for (int n = 0; n < 2; ++n)
            if (lane + 64 * n < d) {
                const int c = g * d + lane + 64 * n;
                if (b.grad_k.p) ((T*)b.grad_k.p)[j * b.grad_k.stride + c] = (T)gk[n];
                if (b.grad_v.p) ((T*)b.grad_v.p)[j * b.grad_v.stride + c] = (T)gv[n];
            }
        __syncthreads();
    }
}

}  // namespace

size_t attention_backward_workspace(const AttentionBackward& b) { return sizeof(float) * (size_t)(b.a.q.rows * b.a.heads); }

int launch_attention_backward(const AttentionBackward& b, void* workspace, hipStream_t s) {
    const Attention& a = b.a;
    float* delta = (float*)workspace;
    const auto grid = [](int64_t n, int64_t most) { return (unsigned)(n < most ? n : most); };
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.q.rows) {
            delta_kernel<T><<<grid((a.q.rows * a.heads + 255) / 256, 4096), 256, 0, s>>>(b, delta);
            if (b.grad_q.p) grad_q_kernel<T><<<dim3(grid(a.q.rows, (1 << 20) / a.heads), (unsigned)a.heads), 64, 0, s>>>(b, delta);
        }
        if (a.k.rows && (b.grad_k.p || b.grad_v.p))
            grad_kv_kernel<T><<<dim3(grid(a.k.rows, (1 << 20) / a.kv_heads), (unsigned)a.kv_heads), 64, 0, s>>>(b, delta);
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
