// Layer norm over the rows of a matrix, and its gradients.
//
// One workgroup per row forward; backward one workgroup per row for grad_x and
// one per column for the sums over the rows.
#include "network.h"

namespace tgs {

namespace {

constexpr int kThreads = 256;

__device__ float block_sum(float v, float* s) {
    __syncthreads();
    s[threadIdx.x] = v;
    __syncthreads();
    for (int n = kThreads / 2; n > 0; n >>= 1) {
        if ((int)threadIdx.x < n) s[threadIdx.x] += s[threadIdx.x + n];
        __syncthreads();
    }
    return s[0];
}

template <class T>
__global__ void __launch_bounds__(kThreads) forward_kernel(LayerNormForward a) {
    __shared__ float s[kThreads];
    const int64_t r = blockIdx.x, n = a.x.cols;
    const T* x = (const T*)a.x.p + r * a.x.stride;
    T* y = (T*)a.y.p + r * a.y.stride;
    float v = 0.0f;
    for (int64_t k = threadIdx.x; k < n; k += kThreads) v += (float)x[k];
    const float mean = block_sum(v, s) / (float)n;
    v = 0.0f;
    for (int64_t k = threadIdx.x; k < n; k += kThreads) {
        const float d = (float)x[k] - mean;
        v = fmaf(d, d, v);
    }
    const float rstd = 1.0f / sqrtf(block_sum(v, s) / (float)n + a.eps);
    for (int64_t k = threadIdx.x; k < n; k += kThreads) {
        const float h = ((float)x[k] - mean) * rstd;
        y[k] = (T)fmaf(h, a.gamma ? a.gamma[k] : 1.0f, a.beta ? a.beta[k] : 0.0f);
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = mean;
        if (a.rstd) a.rstd[r] = rstd;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) backward_rows_kernel(LayerNormBackward a) {
    __shared__ float s[kThreads];
    const int64_t r = blockIdx.x, n = a.x.cols;
    const T* x = (const T*)a.x.p + r * a.x.stride;
    const T* gy = (const T*)a.grad_y.p + r * a.grad_y.stride;
    const T* res = a.residual.p ? (const T*)a.residual.p + r * a.residual.stride : nullptr;
    T* gx = (T*)a.grad_x.p + r * a.grad_x.stride;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float sg = 0.0f, sgh = 0.0f;
    for (int64_t k = threadIdx.x; k < n; k += kThreads) {
        const float h = ((float)x[k] - mean) * rstd, g = (float)gy[k] * (a.gamma ? a.gamma[k] : 1.0f);
        sg += g;
        sgh = fmaf(g, h, sgh);
    }
    sg = block_sum(sg, s) / (float)n;
    sgh = block_sum(sgh, s) / (float)n;
    for (int64_t k = threadIdx.x; k < n; k += kThreads) {
        const float h = ((float)x[k] - mean) * rstd, g = (float)gy[k] * (a.gamma ? a.gamma[k] : 1.0f);
        const float d = rstd * (g - sg - h * sgh);
        gx[k] = (T)(d + (res ? (float)res[k] : 0.0f));
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) backward_columns_kernel(LayerNormBackward a) {
    __shared__ float s[kThreads];
    const int64_t k = blockIdx.x;
    float sg = 0.0f, sb = 0.0f;
    for (int64_t r = threadIdx.x; r < a.x.rows; r += kThreads) {
        const float g = (float)((const T*)a.grad_y.p)[r * a.grad_y.stride + k];
        sb += g;
        sg = fmaf(g, ((float)((const T*)a.x.p)[r * a.x.stride + k] - a.mean[r]) * a.rstd[r], sg);
    }
    sg = block_sum(sg, s);
    sb = block_sum(sb, s);
    if (threadIdx.x == 0) {
        if (a.grad_gamma) a.grad_gamma[k] = sg;
        if (a.grad_beta) a.grad_beta[k] = sb;
    }
}

}  // namespace

size_t layer_norm_backward_workspace(const LayerNormBackward&) { return 0; }

int launch_layer_norm_forward(const LayerNormForward& a, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) { forward_kernel<decltype(t)><<<(unsigned)a.x.rows, kThreads, 0, s>>>(a); });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_layer_norm_backward(const LayerNormBackward& a, void*, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.grad_x.p && a.x.rows) backward_rows_kernel<T><<<(unsigned)a.x.rows, kThreads, 0, s>>>(a);
        if (a.grad_gamma || a.grad_beta) backward_columns_kernel<T><<<(unsigned)a.x.cols, kThreads, 0, s>>>(a);
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
