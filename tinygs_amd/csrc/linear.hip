// Linear layers: y = act(x w^T + bias) + residual and its gradients.
//
// One tiled product serves all three: C(i, j) = sum over k of A(i, k) B(j, k)
// with the operands read through strides, 64 x 64 outputs and 16 of k per step,
// 4 x 4 outputs per thread, products and sums in float.
#include "network.h"

namespace tgs {

namespace {

constexpr int kTileEdge = 64;
constexpr int kDepth = 16;

// An operand element (r, k) at p + r * sr + k * sk; with a second array (z of
// the same strides) it is p's element times act'(z's).
struct Operand {
    const void* p;
    const void* z;
    int64_t sr, sk;
    int64_t r_size;
};

template <class T, int ACT>
__device__ __forceinline__ float operand_at(const Operand& o, int64_t r, int64_t k, int64_t k_size) {
    if (r >= o.r_size || k >= k_size) return 0.0f;
    const float v = (float)((const T*)o.p)[r * o.sr + k * o.sk];
    if constexpr (ACT != kActNone) return v * activate_slope<ACT>((float)((const T*)o.z)[r * o.sr + k * o.sk]);
    return v;
}

struct Epilogue {
    const float* bias;   // per j
    Mat residual, preact, y;
};

// ACT applies to the output; ACT_A to operand A (its slope).
template <class T, int ACT, int ACT_A>
__global__ void __launch_bounds__(256) product_kernel(Operand a, Operand b, int64_t k_size, Epilogue e) {
    __shared__ float sa[kDepth][kTileEdge + 4], sb[kDepth][kTileEdge + 4];
    const int t = threadIdx.x, ti = t >> 4, tj = t & 15;
    const int64_t i0 = (int64_t)blockIdx.x * kTileEdge, j0 = (int64_t)blockIdx.y * kTileEdge;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < k_size; k0 += kDepth) {
        for (int q = t; q < kTileEdge * kDepth; q += 256) {
            const int r = q / kDepth, k = q % kDepth;
            float v = operand_at<T, ACT_A>(a, i0 + r, k0 + k, k_size);
            if constexpr (ACT_A != kActNone) v = (float)(T)v;
            sa[k][r] = v;
            sb[k][r] = operand_at<T, kActNone>(b, j0 + r, k0 + k, k_size);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
            for (int u = 0; u < 4; ++u)
                for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(sa[k][ti * 4 + u], sb[k][tj * 4 + v], acc[u][v]);
        __syncthreads();
    }
    for (int u = 0; u < 4; ++u)
        for (int v = 0; v < 4; ++v) {
            const int64_t i = i0 + ti * 4 + u, j = j0 + tj * 4 + v;
            if (i >= e.y.rows || j >= e.y.cols) continue;
            float z = acc[u][v] + (e.bias ? e.bias[j] : 0.0f);
            if (e.preact.p) ((T*)e.preact.p)[i * e.preact.stride + j] = (T)z;
            z = activate<ACT>(z);
            if (e.residual.p) z += (float)((const T*)e.residual.p)[i * e.residual.stride + j];
            ((T*)e.y.p)[i * e.y.stride + j] = (T)z;
        }
}

template <class T, int ACT>
__global__ void __launch_bounds__(256) bias_gradient_kernel(Mat gy, Mat z, float* out) {
    const int64_t j = blockIdx.x;
    double acc = 0.0;
    for (int64_t r = threadIdx.x; r < gy.rows; r += 256) {
        float v = (float)((const T*)gy.p)[r * gy.stride + j];
        if constexpr (ACT != kActNone) v *= activate_slope<ACT>((float)((const T*)z.p)[r * z.stride + j]);
        acc += v;
    }
    __shared__ double s[256];
    s[threadIdx.x] = acc;
    __syncthreads();
    for (int n = 128; n > 0; n >>= 1) {
        if ((int)threadIdx.x < n) s[threadIdx.x] += s[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[j] = (float)s[0];
}

dim3 grid_of(int64_t i, int64_t j) {
    return dim3((unsigned)((i + kTileEdge - 1) / kTileEdge), (unsigned)((j + kTileEdge - 1) / kTileEdge));
}

template <class T, int ACT>
void forward(const LinearForward& a, hipStream_t s) {
    Operand x{a.x.p, nullptr, a.x.stride, 1, a.x.rows}, w{a.w.p, nullptr, a.w.stride, 1, a.w.rows};
    product_kernel<T, ACT, kActNone><<<grid_of(a.y.rows, a.y.cols), 256, 0, s>>>(x, w, a.x.cols,
                                                                               {a.bias, a.residual, a.preact, a.y});
}

template <class T, int ACT>
void backward(const LinearBackward& a, hipStream_t s) {
    const Mat& g = a.grad_y;
    if (a.grad_x.p && a.grad_x.rows) {
        Operand dz{g.p, a.preact.p, g.stride, 1, g.rows}, w{a.w.p, nullptr, 1, a.w.stride, a.w.cols};
        product_kernel<T, kActNone, ACT><<<grid_of(a.grad_x.rows, a.grad_x.cols), 256, 0, s>>>(
            dz, w, g.cols, {nullptr, {}, {}, a.grad_x});
    }
    if (a.grad_w.p) {
        Operand dz{g.p, a.preact.p, 1, g.stride, g.cols}, x{a.x.p, nullptr, 1, a.x.stride, a.x.cols};
        product_kernel<T, kActNone, ACT><<<grid_of(a.grad_w.rows, a.grad_w.cols), 256, 0, s>>>(
            dz, x, g.rows, {nullptr, {}, {}, a.grad_w});
    }
    if (a.grad_bias) bias_gradient_kernel<T, ACT><<<(unsigned)g.cols, 256, 0, s>>>(g, a.preact, a.grad_bias);
}

}  // namespace

size_t linear_backward_workspace(const LinearBackward&) { return 0; }

int launch_linear_forward(const LinearForward& a, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) {
        by_activation(a.activation, [&](auto act) { forward<decltype(t), decltype(act)::value>(a, s); });
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_linear_backward(const LinearBackward& a, void*, hipStream_t s) {
    by_dtype(a.dtype, [&](auto t) {
        by_activation(a.activation, [&](auto act) { backward<decltype(t), decltype(act)::value>(a, s); });
    });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
