// Muon's update of one matrix after another: momentum, the Newton-Schulz
// steps on the normalised update, the weights.
//
// X is kept with its shorter side as rows (the transpose of a tall matrix), so
// that X X^T is the smaller of the two Gram matrices.
#include "network.h"

namespace tgs {

namespace {

constexpr int kNormBlocks = 64;

template <class G>
__global__ void __launch_bounds__(256) momentum_kernel(MuonMatrix a, MuonStep p, float* x, double* partial) {
    const bool tall = a.w.rows > a.w.cols;
    const int64_t n = a.w.rows * a.w.cols;
    double sum = 0.0;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256) {
        const int64_t r = q / a.w.cols, k = q % a.w.cols;
        const float g = (float)((const G*)a.g.p)[r * a.g.stride + k] * p.grad_scale;
        float* pm = (float*)a.m.p + r * a.m.stride + k;
        const float m = fmaf(p.momentum, *pm, g);
        *pm = m;
        const float u = p.nesterov ? fmaf(p.momentum, m, g) : m;
        x[tall ? k * a.w.rows + r : q] = u;
        sum += (double)u * (double)u;
    }
    __shared__ double s[256];
    s[threadIdx.x] = sum;
    __syncthreads();
    for (int k = 128; k > 0; k >>= 1) {
        if ((int)threadIdx.x < k) s[threadIdx.x] += s[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) partial[blockIdx.x] = s[0];
}

__global__ void __launch_bounds__(256) normalise_kernel(float* x, int64_t n, const double* partial, float epsilon) {
    double sum = 0.0;
    for (int k = 0; k < kNormBlocks; ++k) sum += partial[k];
    const double inv = 1.0 / fmax(sqrt(sum), (double)epsilon);
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256)
        x[q] = (float)((double)x[q] * inv);
}

// out(i, j) = alpha sum over k of a(i, k) b(j, k) + beta c(i, j)
__global__ void __launch_bounds__(256) product_kernel(const float* a, int64_t as, const float* b, int64_t bs,
                                                      int64_t bk, const float* c, float* out, int64_t rows,
                                                      int64_t cols, int64_t depth, float alpha, float beta) {
    __shared__ float sa[32][33], sb[32][33];
    const int ti = threadIdx.x >> 5, tj = threadIdx.x & 31;
    const int64_t i0 = (int64_t)blockIdx.x * 32, j0 = (int64_t)blockIdx.y * 32;
    float acc[4] = {};
    for (int64_t k0 = 0; k0 < depth; k0 += 32) {
        for (int u = 0; u < 4; ++u) {
            const int r = ti + 8 * u;
            const int64_t k = k0 + tj;
            sa[r][tj] = i0 + r < rows && k < depth ? a[(i0 + r) * as + k] : 0.0f;
            sb[r][tj] = j0 + r < cols && k < depth ? b[(j0 + r) * bs + k * bk] : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < 32; ++k)
            for (int u = 0; u < 4; ++u) acc[u] = fmaf(sa[ti + 8 * u][k], sb[tj][k], acc[u]);
        __syncthreads();
    }
    for (int u = 0; u < 4; ++u) {
        const int64_t i = i0 + ti + 8 * u, j = j0 + tj;
        if (i < rows && j < cols)
            out[i * cols + j] = fmaf(alpha, acc[u], c ? beta * c[i * cols + j] : 0.0f);
    }
}

template <class C>
__global__ void __launch_bounds__(256) update_kernel(MuonMatrix a, const float* x, float keep, float step) {
    const bool tall = a.w.rows > a.w.cols;
    const int64_t n = a.w.rows * a.w.cols;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256) {
        const int64_t r = q / a.w.cols, k = q % a.w.cols;
        float* w = (float*)a.w.p + r * a.w.stride + k;
        const float v = fmaf(-step, x[tall ? k * a.w.rows + r : q], keep * *w);
        *w = v;
        if (a.c.p) ((C*)a.c.p)[r * a.c.stride + k] = (C)v;
    }
}

__global__ void __launch_bounds__(256) zero_kernel(Mat m) {
    const int64_t n = m.rows * m.cols;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256)
        ((float*)m.p)[q / m.cols * m.stride + q % m.cols] = 0.0f;
}

}  // namespace

size_t muon_workspace(const MuonMatrix* mats, int count) {
    size_t most = 0;
    for (int i = 0; i < count; ++i) {
        const int64_t n = mats[i].w.rows * mats[i].w.cols;
        const int64_t side = mats[i].w.rows < mats[i].w.cols ? mats[i].w.rows : mats[i].w.cols;
        const size_t need = sizeof(double) * kNormBlocks + sizeof(float) * (size_t)(2 * n + 2 * side * side);
        most = need > most ? need : most;
    }
    return most;
}

int launch_muon_step(const MuonMatrix* mats, int count, const MuonStep& p, void* workspace, hipStream_t s) {
    for (int i = 0; i < count; ++i) {
        const MuonMatrix& a = mats[i];
        const bool tall = a.w.rows > a.w.cols;
        const int64_t n = a.w.rows * a.w.cols, side = tall ? a.w.cols : a.w.rows, length = n / side;
        double* partial = (double*)workspace;
        float* x = (float*)(partial + kNormBlocks);
        float *y = x + n, *gram = y + n, *poly = gram + side * side;
        by_dtype(p.grad_dtype, [&](auto t) {
            momentum_kernel<decltype(t)><<<kNormBlocks, 256, 0, s>>>(a, p, x, partial);
        });
        normalise_kernel<<<256, 256, 0, s>>>(x, n, partial, p.epsilon);
        const dim3 small((unsigned)((side + 31) / 32), (unsigned)((side + 31) / 32));
        const dim3 wide((unsigned)((side + 31) / 32), (unsigned)((length + 31) / 32));
        for (int k = 0; k < p.iterations; ++k) {
            product_kernel<<<small, 256, 0, s>>>(x, length, x, length, 1, nullptr, gram, side, side, length, 1.f, 0.f);
            product_kernel<<<small, 256, 0, s>>>(gram, side, gram, side, 1, gram, poly, side, side, side,
                                                 kNewtonSchulzC, kNewtonSchulzB);
            product_kernel<<<wide, 256, 0, s>>>(poly, side, x, 1, length, x, y, side, length, side, 1.f,
                                                kNewtonSchulzA);
            float* f = x;
            x = y;
            y = f;
        }
        const float step = p.lr * (tall ? sqrtf((float)a.w.rows / (float)a.w.cols) : 1.0f);
        by_dtype(p.copy_dtype, [&](auto t) {
            update_kernel<decltype(t)><<<256, 256, 0, s>>>(a, x, p.keep, step);
        });
    }
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

int launch_zero_matrix(const Mat& m, hipStream_t s) {
    zero_kernel<<<256, 256, 0, s>>>(m);
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
