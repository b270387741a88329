// Attention of a network's rows to an encoder's states: for each row and head
// s = scale q k^T over the states that exist, out = softmax(s) v, lse = log sum exp s.
#include <math.h>

#include "network.h"

namespace tgs {

namespace {

constexpr int kMaxHead = 128;

// One wave a row and head: a lane takes a state of 64 for the scores, then a column or two for the sums.
template <class T>
__global__ void __launch_bounds__(64) attention_kernel(Attention a) {
    __shared__ float q[kMaxHead], p[64];
    const int lane = threadIdx.x, d = a.head, h = blockIdx.y, g = h / (a.heads / a.kv_heads);
    for (int64_t r = blockIdx.x; r < a.q.rows; r += gridDim.x) {
        const int64_t b = r / a.queries;
        const uint8_t* mask = a.mask ? a.mask + b * a.mask_stride : nullptr;
        for (int c = lane; c < d; c += 64) q[c] = (float)((const T*)a.q.p)[r * a.q.stride + h * d + c];
        __syncthreads();
        float top = -INFINITY, sum = 0.0f, o[2] = {0.0f, 0.0f};
        for (int64_t j0 = 0; j0 < a.states; j0 += 64) {
            const int64_t j = j0 + lane;
            float s = -INFINITY;
            if (j < a.states && (!mask || mask[j])) {
                const T* k = (const T*)a.k.p + (b * a.states + j) * a.k.stride + g * d;
                s = 0.0f;
                for (int c = 0; c < d; ++c) s = fmaf(q[c], (float)k[c], s);
                s *= a.scale;
            }
            float m = s;
            for (int k = 32; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
            m = fmaxf(m, top);
            const float from = m == -INFINITY ? 0.0f : m;
            const float e = expf(s - from), keep = expf(top - from);
            top = m;
            float t = e;
            for (int k = 32; k > 0; k >>= 1) t += __shfl_xor(t, k, 64);
            sum = fmaf(sum, keep, t);
            p[lane] = e;
            __syncthreads();
            for (int n = 0; n < 2; ++n) {
                const int c = lane + 64 * n;
                o[n] *= keep;
                if (c < d)
                    for (int k = 0; k < 64 && j0 + k < a.states; ++k)
                        if (!mask || mask[j0 + k])
                            o[n] = fmaf(p[k], (float)((const T*)a.v.p)[(b * a.states + j0 + k) * a.v.stride + g * d + c], o[n]);
            }
            __syncthreads();
        }
        for (int n = 0; n < 2; ++n)
            if (lane + 64 * n < d)
                ((T*)a.out.p)[r * a.out.stride + h * d + lane + 64 * n] = (T)(sum == 0.0f ? 0.0f : o[n] / sum);
        if (a.lse && lane == 0) a.lse[r * a.lse_row_step + h * a.lse_head_step] = sum == 0.0f ? -INFINITY : top + logf(sum);
    }
}

}  // namespace

size_t attention_workspace(const Attention&) { return 0; }

int launch_attention(const Attention& a, void*, hipStream_t s) {
    const int64_t most = (1 << 20) / a.heads;   // a launch of 2^32 threads or more loses what is above
    const dim3 grid((unsigned)(a.q.rows < most ? a.q.rows : most), (unsigned)a.heads);
    by_dtype(a.dtype, [&](auto t) { attention_kernel<decltype(t)><<<grid, 64, 0, s>>>(a); });
    TGS_CHECK_LAUNCH();
    return TGS_OK;
}

}  // namespace tgs
