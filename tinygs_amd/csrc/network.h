// What the attribute network's operators share: element types, activations,
// matrix views and the launchers of linear.hip, layer_norm.hip and muon.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "status.h"

namespace tgs {

// A matrix of a launch: row r at p + r * stride, `cols` elements.
struct Mat {
    void* p = nullptr;
    int64_t rows = 0;
    int64_t cols = 0;
    int64_t stride = 0;
};

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static constexpr int kDtype = TGS_DTYPE_FLOAT32;
};
template <>
struct Elem<_Float16> {
    static constexpr int kDtype = TGS_DTYPE_FLOAT16;
};
template <>
struct Elem<__bf16> {
    static constexpr int kDtype = TGS_DTYPE_BFLOAT16;
};

// Calls f with a value of the element type / with an integral constant.
template <class F>
void by_dtype(int dtype, F f) {
    if (dtype == TGS_DTYPE_FLOAT32) f(float{});
    else if (dtype == TGS_DTYPE_FLOAT16) f(_Float16{});
    else f(__bf16{});
}
template <int N>
struct Constant {
    static constexpr int value = N;
};
template <class F>
void by_activation(int activation, F f) {
    if (activation == 1) f(Constant<1>{});
    else if (activation == 2) f(Constant<2>{});
    else if (activation == 3) f(Constant<3>{});
    else f(Constant<0>{});
}

enum Activation { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// 1 / (1 + 2^t): the logistic of v for t = -v log2 e. Off by |t| 2^-24 of
// itself (t's rounding) and a few units of the last place; where 2^t overflows
// the reciprocal is 0, the limit. A step that put t's rounding back made the
// activations half as long again and moved no stored half.
__device__ __forceinline__ float logistic2(float t) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kGelu1 = 1.5957691216057308f;    // 2 sqrt(2 / pi): 1 + tanh(u) = 2 logistic(2 u)
constexpr float kGelu3 = 0.071354816272600256f;  // 2 sqrt(2 / pi) 0.044715

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == kActRelu) return z < 0.0f ? 0.0f : z;   // NaN stays NaN
    if constexpr (ACT == kActSilu) return z * logistic2(-kLog2E * z);
    if constexpr (ACT == kActGelu) return z * logistic2(z * fmaf(-kLog2E * kGelu3, z * z, -kLog2E * kGelu1));
    return z;
}

// act'(z) = p + z p (1 - p) (d/dz of p's argument). The second term is zero in
// 32 bits well inside the bounds on z and z^2, which keep it from becoming
// 0 * infinity at either end (a preact that left its type's range is infinite);
// p itself keeps a NaN.
template <int ACT>
__device__ __forceinline__ float activate_slope(float z) {
    if constexpr (ACT == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    if constexpr (ACT == kActSilu) {
        const float p = logistic2(-kLog2E * z);
        return fmaf(__builtin_amdgcn_fmed3f(z, -100.0f, 100.0f) * p, 1.0f - p, p);
    }
    if constexpr (ACT == kActGelu) {
        const float q = fminf(z * z, 900.0f);
        const float p = logistic2(z * fmaf(-kLog2E * kGelu3, q, -kLog2E * kGelu1));
        return fmaf(__builtin_amdgcn_fmed3f(z, -30.0f, 30.0f) * (p * (1.0f - p)), fmaf(3.0f * kGelu3, q, kGelu1), p);
    }
    return 1.0f;
}

// ---- linear.hip
struct LinearForward {
    Mat x, w, residual, preact, y;   // residual.p, preact.p may be NULL
    const float* bias;               // may be NULL
    int activation;
    int dtype;
};
struct LinearBackward {
    Mat grad_y, x, w, preact, grad_x, grad_w;   // grad_x.p, grad_w.p may be NULL
    float* grad_bias;                           // may be NULL
    int activation;
    int dtype;
};
size_t linear_backward_workspace(const LinearBackward& a);
size_t linear_forward_workspace(const LinearForward& a);
int launch_linear_forward(const LinearForward& a, void* workspace, hipStream_t s);
int launch_linear_backward(const LinearBackward& a, void* workspace, hipStream_t s);

// ---- linear_few.hip: a few rows
bool linear_forward_is_few(const LinearForward& a);
void launch_linear_few(const LinearForward& a, hipStream_t s);

// ---- linear_rows.hip: many rows of a narrow layer
bool linear_forward_by_rows(const LinearForward& a);
void launch_linear_rows(const LinearForward& a, hipStream_t s);

// ---- linear_narrow.hip: the gradients of a layer whose rows are at most 512
// bytes. Leaves `splits` sets of float sums, each out x in of grad_w and then
// out of grad_bias.
bool linear_backward_is_narrow(const LinearBackward& a);
int narrow_backward_splits(const LinearBackward& a);
void launch_narrow_backward(const LinearBackward& a, float* partial, hipStream_t s);

// ---- layer_norm.hip
struct LayerNormForward {
    Mat x, y;
    const float *gamma, *beta;   // may be NULL
    float eps;
    float *mean, *rstd;          // may be NULL
    int dtype;
};
struct LayerNormBackward {
    Mat grad_y, x, residual, grad_x;            // residual.p, grad_x.p may be NULL
    const float *gamma, *mean, *rstd;           // gamma may be NULL
    float *grad_gamma, *grad_beta;              // may be NULL
    int dtype;
};
size_t layer_norm_backward_workspace(const LayerNormBackward& a);
// Column sums of `blocks` rows of `width` floats: the first n to `first`, the
// others to `second` (each may be NULL), in a fixed order.
void launch_column_sums(const float* partial, int blocks, int64_t n, int64_t width, float* first, float* second,
                        hipStream_t s);
int launch_layer_norm_forward(const LayerNormForward& a, hipStream_t s);
int launch_layer_norm_backward(const LayerNormBackward& a, void* workspace, hipStream_t s);

// ---- muon.hip
constexpr float kNewtonSchulzA = 3.4445f, kNewtonSchulzB = -4.7750f, kNewtonSchulzC = 2.0315f;

// A matrix of the step as the kernels read it, and where its work starts in
// the launches over all matrices (first, by phase).
enum { kMuonPatches = 0, kMuonGram = 1, kMuonUpdate = 2, kMuonSquare = 3 };
struct MuonPart {
    Mat w, g, m, c;              // weights, gradient, momentum, copy (c.p may be NULL)
    int64_t side, length;        // X is side x length, side <= length
    int64_t x_cols, x_stride;    // of X's rows: hi and lo, in halves
    int64_t g_cols, g_stride;    // of the Gram matrix's and the polynomial's
    _Float16 *x[2], *gram, *poly;
    float shape;                 // sqrt(max(1, rows / cols))
    int tall;                    // X is the transpose
    uint32_t first[3];
};
struct MuonPlan {
    uint32_t patches;      // workgroups of the element passes
    uint32_t tiles[2];     // of the products with side x side and side x length outputs
    bool large[2];         // whether those are the large tiles
    bool fits;             // whether the counts fit a launch
    int64_t sums_at, parts_at, firsts_at, bytes;   // in the workspace; firsts: the parts' first[0], then [1], [2]
};
struct MuonStep {
    float momentum, grad_scale;   // grad_scale = (1 - momentum) scale
    float keep, lr;               // 1 - lr weight_decay; lr
    float epsilon;
    int nesterov, iterations;
    int grad_dtype, copy_dtype;
};
// Fills the parts' shapes and places (offsets from the workspace's start,
// which place_muon turns into addresses) from their matrices.
MuonPlan plan_muon(MuonPart* parts, int count);
void place_muon(MuonPart* parts, int count, unsigned char* workspace);
int launch_muon_step(const MuonPlan& plan, int count, const MuonStep& p, unsigned char* workspace, hipStream_t s);
int launch_zero_matrix(const Mat& m, hipStream_t s);

}  // namespace tgs
