// Entry points of the attribute network's operators (include/tinygs_amd.h):
// argument checks, workspaces and the optimiser's handle.
#include <math.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "device_buffer.h"
#include "network.h"

using namespace tgs;

struct tgs_network {
    DevBuf workspace;
};

struct tgs_muon {
    std::vector<MuonPart> mats;
    std::vector<uint32_t> firsts;
    std::vector<std::pair<int64_t, int64_t>> shapes;   // in the caller's order
    bool on_device = false;   // the workspace holds the matrices' table
    MuonPlan plan{};
    int grad_dtype = TGS_DTYPE_FLOAT32;
    int copy_dtype = TGS_DTYPE_FLOAT32;
    tgs_muon_params p{};
    float global_lr = 1.0f;
    DevBuf workspace;
};

namespace {

constexpr int64_t kMaxStride = (int64_t)1 << 21;
constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 1;

int element_size(int dtype) { return dtype == TGS_DTYPE_FLOAT32 ? 4 : 2; }

int check_matrix(const tgs_matrix* m, const char* name) {
    if (!m) return fail(TGS_ERR_INVALID, "%s is NULL", name);
    if (m->dtype != TGS_DTYPE_FLOAT32 && m->dtype != TGS_DTYPE_FLOAT16 && m->dtype != TGS_DTYPE_BFLOAT16)
        return fail(TGS_ERR_UNSUPPORTED, "%s: dtype %d", name, m->dtype);
    if (m->rows < 0 || m->rows > kMaxRows) return fail(TGS_ERR_INVALID, "%s: %lld rows", name, (long long)m->rows);
    if (m->cols < 1 || m->stride < m->cols || m->stride >= kMaxStride)
        return fail(TGS_ERR_INVALID, "%s: %lld columns at a stride of %lld", name, (long long)m->cols,
                    (long long)m->stride);
    if (m->rows > 0 && !m->data) return fail(TGS_ERR_INVALID, "%s: data is NULL", name);
    if ((uintptr_t)m->data % (uintptr_t)element_size(m->dtype))
        return fail(TGS_ERR_INVALID, "%s: data is not aligned to its elements", name);
    return TGS_OK;
}

// The shape and dtype that the call's other matrices ask for.
int check_shape(const tgs_matrix* m, const char* name, int64_t rows, int64_t cols, int dtype) {
    TGS_TRY(check_matrix(m, name));
    if (m->rows != rows || m->cols != cols)
        return fail(TGS_ERR_INVALID, "%s is %lld x %lld, not %lld x %lld", name, (long long)m->rows,
                    (long long)m->cols, (long long)rows, (long long)cols);
    if (m->dtype != dtype) return fail(TGS_ERR_INVALID, "%s: dtype %d, not %d", name, m->dtype, dtype);
    return TGS_OK;
}

// Whether two matrices share elements. Column ranges of one buffer (of the
// same stride in bytes) interleave without sharing any; a single row, whose own
// stride says nothing, lies in the other's.
bool overlap(const tgs_matrix& a, const tgs_matrix& b) {
    if (!a.rows || !b.rows) return false;
    const int64_t sa = element_size(a.dtype), sb = element_size(b.dtype);
    const uintptr_t a0 = (uintptr_t)a.data, b0 = (uintptr_t)b.data;
    const uintptr_t a1 = a0 + (uintptr_t)(((a.rows - 1) * a.stride + a.cols) * sa);
    const uintptr_t b1 = b0 + (uintptr_t)(((b.rows - 1) * b.stride + b.cols) * sb);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.rows == 1 && b.rows == 1) return true;
    const int64_t pitch = a.rows == 1 ? b.stride * sb : a.stride * sa;
    if (a.rows > 1 && b.rows > 1 && pitch != b.stride * sb) return true;
    const int64_t d = (int64_t)((b0 >= a0 ? b0 - a0 : a0 - b0) % (uintptr_t)pitch);
    const int64_t from = b0 >= a0 ? d : (pitch - d) % pitch;   // b's first column after a's, modulo a row
    return from < a.cols * sa || from + b.cols * sb > pitch;
}

bool same_place(const tgs_matrix& a, const tgs_matrix& b) {
    return a.data == b.data && (a.stride == b.stride || a.rows <= 1) && a.dtype == b.dtype;
}

int check_apart(const tgs_matrix* out, const char* out_name, const tgs_matrix* in, const char* in_name) {
    if (out && in && overlap(*out, *in)) return fail(TGS_ERR_INVALID, "%s overlaps %s", out_name, in_name);
    return TGS_OK;
}

int check_vector(const void* p, const char* name) {
    if ((uintptr_t)p & 3u) return fail(TGS_ERR_INVALID, "%s is not aligned to its elements", name);
    return TGS_OK;
}

// A packed float vector as a one-row matrix, for check_apart.
tgs_matrix vector_of(const float* p, int64_t n) {
    return tgs_matrix{(void*)p, p ? 1 : 0, n, n, TGS_DTYPE_FLOAT32};
}

Mat view(const tgs_matrix* m) { return m ? Mat{m->data, m->rows, m->cols, m->stride} : Mat{}; }

int check_activation(int32_t activation) {
    if (activation < TGS_ACTIVATION_NONE || activation > TGS_ACTIVATION_GELU)
        return fail(TGS_ERR_UNSUPPORTED, "activation %d", activation);
    return TGS_OK;
}

int check_muon(const tgs_matrix* weights, const tgs_matrix* grads, const tgs_matrix* momenta,
               const tgs_matrix* copies, int32_t count) {
    if (!weights || !grads || !momenta) return fail(TGS_ERR_INVALID, "weights, grads or momenta is NULL");
    if (count < 1 || count > 4096) return fail(TGS_ERR_INVALID, "%d matrices", count);
    for (int32_t i = 0; i < count; ++i) {
        char name[4][32];
        snprintf(name[0], sizeof(name[0]), "weights[%d]", i);
        snprintf(name[1], sizeof(name[1]), "grads[%d]", i);
        snprintf(name[2], sizeof(name[2]), "momenta[%d]", i);
        snprintf(name[3], sizeof(name[3]), "copies[%d]", i);
        const tgs_matrix& w = weights[i];
        TGS_TRY(check_matrix(&w, name[0]));
        if (w.dtype != TGS_DTYPE_FLOAT32) return fail(TGS_ERR_INVALID, "%s: dtype %d, not float32", name[0], w.dtype);
        if (w.rows < 1 || w.rows >= kMaxStride) return fail(TGS_ERR_INVALID, "%s: %lld rows", name[0], (long long)w.rows);
        TGS_TRY(check_shape(&grads[i], name[1], w.rows, w.cols, grads[0].dtype));
        TGS_TRY(check_shape(&momenta[i], name[2], w.rows, w.cols, TGS_DTYPE_FLOAT32));
        if (copies) TGS_TRY(check_shape(&copies[i], name[3], w.rows, w.cols, copies[0].dtype));
    }
    // what the step writes shares nothing with anything else of the step
    const tgs_matrix* sets[4] = {weights, momenta, copies, grads};
    const char* names[4] = {"weights", "momenta", "copies", "grads"};
    for (int a = 0; a < 3; ++a)
        for (int b = a; b < 4; ++b)
            for (int32_t i = 0; sets[a] && sets[b] && i < count; ++i)
                for (int32_t j = a == b ? i + 1 : 0; j < count; ++j)
                    if (overlap(sets[a][i], sets[b][j]))
                        return fail(TGS_ERR_INVALID, "%s[%d] overlaps %s[%d]", names[a], i, names[b], j);
    return TGS_OK;
}

void bind_muon(tgs_muon* m, const tgs_matrix* weights, const tgs_matrix* grads, const tgs_matrix* momenta,
               const tgs_matrix* copies, int32_t count) {
    for (int32_t i = 0; i < count; ++i) {
        MuonPart& a = m->mats[(size_t)i];
        a.w = view(&weights[i]);
        a.g = view(&grads[i]);
        a.m = view(&momenta[i]);
        a.c = view(copies ? &copies[i] : nullptr);
    }
    // a step's launches take the larger matrices first
    std::sort(m->mats.begin(), m->mats.end(), [](const MuonPart& x, const MuonPart& y) {
        return x.w.rows * x.w.cols > y.w.rows * y.w.cols;
    });
    m->plan = plan_muon(m->mats.data(), count);
    m->on_device = false;
    m->grad_dtype = grads[0].dtype;
    m->copy_dtype = copies ? copies[0].dtype : TGS_DTYPE_FLOAT32;
}

}  // namespace

extern "C" {

int tgs_network_create(tgs_network** out) {
    if (!out) return fail(TGS_ERR_INVALID, "out is NULL");
    *out = new (std::nothrow) tgs_network();
    if (!*out) return fail(TGS_ERR_STATE, "out of host memory");
    return TGS_OK;
}

int tgs_network_destroy(tgs_network* n) {
    if (!n) return TGS_OK;
    release(n->workspace);
    delete n;
    return TGS_OK;
}

int tgs_linear_forward(tgs_network* n, const tgs_matrix* x, const tgs_matrix* w, const float* bias,
                       int32_t activation, const tgs_matrix* residual, const tgs_matrix* preact, const tgs_matrix* y,
                       void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    TGS_TRY(check_matrix(x, "x"));
    TGS_TRY(check_matrix(w, "w"));
    if (w->rows < 1) return fail(TGS_ERR_INVALID, "w has no rows");
    TGS_TRY(check_shape(w, "w", w->rows, x->cols, x->dtype));
    TGS_TRY(check_shape(y, "y", x->rows, w->rows, x->dtype));
    if (residual) TGS_TRY(check_shape(residual, "residual", x->rows, w->rows, x->dtype));
    if (preact) TGS_TRY(check_shape(preact, "preact", x->rows, w->rows, x->dtype));
    TGS_TRY(check_vector(bias, "bias"));
    TGS_TRY(check_activation(activation));
    const tgs_matrix b = vector_of(bias, w->rows);
    for (int k = 0; k < 2; ++k) {
        const tgs_matrix* out = k ? preact : y;
        const char* name = k ? "preact" : "y";
        TGS_TRY(check_apart(out, name, x, "x"));
        TGS_TRY(check_apart(out, name, w, "w"));
        TGS_TRY(check_apart(out, name, &b, "bias"));
        if (residual && (k || !same_place(*y, *residual))) TGS_TRY(check_apart(out, name, residual, "residual"));
    }
    TGS_TRY(check_apart(preact, "preact", y, "y"));
    if (x->rows == 0) return TGS_OK;
    const LinearForward a{view(x), view(w), view(residual), view(preact), view(y), bias, activation, x->dtype};
    const size_t bytes = linear_forward_workspace(a);
    if (bytes) TGS_TRY(ensure(n->workspace, bytes, (hipStream_t)stream));
    return launch_linear_forward(a, n->workspace.p, (hipStream_t)stream);
}

int tgs_linear_backward(tgs_network* n, const tgs_matrix* grad_y, const tgs_matrix* x, const tgs_matrix* w,
                        const tgs_matrix* preact, int32_t activation, const tgs_matrix* grad_x,
                        const tgs_matrix* grad_w, float* grad_bias, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    TGS_TRY(check_matrix(x, "x"));
    TGS_TRY(check_matrix(w, "w"));
    if (w->rows < 1) return fail(TGS_ERR_INVALID, "w has no rows");
    TGS_TRY(check_shape(w, "w", w->rows, x->cols, x->dtype));
    TGS_TRY(check_shape(grad_y, "grad_y", x->rows, w->rows, x->dtype));
    TGS_TRY(check_activation(activation));
    if (activation != TGS_ACTIVATION_NONE) TGS_TRY(check_shape(preact, "preact", x->rows, w->rows, x->dtype));
    if (grad_x) TGS_TRY(check_shape(grad_x, "grad_x", x->rows, x->cols, x->dtype));
    if (grad_w) TGS_TRY(check_shape(grad_w, "grad_w", w->rows, w->cols, x->dtype));
    TGS_TRY(check_vector(grad_bias, "grad_bias"));
    const tgs_matrix gb = vector_of(grad_bias, w->rows);
    const tgs_matrix* outs[3] = {grad_x, grad_w, grad_bias ? &gb : nullptr};
    const char* names[3] = {"grad_x", "grad_w", "grad_bias"};
    for (int k = 0; k < 3; ++k) {
        TGS_TRY(check_apart(outs[k], names[k], grad_y, "grad_y"));
        TGS_TRY(check_apart(outs[k], names[k], x, "x"));
        TGS_TRY(check_apart(outs[k], names[k], w, "w"));
        if (activation != TGS_ACTIVATION_NONE) TGS_TRY(check_apart(outs[k], names[k], preact, "preact"));
        for (int j = 0; j < k; ++j) TGS_TRY(check_apart(outs[k], names[k], outs[j], names[j]));
    }
    const LinearBackward a{view(grad_y), view(x), view(w), activation != TGS_ACTIVATION_NONE ? view(preact) : Mat{},
                           view(grad_x), view(grad_w), grad_bias, activation, x->dtype};
    TGS_TRY(ensure(n->workspace, linear_backward_workspace(a), (hipStream_t)stream));
    return launch_linear_backward(a, n->workspace.p, (hipStream_t)stream);
}

int tgs_layer_norm_forward(tgs_network* n, const tgs_matrix* x, const float* gamma, const float* beta, float epsilon,
                           const tgs_matrix* y, float* mean, float* rstd, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    TGS_TRY(check_matrix(x, "x"));
    TGS_TRY(check_shape(y, "y", x->rows, x->cols, x->dtype));
    if (!(epsilon >= 0.0f) || !isfinite(epsilon)) return fail(TGS_ERR_INVALID, "epsilon %g", epsilon);
    const tgs_matrix in[2] = {vector_of(gamma, x->cols), vector_of(beta, x->cols)};
    const tgs_matrix out[2] = {vector_of(mean, x->rows), vector_of(rstd, x->rows)};
    const char* in_names[2] = {"gamma", "beta"};
    const char* out_names[2] = {"mean", "rstd"};
    for (int k = 0; k < 2; ++k) {
        TGS_TRY(check_vector(in[k].data, in_names[k]));
        TGS_TRY(check_vector(out[k].data, out_names[k]));
        TGS_TRY(check_apart(y, "y", &in[k], in_names[k]));
        TGS_TRY(check_apart(&out[k], out_names[k], x, "x"));
        TGS_TRY(check_apart(&out[k], out_names[k], y, "y"));
        for (int j = 0; j < 2; ++j) TGS_TRY(check_apart(&out[k], out_names[k], &in[j], in_names[j]));
    }
    TGS_TRY(check_apart(&out[0], "mean", &out[1], "rstd"));
    if (!same_place(*x, *y)) TGS_TRY(check_apart(y, "y", x, "x"));
    if (x->rows == 0) return TGS_OK;
    return launch_layer_norm_forward({view(x), view(y), gamma, beta, epsilon, mean, rstd, x->dtype},
                                     (hipStream_t)stream);
}

int tgs_layer_norm_backward(tgs_network* n, const tgs_matrix* grad_y, const tgs_matrix* x, const float* gamma,
                            const float* mean, const float* rstd, const tgs_matrix* residual_grad,
                            const tgs_matrix* grad_x, float* grad_gamma, float* grad_beta, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    TGS_TRY(check_matrix(x, "x"));
    TGS_TRY(check_shape(grad_y, "grad_y", x->rows, x->cols, x->dtype));
    if (x->rows > 0 && (!mean || !rstd)) return fail(TGS_ERR_INVALID, "mean or rstd is NULL");
    if (residual_grad) TGS_TRY(check_shape(residual_grad, "residual_grad", x->rows, x->cols, x->dtype));
    if (residual_grad && !grad_x) return fail(TGS_ERR_INVALID, "residual_grad without grad_x");
    if (grad_x) TGS_TRY(check_shape(grad_x, "grad_x", x->rows, x->cols, x->dtype));
    const tgs_matrix in[3] = {vector_of(gamma, x->cols), vector_of(mean, x->rows), vector_of(rstd, x->rows)};
    const tgs_matrix out[2] = {vector_of(grad_gamma, x->cols), vector_of(grad_beta, x->cols)};
    const char* in_names[3] = {"gamma", "mean", "rstd"};
    const char* out_names[2] = {"grad_gamma", "grad_beta"};
    for (int j = 0; j < 3; ++j) {
        TGS_TRY(check_vector(in[j].data, in_names[j]));
        TGS_TRY(check_apart(grad_x, "grad_x", &in[j], in_names[j]));
    }
    for (int k = 0; k < 2; ++k) {
        TGS_TRY(check_vector(out[k].data, out_names[k]));
        TGS_TRY(check_apart(&out[k], out_names[k], x, "x"));
        TGS_TRY(check_apart(&out[k], out_names[k], grad_y, "grad_y"));
        TGS_TRY(check_apart(&out[k], out_names[k], residual_grad, "residual_grad"));
        TGS_TRY(check_apart(&out[k], out_names[k], grad_x, "grad_x"));
        for (int j = 0; j < 3; ++j) TGS_TRY(check_apart(&out[k], out_names[k], &in[j], in_names[j]));
    }
    TGS_TRY(check_apart(&out[0], "grad_gamma", &out[1], "grad_beta"));
    TGS_TRY(check_apart(grad_x, "grad_x", x, "x"));
    if (grad_x && !same_place(*grad_x, *grad_y)) TGS_TRY(check_apart(grad_x, "grad_x", grad_y, "grad_y"));
    if (grad_x && residual_grad && !same_place(*grad_x, *residual_grad))
        TGS_TRY(check_apart(grad_x, "grad_x", residual_grad, "residual_grad"));
    const LayerNormBackward a{view(grad_y), view(x), view(residual_grad), view(grad_x), gamma, mean, rstd,
                              grad_gamma, grad_beta, x->dtype};
    TGS_TRY(ensure(n->workspace, layer_norm_backward_workspace(a), (hipStream_t)stream));
    return launch_layer_norm_backward(a, n->workspace.p, (hipStream_t)stream);
}

// ------------------------------------------------------------------ Muon

int tgs_muon_create(const tgs_matrix* weights, const tgs_matrix* grads, const tgs_matrix* momenta,
                    const tgs_matrix* copies, int32_t count, tgs_muon** out) {
    if (!out) return fail(TGS_ERR_INVALID, "out is NULL");
    *out = nullptr;
    TGS_TRY(check_muon(weights, grads, momenta, copies, count));
    tgs_muon* m = new (std::nothrow) tgs_muon();
    if (!m) return fail(TGS_ERR_STATE, "out of host memory");
    try {
        m->mats.resize((size_t)count);
        m->firsts.resize((size_t)count * 3);
        for (int32_t i = 0; i < count; ++i) m->shapes.emplace_back(weights[i].rows, weights[i].cols);
    } catch (...) {
        delete m;
        return fail(TGS_ERR_STATE, "out of host memory");
    }
    m->p = tgs_muon_params{0.02f, 0.95f, 0.0f, 1e-12f, 1, 5};
    bind_muon(m, weights, grads, momenta, copies, count);
    if (!m->plan.fits) {
        delete m;
        return fail(TGS_ERR_INVALID, "the matrices are too large for one step");
    }
    *out = m;
    return TGS_OK;
}

int tgs_muon_destroy(tgs_muon* m) {
    if (!m) return TGS_OK;
    release(m->workspace);
    delete m;
    return TGS_OK;
}

int tgs_muon_set_matrices(tgs_muon* m, const tgs_matrix* weights, const tgs_matrix* grads, const tgs_matrix* momenta,
                          const tgs_matrix* copies, int32_t count) {
    if (!m) return fail(TGS_ERR_INVALID, "optimizer is NULL");
    if (count != (int32_t)m->mats.size())
        return fail(TGS_ERR_INVALID, "%d matrices, not %d", count, (int)m->mats.size());
    TGS_TRY(check_muon(weights, grads, momenta, copies, count));
    const bool had_copies = m->mats[0].c.p != nullptr;
    if (grads[0].dtype != m->grad_dtype || (copies != nullptr) != had_copies ||
        (copies && copies[0].dtype != m->copy_dtype))
        return fail(TGS_ERR_INVALID, "the gradients' or copies' dtype is not that of the creation");
    for (int32_t i = 0; i < count; ++i)
        if (weights[i].rows != m->shapes[(size_t)i].first || weights[i].cols != m->shapes[(size_t)i].second)
            return fail(TGS_ERR_INVALID, "weights[%d] is not of its shape at creation", i);
    bind_muon(m, weights, grads, momenta, copies, count);
    return TGS_OK;
}

int tgs_muon_set_params(tgs_muon* m, const tgs_muon_params* p) {
    if (!m || !p) return fail(TGS_ERR_INVALID, "optimizer or params is NULL");
    if (p->iterations < 0 || p->iterations > 32) return fail(TGS_ERR_INVALID, "%d iterations", p->iterations);
    if (!isfinite(p->lr) || !isfinite(p->weight_decay) || !(p->momentum >= 0.0f && p->momentum < 1.0f) ||
        !(p->epsilon > 0.0f) || !isfinite(p->epsilon))
        return fail(TGS_ERR_INVALID, "lr %g, momentum %g, weight decay %g, epsilon %g", p->lr, p->momentum,
                    p->weight_decay, p->epsilon);
    m->p = *p;
    return TGS_OK;
}

int tgs_muon_get_params(tgs_muon* m, tgs_muon_params* p) {
    if (!m || !p) return fail(TGS_ERR_INVALID, "optimizer or params is NULL");
    *p = m->p;
    return TGS_OK;
}

int tgs_muon_set_lr(tgs_muon* m, float global_lr) {
    if (!m) return fail(TGS_ERR_INVALID, "optimizer is NULL");
    m->global_lr = global_lr;
    return TGS_OK;
}

float tgs_muon_get_lr(tgs_muon* m) { return m ? m->global_lr : 0.0f; }

int tgs_muon_step(tgs_muon* m, float scale, void* stream) {
    if (!m) return fail(TGS_ERR_INVALID, "optimizer is NULL");
    const float lr = m->p.lr * m->global_lr;
    MuonStep p{};
    p.momentum = m->p.momentum;
    p.grad_scale = (1.0f - m->p.momentum) * scale;
    p.keep = 1.0f - lr * m->p.weight_decay;
    p.lr = lr;
    p.epsilon = m->p.epsilon;
    p.nesterov = m->p.nesterov != 0;
    p.iterations = m->p.iterations;
    p.grad_dtype = m->grad_dtype;
    p.copy_dtype = m->copy_dtype;
    hipStream_t s = (hipStream_t)stream;
    const int count = (int)m->mats.size();
    if (!m->on_device) {   // the first step, or the first after a rebinding
        const MuonPlan plan = plan_muon(m->mats.data(), count);
        TGS_TRY(ensure(m->workspace, (size_t)plan.bytes, s));
        unsigned char* at = m->workspace.as<unsigned char>();
        place_muon(m->mats.data(), count, at);
        for (int k = 0; k < 3; ++k)
            for (int i = 0; i < count; ++i) m->firsts[(size_t)(k * count + i)] = m->mats[(size_t)i].first[k];
        TGS_HIP(hipMemcpyAsync(at + plan.parts_at, m->mats.data(), sizeof(MuonPart) * (size_t)count,
                               hipMemcpyHostToDevice, s));
        TGS_HIP(hipMemcpyAsync(at + plan.firsts_at, m->firsts.data(), sizeof(uint32_t) * m->firsts.size(),
                               hipMemcpyHostToDevice, s));
        TGS_HIP(hipStreamSynchronize(s));
        m->plan = plan;
        m->on_device = true;
    }
    return launch_muon_step(m->plan, count, p, m->workspace.as<unsigned char>(), s);
}

int tgs_muon_reset(tgs_muon* m, void* stream) {
    if (!m) return fail(TGS_ERR_INVALID, "optimizer is NULL");
    for (const MuonPart& a : m->mats) TGS_TRY(launch_zero_matrix(a.m, (hipStream_t)stream));
    return TGS_OK;
}

}  // extern "C"
