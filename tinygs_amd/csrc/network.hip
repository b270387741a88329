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
    static constexpr int kDevices = 16;
    DevBuf workspaces[kDevices];   // of each device that calls ran on
    std::vector<DevBuf> outgrown;  // which captured calls may still use
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

struct tgs_gradient_clip {
    std::vector<ClipPart> parts;
    std::vector<uint32_t> firsts;
    bool apart = false;
    bool on_device = false;   // the workspace holds the table
    ClipPlan plan{};
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

// The current device's workspace, of `bytes` or more; NULL for none.
int workspace_of(tgs_network* n, size_t bytes, void* stream, void*& p) {
    p = nullptr;
    if (!bytes) return TGS_OK;
    int device = 0;
    TGS_HIP(hipGetDevice(&device));
    if (device < 0 || device >= tgs_network::kDevices) return fail(TGS_ERR_UNSUPPORTED, "device %d", device);
    DevBuf& b = n->workspaces[device];
    if (b.p && b.bytes < bytes) {
        try {
            n->outgrown.push_back(b);
        } catch (...) {
            return fail(TGS_ERR_STATE, "out of host memory");
        }
        b = DevBuf{};
    }
    TGS_TRY(ensure(b, bytes, (hipStream_t)stream));
    p = b.p;
    return TGS_OK;
}

// out does not lie on the mask's bytes.
int check_mask(const tgs_matrix* out, const char* name, const tgs_attention& a, int64_t states) {
    if (!out || !a.mask || !out->rows) return TGS_OK;
    const uintptr_t m0 = (uintptr_t)a.mask, m1 = m0 + (uintptr_t)((a.batch - 1) * a.mask_stride + states);
    const uintptr_t o0 = (uintptr_t)out->data;
    const uintptr_t o1 = o0 + (uintptr_t)(((out->rows - 1) * out->stride + out->cols) * element_size(out->dtype));
    if (o0 < m1 && m0 < o1) return fail(TGS_ERR_INVALID, "%s overlaps the mask", name);
    return TGS_OK;
}

constexpr int kMaxAttentionHead = 128, kMaxNormHead = 256, kMaxHeads = 4096;

int check_attention(const tgs_matrix* q, const tgs_matrix* k, const tgs_matrix* v, const tgs_attention* a, Attention& to) {
    TGS_TRY(check_matrix(q, "q"));
    TGS_TRY(check_matrix(k, "k"));
    if (!a) return fail(TGS_ERR_INVALID, "attention is NULL");
    if (a->heads < 1 || a->heads > kMaxHeads || q->cols % a->heads)
        return fail(TGS_ERR_INVALID, "%d heads of %lld columns", a->heads, (long long)q->cols);
    const int64_t head = q->cols / a->heads;
    if (head > kMaxAttentionHead) return fail(TGS_ERR_UNSUPPORTED, "heads of %lld columns", (long long)head);
    if (a->kv_heads < 1 || a->heads % a->kv_heads)
        return fail(TGS_ERR_INVALID, "%d heads do not share %d", a->heads, a->kv_heads);
    if (a->batch < 1 || q->rows % a->batch || k->rows % a->batch)
        return fail(TGS_ERR_INVALID, "a batch of %lld, %lld queries, %lld states", (long long)a->batch,
                    (long long)q->rows, (long long)k->rows);
    // times log2 e it is still a float
    if (!(a->scale >= 0.0f) || a->scale > 0x1p127f) return fail(TGS_ERR_INVALID, "scale %g", a->scale);
    TGS_TRY(check_shape(k, "k", k->rows, head * a->kv_heads, q->dtype));
    TGS_TRY(check_shape(v, "v", k->rows, head * a->kv_heads, q->dtype));
    const int64_t states = k->rows / a->batch;
    if (a->mask && (a->mask_stride < 0 || a->mask_stride > ((int64_t)1 << 40)))
        return fail(TGS_ERR_INVALID, "a mask's stride of %lld", (long long)a->mask_stride);
    to = Attention{view(q), view(k), view(v), Mat{}, nullptr, 0, 0, a->mask, a->mask_stride, a->batch, q->rows / a->batch, states,
                   a->heads, a->kv_heads, (int)head, a->scale, q->dtype};
    return TGS_OK;
}

// The places of rows x heads floats, in rows of heads or heads of rows, as one vector that holds them.
int check_lse(const float* lse, int64_t row_step, int64_t head_step, int64_t rows, int64_t heads, tgs_matrix& span) {
    span = vector_of(nullptr, 1);
    if (!lse) return TGS_OK;
    TGS_TRY(check_vector(lse, "lse"));
    const int64_t most = (int64_t)1 << 40;
    if (row_step < 1 || head_step < 1 || row_step > most || head_step > most ||
        (rows > 1 && heads > 1 && row_step < heads * head_step && head_step < rows * row_step))
        return fail(TGS_ERR_INVALID, "lse's steps %lld and %lld", (long long)row_step, (long long)head_step);
    if (rows > 0) span = vector_of(lse, (rows - 1) * row_step + (heads - 1) * head_step + 1);
    return TGS_OK;
}

int check_head_norm(const tgs_matrix* x, int32_t heads, const float* gamma, const tgs_turn* turn, float epsilon,
                    HeadNorm& to) {
    TGS_TRY(check_matrix(x, "x"));
    if (heads < 1 || heads > kMaxHeads || x->cols % heads)
        return fail(TGS_ERR_INVALID, "%d heads of %lld columns", heads, (long long)x->cols);
    const int64_t head = x->cols / heads;
    if (head > kMaxNormHead) return fail(TGS_ERR_UNSUPPORTED, "heads of %lld columns", (long long)head);
    TGS_TRY(check_vector(gamma, "gamma"));
    if (!(epsilon >= 0.0f) || !isfinite(epsilon)) return fail(TGS_ERR_INVALID, "epsilon %g", epsilon);
    to = HeadNorm{view(x), Mat{}, Mat{}, Mat{}, Mat{}, gamma, nullptr, heads, (int)head, epsilon, x->dtype};
    if (!turn) return TGS_OK;
    TGS_TRY(check_matrix(&turn->positions, "positions"));
    TGS_TRY(check_matrix(&turn->frequencies, "frequencies"));
    const int64_t axes = turn->positions.cols;
    if (axes > 4) return fail(TGS_ERR_UNSUPPORTED, "positions of %lld axes", (long long)axes);
    TGS_TRY(check_shape(&turn->positions, "positions", x->rows, axes, TGS_DTYPE_FLOAT32));
    TGS_TRY(check_shape(&turn->frequencies, "frequencies", turn->frequencies.rows, axes, TGS_DTYPE_FLOAT32));
    if (turn->frequencies.rows < 1 || turn->frequencies.rows > head / 2)
        return fail(TGS_ERR_INVALID, "%lld pairs in heads of %lld columns", (long long)turn->frequencies.rows,
                    (long long)head);
    to.positions = view(&turn->positions);
    to.frequencies = view(&turn->frequencies);
    return TGS_OK;
}

int check_clip(const tgs_matrix* grads, const tgs_matrix* clipped, int32_t count) {
    if (!grads) return fail(TGS_ERR_INVALID, "grads is NULL");
    if (count < 1 || count > 4096) return fail(TGS_ERR_INVALID, "%d matrices", count);
    const auto name = [](char (&to)[32], bool out, int32_t i) {
        snprintf(to, sizeof(to), out ? "clipped[%d]" : "grads[%d]", i);
        return to;
    };
    char x[32], y[32];
    for (int32_t i = 0; i < count; ++i) {
        TGS_TRY(check_matrix(&grads[i], name(x, false, i)));
        if (clipped) {
            TGS_TRY(check_matrix(&clipped[i], name(x, true, i)));
            TGS_TRY(check_shape(&clipped[i], name(x, true, i), grads[i].rows, grads[i].cols, clipped[i].dtype));
        }
    }
    // no element counts twice, and what is written shares nothing with the rest: in the order of their addresses, each
    // is held against those that begin before it ends
    struct Place {
        const tgs_matrix* m;
        int32_t i;
        bool out;
    };
    std::vector<Place> places;
    try {
        places.reserve((size_t)count * 2);
    } catch (...) {
        return fail(TGS_ERR_STATE, "out of host memory");
    }
    for (int32_t i = 0; i < count; ++i) {
        if (grads[i].rows) places.push_back({&grads[i], i, false});
        if (clipped && clipped[i].rows) places.push_back({&clipped[i], i, true});
    }
    std::sort(places.begin(), places.end(),
              [](const Place& p, const Place& q) { return (uintptr_t)p.m->data < (uintptr_t)q.m->data; });
    for (size_t p = 0; p < places.size(); ++p) {
        const tgs_matrix& a = *places[p].m;
        const uintptr_t end = (uintptr_t)a.data + (uintptr_t)(((a.rows - 1) * a.stride + a.cols) * element_size(a.dtype));
        for (size_t q = p + 1; q < places.size() && (uintptr_t)places[q].m->data < end; ++q) {
            if (!overlap(a, *places[q].m)) continue;
            // the output, or the later one, comes first
            const bool turned = places[p].out == places[q].out ? places[p].i > places[q].i : places[p].out;
            const Place &u = places[turned ? p : q], &v = places[turned ? q : p];
            return fail(TGS_ERR_INVALID, "%s overlaps %s", name(x, u.out, u.i), name(y, v.out, v.i));
        }
    }
    return TGS_OK;
}

int bind_clip(tgs_gradient_clip* c, const tgs_matrix* grads, const tgs_matrix* clipped, int32_t count) {
    std::vector<ClipPart> parts;
    std::vector<uint32_t> firsts;
    try {
        parts.resize((size_t)count);
        firsts.resize((size_t)count);
    } catch (...) {
        return fail(TGS_ERR_STATE, "out of host memory");
    }
    for (int32_t i = 0; i < count; ++i) {
        const tgs_matrix& g = grads[i];
        const tgs_matrix& to = clipped ? clipped[i] : g;
        // a single row's stride says nothing
        parts[(size_t)i] = ClipPart{g.data, to.data, g.rows * g.cols, g.cols, g.rows > 1 ? g.stride : g.cols,
                                    g.rows > 1 ? to.stride : g.cols, g.dtype, to.dtype};
    }
    const ClipPlan plan = plan_clip(parts.data(), count, firsts.data());
    if (plan.chunks == 0x7fffffffu) return fail(TGS_ERR_INVALID, "too many elements for one norm");
    c->parts.swap(parts);
    c->firsts.swap(firsts);
    c->plan = plan;
    c->apart = clipped != nullptr;
    c->on_device = false;
    return TGS_OK;
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
    for (DevBuf& b : n->workspaces) release(b);
    for (DevBuf& b : n->outgrown) release(b);
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
    void* workspace;
    TGS_TRY(workspace_of(n, linear_forward_workspace(a), stream, workspace));
    return launch_linear_forward(a, workspace, (hipStream_t)stream);
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
    void* workspace;
    TGS_TRY(workspace_of(n, linear_backward_workspace(a), stream, workspace));
    return launch_linear_backward(a, workspace, (hipStream_t)stream);
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
    void* workspace;
    TGS_TRY(workspace_of(n, layer_norm_backward_workspace(a), stream, workspace));
    return launch_layer_norm_backward(a, workspace, (hipStream_t)stream);
}

// ------------------------------------------------------------------ attention

int tgs_attention_forward(tgs_network* n, const tgs_matrix* q, const tgs_matrix* k, const tgs_matrix* v,
                          const tgs_attention* a, const tgs_matrix* out, float* lse, int64_t lse_row_step,
                          int64_t lse_head_step, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    Attention to;
    TGS_TRY(check_attention(q, k, v, a, to));
    TGS_TRY(check_shape(out, "out", q->rows, q->cols, q->dtype));
    tgs_matrix l;
    TGS_TRY(check_lse(lse, lse_row_step, lse_head_step, q->rows, a->heads, l));
    const tgs_matrix* outs[2] = {out, &l};
    const char* names[2] = {"out", "lse"};
    for (int i = 0; i < 2; ++i) {
        TGS_TRY(check_apart(outs[i], names[i], q, "q"));
        TGS_TRY(check_apart(outs[i], names[i], k, "k"));
        TGS_TRY(check_apart(outs[i], names[i], v, "v"));
        TGS_TRY(check_mask(outs[i], names[i], *a, to.states));
    }
    TGS_TRY(check_apart(&l, "lse", out, "out"));
    if (q->rows == 0) return TGS_OK;
    to.out = view(out);
    to.lse = lse;
    to.lse_row_step = lse_row_step;
    to.lse_head_step = lse_head_step;
    void* workspace;
    TGS_TRY(workspace_of(n, attention_workspace(to), stream, workspace));
    return launch_attention(to, workspace, (hipStream_t)stream);
}

int tgs_attention_backward(tgs_network* n, const tgs_matrix* grad_out, const tgs_matrix* q, const tgs_matrix* k,
                           const tgs_matrix* v, const tgs_matrix* out, const float* lse, int64_t lse_row_step,
                           int64_t lse_head_step, const tgs_attention* a, const tgs_matrix* grad_q,
                           const tgs_matrix* grad_k, const tgs_matrix* grad_v, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    AttentionBackward to{};
    TGS_TRY(check_attention(q, k, v, a, to.a));
    TGS_TRY(check_shape(grad_out, "grad_out", q->rows, q->cols, q->dtype));
    TGS_TRY(check_shape(out, "out", q->rows, q->cols, q->dtype));
    if (q->rows > 0 && !lse) return fail(TGS_ERR_INVALID, "lse is NULL");
    tgs_matrix l;
    TGS_TRY(check_lse(lse, lse_row_step, lse_head_step, q->rows, a->heads, l));
    if (grad_q) TGS_TRY(check_shape(grad_q, "grad_q", q->rows, q->cols, q->dtype));
    if (grad_k) TGS_TRY(check_shape(grad_k, "grad_k", k->rows, k->cols, q->dtype));
    if (grad_v) TGS_TRY(check_shape(grad_v, "grad_v", k->rows, k->cols, q->dtype));
    const tgs_matrix* outs[3] = {grad_q, grad_k, grad_v};
    const char* names[3] = {"grad_q", "grad_k", "grad_v"};
    const tgs_matrix* ins[6] = {grad_out, q, k, v, out, &l};
    const char* in_names[6] = {"grad_out", "q", "k", "v", "out", "lse"};
    for (int i = 0; i < 3; ++i) {
        for (int j = 0; j < 6; ++j) TGS_TRY(check_apart(outs[i], names[i], ins[j], in_names[j]));
        for (int j = 0; j < i; ++j) TGS_TRY(check_apart(outs[i], names[i], outs[j], names[j]));
        TGS_TRY(check_mask(outs[i], names[i], *a, to.a.states));
    }
    to.a.out = view(out);
    to.a.lse = const_cast<float*>(lse);
    to.a.lse_row_step = lse_row_step;
    to.a.lse_head_step = lse_head_step;
    to.grad_out = view(grad_out);
    to.grad_q = view(grad_q);
    to.grad_k = view(grad_k);
    to.grad_v = view(grad_v);
    void* workspace;
    TGS_TRY(workspace_of(n, attention_backward_workspace(to), stream, workspace));
    return launch_attention_backward(to, workspace, (hipStream_t)stream);
}

int tgs_head_norm_forward(tgs_network* n, const tgs_matrix* x, int32_t heads, const float* gamma, const tgs_turn* turn,
                          float epsilon, const tgs_matrix* y, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    HeadNorm to;
    TGS_TRY(check_head_norm(x, heads, gamma, turn, epsilon, to));
    TGS_TRY(check_shape(y, "y", x->rows, x->cols, x->dtype));
    const tgs_matrix g = vector_of(gamma, to.head);
    TGS_TRY(check_apart(y, "y", &g, "gamma"));
    if (turn) {
        TGS_TRY(check_apart(y, "y", &turn->positions, "positions"));
        TGS_TRY(check_apart(y, "y", &turn->frequencies, "frequencies"));
    }
    if (!same_place(*x, *y)) TGS_TRY(check_apart(y, "y", x, "x"));
    if (x->rows == 0) return TGS_OK;
    to.y = view(y);
    return launch_head_norm(to, (hipStream_t)stream);
}

int tgs_head_norm_backward(tgs_network* n, const tgs_matrix* grad_y, const tgs_matrix* x, int32_t heads,
                           const float* gamma, const tgs_turn* turn, float epsilon, const tgs_matrix* grad_x,
                           float* grad_gamma, void* stream) {
    if (!n) return fail(TGS_ERR_INVALID, "network is NULL");
    HeadNorm to;
    TGS_TRY(check_head_norm(x, heads, gamma, turn, epsilon, to));
    TGS_TRY(check_shape(grad_y, "grad_y", x->rows, x->cols, x->dtype));
    if (grad_x) TGS_TRY(check_shape(grad_x, "grad_x", x->rows, x->cols, x->dtype));
    TGS_TRY(check_vector(grad_gamma, "grad_gamma"));
    const tgs_matrix g = vector_of(gamma, to.head), gg = vector_of(grad_gamma, to.head);
    const tgs_matrix* outs[2] = {grad_x, &gg};
    const char* names[2] = {"grad_x", "grad_gamma"};
    for (int i = 0; i < 2; ++i) {
        TGS_TRY(check_apart(outs[i], names[i], x, "x"));
        TGS_TRY(check_apart(outs[i], names[i], &g, "gamma"));
        if (!turn) continue;
        TGS_TRY(check_apart(outs[i], names[i], &turn->positions, "positions"));
        TGS_TRY(check_apart(outs[i], names[i], &turn->frequencies, "frequencies"));
    }
    TGS_TRY(check_apart(&gg, "grad_gamma", grad_y, "grad_y"));
    TGS_TRY(check_apart(&gg, "grad_gamma", grad_x, "grad_x"));
    if (grad_x && !same_place(*grad_x, *grad_y)) TGS_TRY(check_apart(grad_x, "grad_x", grad_y, "grad_y"));
    to.grad_y = view(grad_y);
    to.y = view(grad_x);
    to.grad_gamma = grad_gamma;
    void* workspace;
    TGS_TRY(workspace_of(n, head_norm_backward_workspace(to), stream, workspace));
    return launch_head_norm_backward(to, workspace, (hipStream_t)stream);
}

// ------------------------------------------------------------------ clipping

int tgs_gradient_clip_create(const tgs_matrix* grads, const tgs_matrix* clipped, int32_t count,
                             tgs_gradient_clip** out) {
    if (!out) return fail(TGS_ERR_INVALID, "out is NULL");
    *out = nullptr;
    TGS_TRY(check_clip(grads, clipped, count));
    tgs_gradient_clip* c = new (std::nothrow) tgs_gradient_clip();
    if (!c) return fail(TGS_ERR_STATE, "out of host memory");
    const int rc = bind_clip(c, grads, clipped, count);
    if (rc != TGS_OK) {
        delete c;
        return rc;
    }
    *out = c;
    return TGS_OK;
}

int tgs_gradient_clip_destroy(tgs_gradient_clip* c) {
    if (!c) return TGS_OK;
    release(c->workspace);
    delete c;
    return TGS_OK;
}

int tgs_gradient_clip_set_matrices(tgs_gradient_clip* c, const tgs_matrix* grads, const tgs_matrix* clipped,
                                   int32_t count) {
    if (!c) return fail(TGS_ERR_INVALID, "gradient clip is NULL");
    TGS_TRY(check_clip(grads, clipped, count));
    return bind_clip(c, grads, clipped, count);
}

int tgs_gradient_clip_run(tgs_gradient_clip* c, float max_norm, float scale, float epsilon, float* norm, void* stream) {
    if (!c) return fail(TGS_ERR_INVALID, "gradient clip is NULL");
    if (!(max_norm >= 0.0f)) return fail(TGS_ERR_INVALID, "max_norm %g", max_norm);
    if (!(scale > 0.0f) || !isfinite(scale)) return fail(TGS_ERR_INVALID, "scale %g", scale);
    if (!(epsilon >= 0.0f) || !isfinite(epsilon)) return fail(TGS_ERR_INVALID, "epsilon %g", epsilon);
    TGS_TRY(check_vector(norm, "norm"));
    const tgs_matrix v = vector_of(norm, 1);
    for (const ClipPart& a : c->parts) {
        const tgs_matrix g{const_cast<void*>(a.g), a.count / a.cols, a.cols, a.stride, a.dtype};
        const tgs_matrix to{a.c, g.rows, a.cols, a.c_stride, a.c_dtype};
        TGS_TRY(check_apart(&v, "norm", &g, "a gradient"));
        TGS_TRY(check_apart(&v, "norm", &to, "a clipped gradient"));
    }
    hipStream_t s = (hipStream_t)stream;
    const int count = (int)c->parts.size();
    if (!c->on_device) {   // the first run, or the first after a rebinding
        TGS_TRY(ensure(c->workspace, (size_t)c->plan.bytes, s));
        unsigned char* at = c->workspace.as<unsigned char>();
        TGS_HIP(hipMemcpyAsync(at + c->plan.parts_at, c->parts.data(), sizeof(ClipPart) * (size_t)count,
                               hipMemcpyHostToDevice, s));
        TGS_HIP(hipMemcpyAsync(at + c->plan.firsts_at, c->firsts.data(), sizeof(uint32_t) * (size_t)count,
                               hipMemcpyHostToDevice, s));
        TGS_HIP(hipStreamSynchronize(s));
        c->on_device = true;
    }
    return launch_clip(c->plan, count, {max_norm, scale, epsilon, norm, c->apart}, c->workspace.as<unsigned char>(), s);
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
