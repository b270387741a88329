// The attention of a few rows to states of another number through the C++
// interface: head norms with turned pairs, attention with a mask and shared
// heads, the gradients of all of them, and clipping, each checked against loops
// in double. Prints "attention ok" or the first difference.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "tinygs_amd/tinygs.hpp"

using namespace tinygs_amd;

namespace {

using Vec = std::vector<double>;

DeviceArray<float> random(int64_t n, uint32_t s, float scale, Vec& host) {
    std::vector<float> v((size_t)n);
    host.resize((size_t)n);
    for (int64_t k = 0; k < n; ++k) {
        s = s * 1664525u + 1013904223u;
        host[(size_t)k] = v[(size_t)k] = scale * (((float)(s >> 8) / 8388608.0f) - 1.0f);
    }
    DeviceArray<float> d;
    d.copy_from_host(v.data(), v.size());
    return d;
}

void check(const char* what, const std::vector<float>& g, const Vec& want, double bound) {
    double off = 0.0, norm = 0.0;
    for (size_t k = 0; k < g.size(); ++k) {
        off += (g[k] - want[k]) * (g[k] - want[k]);
        norm += want[k] * want[k];
    }
    off = std::sqrt(off / norm);
    std::printf("%s: %.2g off\n", what, off);
    if (g.size() != want.size() || !(off <= bound)) {
        std::printf("FAILED: %s\n", what);
        std::exit(1);
    }
}

// Head norms: h = x / root, u = h gamma, pairs turned.
struct HeadNormed {
    Vec y, h, root, cosine, sine;
};
HeadNormed head_norm(const Vec& x, const Vec& gamma, const Vec& pos, const Vec& freq, int rows, int heads, int d, int axes,
                     double eps) {
    HeadNormed o{Vec(x.size()), Vec(x.size()), Vec((size_t)rows * heads), Vec((size_t)rows * d / 2), Vec((size_t)rows * d / 2)};
    for (int r = 0; r < rows; ++r) {
        for (int p = 0; p < d / 2; ++p) {
            double t = 0.0;
            for (int k = 0; k < axes; ++k) t += pos[(size_t)r * axes + k] * freq[(size_t)p * axes + k];
            o.cosine[(size_t)r * d / 2 + p] = std::cos(t);
            o.sine[(size_t)r * d / 2 + p] = std::sin(t);
        }
        for (int h = 0; h < heads; ++h) {
            const size_t at = ((size_t)r * heads + h) * d;
            double s = 0.0;
            for (int c = 0; c < d; ++c) s += x[at + c] * x[at + c] / d;
            const double root = o.root[(size_t)r * heads + h] = std::sqrt(s + eps);
            for (int c = 0; c < d; ++c) o.h[at + c] = x[at + c] / root;
            for (int p = 0; p < d / 2; ++p) {
                const double a = o.h[at + 2 * p] * gamma[2 * p], b = o.h[at + 2 * p + 1] * gamma[2 * p + 1];
                const double co = o.cosine[(size_t)r * d / 2 + p], si = o.sine[(size_t)r * d / 2 + p];
                o.y[at + 2 * p] = a * co - b * si;
                o.y[at + 2 * p + 1] = a * si + b * co;
            }
        }
    }
    return o;
}

}  // namespace

int main() {
    const int rows = 37, states = 51, heads = 4, kv = 2, d = 24, axes = 3, shared = heads / kv;
    const double eps = 1e-6, scale = 1.0 / std::sqrt((double)d);
    Vec x, k, v, gamma, pos, freq, go;
    const auto dx = random(rows * heads * d, 1, 1.5f, x), dk = random(states * kv * d, 2, 1.5f, k),
               dv = random(states * kv * d, 3, 1.0f, v), dg = random(d, 4, 1.0f, gamma), dp = random(rows * axes, 5, 4.0f, pos),
               df = random(d / 2 * axes, 6, 2.0f, freq), dgo = random(rows * heads * d, 7, 0.1f, go);
    std::vector<uint8_t> mask((size_t)states);
    for (int j = 0; j < states; ++j) mask[(size_t)j] = j % 5 != 2;
    DeviceArray<uint8_t> dm;
    dm.copy_from_host(mask.data(), mask.size());
    const auto mat = [](const DeviceArray<float>& a, int64_t r, int64_t c) { return matrix((void*)a.data(), r, c); };
    const int wide = heads * d, narrow = kv * d;
    DeviceArray<float> q(rows * wide), out(rows * wide), lse(rows * heads), gq(rows * wide), gk(states * narrow),
        gv(states * narrow), gx(rows * wide), gg(d);
    const tgs_turn turn{mat(dp, rows, axes), mat(df, d / 2, axes)};
    const tgs_matrix mx = mat(dx, rows, wide), mq = mat(q, rows, wide), mk = mat(dk, states, narrow),
                     mv = mat(dv, states, narrow), mo = mat(out, rows, wide), mgo = mat(dgo, rows, wide),
                     mgq = mat(gq, rows, wide), mgk = mat(gk, states, narrow), mgv = mat(gv, states, narrow),
                     mgx = mat(gx, rows, wide);
    const tgs_attention a = attention_of(1, heads, kv, (float)scale, dm.data());
    LayerOps ops;
    ops.head_norm(mx, heads, dg.data(), &turn, (float)eps, mq);
    ops.attention(mq, mk, mv, a, mo, lse.data());
    ops.attention_backward(mgo, mq, mk, mv, mo, lse.data(), a, &mgq, &mgk, &mgv);
    ops.head_norm_backward(mgq, mx, heads, dg.data(), &turn, (float)eps, &mgx, gg.data());
    hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");

    const HeadNormed n = head_norm(x, gamma, pos, freq, rows, heads, d, axes, eps);
    check("head norm", q.to_host(), n.y, 1e-6);
    Vec o(x.size()), l((size_t)rows * heads), wq(x.size()), wk(k.size()), wv(v.size());
    for (int r = 0; r < rows; ++r)
        for (int h = 0; h < heads; ++h) {
            const double* qr = &n.y[((size_t)r * heads + h) * d];
            const double* g = &go[((size_t)r * heads + h) * d];
            Vec p((size_t)states, 0.0), dp2((size_t)states, 0.0);
            double sum = 0.0, delta = 0.0;
            for (int j = 0; j < states; ++j) {
                if (!mask[(size_t)j]) continue;
                const size_t at = ((size_t)j * kv + h / shared) * d;
                double s = 0.0;
                for (int c = 0; c < d; ++c) {
                    s += qr[c] * k[at + c];
                    dp2[(size_t)j] += g[c] * v[at + c];
                }
                sum += p[(size_t)j] = std::exp(s * scale);
            }
            l[(size_t)h * rows + r] = std::log(sum);
            for (int j = 0; j < states; ++j) {
                p[(size_t)j] /= sum;
                delta += p[(size_t)j] * dp2[(size_t)j];
            }
            for (int j = 0; j < states; ++j) {
                const size_t at = ((size_t)j * kv + h / shared) * d;
                const double ds = p[(size_t)j] * (dp2[(size_t)j] - delta) * scale;
                for (int c = 0; c < d; ++c) {
                    o[((size_t)r * heads + h) * d + c] += p[(size_t)j] * v[at + c];
                    wq[((size_t)r * heads + h) * d + c] += ds * k[at + c];
                    wk[at + c] += ds * qr[c];
                    wv[at + c] += p[(size_t)j] * g[c];
                }
            }
        }
    check("attention", out.to_host(), o, 2e-6);
    check("lse", lse.to_host(), l, 1e-6);
    check("grad q", gq.to_host(), wq, 5e-6);
    check("grad k", gk.to_host(), wk, 5e-6);
    check("grad v", gv.to_host(), wv, 5e-6);
    Vec wx(x.size()), wg((size_t)d, 0.0);
    for (int r = 0; r < rows; ++r)
        for (int h = 0; h < heads; ++h) {
            const size_t at = ((size_t)r * heads + h) * d;
            Vec u((size_t)d);
            double dot = 0.0;
            for (int p = 0; p < d / 2; ++p) {
                const double co = n.cosine[(size_t)r * d / 2 + p], si = n.sine[(size_t)r * d / 2 + p];
                u[2 * p] = wq[at + 2 * p] * co + wq[at + 2 * p + 1] * si;
                u[2 * p + 1] = wq[at + 2 * p + 1] * co - wq[at + 2 * p] * si;
            }
            for (int c = 0; c < d; ++c) {
                wg[(size_t)c] += u[(size_t)c] * n.h[at + c];
                dot += u[(size_t)c] * gamma[(size_t)c] * n.h[at + c] / d;
            }
            for (int c = 0; c < d; ++c)
                wx[at + c] = (u[(size_t)c] * gamma[(size_t)c] - n.h[at + c] * dot) / n.root[(size_t)r * heads + h];
        }
    check("grad x", gx.to_host(), wx, 1e-5);
    check("grad gamma", gg.to_host(), wg, 1e-5);

    double norm = 0.0;
    for (double w : wx) norm += w * w;
    for (double w : wk) norm += w * w;
    norm = std::sqrt(norm);
    DeviceArray<float> got(1);
    GradientClip clip({mgx, mgk});
    clip.clip((float)(0.25 * norm), 1.0f, 0.0f, got.data());
    hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");
    check("norm", got.to_host(), Vec{norm}, 1e-5);
    for (double& w : wx) w *= 0.25;
    for (double& w : wk) w *= 0.25;
    check("clipped grad x", gx.to_host(), wx, 2e-5);
    check("clipped grad k", gk.to_host(), wk, 2e-5);
    try {
        ops.attention(mq, mk, mv, attention_of(1, heads, 3, 1.0f), mo);
        std::printf("FAILED: no refusal\n");
        return 1;
    } catch (const std::runtime_error& e) {
        std::printf("refused: %s\n", e.what());
    }
    std::printf("attention ok\n");
    return 0;
}
