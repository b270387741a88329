// One training step of a residual block through the C++ interface: layer norm,
// two linear layers with bias, activation and residual, their gradients and
// Muon on the two matrices, each checked against loops in double. Prints
// "network ok" or the first difference.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "tinygs_amd/tinygs.hpp"

using namespace tinygs_amd;

namespace {

using Vec = std::vector<double>;

float noise(uint32_t& s) {
    s = s * 1664525u + 1013904223u;
    return ((float)(s >> 8) / 8388608.0f) - 1.0f;
}

DeviceArray<float> random(int64_t n, uint32_t seed, float scale, Vec& host) {
    std::vector<float> v((size_t)n);
    host.resize((size_t)n);
    for (int64_t k = 0; k < n; ++k) host[(size_t)k] = v[(size_t)k] = scale * noise(seed);
    DeviceArray<float> d;
    d.copy_from_host(v.data(), v.size());
    return d;
}

void check(const char* what, const DeviceArray<float>& got, const Vec& want, double bound) {
    const std::vector<float> g = got.to_host();
    double off = 0.0, norm = 0.0;
    for (size_t k = 0; k < g.size(); ++k) {
        off += (g[k] - want[k]) * (g[k] - want[k]);
        norm += want[k] * want[k];
    }
    off = std::sqrt(off / norm);
    std::printf("%s: %.2g off\n", what, off);
    if (!(off <= bound)) {
        std::printf("FAILED: %s\n", what);
        std::exit(1);
    }
}

double silu(double z) { return z / (1.0 + std::exp(-z)); }
double silu_slope(double z) {
    const double p = 1.0 / (1.0 + std::exp(-z));
    return p * (1.0 + z * (1.0 - p));
}

// c (m x n) = a (m x k) b^T (n x k)
Vec product(const Vec& a, const Vec& b, int m, int n, int k) {
    Vec c((size_t)m * n);
    for (int i = 0; i < m; ++i)
        for (int j = 0; j < n; ++j) {
            double v = 0.0;
            for (int q = 0; q < k; ++q) v += a[(size_t)i * k + q] * b[(size_t)j * k + q];
            c[(size_t)i * n + j] = v;
        }
    return c;
}
Vec transposed(const Vec& a, int m, int n) {
    Vec t((size_t)m * n);
    for (int i = 0; i < m; ++i)
        for (int j = 0; j < n; ++j) t[(size_t)j * m + i] = a[(size_t)i * n + j];
    return t;
}

Vec muon_update(const Vec& u, int rows, int cols) {   // X after five steps, rows <= cols
    double norm = 0.0;
    for (double v : u) norm += v * v;
    Vec x = u;
    for (double& v : x) v /= std::sqrt(norm);
    for (int it = 0; it < 5; ++it) {
        const Vec a = product(x, x, rows, rows, cols), a2 = product(a, a, rows, rows, rows);
        Vec p = a;
        for (size_t k = 0; k < p.size(); ++k) p[k] = -4.7750 * a[k] + 2.0315 * a2[k];
        const Vec y = product(p, transposed(x, rows, cols), rows, cols, rows);
        for (size_t k = 0; k < x.size(); ++k) x[k] = 3.4445 * x[k] + y[k];
    }
    return x;
}

}  // namespace

int main() {
    const int rows = 75, width = 40, hidden = 72;
    const double eps = 1e-5;
    Vec x, w1, w2, b1, b2, gamma, beta, gy;
    const auto dx = random(rows * width, 1, 1.0f, x), dw1 = random(hidden * width, 2, 0.3f, w1);
    auto mw1 = random(hidden * width, 2, 0.3f, w1), mw2 = random(width * hidden, 3, 0.3f, w2);
    const auto dw2 = random(width * hidden, 3, 0.3f, w2), db1 = random(hidden, 4, 0.2f, b1),
               db2 = random(width, 5, 0.2f, b2), dgamma = random(width, 6, 1.0f, gamma),
               dbeta = random(width, 7, 0.3f, beta), dgy = random(rows * width, 8, 0.1f, gy);
    const auto mat = [](const DeviceArray<float>& a, int64_t r, int64_t c) { return matrix((void*)a.data(), r, c); };
    DeviceArray<float> n(rows * width), mean(rows), rstd(rows), z(rows * hidden), a(rows * hidden), y(rows * width);
    LayerOps ops;
    const tgs_matrix mx = mat(dx, rows, width), mn = mat(n, rows, width), mz = mat(z, rows, hidden),
                     ma = mat(a, rows, hidden), my = mat(y, rows, width), m1 = mat(dw1, hidden, width),
                     m2 = mat(dw2, width, hidden), mgy = mat(dgy, rows, width);
    ops.layer_norm(mx, dgamma.data(), dbeta.data(), (float)eps, mn, mean.data(), rstd.data());
    ops.linear(mn, m1, db1.data(), Activation::Silu, nullptr, &mz, ma);
    ops.linear(ma, m2, db2.data(), Activation::None, &mx, nullptr, my);
    DeviceArray<float> ga(rows * hidden), gn(rows * width), gx(rows * width), gw1(hidden * width), gw2(width * hidden),
        gb1(hidden), gb2(width), ggamma(width), gbeta(width);
    const tgs_matrix mga = mat(ga, rows, hidden), mgn = mat(gn, rows, width), mgx = mat(gx, rows, width),
                     mg1 = mat(gw1, hidden, width), mg2 = mat(gw2, width, hidden);
    ops.linear_backward(mgy, ma, m2, nullptr, Activation::None, &mga, &mg2, gb2.data());
    ops.linear_backward(mga, mn, m1, &mz, Activation::Silu, &mgn, &mg1, gb1.data());
    ops.layer_norm_backward(mgn, mx, dgamma.data(), mean.data(), rstd.data(), &mgy, &mgx, ggamma.data(), gbeta.data());
    DeviceArray<float> mom1(hidden * width), mom2(width * hidden);
    hip_check(hipMemset(mom1.data(), 0, mom1.bytes()), "hipMemset");
    hip_check(hipMemset(mom2.data(), 0, mom2.bytes()), "hipMemset");
    Muon muon({mat(mw1, hidden, width), mat(mw2, width, hidden)}, {mg1, mg2},
              {mat(mom1, hidden, width), mat(mom2, width, hidden)});
    muon.set_params({{"lr", 0.1}, {"weight_decay", 0.5}});
    muon.step(1.0f);
    hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");

    // in double
    Vec h(x.size()), rs((size_t)rows), nn(x.size());
    for (int r = 0; r < rows; ++r) {
        double m = 0.0, v = 0.0;
        for (int k = 0; k < width; ++k) m += x[(size_t)r * width + k] / width;
        for (int k = 0; k < width; ++k) v += std::pow(x[(size_t)r * width + k] - m, 2) / width;
        rs[(size_t)r] = 1.0 / std::sqrt(v + eps);
        for (int k = 0; k < width; ++k) {
            const size_t q = (size_t)r * width + k;
            h[q] = (x[q] - m) * rs[(size_t)r];
            nn[q] = h[q] * gamma[(size_t)k] + beta[(size_t)k];
        }
    }
    check("layer norm", n, nn, 1e-6);
    Vec zz = product(nn, w1, rows, hidden, width), aa(zz.size());
    for (size_t q = 0; q < zz.size(); ++q) {
        zz[q] += b1[q % hidden];
        aa[q] = silu(zz[q]);
    }
    check("preact", z, zz, 1e-6);
    check("activation", a, aa, 1e-6);
    Vec yy = product(aa, w2, rows, width, hidden);
    for (size_t q = 0; q < yy.size(); ++q) yy[q] += b2[q % width] + x[q];
    check("block", y, yy, 1e-6);
    const Vec gaa = product(gy, transposed(w2, width, hidden), rows, hidden, width);
    check("grad a", ga, gaa, 1e-6);
    const Vec g2 = product(transposed(gy, rows, width), transposed(aa, rows, hidden), width, hidden, rows);
    check("grad w2", gw2, g2, 1e-6);
    Vec dz = gaa, sb1((size_t)hidden, 0.0);
    for (size_t q = 0; q < dz.size(); ++q) {
        dz[q] *= silu_slope(zz[q]);
        sb1[q % hidden] += dz[q];
    }
    check("grad b1", gb1, sb1, 1e-6);
    const Vec g1 = product(transposed(dz, rows, hidden), transposed(nn, rows, width), hidden, width, rows);
    check("grad w1", gw1, g1, 1e-6);
    const Vec gnn = product(dz, transposed(w1, hidden, width), rows, width, hidden);
    check("grad norm", gn, gnn, 1e-6);
    Vec gxx(x.size()), sg((size_t)width, 0.0);
    for (int r = 0; r < rows; ++r) {
        double c1 = 0.0, c2 = 0.0;
        for (int k = 0; k < width; ++k) {
            const size_t q = (size_t)r * width + k;
            c1 += gnn[q] * gamma[(size_t)k] / width;
            c2 += gnn[q] * gamma[(size_t)k] * h[q] / width;
            sg[(size_t)k] += gnn[q] * h[q];
        }
        for (int k = 0; k < width; ++k) {
            const size_t q = (size_t)r * width + k;
            gxx[q] = rs[(size_t)r] * (gnn[q] * gamma[(size_t)k] - c1 - h[q] * c2) + gy[q];
        }
    }
    check("grad x", gx, gxx, 2e-6);
    check("grad gamma", ggamma, sg, 2e-6);
    // zero momenta: the update is the gradient's own direction. w1 is tall: the transpose's, and sqrt(rows / cols)
    const Vec x1 = transposed(muon_update(transposed(g1, hidden, width), width, hidden), width, hidden);
    const Vec x2 = muon_update(g2, width, hidden);
    Vec u1 = w1, u2 = w2;
    for (size_t q = 0; q < u1.size(); ++q) u1[q] = 0.95 * w1[q] - 0.1 * std::sqrt((double)hidden / width) * x1[q];
    for (size_t q = 0; q < u2.size(); ++q) u2[q] = 0.95 * w2[q] - 0.1 * x2[q];
    check("muon w1", mw1, u1, 1e-4);
    check("muon w2", mw2, u2, 1e-4);
    try {
        ops.linear(mx, m2, nullptr, Activation::None, nullptr, nullptr, my);
        std::printf("FAILED: no refusal\n");
        return 1;
    } catch (const std::runtime_error& e) {
        std::printf("refused: %s\n", e.what());
    }
    std::printf("network ok\n");
    return 0;
}
