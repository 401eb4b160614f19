// Layer norm of the C++ host layer with one of its two parameters or neither: a gradient for each that is there, of length 0 for the other.  `gpu`: against double, values
// below 16 that a few dozen roundings to f32 (2^-24 of them each) lead to: 1e-5.
#include <cmath>
#include <cstdio>

#include "autograph_hip.hpp"

using namespace agh;

#define REQUIRE(cond)                                                             \
    do {                                                                          \
        if (!(cond)) {                                                            \
            std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #cond);       \
            return 1;                                                             \
        }                                                                         \
    } while (0)

static int run_gpu() {
    Device device(0);
    const int64_t m = 6, k = 40;
    std::vector<float> x((size_t)(m * k)), dy((size_t)(m * k)), g((size_t)k), b((size_t)k);
    for (size_t i = 0; i < x.size(); ++i) x[i] = (float)((i * 7) % 23) / 4.0f - 2.0f, dy[i] = (float)((i * 13) % 17) / 8.0f - 1.0f;
    for (size_t j = 0; j < g.size(); ++j) g[j] = 1.0f + (float)(j % 5) / 8.0f, b[j] = (float)(j % 3) - 1.0f;
    const Tensor<float> tx = Tensor<float>::from_vec({m, k}, x), tdy = Tensor<float>::from_vec({m, k}, dy);
    const auto tg = std::make_shared<Tensor<float>>(Tensor<float>::from_vec({k}, g)), tb = std::make_shared<Tensor<float>>(Tensor<float>::from_vec({k}, b));
    for (int which = 0; which < 4; ++which) {
        const LayerNorm<float> norm{which & 1 ? tg : nullptr, which & 2 ? tb : nullptr};
        const auto fwd = norm.forward_train(tx);
        const auto grads = norm.backward(tx, tdy, fwd.mean, fwd.rstd);
        REQUIRE(grads.weight.len() == (which & 1 ? k : 0) && grads.bias.len() == (which & 2 ? k : 0));
        const std::vector<float> y = fwd.y.into_vec(), dx = grads.input.into_vec(), dg = grads.weight.into_vec(), db = grads.bias.into_vec();
        std::vector<double> sg((size_t)k), sb((size_t)k);
        for (int64_t i = 0; i < m; ++i) {
            double mean = 0, var = 0, s1 = 0, s2 = 0;
            const size_t row = (size_t)(i * k);
            const auto factor = [&](int64_t j) { return which & 1 ? (double)g[(size_t)j] : 1.0; };
            for (int64_t j = 0; j < k; ++j) mean += x[row + (size_t)j] / (double)k;
            for (int64_t j = 0; j < k; ++j) var += (x[row + (size_t)j] - mean) * (x[row + (size_t)j] - mean) / (double)k;
            const double rstd = 1 / std::sqrt(var + 1e-5);
            for (int64_t j = 0; j < k; ++j) {
                const double h = (x[row + (size_t)j] - mean) * rstd, q = dy[row + (size_t)j] * factor(j);
                REQUIRE(std::fabs(y[row + (size_t)j] - (h * factor(j) + (which & 2 ? b[(size_t)j] : 0.0f))) < 1e-5);
                s1 += q / (double)k, s2 += q * h / (double)k, sg[(size_t)j] += dy[row + (size_t)j] * h, sb[(size_t)j] += dy[row + (size_t)j];
            }
            for (int64_t j = 0; j < k; ++j) {
                const double h = (x[row + (size_t)j] - mean) * rstd, q = dy[row + (size_t)j] * factor(j);
                REQUIRE(std::fabs(dx[row + (size_t)j] - rstd * (q - s1 - h * s2)) < 1e-5);
            }
        }
        for (size_t j = 0; j < dg.size(); ++j) REQUIRE(std::fabs(dg[j] - sg[j]) < 1e-5);
        for (size_t j = 0; j < db.size(); ++j) REQUIRE(std::fabs(db[j] - sb[j]) < 1e-5);
    }
    std::puts("gpu ok");
    return 0;
}

int main(int argc, char **argv) {
    try {
        if (argc == 2 && std::string(argv[1]) == "gpu") return run_gpu();
    } catch (const Error &e) {
        std::fprintf(stderr, "agh::Error [%d]: %s\n", e.code(), e.what());
        return 3;
    }
    std::fprintf(stderr, "usage: layer_norm_parameters_test gpu\n");
    return 64;
}
