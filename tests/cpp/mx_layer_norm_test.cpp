// Layer norm and MXFP4 through the C++ host layer (include/autograph_hip.hpp).  `cpu`: sizes and refusals, without a device; `gpu`: every result against the same
// formulas in double, on values that the format holds exactly, so that only the order of f32 sums is left.
#include <cmath>
#include <cstdio>
#include <cstdlib>

#include "autograph_hip.hpp"

using namespace agh;

#define REQUIRE(cond)                                                             \
    do {                                                                          \
        if (!(cond)) {                                                            \
            std::fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #cond);       \
            return 1;                                                             \
        }                                                                         \
    } while (0)

template <typename F> static bool refused(F f) {
    try {
        f();
    } catch (const Error &e) {
        return e.code() == AGH_EINVAL;
    }
    return false;
}

static int run_cpu() {
    size_t codes = 0, scales = 0;
    check(agh_mxfp4_bytes(17, 129, &codes, &scales));
    REQUIRE(codes == 2 * 2 * 1024 && scales == 1 * 2 * 256);
    REQUIRE(refused([&] { check(agh_mxfp4_bytes(-1, 1, &codes, &scales)); }));
    REQUIRE(refused([] { MxTensor(3, 4, 2); }));
    std::puts("cpu ok");
    return 0;
}

static int run_gpu() {
    Device device(0);
    const int64_t m = 37, k = 96, n = 50;
    // small integers with a 4 in every block: what they stand for in the format is themselves
    std::vector<float> x((size_t)(m * k)), w((size_t)(k * n)), b((size_t)n);
    for (int64_t i = 0; i < m; ++i)
        for (int64_t j = 0; j < k; ++j) x[(size_t)(i * k + j)] = j % 32 == 0 ? 4.0f : (float)((i * 7 + j * 3) % 5) - 2.0f;
    for (int64_t i = 0; i < k; ++i)
        for (int64_t j = 0; j < n; ++j) w[(size_t)(i * n + j)] = i % 32 == 0 ? -4.0f : (float)((i * 5 + j * 11) % 7) / 2.0f - 1.5f;
    for (int64_t j = 0; j < n; ++j) b[(size_t)j] = (float)(j % 9) - 4.0f;
    for (float &v : w)
        if (std::fabs(v) == 1.5f) v = 1.0f;
    const Tensor<float> tx = Tensor<float>::from_vec({m, k}, x), tw = Tensor<float>::from_vec({k, n}, w);
    const auto tb = std::make_shared<Tensor<float>>(Tensor<float>::from_vec({n}, b));
    const MxTensor qx = tx.quantize_mxfp4(), qw = tw.quantize_mxfp4(0);
    REQUIRE(qx.dequantize<float>().into_vec() == x && qw.dequantize<float>().into_vec() == w);
    REQUIRE(qw.t().dequantize<float>().into_vec() == tw.t().into_vec());
    std::vector<float> want((size_t)(m * n));
    for (int64_t i = 0; i < m; ++i)
        for (int64_t j = 0; j < n; ++j) {
            double s = b[(size_t)j];
            for (int64_t l = 0; l < k; ++l) s += (double)x[(size_t)(i * k + l)] * w[(size_t)(l * n + j)];
            want[(size_t)(i * n + j)] = s > 0 ? (float)s : 0.0f;
        }
    REQUIRE(qx.dot<float>(qw, tb.get(), true).into_vec() == want);  // sums of halves below 2^24: exact
    const MxDense<float> layer{qw, tb};
    REQUIRE(layer.forward(tx, true).into_vec() == want);
    const std::vector<bf16> half = qx.dot<bf16>(qw).into_vec();
    const std::vector<float> whole = qx.dot<float>(qw).into_vec();
    for (size_t i = 0; i < half.size(); ++i) REQUIRE(half[i].bits == bf16::from_f32(whole[i]).bits);
    REQUIRE(refused([&] { qx.dot<float>(qw.t()); }) && refused([&] { qw.dot<float>(qx); }) && refused([&] { layer.forward(tx.t()); }) && refused([&] { tb->quantize_mxfp4(); }));

    // layer norm: gradients against double
    std::vector<float> g((size_t)k), h((size_t)k), dy((size_t)(m * k));
    for (int64_t j = 0; j < k; ++j) g[(size_t)j] = 1.0f + (float)(j % 5) / 8.0f, h[(size_t)j] = (float)(j % 3) - 1.0f;
    for (size_t i = 0; i < dy.size(); ++i) dy[i] = (float)((i * 13) % 17) / 8.0f - 1.0f;
    const LayerNorm<float> norm{std::make_shared<Tensor<float>>(Tensor<float>::from_vec({k}, g)), std::make_shared<Tensor<float>>(Tensor<float>::from_vec({k}, h))};
    const auto fwd = norm.forward_train(tx);
    REQUIRE(norm.forward(tx).into_vec() == fwd.y.into_vec());
    const auto grads = tx.layer_norm_backward(Tensor<float>::from_vec({m, k}, dy), *norm.weight, fwd.mean, fwd.rstd);
    const std::vector<float> y = fwd.y.into_vec(), dx = grads.input.into_vec(), dg = grads.weight.into_vec(), dh = grads.bias.into_vec();
    std::vector<double> sg((size_t)k), sh((size_t)k);
    for (int64_t i = 0; i < m; ++i) {
        double mean = 0, var = 0, s1 = 0, s2 = 0;
        for (int64_t j = 0; j < k; ++j) mean += x[(size_t)(i * k + j)] / (double)k;
        for (int64_t j = 0; j < k; ++j) var += (x[(size_t)(i * k + j)] - mean) * (x[(size_t)(i * k + j)] - mean) / (double)k;
        const double rstd = 1 / std::sqrt(var + 1e-5);
        for (int64_t j = 0; j < k; ++j) {
            const size_t at = (size_t)(i * k + j);
            const double e = (x[at] - mean) * rstd, q = (double)dy[at] * g[(size_t)j];
            REQUIRE(std::fabs(y[at] - (e * g[(size_t)j] + h[(size_t)j])) < 1e-5);
            s1 += q / (double)k, s2 += q * e / (double)k, sg[(size_t)j] += dy[at] * e, sh[(size_t)j] += dy[at];
        }
        for (int64_t j = 0; j < k; ++j) {
            const size_t at = (size_t)(i * k + j);
            const double e = (x[at] - mean) * rstd, q = (double)dy[at] * g[(size_t)j];
            REQUIRE(std::fabs(dx[at] - rstd * (q - s1 - e * s2)) < 1e-5);
        }
    }
    for (size_t j = 0; j < sg.size(); ++j) REQUIRE(std::fabs(dg[j] - sg[j]) < 1e-4 && std::fabs(dh[j] - sh[j]) < 1e-4);
    REQUIRE(refused([&] { tx.layer_norm(tb.get(), nullptr); }) && refused([&] { tx.layer_norm_backward(tw, *norm.weight, fwd.mean, fwd.rstd); }));
    std::puts("gpu ok");
    return 0;
}

int main(int argc, char **argv) {
    try {
        if (argc == 2 && std::string(argv[1]) == "cpu") return run_cpu();
        if (argc == 2 && std::string(argv[1]) == "gpu") return run_gpu();
    } catch (const Error &e) {
        std::fprintf(stderr, "agh::Error [%d]: %s\n", e.code(), e.what());
        return 3;
    }
    std::fprintf(stderr, "usage: mx_layer_norm_test cpu | gpu\n");
    return 64;
}
