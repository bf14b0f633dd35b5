// Top-k, sampling and distillation through the C++ host side (include/hpt_hip.hpp), on a device, against plain loops in double.
// Prints one line per failure; exit status 0 when all pass.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <numeric>
#include <random>

#include "hpt_hip.hpp"

using hpt::Tensor;
static int failures = 0, checks = 0;

// Tolerances: an f32 rounding is 6e-8 of the value; a sum of exponentials of n terms is off by at most n of them of itself (rows of 200 terms here), and
// exp adds its argument's rounding, 6e-8 times an argument below 16.
static void near(double got, double want, double tol, const char* what, size_t at) {
    ++checks;
    if (std::fabs(got - want) <= tol) return;
    if (++failures <= 20) printf("FAIL %s at %zu: got %.9g, want %.9g, tolerance %g\n", what, at, got, want, tol);
}
template <class F> static void expect_error(hpt::ErrorKind kind, const char* text, F f) {
    ++checks;
    try {
        f();
    } catch (const hpt::TensorError& e) {
        if (e.kind == kind && std::string(e.what()).find(text) != std::string::npos) return;
        printf("FAIL wrong error: kind %d, text '%s'\n", (int)e.kind, e.what());
        ++failures;
        return;
    }
    ++failures;
    printf("FAIL no error with '%s'\n", text);
}

int main() {
    const int64_t R = 6, V = 200, K = 9;
    const double tau = 1.5;
    std::mt19937 gen(7);
    std::normal_distribution<float> normal(0, 3);
    std::vector<float> x(R * V), t(R * V), u = {0.01f, 0.2f, 0.5f, 0.7f, 0.9f, 0.99f};
    for (float& v : x) v = normal(gen);
    for (float& v : t) v = normal(gen);
    auto tx = Tensor<float>::from_host(x, {R, V}), tt = Tensor<float>::from_host(t, {R, V}), tu = Tensor<float>::from_host(u, {R});

    auto [value, index, lse] = tt.topk_lse(K, tau);
    const auto vh = value.to_host(), lh = lse.to_host();
    const auto ih = index.to_host(), again = tt.topk(K).second.to_host();
    for (int64_t r = 0; r < R; ++r) {
        std::vector<int64_t> at(V);
        std::iota(at.begin(), at.end(), 0);
        std::stable_sort(at.begin(), at.end(), [&](int64_t a, int64_t b) { return t[r * V + a] > t[r * V + b]; });
        double sum = 0;
        for (int64_t j = 0; j < V; ++j) sum += std::exp(t[r * V + j] / tau);
        near(lh[r], std::log(sum), 2e-5, "lse", r);
        for (int64_t j = 0; j < K; ++j) {
            near((double)ih[r * K + j], (double)at[j], 0, "topk index", r * K + j);
            near((double)again[r * K + j], (double)at[j], 0, "topk index alone", r * K + j);
            near(vh[r * K + j], t[r * V + at[j]], 0, "topk value", r * K + j);
        }
    }

    hpt::SampleSettings settings;
    settings.temperature = 0.8, settings.top_k = 20, settings.top_p = 0.9;
    auto [token, logp] = tx.sample(tu, settings);
    std::vector<float> ps(R, 0.9f);
    auto tp = Tensor<float>::from_host(ps, {R});
    settings.top_ps = &tp, settings.top_p = 0.1;  // (the number is not looked at)
    const auto th = token.to_host(), th2 = tx.sample(tu, settings).first.to_host();
    const auto ph = logp.to_host();
    for (int64_t r = 0; r < R; ++r) {
        std::vector<int64_t> at(V);
        std::iota(at.begin(), at.end(), 0);
        std::stable_sort(at.begin(), at.end(), [&](int64_t a, int64_t b) { return x[r * V + a] > x[r * V + b]; });
        const double most = x[r * V + at[0]];
        auto weight = [&](int64_t i) { return std::exp((x[r * V + i] - most) / 0.8); };
        double all = 0, kept = 0, sum = 0;
        for (int j = 0; j < 20; ++j) all += weight(at[j]);
        size_t n = 0;
        while (kept < 0.9 * all) kept += weight(at[n++]);
        at.resize(n);
        std::sort(at.begin(), at.end());
        size_t k = 0;
        while (sum + weight(at[k]) <= u[r] * kept) sum += weight(at[k++]);
        near((double)th[r], (double)at[k], 0, "token", r);
        near((double)th2[r], (double)at[k], 0, "token by a row's own probability (f32)", r);
        near(ph[r], std::log(weight(at[k]) / kept), 1e-6, "logp", r);
    }

    std::vector<float> mask = {1, 0, 0.5f, 1, 1, 2};
    auto tm = Tensor<float>::from_host(mask, {R});
    for (int rest = 0; rest < 2; ++rest) {
        hpt::DistillTerms terms;
        terms.mask = &tm, terms.temperature = tau;
        if (rest) terms.teacher_lse = &lse;
        auto loss = tx.distill_loss(value, index, terms);
        const auto gh = tx.distill_loss_backward(value, index, loss.terms, tau, 2.0).to_host(), kh = loss.kl.to_host();
        double total = 0;
        for (int64_t r = 0; r < R; ++r) {
            if (mask[r] == 0) {
                near(kh[r], 0, 0, "kl of a row that does not count", r);
                continue;
            }
            double sum = 0, known = 0, left = 0, kl = 0;
            std::vector<double> p(V), q(V, 0.0), d(V);
            std::vector<char> named(V, 0);
            for (int64_t j = 0; j < V; ++j) sum += p[j] = std::exp(x[r * V + j] / tau);
            for (int64_t j = 0; j < K; ++j) {
                named[ih[r * K + j]] = 1;
                known += q[ih[r * K + j]] = std::exp(vh[r * K + j] / tau - (rest ? lh[r] : 0));
            }
            for (int64_t j = 0; j < V; ++j) {
                p[j] /= sum;
                if (!rest) q[j] /= known;
                if (!named[j]) left += p[j];
                if (q[j] > 0) kl += q[j] * std::log(q[j] / p[j]);
            }
            const double more = rest ? 1 - known : 0;
            if (more > 0) kl += more * std::log(more / left);
            total += mask[r] * kl;
            near(kh[r], kl, 5e-5, "kl", r);
            for (int64_t j = 0; j < V; ++j) {
                d[j] = p[j] - q[j] - (named[j] ? 0 : more * p[j] / left);
                near(gh[r * V + j], 2 * mask[r] * tau / 5.5 * d[j], 5e-5, "gradient of the logits", r * V + j);
            }
        }
        near(loss.loss.to_host()[0], tau * tau * total / 5.5, 2e-4, "loss", 0);
    }
    expect_error(hpt::ErrorKind::Param, "k is 201", [&] { tx.topk(201); });
    expect_error(hpt::ErrorKind::Param, "temperature", [&] {
        hpt::SampleSettings bad;
        bad.temperature = -1;
        tx.sample(tu, bad);
    });
    expect_error(hpt::ErrorKind::Shape, "Size mismatch", [&] { tx.distill_loss(value, Tensor<int64_t>::empty({R, K + 1})); });
    printf("%d checks, %d failures\n", checks, failures);
    return failures != 0;
}
