// The operators around a transformer's blocks through the C++ host side (include/hpt_hip.hpp), on a device, against plain loops in
// double. Prints one line per failure; exit status 0 when all pass.
#include <cmath>
#include <cstdio>
#include <random>

#include "hpt_hip.hpp"

using hpt::Tensor;
static int failures = 0, checks = 0;

// Tolerances: an f32 rounding is 6e-8 of the value; a sum of n terms is off by at most n of them of the sum of the terms' sizes
// (rows of at most 100 terms here, of size 5 at most), and exp adds its argument's rounding, 6e-8 times an argument below 16.
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

static std::mt19937 gen(7);
static std::vector<float> normal(size_t n, float mean = 0, float sd = 1) {
    std::normal_distribution<float> d(mean, sd);
    std::vector<float> v(n);
    for (float& x : v) x = d(gen);
    return v;
}

static void norm() {
    const int64_t R = 7, C = 100;
    const auto x = normal(R * C), r = normal(R * C), g = normal(C, 1, 0.2f), gy = normal(R * C);
    auto tx = Tensor<float>::from_host(x, {R, C}), tr = Tensor<float>::from_host(r, {R, C}), tg = Tensor<float>::from_host(g, {C}), ty = Tensor<float>::from_host(gy, {R, C});
    auto [y, h] = tx.add_rms_norm(tr, {C}, &tg);
    auto plain = tx.rms_norm({C}, nullptr).to_host();
    auto [q, s] = tx.rms_norm_quant<int8_t>({C}, &tg, 1e-6, 25);
    auto [q8, s8] = tx.rms_norm_quant<uint8_t>({C}, &tg);
    auto [gx, gg] = tx.rms_norm_backward(ty, {C}, &tg, 1e-6, &tr);
    const auto yh = y.to_host(), hh = h.to_host(), gxh = gx.to_host(), ggh = gg.to_host(), sh = s.to_host(), s8h = s8.to_host();
    const auto qh = q.to_host();
    std::vector<double> want(C, 0.0);
    for (int64_t i = 0; i < R; ++i) {
        double sx = 0, shh = 0, c = 0, most = 0;
        for (int64_t j = 0; j < C; ++j) {
            const size_t k = i * C + j;
            near(hh[k], (float)(x[k] + r[k]), 0, "sum", k);
            sx += (double)x[k] * x[k], shh += (double)hh[k] * hh[k], c += (double)gy[k] * g[j] * x[k];
        }
        const double rx = 1 / std::sqrt(sx / C + 1e-6), rh = 1 / std::sqrt(shh / C + 1e-6);
        for (int64_t j = 0; j < C; ++j) {
            const size_t k = i * C + j;
            near(yh[k], hh[k] * rh * g[j], 64 * 6e-8 * std::fabs(hh[k] * rh * g[j]), "add_rms_norm", k);
            near(plain[k], x[k] * rx, 64 * 6e-8 * std::fabs(x[k] * rx), "rms_norm", k);
            const double d = rx * (gy[k] * (double)g[j] - x[k] * rx * rx * c / C) + r[k];
            near(gxh[k], d, 128 * 6e-8 * (4 + std::fabs(d)), "gradient", k);
            want[j] += gy[k] * (double)x[k] * rx;
            const double v = x[k] * rx * g[j], step = sh[i * 4 + j / 25];
            near(qh[k] * step, v, step * 0.5001 + 1e-5, "8 bits", k);
            most = std::fmax(most, std::fabs(v));
        }
        near(s8h[i], most / 448, most / 448 * 1e-5, "scale of e4m3", i);
    }
    for (int64_t j = 0; j < C; ++j) near(ggh[j], want[j], 1e-4, "gradient of gamma", j);
    expect_error(hpt::ErrorKind::Shape, "normalized dims", [&] { tx.rms_norm({C + 1}, nullptr); });
    expect_error(hpt::ErrorKind::Param, "eps", [&] { tx.rms_norm({C}, nullptr, 0.0); });
}

static void bias() {
    const int64_t H = 2, Q = 9, K = 13, N = 8;
    const auto x = normal(H * Q * K, 0, 3), t = normal(N * H), g = normal(H * Q * K);
    auto tx = Tensor<float>::from_host(x, {H, Q, K}), tt = Tensor<float>::from_host(t, {N, H}), tg = Tensor<float>::from_host(g, {H, Q, K});
    hpt::PositionBias b;
    b.scale = 0.5, b.bidirectional = false, b.max_distance = 9, b.query_offset = 4, b.causal = true;
    auto p = tx.softmax_bias(tt, b);
    auto [gs, gt] = p.softmax_bias_backward(tg, N, b);
    const auto ph = p.to_host(), gsh = gs.to_host(), gth = gt.to_host();
    std::vector<double> table(N * H, 0.0);
    for (int64_t h = 0; h < H; ++h)
        for (int64_t i = 0; i < Q; ++i) {
            const int64_t live = std::min(K, i + 5);
            std::vector<double> e(K, 0.0);
            std::vector<int64_t> at(K, 0);
            double sum = 0, dot = 0;
            for (int64_t j = 0; j < live; ++j) {
                const int64_t d = i + 4 - j;  // four buckets of one distance, four that grow to 9
                at[j] = d < 4 ? d : std::min<int64_t>(7, 4 + (int64_t)std::floor(std::log(d / 4.0) / std::log(9 / 4.0) * 4 + 1e-9));
                e[j] = std::exp(0.5 * x[(h * Q + i) * K + j] + t[at[j] * H + h]);
                sum += e[j];
            }
            for (int64_t j = 0; j < K; ++j) dot += ph[(h * Q + i) * K + j] * (double)g[(h * Q + i) * K + j];
            for (int64_t j = 0; j < K; ++j) {
                const size_t k = (h * Q + i) * K + j;
                near(ph[k], e[j] / sum, 1e-5 * e[j] / sum, "softmax_bias", k);
                const double d = ph[k] * (g[k] - dot);
                near(gsh[k], 0.5 * d, 4e-6, "gradient of the scores", k);
                if (j < live) table[at[j] * H + h] += d;
            }
        }
    for (size_t k = 0; k < table.size(); ++k) near(gth[k], table[k], 1e-5, "gradient of the table", k);
    expect_error(hpt::ErrorKind::Param, "max_distance", [&] {
        hpt::PositionBias bad;
        bad.max_distance = 1;
        tx.softmax_bias(tt, bad);
    });
}

static void policy() {
    const int64_t R = 5, V = 37;
    const auto x = normal(R * V, 0, 2), adv = normal(R), shift = normal(R, 0, 0.3f);
    std::vector<int64_t> token = {3, 0, 36, 11, -100};
    std::vector<float> mask = {1, 1, 0.5f, 1, 0}, old(R), ref(R);
    auto tx = Tensor<float>::from_host(x, {R, V});
    auto tok = Tensor<int64_t>::from_host(token, {R});
    auto [lp, ls] = tx.token_logp(tok);
    const auto lph = lp.to_host();
    for (int64_t i = 0; i < R; ++i) old[i] = token[i] < 0 ? 0 : lph[i] + shift[i], ref[i] = old[i] - 0.5f * shift[i];
    auto to = Tensor<float>::from_host(old, {R}), ta = Tensor<float>::from_host(adv, {R}), tr = Tensor<float>::from_host(ref, {R}), tm = Tensor<float>::from_host(mask, {R});
    hpt::PolicyTerms terms;
    terms.reference = &tr, terms.mask = &tm, terms.kl_weight = 0.1;
    auto loss = tx.policy_loss(tok, to, ta, terms);
    auto grad = tx.policy_loss_backward(tok, loss.lse, loss.weight, 2.0);
    const auto gh = grad.to_host(), wh = loss.weight.to_host();
    double want = 0;
    for (int64_t i = 0; i < R; ++i) {
        if (token[i] < 0) {
            near(wh[i], 0, 0, "weight of a row that does not count", i);
            continue;
        }
        double sum = 0;
        for (int64_t j = 0; j < V; ++j) sum += std::exp((double)x[i * V + j]);
        const double logp = x[i * V + token[i]] - std::log(sum), ratio = std::exp(logp - old[i]), k = ref[i] - logp;
        const double free = ratio * adv[i], held = std::fmin(std::fmax(ratio, 0.8), 1.2) * adv[i];
        want += mask[i] * (-std::fmin(free, held) + 0.1 * (std::exp(k) - k - 1)) / 3.5;
        const double w = mask[i] * ((free <= held ? -free : 0.0) + 0.1 * (1 - std::exp(k))) / 3.5;
        near(lph[i], logp, 1e-5, "token_logp", i);
        near(wh[i], w, 1e-5, "weight", i);
        for (int64_t j = 0; j < V; ++j) near(gh[i * V + j], 2 * w * ((j == token[i]) - std::exp((double)x[i * V + j]) / sum), 2e-5, "gradient of the logits", i * V + j);
    }
    near(loss.loss.to_host()[0], want, 1e-5, "loss", 0);
}

int main() {
    norm();
    bias();
    policy();
    printf("%d checks, %d failures\n", checks, failures);
    return failures != 0;
}
