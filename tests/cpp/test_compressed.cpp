// test_compressed.cpp -- the decode operators on compressed data called through the
// C++20 header alpakann_b200/onHost.hpp: rotary, the 8-bit KV cache, 4-bit linear
// layers, against host loops in double, and their refusals. Needs a GPU.
#include <alpakann_b200/onHost.hpp>

#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

namespace b200 = alpaka::nn::b200;
namespace nn = alpaka::nn::onHost::nn;

static int g_failures = 0, g_checks = 0;

static void near(double actual, double expected, double tolerance, char const* what) {
    ++g_checks;
    if (!(std::fabs(actual - expected) <= tolerance) && ++g_failures < 20)
        std::fprintf(stderr, "FAIL %s: %.9g vs %.9g\n", what, actual, expected);
}

template <typename F>
static void refused(F&& f, char const* what) {
    ++g_checks;
    try {
        f();
    } catch (std::invalid_argument const&) {
        return;
    }
    ++g_failures;
    std::fprintf(stderr, "FAIL %s: not refused\n", what);
}

template <typename T>
struct Buffer {
    std::vector<T> host;
    T* dev = nullptr;
    explicit Buffer(std::size_t n, T fill = T{}) : host(n, fill) { cudaMalloc(&dev, n * sizeof(T)); }
    ~Buffer() { cudaFree(dev); }
    Buffer(Buffer const&) = delete;
    void upload() { cudaMemcpy(dev, host.data(), host.size() * sizeof(T), cudaMemcpyHostToDevice); }
    void download() { cudaMemcpy(host.data(), dev, host.size() * sizeof(T), cudaMemcpyDeviceToHost); }
};

int main() {
    int n = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        std::fprintf(stderr, "no CUDA device\n");
        return 2;
    }
    b200::Queue queue(0);
    std::mt19937 rng(5);
    std::normal_distribution<float> normal;
    constexpr int64_t B = 2, Hq = 4, Hkv = 2, D = 64, T = 48, block = 16, P = 16;
    int const exec = 0;

    // rotary of one new token, in place
    Buffer<float> q(B * Hq * D), k(B * Hkv * D), v(B * Hkv * D);
    for (auto* b : {&q, &k, &v})
        for (auto& x : b->host) x = normal(rng);
    q.upload(), k.upload(), v.upload();
    std::vector<float> const q0 = q.host, k0 = k.host;
    Buffer<int32_t> pos(B), len(B);
    pos.host = {20, 0};
    len.host = {21, 1};
    pos.upload(), len.upload();
    Buffer<double> freq(P);
    auto qv = b200::makeView<float, 4>(q.dev, {B, 1, Hq, D}), kv = b200::makeView<float, 4>(k.dev, {B, 1, Hkv, D});
    auto vv = b200::makeView<float, 4>(v.dev, {B, 1, Hkv, D});
    auto fv = b200::makeView<double, 1>(freq.dev, {P});
    auto pv = b200::makeView<int32_t, 2>(pos.dev, {B, 1});
    auto lv = b200::makeView<int32_t, 1>(len.dev, {B}), sv = b200::makeView<int32_t, 1>(pos.dev, {B});
    nn::rotaryFrequencies(queue, exec, fv);
    nn::rotary<float>(queue, exec, qv, kv, pv, fv, qv, kv, nn::RotaryPairs::halves);
    queue.wait(), q.download(), k.download(), freq.download();
    for (int64_t p = 0; p < P; ++p) near(freq.host[p], std::pow(1e4, -double(p) / P), 1e-12, "frequency");
    auto turned = [&](std::vector<float> const& x, int64_t row, int64_t b, int64_t d) {
        if (d >= 2 * P) return double(x[row * D + d]);
        double const a = pos.host[b] * freq.host[d % P], x1 = x[row * D + d % P], x2 = x[row * D + P + d % P];
        return d < P ? x1 * std::cos(a) - x2 * std::sin(a) : x1 * std::sin(a) + x2 * std::cos(a);
    };
    for (int64_t b = 0; b < B; ++b)
        for (int64_t d = 0; d < D; ++d) {
            for (int64_t h = 0; h < Hq; ++h) near(q.host[(b * Hq + h) * D + d], turned(q0, b * Hq + h, b, d), 4e-6, "rotary q");
            for (int64_t h = 0; h < Hkv; ++h) near(k.host[(b * Hkv + h) * D + d], turned(k0, b * Hkv + h, b, d), 4e-6, "rotary k");
        }

    // append to a part-filled cache, read back, attend
    Buffer<int8_t> kc(B * Hkv * T * D), vc(B * Hkv * T * D);
    Buffer<float> ks(B * Hkv * T / block, 0.01f), vs(B * Hkv * T / block, 0.02f);
    for (auto* c : {&kc, &vc})
        for (auto& x : c->host) x = static_cast<int8_t>(static_cast<int>(rng() % 255) - 127);
    kc.upload(), vc.upload(), ks.upload(), vs.upload();
    auto kcv = b200::makeView<int8_t, 4>(kc.dev, {B, Hkv, T, D}), vcv = b200::makeView<int8_t, 4>(vc.dev, {B, Hkv, T, D});
    auto ksv = b200::makeView<float, 3>(ks.dev, {B, Hkv, T / block}), vsv = b200::makeView<float, 3>(vs.dev, {B, Hkv, T / block});
    nn::kvCacheAppendQ8(queue, exec, kv, vv, kcv, vcv, ksv, vsv, sv, block);
    Buffer<float> ko(B * Hkv * T * D), vo(B * Hkv * T * D), out(B * Hq * D);
    auto kov = b200::makeView<float, 4>(ko.dev, {B, Hkv, T, D}), vov = b200::makeView<float, 4>(vo.dev, {B, Hkv, T, D});
    auto ov = b200::makeView<float, 4>(out.dev, {B, 1, Hq, D});
    nn::kvCacheReadQ8(queue, exec, kcv, vcv, ksv, vsv, kov, vov, block, &lv);
    nn::attentionDecodeQ8(queue, exec, qv, kcv, vcv, ksv, vsv, ov, block, &lv, 0.125f, 2u);
    queue.wait(), ko.download(), vo.download(), out.download(), ks.download();
    for (int64_t b = 0; b < B; ++b)
        for (int64_t h = 0; h < Hkv; ++h)
            for (int64_t d = 0; d < D; ++d) {
                int64_t const t = pos.host[b], at = ((b * Hkv + h) * T + t) * D + d;
                float const step = ks.host[(b * Hkv + h) * (T / block) + t / block];
                near(ko.host[at], k.host[(b * Hkv + h) * D + d], 0.501 * step, "appended row");
            }
    for (int64_t b = 0; b < B; ++b)
        for (int64_t h = 0; h < Hq; ++h) {
            std::vector<double> s(len.host[b]), o(D);
            double sum = 0;
            for (int64_t j = 0; j < len.host[b]; ++j) {
                for (int64_t d = 0; d < D; ++d)
                    s[j] += double(q.host[(b * Hq + h) * D + d]) * ko.host[((b * Hkv + h / 2) * T + j) * D + d];
                sum += s[j] = std::exp(0.125 * s[j]);
            }
            for (int64_t j = 0; j < len.host[b]; ++j)
                for (int64_t d = 0; d < D; ++d) o[d] += s[j] / sum * vo.host[((b * Hkv + h / 2) * T + j) * D + d];
            for (int64_t d = 0; d < D; ++d) near(out.host[(b * Hq + h) * D + d], o[d], 1e-4, "attention");
        }

    // a 4-bit layer with bias, activation and residual
    constexpr int64_t K = 96, N = 20, group = 32;
    Buffer<float> w(K * N), sc(K / group * N), x(2 * K), bias(N, 0.25f), y(2 * N, 1.0f);
    Buffer<int32_t> packed(K / 8 * N);
    for (auto& e : w.host) e = normal(rng);
    for (auto& e : x.host) e = normal(rng);
    w.upload(), x.upload(), bias.upload(), y.upload();
    auto wv = b200::makeView<float, 2>(w.dev, {K, N}), scv = b200::makeView<float, 2>(sc.dev, {K / group, N});
    auto packedv = b200::makeView<int32_t, 2>(packed.dev, {K / 8, N});
    auto xv = b200::makeView<float, 2>(x.dev, {2, K}), yv = b200::makeView<float, 2>(y.dev, {2, N});
    auto biasv = b200::makeView<float, 1>(bias.dev, {N});
    nn::packWeightQ4(queue, exec, wv, packedv, scv, group);
    nn::linearQ4(queue, exec, xv, packedv, scv, yv, group, &biasv, nn::Activation::relu, &yv);
    queue.wait(), packed.download(), sc.download(), y.download();
    for (int64_t m = 0; m < 2; ++m)
        for (int64_t c = 0; c < N; ++c) {
            double sum = 0.25;
            for (int64_t i = 0; i < K; ++i) {
                int const u = static_cast<int>(static_cast<uint32_t>(packed.host[i / 8 * N + c]) >> (4 * (i % 8)) & 15u);
                float const s = sc.host[i / group * N + c];
                if (m == 0) near((u - 8) * s, w.host[i * N + c], 0.501 * s, "packed weight");
                sum += double(x.host[m * K + i]) * (u - 8) * s;
            }
            near(y.host[m * N + c], (sum > 0 ? sum : 0) + 1, 1e-4, "linear");
        }

    refused([&] { nn::linearQ4(queue, exec, xv, packedv, scv, yv, 64u); }, "group size");
    refused([&] { nn::attentionDecodeQ8(queue, exec, qv, kcv, vcv, ksv, vsv, ov, 32u, &lv, 0.1f, 2u); }, "tokens a scale");
    refused([&] { nn::kvCacheAppendQ8(queue, exec, qv, vv, kcv, vcv, ksv, vsv, sv, block); }, "row heads");
    std::printf("%d checks, %d failures\n", g_checks, g_failures);
    return g_failures == 0 ? 0 : 1;
}
