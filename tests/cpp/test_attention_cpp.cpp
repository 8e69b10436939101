// The attention operators of the C++ interface (include/t2h.hpp, t2h::gpu)
// against their definitions in double. Errors are compared with a share of
// the sum of the terms' magnitudes: f16 rounds each probability and the output
// by at most 2^-11 of it, so 2^-9 holds them with the f32 arithmetic. An output
// below 2^-14 is stored in steps of 2^-24 whatever the terms are, off by at most
// 2^-25 (dv of one query and 200 keys: P dout is mostly below 1e-4).
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <random>
#include <string>
#include <vector>

#include "t2h.hpp"

using namespace t2h;

namespace {

int failed = 0;

void expect(bool ok, const std::string& what) {
    if (!ok) {
        std::printf("FAIL %s\n", what.c_str());
        ++failed;
    }
}

std::vector<float> randn(int64_t n, int seed, float std = 1.0f) {
    std::mt19937 g(seed);
    std::normal_distribution<float> d(0.0f, std);
    std::vector<float> v((size_t)n);
    for (float& x : v) x = d(g);
    return v;
}

struct Problem {
    int64_t rows, keys, h, kvh, d;
    Tensor q, k, v, g;
    std::vector<float> hq, hk, hv, hg;
    Problem(int64_t rows_, int64_t keys_, int64_t h_, int64_t kvh_, int64_t d_)
        : rows(rows_), keys(keys_), h(h_), kvh(kvh_), d(d_) {
        q = Tensor::from_host(randn(rows * h * d, 1).data(), {rows, h, d}, F16);
        k = Tensor::from_host(randn(keys * kvh * d, 2).data(), {keys, kvh, d}, F16);
        v = Tensor::from_host(randn(keys * kvh * d, 3).data(), {keys, kvh, d}, F16);
        g = Tensor::from_host(randn(rows * h * d, 4, 0.5f).data(), {rows, h, d}, F16);
        hq = q.to_host();
        hk = k.to_host();
        hv = v.to_host();
        hg = g.to_host();
    }
};

void near(const std::vector<float>& got, const std::vector<double>& want, const std::vector<double>& size,
          const std::string& what) {
    double worst = 0;
    for (size_t i = 0; i < got.size(); ++i) {
        const double e = std::max(0.0, std::fabs(got[i] - want[i]) - std::ldexp(1.0, -25)) / (size[i] + 1e-12);
        if (!(e <= worst)) worst = e;
    }
    std::printf("%s: worst %.2e of the terms\n", what.c_str(), worst);
    expect(worst <= 1.0 / 512, what);
}

void attention_and_gradients(int64_t rows, int64_t keys, int64_t h, int64_t kvh, int64_t d) {
    const std::string name = "attention " + std::to_string(rows) + "x" + std::to_string(keys);
    Problem p(rows, keys, h, kvh, d);
    const gpu::Attention a = gpu::attention(p.q, p.k, p.v);
    const std::vector<float> out = a.out.to_host(), lse = a.lse.to_host();
    const double scale = 1.0 / std::sqrt((double)d);
    std::vector<double> o(out.size()), os(out.size()), dq(out.size()), dqs(out.size());
    std::vector<double> dk(p.hk.size()), dks(p.hk.size()), dv(p.hv.size()), dvs(p.hv.size());
    for (int64_t i = 0; i < rows; ++i)
        for (int64_t hh = 0; hh < h; ++hh) {
            const float* qi = &p.hq[(size_t)((i * h + hh) * d)];
            const float* gi = &p.hg[(size_t)((i * h + hh) * d)];
            const int64_t j2 = hh / (h / kvh);
            std::vector<double> s((size_t)keys);
            double top = -1e300, sum = 0;
            for (int64_t j = 0; j < keys; ++j) {
                const float* kj = &p.hk[(size_t)((j * kvh + j2) * d)];
                double x = 0;
                for (int64_t e = 0; e < d; ++e) x += (double)qi[e] * kj[e];
                s[(size_t)j] = x * scale;
                top = std::max(top, s[(size_t)j]);
            }
            for (double x : s) sum += std::exp(x - top);
            const double l = top + std::log(sum);
            expect(std::fabs(l - lse[(size_t)(hh * rows + i)]) < 1e-4, name + " lse");
            double delta = 0, mag = 0;
            for (int64_t e = 0; e < d; ++e) {
                const double x = (double)gi[e] * out[(size_t)((i * h + hh) * d + e)];
                delta += x;
                mag += std::fabs(x);
            }
            for (int64_t j = 0; j < keys; ++j) {
                const double pr = std::exp(s[(size_t)j] - l);
                const size_t kr = (size_t)((j * kvh + j2) * d), qr = (size_t)((i * h + hh) * d);
                double dp = 0, m = mag;
                for (int64_t e = 0; e < d; ++e) {
                    dp += (double)gi[e] * p.hv[kr + (size_t)e];
                    m += std::fabs((double)gi[e] * p.hv[kr + (size_t)e]);
                }
                const double ds = pr * (dp - delta) * scale, dm = pr * m * scale;
                for (int64_t e = 0; e < d; ++e) {
                    o[qr + (size_t)e] += pr * p.hv[kr + (size_t)e];
                    os[qr + (size_t)e] += pr * std::fabs(p.hv[kr + (size_t)e]);
                    dq[qr + (size_t)e] += ds * p.hk[kr + (size_t)e];
                    dqs[qr + (size_t)e] += dm * std::fabs(p.hk[kr + (size_t)e]);
                    dk[kr + (size_t)e] += ds * qi[e];
                    dks[kr + (size_t)e] += dm * std::fabs(qi[e]);
                    dv[kr + (size_t)e] += pr * gi[e];
                    dvs[kr + (size_t)e] += pr * std::fabs(gi[e]);
                }
            }
        }
    near(out, o, os, name + " out");
    const gpu::AttentionGrads g = gpu::attention_backward(p.g, p.q, p.k, p.v, a);
    near(g.dq.to_host(), dq, dqs, name + " dq");
    near(g.dk.to_host(), dk, dks, name + " dk");
    near(g.dv.to_host(), dv, dvs, name + " dv");
}

void head_major_operands() {
    const int64_t rows = 100, h = 4, d = 64, mp = 128;
    const Tensor qkv = Tensor::from_host(randn(rows * 3 * h * d, 7).data(), {rows, 3 * h * d}, F16);
    const gpu::AttnOperands o = gpu::attn_pack(qkv, (int32_t)h, Tensor(), Tensor(), Tensor(), gpu::Rope(), mp, mp, false);
    const gpu::Attention a = gpu::attention(o, rows);
    // the same rows, token-major; 1 / sqrt(64) is a power of two, so the packed q is exact
    const std::vector<float> all = qkv.to_host();
    std::vector<float> part[3];
    for (int t = 0; t < 3; ++t)
        for (int64_t r = 0; r < rows; ++r)
            for (int64_t e = 0; e < h * d; ++e) part[t].push_back(all[(size_t)((r * 3 + t) * h * d + e)]);
    const gpu::Attention b = gpu::attention(Tensor::from_values({rows, h, d}, part[0], F16),
                                            Tensor::from_values({rows, h, d}, part[1], F16),
                                            Tensor::from_values({rows, h, d}, part[2], F16));
    const std::vector<float> x = a.out.to_host(), y = b.out.to_host();
    expect(std::memcmp(x.data(), y.data(), x.size() * 4) == 0, "head-major operands");
}

void epilogue_gradient() {
    const int64_t rows = 50, h = 4, d = 64;
    const Tensor x = Tensor::from_host(randn(rows * h * d, 8).data(), {rows, h, d});
    const Tensor dy = Tensor::from_host(randn(rows * h * d, 9).data(), {rows, h, d});
    const Tensor gamma = Tensor::from_host(randn(h * d, 10).data(), {h, d});
    const gpu::QkGrads g = gpu::qk_rmsnorm_rope_backward(dy, x, gamma);
    const std::vector<float> hx = x.to_host(), hy = dy.to_host(), hg = gamma.to_host();
    const std::vector<float> dx = g.dx.to_host(), dg = g.dgamma.to_host();
    expect(!g.dbias.defined(), "no bias, no gradient of it");
    std::vector<double> sum((size_t)(h * d));
    double worst = 0;
    for (int64_t r = 0; r < rows; ++r)
        for (int64_t i = 0; i < h; ++i) {
            const size_t at = (size_t)((r * h + i) * d);
            double n = 0, dot = 0;
            for (int64_t e = 0; e < d; ++e) n += (double)hx[at + (size_t)e] * hx[at + (size_t)e];
            n = std::sqrt(n);
            const double sc = std::sqrt((double)d);
            for (int64_t e = 0; e < d; ++e) dot += hy[at + (size_t)e] * hg[(size_t)(i * d + e)] * sc * hx[at + (size_t)e] / n;
            for (int64_t e = 0; e < d; ++e) {
                const double xh = hx[at + (size_t)e] / n;
                const double want = (hy[at + (size_t)e] * hg[(size_t)(i * d + e)] * sc - xh * dot) / n;
                worst = std::max(worst, std::fabs(want - dx[at + (size_t)e]));
                sum[(size_t)(i * d + e)] += hy[at + (size_t)e] * xh * sc;
            }
        }
    for (size_t c = 0; c < sum.size(); ++c) worst = std::max(worst, std::fabs(sum[c] - dg[c]));
    std::printf("epilogue gradients: worst %.2e\n", worst);
    expect(worst < 1e-4, "epilogue gradients");     // values up to 20, f32 sums of 64 terms
}

void errors(bool device) {
    const auto throws = [](const std::function<void()>& f) {
        try {
            f();
        } catch (const Error&) {
            return true;
        }
        return false;
    };
    expect(throws([] { gpu::detail::workspace(t2h_attention_workspace(-1, 1, 1, 1, 64, 1)); }), "negative rows");
    expect(throws([] { gpu::detail::workspace(t2h_attention_backward_workspace(1, 1, 3, 2, 64, 1)); }), "heads over kv heads");
    if (!device) return;
    const Tensor q = Tensor::zeros({4, 2, 64}, F16), k = Tensor::zeros({4, 2, 64}, F16), f = Tensor::zeros({4, 2, 64});
    expect(throws([&] { gpu::attention(q, k, f); }), "types differ");
    expect(throws([&] { gpu::attention(f, f, f); }), "f32 operands");
    expect(throws([&] { gpu::attention(q, k, k, -1.0f); }), "negative scale");
}

}  // namespace

int main(int argc, char** argv) {
    const bool host = argc > 1 && std::strcmp(argv[1], "--host") == 0;
    errors(!host);
    if (!host) {
        check(t2h_device_init(0));
        attention_and_gradients(70, 90, 2, 1, 64);
        attention_and_gradients(1, 200, 2, 2, 128);
        attention_and_gradients(33, 17, 2, 2, 128);
        head_major_operands();
        epilogue_gradient();
    }
    std::printf(failed ? "%d failed\n" : "all passed\n", failed);
    return failed != 0;
}
