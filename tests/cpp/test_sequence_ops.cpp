// The gated recurrence, 8-bit checkpoints and the softmax cross-entropy through the C++ host mirror.
// Exit code 0 = all passed; prints the first failure otherwise.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "rtensors_b200.hpp"

using namespace rtb200;
template <typename T> using Tensor = TensorBase<T>;

static int g_checks = 0;
#define ASSERT_TRUE(x)                                                              \
    do {                                                                            \
        ++g_checks;                                                                 \
        if (!(x)) { std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #x); std::exit(1); } \
    } while (0)

static double value(int i) { return std::sin(0.7 * i) * 2.0; }

int main() {
    Cuda cuda(0);
    const size_t B = 2, S = 9, D = 5;
    std::vector<double> x, a, h0;
    for (size_t i = 0; i < B * S * D; ++i) x.push_back(value((int)i)), a.push_back(0.5 + 0.4 * std::cos(0.3 * i));
    for (size_t i = 0; i < B * D; ++i) h0.push_back(value((int)i + 1000));
    auto tx = Tensor<double>::from_buf(cuda, x, {B, S, D}), ta = Tensor<double>::from_buf(cuda, a, {B, S, D});
    auto t0 = Tensor<double>::from_buf(cuda, h0, {B, 1, D});
    {  // both directions, coupled and not, against the loop
        for (int flags = 0; flags < 4; ++flags) {
            const auto got = tx.gated_scan_at(1, ta, &t0, flags).cpu();
            for (size_t b = 0; b < B; ++b)
                for (size_t d = 0; d < D; ++d) {
                    double h = h0[b * D + d];
                    for (size_t k = 0; k < S; ++k) {
                        const size_t s = flags & RTB_SCAN_REVERSE ? S - 1 - k : k, i = (b * S + s) * D + d;
                        h = a[i] * h + (flags & RTB_SCAN_COUPLED ? (1 - a[i]) * x[i] : x[i]);
                        ASSERT_TRUE(std::fabs(got[i] - h) <= 1e-14 * (1 + std::fabs(h)) * S);
                    }
                }
        }
    }
    {  // a gate for each channel, broadcast over batch and time; steps of a state
        const std::vector<double> per(a.begin(), a.begin() + D);
        auto tg = Tensor<double>::from_buf(cuda, per, {D});
        const auto h = tx.gated_scan_at(1, tg).cpu();
        auto state = Tensor<double>::from_buf(cuda, std::vector<double>(B * D, 0.0), {B, D});
        for (size_t s = 0; s < S; ++s) {
            state.gated_step_inplace(tg, tx.slice(1, Slice::range(s, s)));
            const auto now = state.cpu();
            for (size_t i = 0; i < B * D; ++i) {
                const double want = h[(i / D * S + s) * D + i % D];
                ASSERT_TRUE(std::fabs(now[i] - want) <= 1e-14 * (1 + std::fabs(want)) * S);
            }
        }
    }
    {  // codes stand for c m / 127; the map reads them
        const auto ck = Checkpoint8<double>::of(tx);
        const auto r = ck.restore().cpu(), g = ck.grad(RTB_CKPT8_MUL, ta).cpu();
        double m = 0;
        for (double v : x) m = std::fmax(m, std::fabs(v));
        for (size_t i = 0; i < x.size(); ++i) {
            ASSERT_TRUE(std::fabs(r[i] - x[i]) <= m / 254 * (1 + 1e-12));
            ASSERT_TRUE(std::fabs(g[i] - r[i] * a[i]) <= 1e-15 * std::fabs(r[i]));
        }
    }
    {  // the loss of three rows, one of them padding
        auto logits = Tensor<double>::from_buf(cuda, std::vector<double>(x.begin(), x.begin() + 3 * D), {3, D});
        auto targets = Tensor<int64_t>::from_buf(cuda, {2, -1, 4}, {3});
        double want = 0;
        for (size_t r : {(size_t)0, (size_t)2}) {
            double sum = 0;
            for (size_t j = 0; j < D; ++j) sum += std::exp(x[r * D + j]);
            want += std::log(sum) - x[r * D + (r == 0 ? 2 : 4)];
        }
        ASSERT_TRUE(std::fabs(cross_entropy_loss(logits, targets).cpu()[0] - want / 2) <= 1e-14 * (1 + std::fabs(want)));
    }
    {  // refusals carry the library's codes
        int code = 0;
        try { tx.gated_scan_at(3, ta); } catch (const TensorError &e) { code = e.code; }
        ASSERT_TRUE(code == RTB_ERR_DIM);
        try { tx.gated_scan_at(1, ta, &tx); } catch (const TensorError &e) { code = e.code; }
        ASSERT_TRUE(code == RTB_ERR_SHAPE);
    }
    std::printf("ok: %d checks\n", g_checks);
    return 0;
}
