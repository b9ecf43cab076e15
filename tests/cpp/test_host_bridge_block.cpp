// GPU test of the bridge's fused block operators (bee_b200/host/tensor_cuda.hpp):
// known answers through the C++ calls and the error of a refused one.  Exits 0
// on success.  Run by tests/test_gpu_block.py.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "tensor_cuda.hpp"

namespace tc = bee_b200::tensor_cuda;

static int failures = 0;
#define CHECK(cond, what)                                                    \
    do {                                                                     \
        if (!(cond)) {                                                       \
            std::fprintf(stderr, "FAIL %s:%d: %s\n", __FILE__, __LINE__, what); \
            ++failures;                                                      \
        }                                                                    \
    } while (0)

template <typename T> static T* upload(const std::vector<T>& v) {
    auto r = tc::allocate(v.size() * sizeof(T), 64);
    if (!r || !tc::memcpy_h2d(*r, v.data(), v.size() * sizeof(T))) std::exit(2);
    return static_cast<T*>(*r);
}
template <typename T> static std::vector<T> download(const T* p, size_t n) {
    std::vector<T> v(n);
    if (!tc::memcpy_d2h(v.data(), p, n * sizeof(T))) std::exit(2);
    return v;
}
static bool near(float a, float b, float tol) { return std::fabs(a - b) <= tol; }

int main() {
    constexpr int F32 = 4, I32 = 2, BF16 = 8;
    constexpr std::uint16_t kOne = 0x3f80;  // 1.0 in bf16

    // rows of one value v: rmsnorm gives sign(v), so x' = 2 x + 0.5 * gate * sign(h), y = sign(x')
    const size_t rows = 3, cols = 40;
    std::vector<float> h(rows * cols), x(rows * cols), ones(cols, 1.f), gate(cols, 4.f);
    for (size_t i = 0; i < rows * cols; ++i) h[i] = -3.f * static_cast<float>(1 + i / cols), x[i] = static_cast<float>(i / cols) + 2.f;
    float *dh = upload(h), *dx = upload(x), *dw = upload(ones), *dg = upload(gate), *dxo = upload(x), *dy = upload(x);
    CHECK(tc::norm_gate_residual(F32, dh, dx, dw, dg, dw, dxo, dy, rows, cols, 0, 2.f, 0.5f, 0.f).has_value(), "norm_gate_residual");
    auto xo = download(dxo, rows * cols), y = download(dy, rows * cols);
    for (size_t i = 0; i < rows * cols; ++i) CHECK(near(xo[i], 2.f * x[i] - 2.f, 1e-5f) && near(y[i], 1.f, 1e-6f), "x_out, y");
    // constant rows do not change under rmsnorm: dh = 0 and dx = 2 dx_out
    float *gh = upload(h), *gx = upload(x), *gw = upload(ones), *gg = upload(ones), *gp = upload(ones);
    CHECK(tc::norm_gate_residual_backward(F32, dh, dx, dw, dg, dw, dx, dxo, gh, gx, gw, gg, gp, rows, cols, 0, 2.f, 0.5f, 0.f).has_value(),
          "norm_gate_residual_backward");
    auto rh = download(gh, rows * cols), rx = download(gx, rows * cols), rg = download(gg, cols);
    for (size_t i = 0; i < rows * cols; ++i) CHECK(near(rh[i], 0.f, 1e-5f) && near(rx[i], 2.f * x[i], 1e-4f), "dh, dx");
    for (size_t i = 0; i < cols; ++i) CHECK(near(rg[i], -0.5f * (2.f + 3.f + 4.f), 1e-4f), "dgate");
    auto bad = tc::norm_gate_residual(I32, dh, dx, dw, dg, dw, dxo, dy, rows, cols, 0, 1.f, 1.f, 0.f);
    CHECK(!bad.has_value() && bad.error().errc == 1, "a refused dtype is an error");

    // x = ones [2, 8], Wg = Wu = ones [8, 16] / 8 (0x3e00 = 0.125): g = u = 1, out = silu(1)
    const size_t M = 2, D = 8, F = 16;
    std::uint16_t *mx = upload(std::vector<std::uint16_t>(M * D, kOne)), *mw = upload(std::vector<std::uint16_t>(D * F, 0x3e00));
    std::uint16_t *out = upload(std::vector<std::uint16_t>(M * F)), *g = upload(std::vector<std::uint16_t>(M * F)),
                  *u = upload(std::vector<std::uint16_t>(M * F));
    CHECK(tc::gated_linear(BF16, 0, mx, D, mw, mw, F, false, out, g, u, M, D, F).has_value(), "gated_linear");
    for (auto v : download(g, M * F)) CHECK(v == kOne, "g");
    for (auto v : download(out, M * F)) CHECK(v == 0x3f3b, "silu(1) = 0.7311 in bf16");
    std::uint16_t *mdx = upload(std::vector<std::uint16_t>(M * D)), *wg = upload(std::vector<std::uint16_t>(D * F)),
                  *wu = upload(std::vector<std::uint16_t>(D * F));
    CHECK(tc::gated_linear_backward(BF16, 0, mx, D, mw, mw, F, false, g, u, g, mdx, wg, wu, F, M, D, F).has_value(), "gated_linear_backward");
    for (auto v : download(wu, D * F)) CHECK(v == 0x3fbb, "dWu = 2 silu(1), from du rounded to bf16");

    // equal logits over 50 tokens
    const size_t V = 50;
    float* logits = upload(std::vector<float>(2 * V, 0.25f));
    int* targets = upload(std::vector<int>{7, -1});
    float *lp = upload(std::vector<float>(2)), *ent = upload(std::vector<float>(2)), *mx2 = upload(std::vector<float>(2)),
          *ls = upload(std::vector<float>(2)), *top = upload(std::vector<float>(6)), *dl = upload(std::vector<float>(2 * V));
    std::int32_t* ids = upload(std::vector<std::int32_t>(6));
    CHECK(tc::token_logprobs(F32, logits, V, I32, targets, 2, V, 1.f, lp, ent, mx2, ls, 3, ids, top).has_value(), "token_logprobs");
    const float lv = std::log(50.f);
    auto vlp = download(lp, 2), vent = download(ent, 2);
    CHECK(near(vlp[0], -lv, 1e-5f) && vlp[1] == 0.f && near(vent[0], lv, 1e-5f) && near(vent[1], lv, 1e-5f), "logprob, entropy");
    auto vids = download(ids, 6);
    for (int i = 0; i < 6; ++i) CHECK(vids[i] == i % 3, "equal logits: the lowest indices");
    CHECK(tc::token_logprobs_backward(F32, logits, V, I32, targets, 2, V, 1.f, mx2, ls, ent, lp, nullptr, dl, V).has_value(), "backward");
    auto vdl = download(dl, 2 * V);
    CHECK(near(vdl[7], -lv * 0.98f, 1e-5f) && near(vdl[0], lv * 0.02f, 1e-5f) && vdl[V + 3] == 0.f, "dlogits");

    if (failures) return 1;
    std::printf("host bridge block ok\n");
    return 0;
}
