// GPU: rms_norm_add and rms_norm_add_w8a8_quantize of the C++ surface against the separate calls on the sum of the rows, made on
// the host (fp16 to nearest even): every output bit-identical, with the sum in a tensor of its own and in either input's place;
// and what they refuse.
#include "minicpmv/hip_context.h"
#include "minicpmv/ops.h"
#include "test_common.h"

#include <stdexcept>

using namespace minicpmv;

namespace {

Tensor device(const std::vector<uint16_t>& v, std::vector<int64_t> shape) {
    Tensor t(std::move(shape), DType::Float16);
    t.copy_from_host(v.data(), v.size() * 2);
    return t;
}
Tensor empty(std::vector<int64_t> shape, DType dtype) {
    Tensor t(std::move(shape), dtype);
    t.allocate();
    return t;
}
template <typename T>
std::vector<T> host(const Tensor& t) {
    std::vector<T> v(static_cast<size_t>(t.numel()));
    t.copy_to_host(v.data(), v.size() * sizeof(T));
    return v;
}
template <typename Call>
bool refuses(Call call) {
    try {
        call();
    } catch (const std::runtime_error&) {
        return true;
    }
    return false;
}

}  // namespace

int main() {
    HipContext ctx(0);
    int bad = 0;
    uint32_t seed = 1;
    auto next = [&] {
        seed = seed * 1664525u + 1013904223u;
        return t::f2h_rne((static_cast<float>(seed >> 8) / 8388608.0f - 1.0f) * 3.0f);
    };
    const double eps = 1e-6;
    for (const auto& [M, H] : {std::pair<int64_t, int64_t>{1, 1}, {1, 1024}, {5, 200}, {3, 1021}, {33, 3592}, {2, 9000}}) {
        std::vector<uint16_t> x(M * H), r(M * H), g(H), sum(M * H);
        for (auto* v : {&x, &r, &g})
            for (auto& e : *v) e = next();
        for (size_t i = 0; i < sum.size(); ++i) sum[i] = t::f2h_rne(t::h2f(x[i]) + t::h2f(r[i]));
        const Tensor gamma = device(g, {H}), total = device(sum, {M, H});
        Tensor out = empty({M, H}, DType::Float16), normed = empty({M, H}, DType::Float16), q = empty({M, H}, DType::Int8), s = empty({M}, DType::Float32);
        rms_norm(total, gamma, out, eps, ctx.stream());
        rms_norm_w8a8_quantize(total, gamma, eps, &normed, q, s, ctx.stream());
        const auto want = host<uint16_t>(out);
        const auto want_q = host<int8_t>(q);
        const auto want_s = host<float>(s);
        for (int place = 0; place < 3; ++place) {
            Tensor xd = device(x, {M, H}), rd = device(r, {M, H}), own = empty({M, H}, DType::Float16), y = empty({M, H}, DType::Float16);
            Tensor& to = place == 0 ? own : place == 1 ? xd : rd;
            rms_norm_add(xd, rd, gamma, y, to, eps, ctx.stream());
            bad += host<uint16_t>(y) != want || host<uint16_t>(to) != sum;
            xd = device(x, {M, H}), rd = device(r, {M, H});
            Tensor yq = empty({M, H}, DType::Int8), ys = empty({M}, DType::Float32);
            rms_norm_add_w8a8_quantize(xd, rd, gamma, eps, place ? &y : nullptr, yq, ys, to, ctx.stream());
            bad += host<int8_t>(yq) != want_q || host<float>(ys) != want_s || host<uint16_t>(to) != sum || (place && host<uint16_t>(y) != want);
        }
    }
    Tensor a = empty({2, 64}, DType::Float16), b = empty({2, 64}, DType::Float16), c = empty({2, 64}, DType::Float16), d = empty({2, 64}, DType::Float16);
    Tensor g = empty({64}, DType::Float16), short_rows = empty({2, 63}, DType::Float16), wide = empty({2, 64}, DType::Float32), q = empty({2, 64}, DType::Int8),
           s = empty({2}, DType::Float32);
    bad += !refuses([&] { rms_norm_add(a, short_rows, g, c, d, eps, ctx.stream()); });
    bad += !refuses([&] { rms_norm_add(a, b, g, c, short_rows, eps, ctx.stream()); });
    bad += !refuses([&] { rms_norm_add(wide, b, g, c, d, eps, ctx.stream()); });
    bad += !refuses([&] { rms_norm_add(a, b, s, c, d, eps, ctx.stream()); });
    bad += !refuses([&] { rms_norm_add_w8a8_quantize(a, b, g, eps, &short_rows, q, s, d, ctx.stream()); });
    bad += !refuses([&] { rms_norm_add_w8a8_quantize(a, b, g, eps, nullptr, q, g, d, ctx.stream()); });
    bad += !refuses([&] { rms_norm_add_w8a8_quantize(a, short_rows, g, eps, nullptr, q, s, d, ctx.stream()); });
    std::printf("%d wrong\n%s\n", bad, bad ? "FAILED" : "ok");
    return bad != 0;
}
