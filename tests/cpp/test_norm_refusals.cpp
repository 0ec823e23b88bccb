// CPU: rows of no elements are refused by rms_norm, rms_norm_add and rms_norm_add_w8a8_quantize of the C++ surface, before any
// device is asked for.
#include "minicpmv/ops.h"

#include <cstdio>
#include <stdexcept>

using namespace minicpmv;

namespace {

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
    int bad = 0;
    for (int64_t rows : {0, 1, 3}) {
        Tensor x({rows, 0}, DType::Float16), r({rows, 0}, DType::Float16), g(std::vector<int64_t>{0}, DType::Float16), y({rows, 0}, DType::Float16),
            sum({rows, 0}, DType::Float16), q({rows, 0}, DType::Int8), s(std::vector<int64_t>{rows}, DType::Float32);
        bad += !refuses([&] { rms_norm(x, g, y, 1e-6, nullptr); });
        bad += !refuses([&] { rms_norm_add(x, r, g, y, sum, 1e-6, nullptr); });
        bad += !refuses([&] { rms_norm_add_w8a8_quantize(x, r, g, 1e-6, nullptr, q, s, sum, nullptr); });
    }
    std::printf("%d wrong\n%s\n", bad, bad ? "FAILED" : "ok");
    return bad != 0;
}
