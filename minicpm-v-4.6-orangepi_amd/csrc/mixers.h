// mixers.h -- argument checks shared by the token mixers' entry points.
#pragma once

#include <initializer_list>

#include "common.h"
#include "mcv_mixers.h"

namespace mcv {

// 16-byte accesses: an aligned pointer and strides of whole chunks of 8 fp16 values.
inline bool chunked16(const void* p, std::initializer_list<int64_t> strides) {
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    for (int64_t s : strides)
        if (s % 8 != 0) return false;
    return true;
}

}  // namespace mcv
