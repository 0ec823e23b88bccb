// rotary.hip -- rotary positions with several axes, alone or written with v into a
// paged cache, gfx950.
//
// The angle positions[axis[i]][t] freq[i] is computed and reduced to one turn in 64
// bits (32 bits lose 0.06 rad at position 10^6) and shared by all heads of a token: a
// workgroup fills LDS with the cosines and sines of its tokens, then its threads turn
// 8 pairs each in 16-byte accesses (VEC: rot a multiple of 16), or one pair.
#include "mixers.h"

namespace mcv {
namespace {

struct RotaryArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int64_t* pos;
    const double* freq;
    const int32_t* axis;
    const int64_t* slots;
    uint16_t* q_out;
    uint16_t* k_out;
    uint16_t* v_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, pos_axis, pos_token;
    int64_t qo_row, qo_head, ko_page, ko_row, ko_head, vo_page, vo_row, vo_head, n_slots;
    int axes, T, Hq, Hkv, D, rot, page_size;
};

__device__ __forceinline__ void turn(float a, float b, float c, float s, uint16_t& x, uint16_t& y) {
    x = f2h(a * c - b * s);
    y = f2h(b * c + a * s);
}

// One token a workgroup.
template <bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
    constexpr int W = VEC ? 8 : 1;
    const int t = blockIdx.x, half = p.rot / 2;
    __shared__ float cs[256], sn[256];
    for (int i = threadIdx.x; i < half; i += 256) {
        int a = p.axis[i];
        a = a < 0 ? 0 : a >= p.axes ? p.axes - 1 : a;
        const double x = static_cast<double>(p.pos[a * p.pos_axis + t * p.pos_token]) * p.freq[i] * 0.15915494309189533577;
        const float turns = static_cast<float>(x - rint(x));
        sincospif(2.0f * turns, &sn[i], &cs[i]);
    }
    __syncthreads();
    const int pairs = half / W, rest = (p.D - p.rot) / W, per = pairs + rest, vper = p.D / 8;
    const int nq = p.Hq * per, nk = p.Hkv * per, nv = p.v ? p.Hkv * vper : 0;
    int64_t page = 0, row = t;
    bool keep = true;
    if (p.slots) {
        const int64_t slot = p.slots[t];
        keep = slot >= 0 && slot < p.n_slots;
        page = keep ? slot / p.page_size : 0;
        row = keep ? slot % p.page_size : 0;
    }
    for (int n = threadIdx.x; n < nq + nk + nv; n += 256) {
        if (n >= nq + nk) {
            const int m = n - nq - nk, h = m / vper, e = 8 * (m % vper);
            if (keep)
                *reinterpret_cast<uint4*>(p.v_out + page * p.vo_page + row * p.vo_row + h * p.vo_head + e) =
                    *reinterpret_cast<const uint4*>(p.v + t * p.v_row + h * p.v_head + e);
            continue;
        }
        const bool isq = n < nq;
        const int m = isq ? n : n - nq, h = m / per, i = m % per;
        const uint16_t* src = isq ? p.q + t * p.q_row + h * p.q_head : p.k + t * p.k_row + h * p.k_head;
        uint16_t* dst = isq ? p.q_out + t * p.qo_row + h * p.qo_head : p.k_out + page * p.ko_page + row * p.ko_row + h * p.ko_head;
        if (!isq && !keep) continue;
        if (i >= pairs) {
            const int e = p.rot + W * (i - pairs);
            if constexpr (VEC) *reinterpret_cast<uint4*>(dst + e) = *reinterpret_cast<const uint4*>(src + e);
            else dst[e] = src[e];
            continue;
        }
        const int e = W * i;
        if constexpr (VEC) {
            uint16_t a[8], b[8];
            *reinterpret_cast<uint4*>(a) = *reinterpret_cast<const uint4*>(src + e);
            *reinterpret_cast<uint4*>(b) = *reinterpret_cast<const uint4*>(src + half + e);
            for (int x = 0; x < 8; ++x) turn(h2f(a[x]), h2f(b[x]), cs[e + x], sn[e + x], a[x], b[x]);
            *reinterpret_cast<uint4*>(dst + e) = *reinterpret_cast<uint4*>(a);
            *reinterpret_cast<uint4*>(dst + half + e) = *reinterpret_cast<uint4*>(b);
        } else {
            uint16_t x, y;
            turn(h2f(src[e]), h2f(src[half + e]), cs[e], sn[e], x, y);
            dst[e] = x;
            dst[half + e] = y;
        }
    }
}

int check_rotary(const char* who, const RotaryArgs& a, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, int64_t axes) {
    if (!a.q || !a.k || !a.pos || !a.freq || !a.axis || !a.q_out || !a.k_out) return fail(MCV_ERR_INVALID_ARG, "%s: null pointer", who);
    if (T <= 0 || T > 0x7fffffff || Hq <= 0 || Hkv <= 0 || Hq > 65535 || Hkv > 65535 || axes <= 0 || axes > 16)
        return fail(MCV_ERR_SHAPE, "%s: bad shape T=%lld Hq=%lld Hkv=%lld axes=%lld", who, (long long)T, (long long)Hq,
                    (long long)Hkv, (long long)axes);
    if (D <= 0 || D % 8 != 0 || D > 512 || rot < 2 || rot % 2 != 0 || rot > D)
        return fail(MCV_ERR_SHAPE, "%s: D must be a multiple of 8 up to 512 and rot even, 2 <= rot <= D (D=%lld rot=%lld)", who,
                    (long long)D, (long long)rot);
    for (int64_t s : {a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.pos_axis, a.pos_token, a.qo_row, a.qo_head,
                      a.ko_page, a.ko_row, a.ko_head, a.vo_page, a.vo_row, a.vo_head})
        if (s < 0) return fail(MCV_ERR_SHAPE, "%s: negative stride", who);
    if (!chunked16(a.q, {a.q_row, a.q_head}) || !chunked16(a.k, {a.k_row, a.k_head}) || !chunked16(a.v, {a.v_row, a.v_head}) ||
        !chunked16(a.q_out, {a.qo_row, a.qo_head}) || !chunked16(a.k_out, {a.ko_page, a.ko_row, a.ko_head}) ||
        !chunked16(a.v_out, {a.vo_page, a.vo_row, a.vo_head}))
        return fail(MCV_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned, strides multiples of 8 elements", who);
    return MCV_OK;
}

int launch_rotary(const RotaryArgs& a, mcv_stream_t stream) {
    int rc = require_device();
    if (rc != MCV_OK) return rc;
    hipLaunchKernelGGL(a.rot % 16 == 0 ? rotary_kernel<true> : rotary_kernel<false>, dim3(static_cast<unsigned>(a.T)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), a);
    return check_launch("rotary_kernel");
}

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int mcv_rotary_axes(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                    const void* positions, int64_t pos_axis, int64_t pos_token, int64_t axes, const void* freq,
                    const void* axis, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, void* q_out,
                    int64_t qo_row, int64_t qo_head, void* k_out, int64_t ko_row, int64_t ko_head,
                    mcv_stream_t stream) {
    RotaryArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), nullptr,
                 static_cast<const int64_t*>(positions), static_cast<const double*>(freq), static_cast<const int32_t*>(axis),
                 nullptr, static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_out), nullptr,
                 q_row, q_head, k_row, k_head, 0, 0, pos_axis, pos_token,
                 qo_row, qo_head, 0, ko_row, ko_head, 0, 0, 0, 0,
                 static_cast<int>(axes), static_cast<int>(T), static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(D),
                 static_cast<int>(rot), 1};
    int rc = check_rotary("rotary_axes", a, T, Hq, Hkv, D, rot, axes);
    return rc != MCV_OK ? rc : launch_rotary(a, stream);
}

int mcv_rotary_axes_cached(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                           const void* v, int64_t v_row, int64_t v_head, const void* positions, int64_t pos_axis,
                           int64_t pos_token, int64_t axes, const void* freq, const void* axis, int64_t T, int64_t Hq,
                           int64_t Hkv, int64_t D, int64_t rot, void* q_out, int64_t qo_row, int64_t qo_head,
                           void* k_cache, int64_t k_page, int64_t k_token, int64_t kc_head, void* v_cache,
                           int64_t v_page, int64_t v_token, int64_t vc_head, int64_t pages, int64_t page_size,
                           const void* slots, mcv_stream_t stream) {
    if (!v || !v_cache || !slots) return fail(MCV_ERR_INVALID_ARG, "rotary_axes_cached: null pointer");
    if (pages <= 0 || page_size <= 0 || page_size > 0x7fffffff || pages > 0x7fffffff)
        return fail(MCV_ERR_SHAPE, "rotary_axes_cached: bad cache pages=%lld page_size=%lld", (long long)pages, (long long)page_size);
    RotaryArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                 static_cast<const int64_t*>(positions), static_cast<const double*>(freq), static_cast<const int32_t*>(axis),
                 static_cast<const int64_t*>(slots), static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_cache),
                 static_cast<uint16_t*>(v_cache), q_row, q_head, k_row, k_head, v_row, v_head, pos_axis, pos_token,
                 qo_row, qo_head, k_page, k_token, kc_head, v_page, v_token, vc_head, pages * page_size,
                 static_cast<int>(axes), static_cast<int>(T), static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(D),
                 static_cast<int>(rot), static_cast<int>(page_size)};
    int rc = check_rotary("rotary_axes_cached", a, T, Hq, Hkv, D, rot, axes);
    return rc != MCV_OK ? rc : launch_rotary(a, stream);
}

}  // extern "C"
