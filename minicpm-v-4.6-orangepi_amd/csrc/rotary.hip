// rotary.hip -- rotary positions with several axes, alone or written with v into a
// paged cache, gfx950.
//
// The angle positions[axis[i]][t] freq[i] is computed and reduced to one turn in 64
// bits (32 bits lose 0.06 rad at position 10^6) and shared by all heads of a token.
// Bound by memory, so the data is on its way while the angles are made: a thread has 32
// bytes of the same place in a head (two chunks that turn into one another, or two that
// are copied) of one or four tokens in registers before the workgroup's angles meet in LDS.
// MI355X, 8 + 2 heads of 256, 64 turned, with the cache: 8192 tokens 20.9 us, 4.8 TB/s (a
// copy of 1 GiB 5.2); one token 4.2 us, the host's part of a call.
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
    uint32_t pairs_inv, rest_inv, per_inv;       // ceil(2^32 / n) for the chunk kernel's divisions, 0 for n = 1
};

__device__ __forceinline__ void turn(float a, float b, float c, float s, uint16_t& x, uint16_t& y) {
    x = f2h(a * c - b * s);
    y = f2h(b * c + a * s);
}

// Angle i of token t: its quarter turns and what is left of it, an eighth of a turn at most, are found in 64 bits, so
// that the sine and the cosine are both within 32-bit roundings of themselves.  (In 32 bits a turn next to a half or a
// quarter has lost the last bits of the smaller of the two.)
__device__ __forceinline__ void angle_of(const RotaryArgs& p, int t, int i, float& c, float& s) {
    int a = p.axis[i];
    a = a < 0 ? 0 : a >= p.axes ? p.axes - 1 : a;
    double x = static_cast<double>(p.pos[a * p.pos_axis + t * p.pos_token]) * p.freq[i] * 0.15915494309189533577;
    x -= rint(x);
    const double quarter = rint(4.0 * x);
    const int n = static_cast<int>(quarter);
    float sy, cy;
    sincospif(2.0f * static_cast<float>(fma(quarter, -0.25, x)), &sy, &cy);
    s = n & 1 ? cy : sy;
    c = n & 1 ? sy : cy;
    s = n & 2 ? -s : s;
    c = (n + 1) & 2 ? -c : c;
}

// Where token t's k and v go: page and row, or nowhere.
struct Place {
    int64_t page, row;
    bool keep;
};
__device__ __forceinline__ Place place_of(const RotaryArgs& p, int t) {
    if (!p.slots) return {0, t, true};
    const int64_t slot = p.slots[t];
    if (slot < 0 || slot >= p.n_slots) return {0, 0, false};
    if (p.n_slots <= 0x7fffffff) {
        const uint32_t s = static_cast<uint32_t>(slot), page = s / static_cast<uint32_t>(p.page_size);
        return {page, s - page * static_cast<uint32_t>(p.page_size), true};
    }
    return {slot / p.page_size, slot % p.page_size, true};
}

// m / n, n's inverse as above, m n < 2^32.
__device__ __forceinline__ int over(int m, uint32_t inv) { return inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(m), inv)) : m; }

// Of values, all of them read: a choice between reads becomes a read of a chosen address, and what it chooses from
// would lie in scratch memory.
template <class V>
__device__ __forceinline__ V pick(int kind, V a, V b, V c) {
    return kind == 0 ? a : kind == 1 ? b : c;
}

// D and rot multiples of 16: TT tokens a workgroup, blockDim.x threads over their (head, 32 bytes),
// those that turn first: then few waves have any.
template <int TT>
__global__ __launch_bounds__(256) void rotary_chunk_kernel(RotaryArgs p) {
    const int t0 = blockIdx.x * TT, half = p.rot / 2, per = p.D / 16, pairs = half / 8, rest = per - pairs;
    const int turning = (p.Hq + p.Hkv) * pairs, ends = (p.Hq + p.Hkv) * per, items = ends + (p.v ? p.Hkv * per : 0);
    __shared__ float cs[TT][256], sn[TT][256];
    __shared__ int64_t k_to[TT], v_to[TT];       // -1: nowhere
    uint4 x[TT], y[TT];
    int head, lo, hi, kind;                      // 0 q, 1 k, 2 v; the elements at lo and hi
    auto load = [&](int m) {
        const int group = m < turning ? 0 : m < ends ? 1 : 2, at = m - pick(group, 0, turning, ends);
        const int h = over(at, pick(group, p.pairs_inv, p.rest_inv, p.per_inv)), i = at - h * pick(group, pairs, rest, per);
        kind = group == 2 ? 2 : h < p.Hq ? 0 : 1;
        head = h - pick(kind, 0, p.Hq, 0);
        lo = pick(group, 8 * i, p.rot + 16 * i, 16 * i);
        hi = lo + pick(group, half, 8, 8);
        const uint16_t* base = pick(kind, p.q, p.k, p.v);
        const int64_t row = pick(kind, p.q_row, p.k_row, p.v_row);
        base += head * pick(kind, p.q_head, p.k_head, p.v_head);
#pragma unroll
        for (int n = 0; n < TT; ++n) {
            const uint16_t* at = base + (t0 + n < p.T ? t0 + n : p.T - 1) * row;
            x[n] = *reinterpret_cast<const uint4*>(at + lo);
            y[n] = *reinterpret_cast<const uint4*>(at + hi);
        }
    };
    int m = threadIdx.x;
    if (m < items) load(m);
    for (int n = threadIdx.x; n < TT * half; n += blockDim.x) {
        const int t = TT == 1 ? 0 : n / half, i = n - t * half;
        if (t0 + t < p.T) angle_of(p, t0 + t, i, cs[t][i], sn[t][i]);
    }
    if (threadIdx.x < TT && t0 + static_cast<int>(threadIdx.x) < p.T) {
        const Place at = place_of(p, t0 + threadIdx.x);
        k_to[threadIdx.x] = at.keep ? at.page * p.ko_page + at.row * p.ko_row : -1;
        v_to[threadIdx.x] = at.keep ? at.page * p.vo_page + at.row * p.vo_row : -1;
    }
    __syncthreads();
    while (m < items) {
        uint16_t* const out = pick(kind, p.q_out, p.k_out, p.v_out);
        const int64_t head_at = head * pick(kind, p.qo_head, p.ko_head, p.vo_head);
#pragma unroll
        for (int n = 0; n < TT; ++n) {
            if (t0 + n >= p.T) break;
            if (m < turning) {
                uint16_t a[8], b[8];
                *reinterpret_cast<uint4*>(a) = x[n];
                *reinterpret_cast<uint4*>(b) = y[n];
#pragma unroll
                for (int e = 0; e < 8; ++e) turn(h2f(a[e]), h2f(b[e]), cs[n][lo + e], sn[n][lo + e], a[e], b[e]);
                x[n] = *reinterpret_cast<uint4*>(a);
                y[n] = *reinterpret_cast<uint4*>(b);
            }
            const int64_t to = kind == 0 ? (t0 + n) * p.qo_row : kind == 1 ? k_to[n] : v_to[n];
            if (to < 0) continue;
            *reinterpret_cast<uint4*>(out + to + head_at + lo) = x[n];
            *reinterpret_cast<uint4*>(out + to + head_at + hi) = y[n];
        }
        m += blockDim.x;
        if (m < items) load(m);
    }
}

// Any even rot: a pair of elements a thread, one token a workgroup.
__global__ __launch_bounds__(256) void rotary_pair_kernel(RotaryArgs p) {
    const int t = blockIdx.x, half = p.rot / 2;
    __shared__ float cs[256], sn[256];
    for (int i = threadIdx.x; i < half; i += 256) angle_of(p, t, i, cs[i], sn[i]);
    __syncthreads();
    const int per = half + p.D - p.rot, vper = p.D / 8;
    const int nq = p.Hq * per, nk = p.Hkv * per, nv = p.v ? p.Hkv * vper : 0;
    const Place at = place_of(p, t);
    for (int n = threadIdx.x; n < nq + nk + nv; n += 256) {
        if (n >= nq && !at.keep) break;
        if (n >= nq + nk) {
            const int m = n - nq - nk, h = m / vper, e = 8 * (m % vper);
            *reinterpret_cast<uint4*>(p.v_out + at.page * p.vo_page + at.row * p.vo_row + h * p.vo_head + e) =
                *reinterpret_cast<const uint4*>(p.v + t * p.v_row + h * p.v_head + e);
            continue;
        }
        const bool isq = n < nq;
        const int m = isq ? n : n - nq, h = m / per, i = m % per;
        const uint16_t* src = isq ? p.q + t * p.q_row + h * p.q_head : p.k + t * p.k_row + h * p.k_head;
        uint16_t* dst = isq ? p.q_out + t * p.qo_row + h * p.qo_head : p.k_out + at.page * p.ko_page + at.row * p.ko_row + h * p.ko_head;
        if (i >= half) {
            dst[i + half] = src[i + half];
            continue;
        }
        uint16_t x, y;
        turn(h2f(src[i]), h2f(src[half + i]), cs[i], sn[i], x, y);
        dst[i] = x;
        dst[half + i] = y;
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

int launch_rotary(RotaryArgs& a, mcv_stream_t stream) {
    int rc = require_device();
    if (rc != MCV_OK) return rc;
    auto inverse = [](int n) { return n > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + n - 1) / n) : 0; };
    a.pairs_inv = inverse(a.rot / 16);
    a.rest_inv = inverse(a.D / 16 - a.rot / 16);
    a.per_inv = inverse(a.D / 16);
    const dim3 one(static_cast<unsigned>(a.T));
    if (a.rot % 16 != 0 || a.D % 16 != 0) {
        hipLaunchKernelGGL(rotary_pair_kernel, one, dim3(256), 0, static_cast<hipStream_t>(stream), a);
        return check_launch("rotary_pair_kernel");
    }
    const int64_t items = (static_cast<int64_t>(a.Hq) + a.Hkv + (a.v ? a.Hkv : 0)) * (a.D / 16);
    const dim3 threads(static_cast<unsigned>(items < 256 ? ceil_div(items, 64) * 64 : 256));
    // Four tokens a workgroup once that still fills the chip.  MI355X, us a pass, one and four tokens: with the cache, 8 + 2
    // heads of 256, 64 turned, 2048 tokens 7.6 8.7, 4096 12.4 12.2, 8192 24.7 20.9; 16 + 4 of 128 without 6.1 7.8, 10.2 10.5,
    // 18.0 15.6; 16 + 16 of 64 without 5.1 6.3, 9.3 9.2, 14.4 12.7.
    if (a.T >= 4096)
        hipLaunchKernelGGL(rotary_chunk_kernel<4>, dim3(static_cast<unsigned>(ceil_div(a.T, 4))), threads, 0, static_cast<hipStream_t>(stream), a);
    else
        hipLaunchKernelGGL(rotary_chunk_kernel<1>, one, threads, 0, static_cast<hipStream_t>(stream), a);
    return check_launch("rotary_chunk_kernel");
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
                 static_cast<int>(rot), 1, 0, 0, 0};
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
                 static_cast<int>(rot), static_cast<int>(page_size), 0, 0, 0};
    int rc = check_rotary("rotary_axes_cached", a, T, Hq, Hkv, D, rot, axes);
    return rc != MCV_OK ? rc : launch_rotary(a, stream);
}

}  // extern "C"
