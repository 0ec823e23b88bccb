// delta_rule.hip -- the gated delta rule, token by token, gfx950.
//
// Per token and value head, S [Dk][Dv] fp32:  with decay e = exp(g), and q, k the
// raw rows with norm factors rq, rk (1 without normalize)
//   a = k . S,  b = q . S,  c = q . k          (sums over Dk)
//   u = beta (v - e rk a),  S' = e S + rk k u,  out = scale rq (e b + rk c u)
// so one pass over S gives everything that S' and out need: out comes from the old
// state and c instead of a second sum over the new one.  One token is bound by the state's
// way in and out, past the caches (non-temporal: 53 sequences of 16 states of 128 x 128 take
// 21.5 us on MI355X, 5.2 TB/s, as fast as a copy; 24.8 through them); more tokens take 1.1
// us each, one after the other.
//
// A workgroup holds DVW columns of one state in registers for the whole sequence:
// 16-byte column chunks over the lanes, R consecutive rows a thread (so its part of
// q and k is one vector load).  Sums over Dk: R rows in the thread, the row groups
// of a wave by lane swaps, the four waves through LDS.
#include "delta_rule.h"

namespace mcv {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMixed = 16;                   // more sequences than these: short ones by the recurrence, long ones in chunks

// Sum over the lanes of one lane % C4 (C4 4 .. 32), in all of them: steps of a butterfly as in wave_butterfly.
template <int C4>
__device__ __forceinline__ float sum_over(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    if constexpr (C4 <= 16) {
        const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
    if constexpr (C4 <= 8) v += row_ror<8>(v);
    if constexpr (C4 <= 4) v += row_ror<4>(v);
    return v;
}

template <int DK, int DVW>
__global__ __launch_bounds__(kThreads) void delta_recurrent_kernel(DeltaArgs p) {
    constexpr int C4 = DVW / 4;                  // lanes over one row's columns
    constexpr int RG = kThreads / C4;            // row groups of the workgroup
    constexpr int R = DK / RG;                   // rows a thread holds
    static_assert(R * RG == DK && R >= 1, "rows");
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int c4 = t % C4, rg = t / C4;
    const int slices = p.Dv / DVW;
    const int slice = blockIdx.x % slices;
    const int bh = blockIdx.x / slices;
    const int h = bh % p.Hv, b = bh / p.Hv, hk = h / p.group;
    int t0, t1;
    delta_span(p, b, t0, t1);
    const int col = slice * DVW + 4 * c4;
    if (p.short_below && t1 - t0 >= p.short_below) return;
    const int64_t at = p.state_index ? p.state_index[b] : b;
    if (at < 0 || at >= p.n_states) {
        if (rg == 0)
            for (int i = t0; i < t1; ++i)
                *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(i) * p.Hv + h) * p.Dv + col) = make_uint2(0, 0);
        return;
    }
    const int64_t base = (at * p.Hv + h) * DK * p.Dv + static_cast<int64_t>(rg * R) * p.Dv + col;
    float4_t S[R];
#pragma unroll
    for (int j = 0; j < R; ++j)
        S[j] = p.state ? __builtin_nontemporal_load(reinterpret_cast<const float4_t*>(p.state + base + static_cast<int64_t>(j) * p.Dv)) : float4_t{0, 0, 0, 0};
    __shared__ float4_t part[2][4][C4][2];
    __shared__ float dots[2][4][3];
    for (int i = t0; i < t1; ++i) {
        float kr[R], qr[R];
        const uint16_t* kp = p.k + i * p.k_row + hk * p.k_head + rg * R;
        const uint16_t* qp = p.q + i * p.q_row + hk * p.q_head + rg * R;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            kr[j] = h2f(kp[j]);
            qr[j] = h2f(qp[j]);
        }
        const uint2 vw = *reinterpret_cast<const uint2*>(p.v + i * p.v_row + h * p.v_head + col);
        const float e = expf(p.g[i * p.g_row + h]), beta = p.beta[i * p.beta_row + h];
        float s[11] = {};
#pragma unroll
        for (int j = 0; j < R; ++j) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[x] = fmaf(kr[j], S[j][x], s[x]);
                s[4 + x] = fmaf(qr[j], S[j][x], s[4 + x]);
            }
            s[8] = fmaf(qr[j], kr[j], s[8]);
            s[9] = fmaf(kr[j], kr[j], s[9]);
            s[10] = fmaf(qr[j], qr[j], s[10]);
        }
#pragma unroll
        for (int x = 0; x < 11; ++x) s[x] = sum_over<C4>(s[x]);
        const int buf = (i - t0) & 1;            // the other buffer may still be read by a slower wave
        if (lane < C4) {
            part[buf][wave][lane][0] = float4_t{s[0], s[1], s[2], s[3]};
            part[buf][wave][lane][1] = float4_t{s[4], s[5], s[6], s[7]};
        }
        if (lane == 0) {
            dots[buf][wave][0] = s[8];
            dots[buf][wave][1] = s[9];
            dots[buf][wave][2] = s[10];
        }
        __syncthreads();
        float4_t a = part[buf][0][c4][0], o = part[buf][0][c4][1];
        float qk = dots[buf][0][0], kk = dots[buf][0][1], qq = dots[buf][0][2];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            a += part[buf][w][c4][0];
            o += part[buf][w][c4][1];
            qk += dots[buf][w][0];
            kk += dots[buf][w][1];
            qq += dots[buf][w][2];
        }
        const float rk = p.normalize ? 1.0f / sqrtf(kk + kDeltaEps) : 1.0f;
        const float rq = p.normalize ? 1.0f / sqrtf(qq + kDeltaEps) : 1.0f;
        const float vs[4] = {h2f(vw.x & 0xffff), h2f(vw.x >> 16), h2f(vw.y & 0xffff), h2f(vw.y >> 16)};
        float4_t u;
#pragma unroll
        for (int x = 0; x < 4; ++x) u[x] = beta * (vs[x] - e * rk * a[x]);
        if (rg == 0) {
            uint16_t r[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) r[x] = f2h(p.scale * rq * fmaf(rk * qk, u[x], e * o[x]));
            *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(i) * p.Hv + h) * p.Dv + col) =
                make_uint2(r[0] | (static_cast<uint32_t>(r[1]) << 16), r[2] | (static_cast<uint32_t>(r[3]) << 16));
        }
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int x = 0; x < 4; ++x) S[j][x] = fmaf(rk * kr[j], u[x], e * S[j][x]);
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
        __builtin_nontemporal_store(S[j], reinterpret_cast<float4_t*>(p.state_out + base + static_cast<int64_t>(j) * p.Dv));
}

// Where the chunked form is faster than 1.1 us a token of the longest sequence.  MI355X, us a pass, recurrence and chunks
// (16 heads of 128): 1 sequence of 8 tokens 11.7 14.5, of 12 16.3 14.6, of 32 39.0 14.6; 4 of 8 on average 26.4 20.3.
// Lengths are the device's, and one sequence may have all tokens but a few: 100 of one token and one of 800 take 1083 us
// by the recurrence and 88 as below.  Both forms launched cost the recurrence's batches 4 to 9 us (41 of two tokens 19.1
// 28.1, 8 of five 9.6 13.9) and save what one longer sequence takes: 40 of one token and one of 20 39.0 38.0, of 40 61.9
// 38.4, of 63 88.2 38.5; 7 and one of 33 41.4 20.3, of 60 72.5 20.4.  From 32 tokens more than sequences on the second
// is the larger of the two that a wrong guess loses.
constexpr int kShort = 10;
bool may_be_long(int64_t B, int64_t T) {
    const int64_t even = kShort * B, skewed = B + 32;
    return T >= (B == 1 || even < skewed ? even : skewed);
}
// Then: whether both forms are launched.  With few sequences not where they may all be long.
bool mixed(int64_t B, int64_t T) { return B > kMixed || (B > 1 && T < kShort * B && T < B + 64); }

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int64_t mcv_delta_rule_workspace_bytes(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv) {
    if (B <= 0 || T <= 0 || Hk <= 0 || Hv <= 0 || (Dk != 64 && Dk != 128) || Dv <= 0 || Dv % 16 != 0 || !may_be_long(B, T)) return 0;
    return delta_chunk_workspace(B, T, Hk, Hv, Dk);
}

int mcv_delta_rule(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                   const void* v, int64_t v_row, int64_t v_head, const void* g, int64_t g_row, const void* beta,
                   int64_t beta_row, const void* state, void* state_out, const void* state_index, int64_t n_states,
                   const void* cu_seqlens, int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv,
                   double scale, int normalize, void* out, void* workspace, int64_t workspace_bytes,
                   mcv_stream_t stream) {
    if (!state_out) return fail(MCV_ERR_INVALID_ARG, "delta_rule: null state_out");
    if (B <= 0 || T < 0 || Hk <= 0 || Hv <= 0 || Hv % Hk != 0 || B > 0x7fffffff || T > 0x7fffffff || Hv > 65535)
        return fail(MCV_ERR_SHAPE, "delta_rule: bad shape B=%lld T=%lld Hk=%lld Hv=%lld", (long long)B, (long long)T,
                    (long long)Hk, (long long)Hv);
    if ((Dk != 64 && Dk != 128) || Dv <= 0 || Dv % 16 != 0 || Dv > 256)
        return fail(MCV_ERR_SHAPE, "delta_rule: Dk must be 64 or 128 and Dv a multiple of 16 up to 256 (Dk=%lld Dv=%lld)",
                    (long long)Dk, (long long)Dv);
    if (!cu_seqlens && T % B != 0)
        return fail(MCV_ERR_SHAPE, "delta_rule: T=%lld is not B=%lld sequences of one length", (long long)T, (long long)B);
    if (T > 0 && (!q || !k || !v || !g || !beta || !out)) return fail(MCV_ERR_INVALID_ARG, "delta_rule: null pointer");
    if (n_states < (state_index ? 1 : B))
        return fail(MCV_ERR_SHAPE, "delta_rule: %lld states for %lld sequences", (long long)n_states, (long long)B);
    if (q_row < 0 || q_head < 0 || k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0 || g_row < 0 || beta_row < 0)
        return fail(MCV_ERR_SHAPE, "delta_rule: negative stride");
    if (!chunked16(q, {q_row, q_head}) || !chunked16(k, {k_row, k_head}) || !chunked16(v, {v_row, v_head}) ||
        !chunked16(out, {}) || !chunked16(state, {}) || !chunked16(state_out, {}))
        return fail(MCV_ERR_UNSUPPORTED, "delta_rule: pointers must be 16-byte aligned, strides multiples of 8 elements");
    int rc = require_device();
    if (rc != MCV_OK) return rc;
    DeltaArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                static_cast<const float*>(g), static_cast<const float*>(beta), static_cast<const float*>(state),
                static_cast<float*>(state_out), static_cast<const int32_t*>(state_index),
                static_cast<const int32_t*>(cu_seqlens), static_cast<uint16_t*>(out), q_row, q_head, k_row, k_head,
                v_row, v_head, g_row, beta_row, n_states, static_cast<int>(T), static_cast<int>(B),
                static_cast<int>(cu_seqlens ? 0 : T / B), static_cast<int>(Hv), static_cast<int>(Hv / Hk),
                static_cast<int>(Dv), static_cast<float>(scale), normalize, 0};
    const bool chunks = (cu_seqlens ? may_be_long(B, T) : T >= kShort * B) && workspace && workspace_bytes >= delta_chunk_workspace(B, T, Hk, Hv, Dk);
    if (chunks) {
        if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
            return fail(MCV_ERR_INVALID_ARG, "delta_rule: workspace must be 256-byte aligned");
        a.short_below = cu_seqlens && mixed(B, T) ? kShort : 0;
        rc = launch_delta_chunk(a, static_cast<int>(Hk), static_cast<int>(Dk), workspace, workspace_bytes, static_cast<hipStream_t>(stream));
        if (rc != MCV_OK || a.short_below == 0) return rc;
    }
    // Columns a workgroup holds: 256 bytes of a row at a time unless that leaves most CUs without work.  MI355X, us a
    // pass of 128 x 128 states, 16 and 64 columns: 16 states 4.2 4.3, 64 5.1 5.2, 256 14.3 7.5, 848 35.5 22.0.
    const int width = Dv % 64 == 0 && B * Hv * (Dv / 64) >= 96 ? 64 : 16;
    const int64_t grid = B * Hv * (Dv / width);
    if (grid > 0x7fffffff) return fail(MCV_ERR_SHAPE, "delta_rule: too many states");
    auto fn = Dk == 64 ? (width == 64 ? delta_recurrent_kernel<64, 64> : delta_recurrent_kernel<64, 16>)
                       : (width == 64 ? delta_recurrent_kernel<128, 64> : delta_recurrent_kernel<128, 16>);
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    return check_launch("delta_recurrent_kernel");
}

}  // extern "C"
