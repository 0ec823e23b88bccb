// row_norm.h -- RMSNorm of fp16 rows, alone (elementwise.hip) or followed by
// the W8A8 activation quantisation (w8a8.hip), and either of them of the sum of two
// rows; one 256-thread workgroup per row, or a wave for short rows of a sum.
#pragma once

#include "common.h"

namespace mcv {

// Two halves of 16 bytes at a time, element e of a chunk.
__device__ __forceinline__ uint16_t chunk_get(const uint4& v, int e) {
    const uint32_t w = e < 4 ? (e < 2 ? v.x : v.y) : (e < 6 ? v.z : v.w);
    return static_cast<uint16_t>(w >> (16 * (e & 1)));
}

// The normed values of a chunk; MAX: m becomes the largest magnitude among them and m.
template <bool MAX>
__device__ __forceinline__ uint4 rms_chunk(const uint4& x, const uint4& g, float rstd, float& m) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const uint16_t a = rms_apply(chunk_get(x, e), rstd, chunk_get(g, e));
        const uint16_t b = rms_apply(chunk_get(x, e + 1), rstd, chunk_get(g, e + 1));
        w[e / 2] = a | (static_cast<uint32_t>(b) << 16);
        if constexpr (MAX) {
            const float va = fabsf(h2f(a)), vb = fabsf(h2f(b));
            m = va > m ? va : m;
            m = vb > m ? vb : m;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// fp16 RNE(a + b).  In 32 bits first, whose 24 bits are enough for the second rounding to find what one would.
__device__ __forceinline__ uint16_t add_f16(uint16_t a, uint16_t b) { return f2h(__fadd_rn(h2f(a), h2f(b))); }
__device__ __forceinline__ uint4 add_chunk(const uint4& a, const uint4& b) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        w[e / 2] = add_f16(chunk_get(a, e), chunk_get(b, e)) | (static_cast<uint32_t>(add_f16(chunk_get(a, e + 1), chunk_get(b, e + 1))) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The other row of a sum, and where the sum goes (either row, or a row of its own); elements from row to row.
struct AddRows {
    const uint16_t* other;
    uint16_t* sum;
    int64_t x_row, other_row, sum_row;
};

// normed = fp16((x * rstd) * gamma), rstd = 1 / sqrt(mean(x^2) + eps); QUANT:
// then the row's int8 values and scale, from the same fp16 values.  Every step
// is an explicitly rounded fp32 operation, and thread t sums the squares of
// elements t, t + 256, ... in that order, so the result does not depend on PER,
// VEC or QUANT.
//
// A row is one memory round trip: every load goes out before the first use
// (PER strided elements a thread for the sum; VEC: x again and gamma as 16-byte
// chunks, chunk t + 256 c, for the output, whose stores are then 16 bytes of
// fp16 and 8 of int8 a thread).  Reloading x and gamma element by element
// after the sum made two and more.  MI355X, us before / after: M=1 H=1024 2.7 /
// 2.4, H=3584 5.1 / 3.6, M=1100 H=1024 4.1 / 3.4, M=3000 7.5 / 6.4; with the
// quantisation M=1 H=1024 3.5 / 3.1, H=2048 4.9 / 3.5.  PER = 0: rows longer than
// 256 * 32, strided loops, each with only the loads and stores it needs (with the
// store conditional inside: M=1 H=16384 27.8 us, now 26.3, as before PER).
// ADD: the row is fp16(x + other), which goes to `sum` too; normed and int8 are what
// they are for a row that holds it.  VEC then loads every element once, as chunks, and
// thread t finds the elements t, t + 256, ... of the sum in LDS: bound by HBM from some
// 1000 rows on.  M=8192 H=1024 12.3 us (5.4 TB/s; each element twice, as without ADD:
// 19.2), M=1024 H=8192 11.3 (5.9 TB/s), M=1100 H=3592 to int8 9.8 (17), M=1 H=1024 2.0.
// Not for PER = 0, whose thread writes the sum element by element and reads it back for
// each pass: M=1024 H=16384 65 us (2.1 TB/s), without ADD 38.
template <int PER, bool VEC, bool QUANT, bool ADD = false>
__global__ __launch_bounds__(256) void rms_row_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ gamma,
                                                      int H, float eps, uint16_t* __restrict__ normed,
                                                      int8_t* __restrict__ xq, float* __restrict__ s32,
                                                      uint16_t* __restrict__ s16, AddRows add) {
    const int row = blockIdx.x;
    const int t = threadIdx.x;
    const uint16_t* xr = x + (ADD ? row * add.x_row : static_cast<int64_t>(row) * H);
    const uint16_t* ar = ADD ? add.other + row * add.other_row : nullptr;
    uint16_t* sr = ADD ? add.sum + row * add.sum_row : nullptr;
    uint16_t* nr = normed ? normed + static_cast<size_t>(row) * H : nullptr;
    int8_t* qr = QUANT ? xq + static_cast<size_t>(row) * H : nullptr;
    float m = 0.f;
    float scale = 0.f;
    if constexpr (PER > 0) {
        constexpr int NC = VEC ? (PER + 7) / 8 : 1;
        uint16_t xs[PER], gs[VEC ? 1 : PER];
        uint4 xv[NC], gv[NC];
        uint16_t as[ADD ? PER : 1];
        if constexpr (ADD && VEC) {
            // each element is loaded once, by the thread that stores its chunk: rows and sum may be one
            __shared__ uint4 sums[256 * NC];
            uint4 av[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int i = 8 * (t + 256 * c);
                xv[c] = i < H ? *reinterpret_cast<const uint4*>(xr + i) : make_uint4(0, 0, 0, 0);
                av[c] = i < H ? *reinterpret_cast<const uint4*>(ar + i) : make_uint4(0, 0, 0, 0);
                gv[c] = i < H ? *reinterpret_cast<const uint4*>(gamma + i) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int i = 8 * (t + 256 * c);
                xv[c] = add_chunk(xv[c], av[c]);
                sums[t + 256 * c] = xv[c];
                if (i < H) *reinterpret_cast<uint4*>(sr + i) = xv[c];
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j) xs[j] = reinterpret_cast<const uint16_t*>(sums)[t + 256 * j];      // (zero past the row)
        } else
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = t + 256 * j;
            xs[j] = i < H ? xr[i] : uint16_t(0);
            if constexpr (ADD) as[j] = i < H ? ar[i] : uint16_t(0);
            if constexpr (!VEC) gs[j] = i < H ? gamma[i] : uint16_t(0);
        }
        if constexpr (VEC && !ADD)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int i = 8 * (t + 256 * c);
                xv[c] = i < H ? *reinterpret_cast<const uint4*>(xr + i) : make_uint4(0, 0, 0, 0);
                gv[c] = i < H ? *reinterpret_cast<const uint4*>(gamma + i) : make_uint4(0, 0, 0, 0);
            }
        // x may be `normed` (or the sum's place): no load may be in flight when another thread stores
        if constexpr (!(ADD && VEC)) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (ADD && !VEC)
#pragma unroll
            for (int j = 0; j < PER; ++j) xs[j] = add_f16(xs[j], as[j]);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float v = h2f(xs[j]);                  // zero past the row: adds nothing
            ss = fmaf(v, v, ss);
        }
        const float rstd = block_rstd(ss, H, eps);
        if constexpr (VEC) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int i = 8 * (t + 256 * c);
                xv[c] = rms_chunk<QUANT>(xv[c], gv[c], rstd, m);          // now the normed chunk
                if (i < H && nr) *reinterpret_cast<uint4*>(nr + i) = xv[c];
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int i = t + 256 * j;
                if constexpr (ADD)
                    if (i < H) sr[i] = xs[j];
                xs[j] = rms_apply(xs[j], rstd, gs[j]);
                if (i < H && nr) nr[i] = xs[j];
                if constexpr (QUANT) {
                    const float v = i < H ? fabsf(h2f(xs[j])) : 0.f;
                    m = v > m ? v : m;
                }
            }
        }
        if constexpr (QUANT) {
            scale = act_scale(row_absmax(m));
            const float inv = __fdiv_rn(1.0f, scale);
            if constexpr (VEC) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int i = 8 * (t + 256 * c);
                    if (i < H) *reinterpret_cast<uint2*>(qr + i) = act_quant8(xv[c], inv);
                }
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int i = t + 256 * j;
                    if (i < H) qr[i] = act_quant(xs[j], inv);
                }
            }
        }
    } else {
        if constexpr (ADD) {                     // each thread reads back what it has written itself
            for (int i = t; i < H; i += blockDim.x) sr[i] = add_f16(xr[i], ar[i]);
            xr = sr;
        }
        const float rstd = row_rstd(xr, H, eps);
        if constexpr (!QUANT) {
            for (int i = t; i < H; i += blockDim.x) nr[i] = rms_apply(xr[i], rstd, gamma[i]);
        } else {
            auto each = [&](auto&& use) {
                for (int i = t; i < H; i += blockDim.x) use(i, rms_apply(xr[i], rstd, gamma[i]));
            };
            auto largest = [&](uint16_t h) {
                const float v = fabsf(h2f(h));
                m = v > m ? v : m;
            };
            if (nr) each([&](int i, uint16_t h) { largest(h); nr[i] = h; });
            else each([&](int, uint16_t h) { largest(h); });
            scale = act_scale(row_absmax(m));
            const float inv = __fdiv_rn(1.0f, scale);
            // the normed row again, from memory only where x is gone (in place)
            if (nr == xr) for (int i = t; i < H; i += blockDim.x) qr[i] = act_quant(nr[i], inv);
            else each([&](int i, uint16_t h) { qr[i] = act_quant(h, inv); });
        }
    }
    if constexpr (QUANT) {
        if (t == 0) {
            if (s32) s32[row] = scale;
            if (s16) s16[row] = f2h(scale);
        }
    }
}

// The sum's norm of rows of up to 256: a wave a row, four to a workgroup, with the sums of rms_row_kernel's four waves one after
// another in one, and no barrier.  M=16384 H=200
// 10.4 us, 15.0 with a workgroup a row; M=8192 H=64 4.5 / 6.2.  (Beyond 256 the chunks' loads are wider than a wave's.)
template <bool QUANT>
__global__ __launch_bounds__(256) void rms_add_short_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ gamma, int M, int H,
                                                            float eps, uint16_t* __restrict__ normed, int8_t* __restrict__ xq,
                                                            float* __restrict__ s32, uint16_t* __restrict__ s16, AddRows add) {
    const int row = 4 * blockIdx.x + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= M) return;
    const uint16_t* xr = x + row * add.x_row;
    const uint16_t* ar = add.other + row * add.other_row;
    uint16_t* sr = add.sum + row * add.sum_row;
    uint16_t xs[4], as[4], gs[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int i = lane + 64 * w;
        xs[w] = i < H ? xr[i] : uint16_t(0);
        as[w] = i < H ? ar[i] : uint16_t(0);
        gs[w] = i < H ? gamma[i] : uint16_t(0);
    }
    float tot = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int i = lane + 64 * w;
        xs[w] = add_f16(xs[w], as[w]);
        if (i < H) sr[i] = xs[w];
        const float v = h2f(xs[w]);                      // zero past the row
        tot += wave_butterfly(fmaf(v, v, 0.f), [](float p, float q) { return p + q; });
    }
    const float rstd = rms_rstd(tot, H, eps);
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int i = lane + 64 * w;
        xs[w] = rms_apply(xs[w], rstd, gs[w]);
        if (i < H && normed) normed[static_cast<int64_t>(row) * H + i] = xs[w];
        const float v = i < H ? fabsf(h2f(xs[w])) : 0.f;
        m = v > m ? v : m;
    }
    if constexpr (QUANT) {
        m = wave_butterfly(m, [](float p, float q) { return q > p ? q : p; });
        const float scale = act_scale(m), inv = __fdiv_rn(1.0f, scale);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int i = lane + 64 * w;
            if (i < H) xq[static_cast<int64_t>(row) * H + i] = act_quant(xs[w], inv);
        }
        if (lane == 0) {
            if (s32) s32[row] = scale;
            if (s16) s16[row] = f2h(scale);
        }
    }
}

using RmsFn = void (*)(const uint16_t*, const uint16_t*, int, float, uint16_t*, int8_t*, float*, uint16_t*, AddRows);

// Launches the kernel for M rows of H; VEC needs whole 16-byte chunks: H a
// multiple of 8 and aligned rows, and more than one element a thread: up to 256
// it loads x twice where the strided form has everything in one load each
// (M=50000 H=128 33.3 us in chunks, 24.3 strided; M=8192 H=256 7.8 / 6.3).  (A wave per row, without barriers, was slower
// below 8192 rows: M=512 H=1024 3.9 us against 3.1, M=2000 H=2048 13.6 / 7.9.)
template <bool QUANT, bool ADD = false>
void launch_rms(const uint16_t* x, const uint16_t* gamma, int64_t M, int64_t H, float eps, uint16_t* normed, int8_t* xq,
                float* s32, uint16_t* s16, hipStream_t stream, const AddRows& add = {}) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gamma) |
                         reinterpret_cast<uintptr_t>(normed) | (reinterpret_cast<uintptr_t>(xq) << 1) |
                         reinterpret_cast<uintptr_t>(add.other) | reinterpret_cast<uintptr_t>(add.sum) |
                         static_cast<uintptr_t>(2 * (add.x_row | add.other_row | add.sum_row));
    const bool vec = H % 8 == 0 && at % 16 == 0;
    const int h = static_cast<int>(H);
    RmsFn fn = rms_row_kernel<0, false, QUANT, ADD>;
    if (H <= 256) {
        if constexpr (ADD) {
            hipLaunchKernelGGL(rms_add_short_kernel<QUANT>, dim3(static_cast<unsigned>(ceil_div(M, 4))), dim3(256), 0, stream, x, gamma, static_cast<int>(M), h, eps,
                               normed, xq, s32, s16, add);
            return;
        } else {
            fn = rms_row_kernel<1, false, QUANT>;
        }
    } else if (H <= 1024) fn = vec ? rms_row_kernel<4, true, QUANT, ADD> : rms_row_kernel<4, false, QUANT, ADD>;
    else if (H <= 2048) fn = vec ? rms_row_kernel<8, true, QUANT, ADD> : rms_row_kernel<8, false, QUANT, ADD>;
    else if (H <= 4096) fn = vec ? rms_row_kernel<16, true, QUANT, ADD> : rms_row_kernel<16, false, QUANT, ADD>;
    else if (H <= 8192) fn = vec ? rms_row_kernel<32, true, QUANT, ADD> : rms_row_kernel<32, false, QUANT, ADD>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(M)), dim3(256), 0, stream, x, gamma, h, eps, normed, xq, s32, s16, add);
}

}  // namespace mcv
