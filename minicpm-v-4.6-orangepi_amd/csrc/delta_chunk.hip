// delta_chunk.hip -- the gated delta rule over chunks of 64 tokens on the matrix cores, gfx950.
//
// Inside a chunk, with G the running sum of g, k^ = rk k and q^ = rq q the (normalised)
// rows and S the state before it, the rule's 64 rank-one updates are
//   (I + L) U = diag(beta) (V - diag(e^G) K^ S),   L[i][j] = beta_i e^(G_i - G_j) k^_i . k^_j, j < i
//   O  = scale (diag(e^G) Q^ S + P U),             P[i][j] = e^(G_i - G_j) q^_i . k^_j, j <= i
//   S' = e^(G_last) S + K^^T diag(e^(G_last - G)) U
// With T = (I + L)^-1:  U = T diag(beta) V - W S,  W = T diag(beta e^G) K^: all but two
// products per chunk need no state.  Two launches:
//   delta_prepare_kernel  every (chunk, value head) at once: L, T, P, W, T diag(beta) V
//   delta_scan_kernel     a workgroup per 16 NT columns of one state walks its chunks
//
// Precision.  The state, G, L, T and all sums are fp32 (G's differences from a sum in 64
// bits; T by substitution, in fp32 products).  Operands of the products that the state
// depends on are two fp16 parts, 22 bits, of which only lo x lo is left out; k and v
// are fp16 as they come.  What only out depends on, one fp16 value itself, takes one
// part: S, U and P rounded once each.  fp16's range: k rows are scaled by the
// power of two next to their norm's factor, q's norm is taken out of P, and the
// scan works on states and values scaled by a power of two that brings the largest to
// 8 .. 16, so that they may grow 4096-fold and a part's last bit is 2^-25 at worst.
//
// Operand order.  v_mfma_f32_16x16x32_f16 leaves lane (c, j) = (lane % 16, lane / 16) column c
// and rows 4j .. 4j + 3 of a 16 x 16 tile; as an operand it wants row (or column) c and eight
// of the 32 summed-over indexes, which may be any eight as long as both operands agree.
// Index 8j + e of a step stands for 4j + e (e < 4) or 16 + 4j + e - 4: two tiles' results
// are then an operand as they lie in the registers.  S, U, W and P pass from product to
// product that way, and everything in the workspace is kept in it, 16 bytes a lane.
#include <algorithm>

#include "delta_rule.h"

namespace mcv {
namespace {

constexpr int kC = 64;                           // tokens of a chunk
constexpr int64_t kSegmentBytes = int64_t(192) << 20;   // workspace of one pass over the chunks
constexpr int kScalars = 256;                    // floats a (chunk, head): ef, eq, osc (64 each), then:
constexpr int kKeep = 192, kVmax = 193;          // e^(G_last), largest |T diag(beta) V| of each wave (4)

struct ChunkArgs {
    DeltaArgs d;
    uint4* W;                                    // [unit][2 parts][4 token tiles][Dk / 32][64]
    uint4* U;                                    // [unit][Dv / 16][4][64] fp32
    uint4* P;                                    // [unit][4][2][64]
    uint4* K;                                    // [slot][Hk][Dk / 16][2][64]
    float* sc;                                   // [unit][kScalars]
    int Hk, slot0, slots;                        // the slots of this pass; unit = slot * Hv + head
};

// Chunk c of sequence b has slot cu[b] / 64 + b + c: no two share one, and there are
// at most T / 64 + B, without a table of chunks.
__device__ __forceinline__ int first_slot(int t0, int b) { return t0 / kC + b; }

// The sequence whose slots include `slot`: the last b whose first slot is not past it.
__device__ __forceinline__ int seq_of_slot(const DeltaArgs& p, int slot) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
        int t0 = 0, t1;
        const int mine = b0 + lane;
        if (mine < p.B) delta_span(p, mine, t0, t1);
        const unsigned long long on = __ballot(mine < p.B && first_slot(t0, mine) <= slot);
        if (on) b = b0 + 63 - __builtin_clzll(on);
        if (on != ~0ull) break;
    }
    return __builtin_amdgcn_readfirstlane(b);
}

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half8_t as_h8(uint4 v) { return __builtin_bit_cast(half8_t, v); }
__device__ __forceinline__ uint4 as_u4(half8_t v) { return __builtin_bit_cast(uint4, v); }
__device__ __forceinline__ float4_t mfma16(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// x in two fp16 parts.  (The empty asm hides the product that x may be: the backend folds one into
// the conversion, rounded once, at one of hi's two uses, and lo no longer belongs to hi.)
__device__ __forceinline__ void split(float x, _Float16& hi, _Float16& lo) {
    asm("" : "+v"(x));
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}
// LDS is ready for the other waves; global loads in flight stay there.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Position of token t's value in row d of a transposed tile [D][64] fp16: operand order,
// 16-byte blocks moved so that neither the pair stores nor the operand loads conflict.
__device__ __forceinline__ int turned(int d, int block) { return d * 64 + ((block ^ d ^ (d >> 3)) & 7) * 8; }
__device__ __forceinline__ int token_block(int t) { return (t / 32) * 4 + (t % 16) / 4; }
__device__ __forceinline__ int token_in_block(int t) { return t % 4 + (t % 32) / 16 * 4; }

template <int DK>
__global__ __launch_bounds__(256, 2) void delta_prepare_kernel(ChunkArgs a) {
    constexpr int KS = DK / 32;
    constexpr int PT = kC + 4;                   // row of L and T in LDS
    const DeltaArgs& p = a.d;
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % p.Hv, local = blockIdx.x / p.Hv, hk = h / p.group;
    const int slot = a.slot0 + local;
    const int b = seq_of_slot(p, slot);
    int t0, t1;
    delta_span(p, b, t0, t1);
    const int chunk = slot - first_slot(t0, b);
    const int64_t start = t0 + static_cast<int64_t>(chunk) * kC;
    if (chunk < 0 || start >= t1) return;
    const int n = t1 - start < kC ? static_cast<int>(t1 - start) : kC;
    const int64_t unit = static_cast<int64_t>(local) * p.Hv + h;

    __shared__ __attribute__((aligned(16))) _Float16 kt[DK * kC], vt[256 * kC / 4];   // v: 64 columns at a time
    __shared__ __attribute__((aligned(16))) float tri[kC][PT];
    __shared__ float gh[kC], gl[kC], bet[kC], rkn[kC], rqn[kC], kk[kC], qq[kC], wsc[kC];
    __shared__ _Float16 kpow[kC];

    const uint16_t* qb = p.q + start * p.q_row + hk * p.q_head;
    const uint16_t* kb = p.k + start * p.k_row + hk * p.k_head;
    const uint16_t* vb = p.v + start * p.v_row + h * p.v_head;
    const uint4 zero = make_uint4(0, 0, 0, 0);

    // products of the raw rows: this wave's 16 tokens against those up to them
    float4_t kkt[4], kqt[4], qqt = {};
    {
        half8_t qf[KS], kw[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int t = 16 * w + c;
            qf[s] = as_h8(t < n ? *reinterpret_cast<const uint4*>(qb + t * p.q_row + 32 * s + 8 * j) : zero);
            kw[s] = as_h8(t < n ? *reinterpret_cast<const uint4*>(kb + t * p.k_row + 32 * s + 8 * j) : zero);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) qqt = mfma16(qf[s], qf[s], qqt);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            kkt[x] = kqt[x] = float4_t{0, 0, 0, 0};
            if (x > w) continue;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int t = 16 * x + c;
                const half8_t kx = as_h8(t < n ? *reinterpret_cast<const uint4*>(kb + t * p.k_row + 32 * s + 8 * j) : zero);
                kkt[x] = mfma16(kw[s], kx, kkt[x]);
                kqt[x] = mfma16(kx, qf[s], kqt[x]);
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (x == w && c == 4 * j + r) {
                    kk[16 * w + c] = kkt[x][r];
                    qq[16 * w + c] = qqt[r];
                }
    }
    if (w == 0) {
        // a decay below e^-200 is none in 32 bits; G's differences want more than a 32-bit sum
        double G = lane < n ? static_cast<double>(fmaxf(p.g[(start + lane) * p.g_row + h], -200.f)) : 0.0;
        for (int m = 1; m < 64; m <<= 1) {
            const double o = __shfl_up(G, m, 64);
            if (lane >= m) G += o;
        }
        gh[lane] = static_cast<float>(G);
        gl[lane] = static_cast<float>(G - static_cast<double>(static_cast<float>(G)));
    } else if (w == 1) {
        bet[lane] = lane < n ? p.beta[(start + lane) * p.beta_row + h] : 0.f;
    }
    __syncthreads();
    float* const sc = a.sc + unit * kScalars;
    if (w == 0) {
        const float k2 = kk[lane], q2 = qq[lane];
        const float rk = p.normalize ? 1.0f / sqrtf(k2 + kDeltaEps) : 1.0f;
        const float pw = p.normalize ? ldexpf(1.0f, ilogbf(rk)) : 1.0f;
        const float rn = q2 > 0.f ? 1.0f / sqrtf(q2) : 0.f;
        const float G = gh[lane], last = gh[kC - 1];
        const float fall = expf((last - G) + (gl[kC - 1] - gl[lane]));
        rkn[lane] = rk;
        rqn[lane] = rn;
        kpow[lane] = static_cast<_Float16>(pw);
        wsc[lane] = bet[lane] * expf(G) * (rk / pw);
        sc[lane] = fall * (rk / pw);
        sc[64 + lane] = expf(G) * rn;
        sc[128 + lane] = p.scale * (p.normalize ? sqrtf(q2 / (q2 + kDeltaEps)) : sqrtf(q2));
        if (lane == 0) sc[kKeep] = expf(last);
    }
    __syncthreads();

    // L into LDS; P, one part, straight out: its tile pairs are operands
    const float ghc = gh[16 * w + c], glc = gl[16 * w + c], rqc = rqn[16 * w + c];
    float4_t pt[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        pt[x] = float4_t{0, 0, 0, 0};
        if (x > w) {
            if (x == w + 1 && (w & 1) == 0)      // the other half of T's own step
#pragma unroll
                for (int r = 0; r < 4; ++r) tri[16 * w + 4 * j + r][16 * x + c] = 0.f;
            continue;
        }
        const float gx = gh[16 * x + c], gxl = gl[16 * x + c], rkx = rkn[16 * x + c];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * w + 4 * j + r;    // L: row i, column 16 x + c
            const float f = bet[i] * expf((gh[i] - gx) + (gl[i] - gxl)) * rkn[i] * rkx;
            tri[i][16 * x + c] = 16 * x + c < i ? f * kkt[x][r] : 0.f;
            const int y = 16 * x + 4 * j + r;    // P: key y, query 16 w + c
            const float e = expf((ghc - gh[y]) + (glc - gl[y])) * rkn[y] * rqc;
            pt[x][r] = y <= 16 * w + c ? e * kqt[x][r] : 0.f;
        }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (2 * s > w) continue;
        half8_t o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = static_cast<_Float16>(pt[2 * s + e / 4][e % 4]);
        a.P[((unit * 4 + w) * 2 + s) * 64 + lane] = as_u4(o);
    }
    // k, scaled, turned: a thread packs two tokens of eight d
    for (int i = threadIdx.x; i < kC / 2 * (DK / 8); i += 256) {
        const int t = 2 * (i / (DK / 8)), ch = i % (DK / 8);
        uint4 x = t < n ? *reinterpret_cast<const uint4*>(kb + t * p.k_row + 8 * ch) : zero;
        uint4 y = t + 1 < n ? *reinterpret_cast<const uint4*>(kb + (t + 1) * p.k_row + 8 * ch) : zero;
        const half8_t hx = as_h8(x) * kpow[t], hy = as_h8(y) * kpow[t + 1];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            *reinterpret_cast<half2_t*>(kt + turned(8 * ch + e, token_block(t)) + token_in_block(t)) = half2_t{hx[e], hy[e]};
    }
    __syncthreads();

    // T: the diagonal blocks by substitution, lane c a column; in place
    {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == c ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < i; ++m) s = fmaf(-tri[16 * w + i][16 * w + m], x[m], s);
            x[i] = s;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i / 4 == j) tri[16 * w + i][16 * w + c] = x[i];
    }
    __syncthreads();
    // ... and block column w under it: T[i][w] = -T[i][i] sum over k of L[i][k] T[k][w]
    float4_t col[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) col[0][r] = tri[16 * w + 4 * j + r][16 * w + c];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        col[i] = float4_t{0, 0, 0, 0};
        if (w + i > 3) continue;
        float4_t s = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < i; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s = __builtin_amdgcn_mfma_f32_16x16x4f32(tri[16 * (w + i) + c][16 * (w + k) + 4 * j + r], col[k][r], s, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            col[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-tri[16 * (w + i) + c][16 * (w + i) + 4 * j + r], s[r], col[i], 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 1; i < 4; ++i)
        if (w + i < 4)
#pragma unroll
            for (int r = 0; r < 4; ++r) tri[16 * (w + i) + 4 * j + r][16 * w + c] = col[i][r];
    __syncthreads();

    // T diag(beta) and T diag(beta e^G f), two parts each, of this wave's rows
    half8_t th[2][2], tw[2][2];                  // [step][part]
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int y = 32 * s + 4 * j + e % 4 + e / 4 * 16;
            const float t = 2 * s <= w ? tri[16 * w + c][y] : 0.f;
            _Float16 hi, lo;
            split(t * bet[y], hi, lo);
            th[s][0][e] = hi;
            th[s][1][e] = lo;
            split(t * wsc[y], hi, lo);
            tw[s][0][e] = hi;
            tw[s][1][e] = lo;
        }
    }
    // -W, turned: rows dk, column token, so that two tiles are an operand of W S
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        half8_t hi, lo;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int d = 32 * s + 16 * x + c;
            float4_t acc = {0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (2 * y > w) continue;
                const half8_t kf = *reinterpret_cast<const half8_t*>(kt + turned(d, 4 * y + j));
                acc = mfma16(kf, tw[y][0], acc);
                acc = mfma16(kf, tw[y][1], acc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                _Float16 u, v;
                split(-acc[r], u, v);
                hi[4 * x + r] = u;
                lo[4 * x + r] = v;
            }
        }
        a.W[((unit * 2 * 4 + w) * KS + s) * 64 + lane] = as_u4(hi);
        a.W[(((unit * 2 + 1) * 4 + w) * KS + s) * 64 + lane] = as_u4(lo);
    }
    if (h % p.group == 0)
        for (int i = w; i < DK / 16 * 2; i += 4)
            a.K[((static_cast<int64_t>(local) * a.Hk + hk) * (DK / 16) * 2 + i) * 64 + lane] =
                *reinterpret_cast<const uint4*>(kt + turned(16 * (i / 2) + c, 4 * (i % 2) + j));
    // T diag(beta) V, 64 columns of v at a time
    float big = 0.f;
    for (int v0 = 0; v0 < p.Dv; v0 += 64) {
        const int width = p.Dv - v0 < 64 ? p.Dv - v0 : 64;
        if (v0) __syncthreads();
        for (int i = threadIdx.x; i < kC / 2 * 8; i += 256) {
            const int t = 2 * (i / 8), ch = i % 8;
            if (8 * ch >= width) continue;
            const uint4 x = t < n ? *reinterpret_cast<const uint4*>(vb + t * p.v_row + v0 + 8 * ch) : zero;
            const uint4 y = t + 1 < n ? *reinterpret_cast<const uint4*>(vb + (t + 1) * p.v_row + v0 + 8 * ch) : zero;
            const half8_t hx = as_h8(x), hy = as_h8(y);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                *reinterpret_cast<half2_t*>(vt + turned(8 * ch + e, token_block(t)) + token_in_block(t)) = half2_t{hx[e], hy[e]};
        }
        __syncthreads();
        for (int x = 0; x < width / 16; ++x) {
            float4_t acc = {0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (2 * y > w) continue;
                const half8_t vf = *reinterpret_cast<const half8_t*>(vt + turned(16 * x + c, 4 * y + j));
                acc = mfma16(th[y][0], vf, acc);
                acc = mfma16(th[y][1], vf, acc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) big = fmaxf(big, fabsf(acc[r]));
            a.U[((unit * (p.Dv / 16) + v0 / 16 + x) * 4 + w) * 64 + lane] = __builtin_bit_cast(uint4, acc);
        }
    }
    big = wave_butterfly(big, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) sc[kVmax + w] = big;
}

// Waves 0 .. 3 carry the state: wave w has rows w DK / 4 .. of it and token tile w of U.
// Waves 4 .. 7 make the outputs of token tile w - 4.
template <int DK, int NT>
__global__ __launch_bounds__(512, 2) void delta_scan_kernel(ChunkArgs a) {
    constexpr int KS = DK / 32, MT = DK / 64;    // steps over dk; 16-row tiles of the state a wave carries
    constexpr int PD = 2;                        // chunks whose operands are in flight
    const DeltaArgs& p = a.d;
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave & 3;
    const int slices = p.Dv / (16 * NT), heads = p.B * p.Hv;
    // all slices of one state on one XCD (workgroup id % 8): they read the same operands
    const int r8 = blockIdx.x / 8, slice = r8 % slices, bh = r8 / slices * 8 + blockIdx.x % 8;
    if (bh >= heads) return;
    const int b = bh / p.Hv, h = bh % p.Hv, hk = h / p.group;
    int t0, t1;
    delta_span(p, b, t0, t1);
    const int s0 = first_slot(t0, b), chunks = (t1 - t0 + kC - 1) / kC;
    int c0 = a.slot0 - s0, c1 = a.slot0 + a.slots - s0;
    c0 = c0 < 0 ? 0 : c0;
    c1 = c1 > chunks ? chunks : c1;
    const bool starts = s0 >= a.slot0 && s0 < a.slot0 + a.slots;
    if (c0 >= c1 && !(chunks == 0 && starts)) return;
    const int dv0 = slice * 16 * NT;
    const int64_t at = p.state_index ? p.state_index[b] : b;
    if (at < 0 || at >= p.n_states) {
        for (int64_t i = threadIdx.x; i < static_cast<int64_t>(c1 - c0) * kC * NT * 2; i += 512) {
            const int64_t t = t0 + static_cast<int64_t>(c0) * kC + i / (NT * 2);
            if (t < t1) *reinterpret_cast<uint4*>(p.out + (t * p.Hv + h) * p.Dv + dv0 + i % (NT * 2) * 8) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    __shared__ __attribute__((aligned(16))) uint2 sf[2][NT][KS][64][2];       // S, two parts, operand order
    __shared__ __attribute__((aligned(16))) uint2 uf[3][NT][2][64][2];        // U; e^(G_last - G) f U in two parts
    __shared__ float maxes[8];

    // the state and the scale of this pass
    const int count = c1 > c0 ? c1 - c0 : 0;
    float4_t S[MT][NT];
    const float* src = starts ? p.state : p.state_out;
    const int64_t base = (at * p.Hv + h) * DK * p.Dv + dv0 + c;
    float big = 0.f;
    if (wave < 4) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = 16 * (MT * w + m) + 4 * j + r;
                    S[m][x][r] = src ? src[base + static_cast<int64_t>(dk) * p.Dv + 16 * x] : 0.f;
                    big = fmaxf(big, fabsf(S[m][x][r]));
                }
    }
    if (count == 0) {                            // no token: the state as it is
        if (wave < 4)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        p.state_out[base + static_cast<int64_t>(16 * (MT * w + m) + 4 * j + r) * p.Dv + 16 * x] = S[m][x][r];
        return;
    }
    const int64_t unit0 = (static_cast<int64_t>(s0 + c0 - a.slot0)) * p.Hv + h;      // unit of chunk c0; the next is Hv on
    for (int i = threadIdx.x; i < (c1 - c0) * 4; i += 512)
        big = fmaxf(big, a.sc[(unit0 + static_cast<int64_t>(i / 4) * p.Hv) * kScalars + kVmax + i % 4]);
    big = wave_butterfly(big, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) maxes[wave] = big;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) big = fmaxf(big, maxes[i]);
    int ex = big > 0.f && big < INFINITY ? 3 - ilogbf(big) : 0;
    ex = ex > 100 ? 100 : ex < -100 ? -100 : ex;
    const float up = ldexpf(1.0f, ex), down = ldexpf(1.0f, -ex);

    if (wave < 4) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < NT; ++x) S[m][x] *= up;
        struct Stage {
            uint4 wf[2][KS], kf[MT][2], u[NT];
            float4_t ef;
            float keep;
        } st[PD];
        auto load = [&](Stage& s, int i) {
            const int64_t unit = unit0 + static_cast<int64_t>(i) * p.Hv;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int k = 0; k < KS; ++k) s.wf[q][k] = a.W[(((unit * 2 + q) * 4 + w) * KS + k) * 64 + lane];
#pragma unroll
            for (int x = 0; x < NT; ++x) s.u[x] = a.U[((unit * (p.Dv / 16) + slice * NT + x) * 4 + w) * 64 + lane];
            const float* sc = a.sc + unit * kScalars;
            s.ef = *reinterpret_cast<const float4_t*>(sc + 16 * w + 4 * j);
            s.keep = sc[kKeep];
            const uint4* kp = a.K + (static_cast<int64_t>(s0 + c0 + i - a.slot0) * a.Hk + hk) * (DK / 16) * 2 * 64 + lane;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q) s.kf[m][q] = kp[((MT * w + m) * 2 + q) * 64];
        };
        auto put_state = [&]() {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    half4_t hi, lo;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        _Float16 u, v;
                        split(S[m][x][r], u, v);
                        hi[r] = u;
                        lo[r] = v;
                    }
                    const int tile = MT * w + m;
                    sf[0][x][tile / 2][lane][tile % 2] = __builtin_bit_cast(uint2, hi);
                    sf[1][x][tile / 2][lane][tile % 2] = __builtin_bit_cast(uint2, lo);
                }
        };
#pragma unroll
        for (int q = 0; q < PD; ++q)
            if (q < count) load(st[q], q);
        put_state();
        for (int i0 = 0; i0 < count; i0 += PD)
#pragma unroll
            for (int q = 0; q < PD; ++q) {
                const int i = i0 + q;
                if (i >= count) break;
                Stage& s = st[q];
                lds_barrier();                   // S is there
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    float4_t u = __builtin_bit_cast(float4_t, s.u[x]) * up, v = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&sf[0][x][k][lane][0]));
                        const half8_t lo = as_h8(*reinterpret_cast<const uint4*>(&sf[1][x][k][lane][0]));
                        u = mfma16(as_h8(s.wf[0][k]), hi, u);
                        v = mfma16(as_h8(s.wf[0][k]), lo, v);
                        v = mfma16(as_h8(s.wf[1][k]), hi, v);
                    }
                    u += v;
                    half4_t o, hi, lo;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        _Float16 y, z;
                        o[r] = static_cast<_Float16>(u[r]);
                        split(s.ef[r] * u[r], y, z);
                        hi[r] = y;
                        lo[r] = z;
                    }
                    uf[0][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, o);
                    uf[1][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, hi);
                    uf[2][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, lo);
                }
                lds_barrier();                   // U is there, S is read
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        S[m][x] *= s.keep;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&uf[1][x][k][lane][0]));
                            const half8_t lo = as_h8(*reinterpret_cast<const uint4*>(&uf[2][x][k][lane][0]));
                            S[m][x] = mfma16(as_h8(s.kf[m][k]), hi, S[m][x]);
                            S[m][x] = mfma16(as_h8(s.kf[m][k]), lo, S[m][x]);
                        }
                    }
                put_state();
                if (i + PD < count) load(s, i + PD);
            }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int dk = 16 * (MT * w + m) + 4 * j + r;
                    p.state_out[base + static_cast<int64_t>(dk) * p.Dv + 16 * x] = S[m][x][r] * down;
                }
    } else {
        struct Stage {
            uint4 pf[2];
            uint2 qf[KS][2];
            float eq, osc;
        } st[PD];
        auto load = [&](Stage& s, int i) {
            const int64_t unit = unit0 + static_cast<int64_t>(i) * p.Hv;
            const int64_t first = t0 + static_cast<int64_t>(c0 + i) * kC;
            int64_t t = first + 16 * w + c;
            t = t < t1 ? t : t1 - 1;             // rows past the end: any, they are not stored
            const uint16_t* qp = p.q + t * p.q_row + hk * p.q_head + 4 * j;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                s.qf[k][0] = *reinterpret_cast<const uint2*>(qp + 32 * k);
                s.qf[k][1] = *reinterpret_cast<const uint2*>(qp + 32 * k + 16);
            }
            s.pf[0] = a.P[((unit * 4 + w) * 2) * 64 + lane];
            if (w >= 2) s.pf[1] = a.P[((unit * 4 + w) * 2 + 1) * 64 + lane];
            s.eq = a.sc[unit * kScalars + 64 + 16 * w + c];
            s.osc = a.sc[unit * kScalars + 128 + 16 * w + c] * down;
        };
#pragma unroll
        for (int q = 0; q < PD; ++q)
            if (q < count) load(st[q], q);
        for (int i0 = 0; i0 < count; i0 += PD)
#pragma unroll
            for (int q = 0; q < PD; ++q) {
                const int i = i0 + q;
                if (i >= count) break;
                Stage& s = st[q];
                lds_barrier();                   // S is there
                float4_t o[NT];
#pragma unroll
                for (int x = 0; x < NT; ++x) {   // rows dv, column token
                    o[x] = float4_t{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&sf[0][x][k][lane][0]));
                        const half8_t qv = as_h8(make_uint4(s.qf[k][0].x, s.qf[k][0].y, s.qf[k][1].x, s.qf[k][1].y));
                        o[x] = mfma16(hi, qv, o[x]);
                    }
                    o[x] *= s.eq;
                }
                lds_barrier();                   // U is there
                const int64_t t = t0 + static_cast<int64_t>(c0 + i) * kC + 16 * w + c;
#pragma unroll
                for (int x = 0; x < NT; ++x) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (2 * k > w) continue;
                        o[x] = mfma16(as_h8(*reinterpret_cast<const uint4*>(&uf[0][x][k][lane][0])), as_h8(s.pf[k]), o[x]);
                    }
                    uint16_t r[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = f2h(o[x][e] * s.osc);
                    if (t < t1)
                        *reinterpret_cast<uint2*>(p.out + (t * p.Hv + h) * p.Dv + dv0 + 16 * x + 4 * j) =
                            make_uint2(r[0] | (static_cast<uint32_t>(r[1]) << 16), r[2] | (static_cast<uint32_t>(r[3]) << 16));
                }
                if (i + PD < count) load(s, i + PD);
            }
    }
}

// Bytes per slot, all heads.
int64_t slot_bytes(int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv) {
    return Hv * (kC * Dk * 4 + kC * Dv * 4 + kC * kC * 2 + kScalars * 4) + Hk * kC * Dk * 2;
}
int64_t all_slots(int64_t B, int64_t T) { return T / kC + B; }
int64_t pass_slots(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv) {
    return std::min(all_slots(B, T), std::max<int64_t>(kSegmentBytes / slot_bytes(Hk, Hv, Dk, Dv), 1));
}

}  // namespace

int64_t delta_chunk_workspace(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv) {
    return pass_slots(B, T, Hk, Hv, Dk, Dv) * slot_bytes(Hk, Hv, Dk, Dv);
}

int launch_delta_chunk(const DeltaArgs& d, int Hk, int Dk, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    ChunkArgs a;
    a.d = d;
    a.Hk = Hk;
    const int64_t total = all_slots(d.B, d.T), per = pass_slots(d.B, d.T, Hk, d.Hv, Dk, d.Dv), units = per * d.Hv;
    uint8_t* at = static_cast<uint8_t*>(workspace);
    auto take = [&](int64_t bytes) {
        uint8_t* was = at;
        at += bytes;
        return was;
    };
    a.W = reinterpret_cast<uint4*>(take(units * kC * Dk * 4));
    a.U = reinterpret_cast<uint4*>(take(units * kC * d.Dv * 4));
    a.P = reinterpret_cast<uint4*>(take(units * kC * kC * 2));
    a.sc = reinterpret_cast<float*>(take(units * kScalars * 4));
    a.K = reinterpret_cast<uint4*>(take(per * Hk * kC * Dk * 2));
    if (at - static_cast<uint8_t*>(workspace) > workspace_bytes) return fail(MCV_ERR_INVALID_ARG, "delta_rule: workspace too small");
    // columns of a state per workgroup: the widest slice that still leaves two workgroups a CU
    const int64_t states = ceil_div(static_cast<int64_t>(d.B) * d.Hv, 8) * 8, tiles = d.Dv / 16;
    int nt = 1;
    for (int x : {2, 4})
        if (tiles % x == 0 && states * (tiles / x) >= 512) nt = x;
    for (int64_t s = 0; s < total; s += per) {
        a.slot0 = static_cast<int>(s);
        a.slots = static_cast<int>(std::min(per, total - s));
        hipLaunchKernelGGL((Dk == 64 ? delta_prepare_kernel<64> : delta_prepare_kernel<128>),
                           dim3(static_cast<unsigned>(a.slots * static_cast<int64_t>(d.Hv))), dim3(256), 0, stream, a);
        int rc = check_launch("delta_prepare_kernel");
        if (rc != MCV_OK) return rc;
        auto fn = Dk == 64 ? (nt == 1 ? delta_scan_kernel<64, 1> : nt == 2 ? delta_scan_kernel<64, 2> : delta_scan_kernel<64, 4>)
                           : (nt == 1 ? delta_scan_kernel<128, 1> : nt == 2 ? delta_scan_kernel<128, 2> : delta_scan_kernel<128, 4>);
        hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(states * (tiles / nt))), dim3(512), 0, stream, a);
        rc = check_launch("delta_scan_kernel");
        if (rc != MCV_OK) return rc;
    }
    return MCV_OK;
}

}  // namespace mcv
