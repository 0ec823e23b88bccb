// delta_chunk.hip -- the gated delta rule over chunks of 64 tokens on the matrix cores, gfx950.
//
// Inside a chunk, with G the running sum of g, k^ = rk k and q^ = rq q the (normalised)
// rows and S the state before it, the rule's 64 rank-one updates are
//   (I + L) U = diag(beta) (V - diag(e^G) K^ S),   L[i][j] = beta_i e^(G_i - G_j) k^_i . k^_j, j < i
//   O  = scale (diag(e^G) Q^ S + P U),             P[i][j] = e^(G_i - G_j) q^_i . k^_j, j <= i
//   S' = e^(G_last) S + K^^T diag(e^(G_last - G)) U
// and with T = (I + L)^-1:  X = diag(beta) (V - diag(e^G) K^ S),  U = T X.  Two launches:
//   delta_prepare_kernel  every (chunk, value head) at once: T, P, the scalars, K turned
//   delta_scan_kernel     a workgroup per 16 NT columns of one state walks its chunks
// The scan takes K and V as they come and applies T, instead of T K and T V made ahead: three
// products that wait for one another in place of two, but 41 KiB a (chunk, head) through
// memory in place of 88, and K, exact in fp16, in place of T K in two parts.
//
// Precision.  The state, G, L, T and all sums are fp32 (G's differences from a sum in 64
// bits; T by substitution, in fp32 products).  Operands of products are two fp16 parts,
// 22 bits, of which only lo x lo is left out; q, k and v are fp16 as they come.  fp16's
// range: turned k rows are scaled by the power of two next to their norm's factor, q's
// norm is taken out of P, and the scan works on states and values scaled by a power of
// two that brings the largest to 8 .. 16, so that they may grow 4096-fold and a part's
// last bit is 2^-25 at worst.
//
// Operand order.  v_mfma_f32_16x16x32_f16 leaves lane (c, j) = (lane % 16, lane / 16) column c
// and rows 4j .. 4j + 3 of a 16 x 16 tile; as an operand it wants row (or column) c and eight
// of the 32 summed-over indexes, which may be any eight as long as both operands agree.
// Two tiles' results, eight rows, are an operand as they lie in the registers: of tokens,
// index 8j + e stands for 4j + e (e < 4) or 16 + 4j + e - 4; of the state, tile m's row 4j + r
// is dk 8j + 4m + r of its 32, so that the other operand is 16 bytes of a row of k or q.
#include <algorithm>

#include "delta_rule.h"

namespace mcv {
namespace {

constexpr int kC = 64;                           // tokens of a chunk
constexpr int64_t kSegmentBytes = int64_t(192) << 20;   // workspace of one pass over the chunks
constexpr int kBet = 0, kBr = 64, kEf = 128, kEq = 192, kOsc = 256;   // of a unit's scalars, 64 each, then:
constexpr int kKeep = 320, kVmax = 321;          // e^(G_last), largest |v| each wave saw (4)
constexpr int kScalars = 352;
constexpr int kTriBytes = 6 * 2 * 64 * 16;       // a triangle of 16 x 32 blocks, two parts

struct ChunkArgs {
    DeltaArgs d;
    uint4* T;                                    // [unit][tri_block][2 parts][64]
    uint4* P;                                    // the same
    uint4* Kt;                                   // [slot][Hk][Dk / 16][2][64]: k turned, scaled
    uint4* K;                                    // [slot][Hk][4 token tiles][Dk / 32][64]
    uint4* Q;                                    // the same
    float* sc;                                   // [unit][kScalars]
    int Hk, slot0, slots;                        // the slots of this pass; unit = slot * Hv + head
};

// Block of row tile w and step s (32 columns) of a lower triangle, s <= w / 2.
__device__ __forceinline__ int tri_block(int w, int s) { return (w < 2 ? w : 2 * w - 2) + s; }

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
typedef float float8_t __attribute__((ext_vector_type(8)));

__device__ __forceinline__ half8_t as_h8(uint4 v) { return __builtin_bit_cast(half8_t, v); }
__device__ __forceinline__ uint4 as_u4(half8_t v) { return __builtin_bit_cast(uint4, v); }
__device__ __forceinline__ float4_t mfma16(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// x in two fp16 parts; the second is rounded from x - hi, which one fused product has exactly.
template <int N, class F, class V>
__device__ __forceinline__ void split(F x, V& hi, V& lo) {
    typedef float floats __attribute__((ext_vector_type(N)));
    hi = __builtin_convertvector(x, V);
    floats l;
#pragma unroll
    for (int e = 0; e < N; ++e) l[e] = fmaf(static_cast<float>(hi[e]), -1.0f, x[e]);
    lo = __builtin_convertvector(l, V);
}
// A product or sum that is split: the backend would fold it into the conversion, rounded once, at one of
// hi's two uses, and lo would no longer belong to hi.
__device__ __forceinline__ float apart(float x) {
    asm("" : "+v"(x));
    return x;
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// LDS is ready for the other waves; global loads in flight stay there.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Position of token t's value in row d of a transposed tile [D][64] fp16: operand order,
// 16-byte blocks moved so that neither the pair stores nor the operand loads conflict.
__device__ __forceinline__ int turned(int d, int block) { return d * 64 + ((block ^ d ^ (d >> 3)) & 7) * 8; }
__device__ __forceinline__ int token_block(int t) { return (t / 32) * 4 + (t % 16) / 4; }
__device__ __forceinline__ int token_in_block(int t) { return t % 4 + (t % 32) / 16 * 4; }

template <int DK>
__global__ __launch_bounds__(256, 3) void delta_prepare_kernel(ChunkArgs a) {
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

    // k and q as rows, 16-byte chunks moved so that operand reads do not conflict; then k turned and L, T
    constexpr int RC = DK / 8;                   // chunks of a row
    __shared__ __attribute__((aligned(16))) uint8_t space[2][kC * PT * 4];
    __shared__ __attribute__((aligned(16))) float gh[kC], gl[kC], bet[kC], rkn[kC], rqn[kC], kk[kC], qq[kC];
    __shared__ __attribute__((aligned(16))) _Float16 kpow[kC];
    half8_t* const kr = reinterpret_cast<half8_t*>(space[0]);
    half8_t* const qr = reinterpret_cast<half8_t*>(space[1]);
    float (*const tri)[PT] = reinterpret_cast<float (*)[PT]>(space[0]);
    _Float16* const kt = reinterpret_cast<_Float16*>(space[1]);
    auto place = [](int t, int ch) { return t * RC + (ch ^ (DK == 128 ? t & 15 : (t >> 1) & 7)); };

    const uint16_t* qb = p.q + start * p.q_row + hk * p.q_head;
    const uint16_t* kb = p.k + start * p.k_row + hk * p.k_head;
    const uint16_t* vb = p.v + start * p.v_row + h * p.v_head;
    float* const sc = a.sc + unit * kScalars;
    auto row = [&](int t) { return t < n ? t : n - 1; };         // rows past the end: read another, made zero
    const half8_t none = {};

    float gate = 0.f;
    if (w == 0) gate = p.g[(start + row(lane)) * p.g_row + h];
    else if (w == 1) gate = p.beta[(start + row(lane)) * p.beta_row + h];
    {
        constexpr int IT = kC * RC / 256;
        half8_t x[IT], y[IT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {           // (operand loads straight from the rows cost four times the lines)
            const int t = (threadIdx.x + 256 * i) / RC, ch = threadIdx.x % RC;
            x[i] = *reinterpret_cast<const half8_t*>(kb + row(t) * p.k_row + 8 * ch);
            y[i] = *reinterpret_cast<const half8_t*>(qb + row(t) * p.q_row + 8 * ch);
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int t = (threadIdx.x + 256 * i) / RC, ch = threadIdx.x % RC;
            kr[place(t, ch)] = t < n ? x[i] : none;
            qr[place(t, ch)] = t < n ? y[i] : none;
        }
    }
    __syncthreads();
    // Products of the raw rows: this wave's 16 tokens against those up to them.
    float4_t kkt[4], kqt[4], qqt = {};
    {
        half8_t qf[KS], kw[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = qr[place(16 * w + c, 4 * s + j)];
            kw[s] = kr[place(16 * w + c, 4 * s + j)];
        }
        if (h % p.group == 0) {
            const int64_t at = ((static_cast<int64_t>(local) * a.Hk + hk) * 4 + w) * KS * 64 + lane;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                a.K[at + s * 64] = as_u4(kw[s]);
                a.Q[at + s * 64] = as_u4(qf[s]);
            }
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) qqt = mfma16(qf[s], qf[s], qqt);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            kkt[x] = kqt[x] = float4_t{0, 0, 0, 0};
            if (x > w) continue;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const half8_t kx = kr[place(16 * x + c, 4 * s + j)];
                kkt[x] = mfma16(kw[s], kx, kkt[x]);
                kqt[x] = mfma16(kx, qf[s], kqt[x]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (x == w && c == 4 * j + r) {
                    kk[16 * w + c] = kkt[x][r];
                    qq[16 * w + c] = qqt[r];
                }
        }
    }
    if (w == 0) {
        // a decay below e^-200 is none in 32 bits; G's differences want more than a 32-bit sum
        double G = lane < n ? static_cast<double>(gate < -200.f ? -200.f : gate) * 1.4426950408889634074 : 0.0;
        for (int m = 1; m < 64; m <<= 1) {
            const double o = __shfl_up(G, m, 64);
            if (lane >= m) G += o;
        }
        gh[lane] = static_cast<float>(G);
        gl[lane] = static_cast<float>(G - static_cast<double>(static_cast<float>(G)));
    } else if (w == 1) {
        bet[lane] = lane < n ? gate : 0.f;
    }
    __syncthreads();
    // k turned: a thread packs two tokens of eight d
    for (int i = threadIdx.x; i < kC / 2 * RC; i += 256) {
        const int t = 2 * (i / RC), ch = i % RC;
        const half8_t x = kr[place(t, ch)], y = kr[place(t + 1, ch)];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            *reinterpret_cast<half2_t*>(kt + turned(8 * ch + e, token_block(t)) + token_in_block(t)) = half2_t{x[e], y[e]};
    }
    if (w == 0) {
        const float k2 = kk[lane], q2 = qq[lane];
        const float rk = p.normalize ? 1.0f / sqrtf(k2 + kDeltaEps) : 1.0f;
        const float pw = p.normalize ? ldexpf(1.0f, ilogbf(rk)) : 1.0f;
        const float rn = q2 > 0.f ? 1.0f / sqrtf(q2) : 0.f;
        const float eg = exp2f(gh[lane] + gl[lane]);
        const float fall = exp2f((gh[kC - 1] - gh[lane]) + (gl[kC - 1] - gl[lane]));
        rkn[lane] = rk;
        rqn[lane] = rn;
        kpow[lane] = static_cast<_Float16>(pw);
        sc[kBet + lane] = bet[lane];
        sc[kBr + lane] = bet[lane] * rk * eg;
        sc[kEf + lane] = fall * (rk / pw);
        sc[kEq + lane] = eg * rn;
        sc[kOsc + lane] = p.scale * (p.normalize ? sqrtf(q2 / (q2 + kDeltaEps)) : sqrtf(q2));
        if (lane == kC - 1) sc[kKeep] = eg;
    }
    __syncthreads();

    // L into LDS; P straight out: its tile pairs are operands
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
            const float f = bet[i] * exp2_of((gh[i] - gx) + (gl[i] - gxl)) * rkn[i] * rkx;
            tri[i][16 * x + c] = 16 * x + c < i ? f * kkt[x][r] : 0.f;
            const int y = 16 * x + 4 * j + r;    // P: key y, query 16 w + c
            const float e = exp2_of((ghc - gh[y]) + (glc - gl[y])) * rkn[y] * rqc;
            pt[x][r] = y <= 16 * w + c ? e * kqt[x][r] : 0.f;
        }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (2 * s > w) continue;
        half8_t hi, lo;
        float8_t x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = apart(pt[2 * s + e / 4][e % 4]);
        split<8>(x, hi, lo);
        uint4* at = a.P + (unit * 6 + tri_block(w, s)) * 2 * 64 + lane;
        at[0] = as_u4(hi);
        at[64] = as_u4(lo);
    }
    // K turned, scaled, in operand order: row c of tile i is dk 32 (i / 2) + 8 (c / 4) + 4 (i % 2) + c % 4
    if (h % p.group == 0)
#pragma unroll
        for (int i = w; i < DK / 16; i += 4) {
            const int d = 32 * (i / 2) + 8 * (c / 4) + 4 * (i % 2) + c % 4;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const half4_t p0 = *reinterpret_cast<const half4_t*>(kpow + 32 * s + 4 * j);
                const half4_t p1 = *reinterpret_cast<const half4_t*>(kpow + 32 * s + 16 + 4 * j);
                const half8_t pw = {p0[0], p0[1], p0[2], p0[3], p1[0], p1[1], p1[2], p1[3]};
                a.Kt[((static_cast<int64_t>(local) * a.Hk + hk) * (DK / 16) * 2 + i * 2 + s) * 64 + lane] =
                    as_u4(*reinterpret_cast<const half8_t*>(kt + turned(d, 4 * s + j)) * pw);
            }
        }
    // the largest |v|, for the scan's scale
    {
        uint32_t most = 0;                       // of fp16 magnitudes as whole numbers; NaN is none
        for (int i = threadIdx.x; i < kC * p.Dv / 8; i += 256) {
            const uint4 v = *reinterpret_cast<const uint4*>(vb + row(i / (p.Dv / 8)) * p.v_row + i % (p.Dv / 8) * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t u = (e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w) & 0x7fff7fffu;
                const uint32_t x = u & 0xffff, y = u >> 16;
                most = x <= 0x7c00 && x > most ? x : most;
                most = y <= 0x7c00 && y > most ? y : most;
            }
        }
        const float big = wave_butterfly(h2f(static_cast<uint16_t>(most)), [](float x, float y) { return fmaxf(x, y); });
        if (lane == 0) sc[kVmax + w] = big;
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
        for (int k = 0; k < i; ++k) {
            const float4_t l = *reinterpret_cast<const float4_t*>(&tri[16 * (w + i) + c][16 * (w + k) + 4 * j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) s = __builtin_amdgcn_mfma_f32_16x16x4f32(l[r], col[k][r], s, 0, 0, 0);
        }
        const float4_t l = *reinterpret_cast<const float4_t*>(&tri[16 * (w + i) + c][16 * (w + i) + 4 * j]);
#pragma unroll
        for (int r = 0; r < 4; ++r) col[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-l[r], s[r], col[i], 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 1; i < 4; ++i)
        if (w + i < 4)
#pragma unroll
            for (int r = 0; r < 4; ++r) tri[16 * (w + i) + 4 * j + r][16 * w + c] = col[i][r];
    __syncthreads();
    // T of this wave's rows, two parts
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (2 * s > w) continue;
        half8_t hi, lo;
        const float4_t x = *reinterpret_cast<const float4_t*>(&tri[16 * w + c][32 * s + 4 * j]);
        const float4_t y = *reinterpret_cast<const float4_t*>(&tri[16 * w + c][32 * s + 16 + 4 * j]);
        split<8>(float8_t{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, hi, lo);
        uint4* at = a.T + (unit * 6 + tri_block(w, s)) * 2 * 64 + lane;
        at[0] = as_u4(hi);
        at[64] = as_u4(lo);
    }
}

// Waves 0 .. 3 carry the state: wave w holds dk MT 16 w .. of it and makes token tile w of X
// and U.  Waves 4 .. 7 make the outputs of token tile w - 4.  A chunk has three barriers:
//   X = beta (V - e^G K S)  |  U = T X  |  S' = e^(G_last) S + K^T (e^(G_last - G) U)
// Column x of lane c is dv NT c + x of the slice.
template <int DK, int NT>
__global__ __launch_bounds__(512, 2) void delta_scan_kernel(ChunkArgs a) {
    constexpr int KS = DK / 32, MT = DK / 64;    // steps over dk; tiles of the state a wave carries
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
    __shared__ __attribute__((aligned(16))) uint2 xf[2][NT][2][64][2];        // X, two parts
    __shared__ __attribute__((aligned(16))) uint2 uf[4][NT][2][64][2];        // U and e^(G_last - G) f U, two parts each
    __shared__ float maxes[8];

    // the state and the scale of this pass
    const int count = c1 > c0 ? c1 - c0 : 0;
    float4_t S[MT][NT];
    const float* src = starts ? p.state : p.state_out;
    // tile i of the state: row 4 j + r is dk 32 (i / 2) + 4 (i % 2) + 8 j + r
    auto at_state = [&](int m, int r) {
        const int i = MT * w + m;
        return (at * p.Hv + h) * DK * p.Dv + static_cast<int64_t>(32 * (i / 2) + 4 * (i % 2) + 8 * j + r) * p.Dv + dv0 + NT * c;
    };
    float big = 0.f;
    if (wave < 4) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    S[m][x][r] = src ? src[at_state(m, r) + x] : 0.f;
                    big = fmaxf(big, fabsf(S[m][x][r]));
                }
    }
    auto store_state = [&](float by) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int x = 0; x < NT; ++x) p.state_out[at_state(m, r) + x] = S[m][x][r] * by;
    };
    if (count == 0) {                            // no token: the state as it is
        if (p.state_out == src) return;
        if (wave < 4) store_state(1.f);
        return;
    }
    const int slot = s0 + c0 - a.slot0;          // of chunk c0 in this pass
    const int64_t unit0 = static_cast<int64_t>(slot) * p.Hv + h;     // its unit; the next is Hv on
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
    const int64_t first = t0 + static_cast<int64_t>(c0) * kC;
    const int n_last = t1 - (first + static_cast<int64_t>(count - 1) * kC) < kC
                           ? static_cast<int>(t1 - (first + static_cast<int64_t>(count - 1) * kC)) : kC;
    auto row = [&](int t, int n) { return static_cast<int64_t>(t < n ? t : n - 1); };

    if (wave < 4) {
        typedef _Float16 vrow __attribute__((ext_vector_type(NT)));
        struct Stage {
            half8_t k[KS], kt[MT][2], t[2][2];
            vrow v[4];
            float4_t bet, br, ef;
            float keep;
        } st[PD];
        // Loads are unconditional (past the last chunk: the last again), so that a wait counts those in flight exactly.
        int64_t voff[4];
        auto rows_of = [&](int n) {
#pragma unroll
            for (int t = 0; t < 4; ++t) voff[t] = row(16 * w + 4 * j + t, n) * p.v_row + NT * c;
        };
        const uint16_t* const vbase = p.v + first * p.v_row + h * p.v_head + dv0;
        auto next = [&](int i) {
            i = i < count ? i : count - 1;
            if (i == count - 1) rows_of(n_last);
            return i;
        };
        auto load_k = [&](Stage& s, int i) {
            const uint4* at = a.K + ((static_cast<int64_t>(slot + i) * a.Hk + hk) * 4 + w) * KS * 64 + lane;
#pragma unroll
            for (int k = 0; k < KS; ++k) s.k[k] = as_h8(at[k * 64]);
        };
        auto load_v = [&](Stage& s, int i) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s.v[r] = *reinterpret_cast<const vrow*>(vbase + static_cast<int64_t>(i) * kC * p.v_row + voff[r]);
            const float* sc = a.sc + (unit0 + static_cast<int64_t>(i) * p.Hv) * kScalars + 16 * w + 4 * j;
            s.bet = *reinterpret_cast<const float4_t*>(sc + kBet);
            s.br = *reinterpret_cast<const float4_t*>(sc + kBr);
        };
        auto load_t = [&](Stage& s, int i) {
            const int64_t unit = unit0 + static_cast<int64_t>(i) * p.Hv;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int part = 0; part < 2; ++part)
                    s.t[q][part] = as_h8(a.T[((unit * 6 + tri_block(w, w < 2 ? 0 : q)) * 2 + part) * 64 + lane]);
            s.ef = *reinterpret_cast<const float4_t*>(a.sc + unit * kScalars + kEf + 16 * w + 4 * j);
        };
        auto load_kt = [&](Stage& s, int i) {
            const uint4* at = a.Kt + (static_cast<int64_t>(slot + i) * a.Hk + hk) * (DK / 16) * 2 * 64 + lane;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q) s.kt[m][q] = as_h8(at[((MT * w + m) * 2 + q) * 64]);
            s.keep = a.sc[(unit0 + static_cast<int64_t>(i) * p.Hv) * kScalars + kKeep];
        };
        auto put_state = [&]() {
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                half4_t hi[MT], lo[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) split<4>(S[m][x], hi[m], lo[m]);
                if constexpr (MT == 2) {
                    *reinterpret_cast<uint4*>(&sf[0][x][w][lane][0]) = as_u4(half8_t{hi[0][0], hi[0][1], hi[0][2], hi[0][3], hi[1][0], hi[1][1], hi[1][2], hi[1][3]});
                    *reinterpret_cast<uint4*>(&sf[1][x][w][lane][0]) = as_u4(half8_t{lo[0][0], lo[0][1], lo[0][2], lo[0][3], lo[1][0], lo[1][1], lo[1][2], lo[1][3]});
                } else {
                    sf[0][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, hi[0]);
                    sf[1][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, lo[0]);
                }
            }
        };
        rows_of(kC);
#pragma unroll
        for (int q = 0; q < PD; ++q) {
            const int i = next(q);
            load_k(st[q], i);
            load_v(st[q], i);
            load_t(st[q], i);
            load_kt(st[q], i);
            asm volatile("" ::: "memory");       // in this order
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < NT; ++x) S[m][x] *= up;
        put_state();
        for (int i0 = 0; i0 < count; i0 += PD)
#pragma unroll
            for (int q = 0; q < PD; ++q) {
                const int i = i0 + q;
                if (i >= count) break;
                Stage& s = st[q];
                const int ahead = next(i + PD);
                const int live = i == count - 1 ? n_last : kC;
                lds_barrier();                   // S is there
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    float4_t ks = {0, 0, 0, 0}, kl = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        ks = mfma16(s.k[k], as_h8(*reinterpret_cast<const uint4*>(&sf[0][x][k][lane][0])), ks);
                        kl = mfma16(s.k[k], as_h8(*reinterpret_cast<const uint4*>(&sf[1][x][k][lane][0])), kl);
                    }
                    ks += kl;
                    float4_t v;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        v[r] = apart(fmaf(s.bet[r] * up, static_cast<float>(s.v[r][x]), -(s.br[r] * ks[r])));
                    if (live < kC)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (16 * w + 4 * j + r >= live) v[r] = 0.f;
                    half4_t hi, lo;
                    split<4>(v, hi, lo);
                    xf[0][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, hi);
                    xf[1][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, lo);
                }
                load_k(s, ahead);
                load_v(s, ahead);
                lds_barrier();                   // X is there
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    float4_t u = {0, 0, 0, 0}, v = {0, 0, 0, 0}, z = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (2 * k > w) continue;
                        const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&xf[0][x][k][lane][0]));
                        const half8_t lo = as_h8(*reinterpret_cast<const uint4*>(&xf[1][x][k][lane][0]));
                        u = mfma16(s.t[k][0], hi, u);
                        v = mfma16(s.t[k][0], lo, v);
                        z = mfma16(s.t[k][1], hi, z);
                    }
                    u += v + z;
                    float4_t eu;
                    half4_t part[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) eu[r] = apart(s.ef[r] * u[r]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) u[r] = apart(u[r]);
                    split<4>(eu, part[2], part[3]);
                    split<4>(u, part[0], part[1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) uf[e][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, part[e]);
                }
                load_t(s, ahead);
                lds_barrier();                   // U is there, S has been read
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int m = 0; m < MT; ++m) S[m][x] *= s.keep;
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&uf[2][x][k][lane][0]));
                        const half8_t lo = as_h8(*reinterpret_cast<const uint4*>(&uf[3][x][k][lane][0]));
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            S[m][x] = mfma16(s.kt[m][k], hi, S[m][x]);
                            S[m][x] = mfma16(s.kt[m][k], lo, S[m][x]);
                        }
                    }
                put_state();
                load_kt(s, ahead);
            }
        store_state(down);
    } else {
        struct Stage {
            half8_t q[KS], pf[2][2];
            float eq, osc;
        } st[PD];
        auto next = [&](int i) { return i < count ? i : count - 1; };
        auto load_q = [&](Stage& s, int i) {
            const uint4* at = a.Q + ((static_cast<int64_t>(slot + i) * a.Hk + hk) * 4 + w) * KS * 64 + lane;
#pragma unroll
            for (int k = 0; k < KS; ++k) s.q[k] = as_h8(at[k * 64]);
        };
        auto load_p = [&](Stage& s, int i) {
            const int64_t unit = unit0 + static_cast<int64_t>(i) * p.Hv;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int part = 0; part < 2; ++part)
                    s.pf[q][part] = as_h8(a.P[((unit * 6 + tri_block(w, w < 2 ? 0 : q)) * 2 + part) * 64 + lane]);
            s.eq = a.sc[unit * kScalars + kEq + 16 * w + c];
            s.osc = a.sc[unit * kScalars + kOsc + 16 * w + c];
        };
#pragma unroll
        for (int q = 0; q < PD; ++q) {
            const int i = next(q);
            load_q(st[q], i);
            load_p(st[q], i);
            asm volatile("" ::: "memory");
        }
        for (int i0 = 0; i0 < count; i0 += PD)
#pragma unroll
            for (int q = 0; q < PD; ++q) {
                const int i = i0 + q;
                if (i >= count) break;
                Stage& s = st[q];
                const int ahead = next(i + PD);
                float4_t o[NT], ol[NT];          // rows dv, column token
                lds_barrier();                   // S is there: for X first
                lds_barrier();
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    o[x] = ol[x] = float4_t{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        o[x] = mfma16(as_h8(*reinterpret_cast<const uint4*>(&sf[0][x][k][lane][0])), s.q[k], o[x]);
                        ol[x] = mfma16(as_h8(*reinterpret_cast<const uint4*>(&sf[1][x][k][lane][0])), s.q[k], ol[x]);
                    }
                }
                load_q(s, ahead);
                lds_barrier();                   // U is there
                const int64_t t = first + static_cast<int64_t>(i) * kC + 16 * w + c;
                uint16_t r[4 * NT];
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    float4_t y = (o[x] + ol[x]) * s.eq, z = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (2 * k > w) continue;
                        const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&uf[0][x][k][lane][0]));
                        const half8_t lo = as_h8(*reinterpret_cast<const uint4*>(&uf[1][x][k][lane][0]));
                        y = mfma16(hi, s.pf[k][0], y);
                        z = mfma16(lo, s.pf[k][0], z);
                        z = mfma16(hi, s.pf[k][1], z);
                    }
                    const float osc = s.osc * down;
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[NT * e + x] = f2h((y[e] + z[e]) * osc);
                }
                load_p(s, ahead);
                if (t < t1) {
                    uint2* at_out = reinterpret_cast<uint2*>(p.out + (t * p.Hv + h) * p.Dv + dv0 + 4 * NT * j);
#pragma unroll
                    for (int x = 0; x < NT; ++x)
                        at_out[x] = make_uint2(r[4 * x] | (static_cast<uint32_t>(r[4 * x + 1]) << 16),
                                               r[4 * x + 2] | (static_cast<uint32_t>(r[4 * x + 3]) << 16));
                }
            }
    }
}

// Bytes per slot, all heads.
int64_t slot_bytes(int64_t Hk, int64_t Hv, int64_t Dk) {
    return Hv * (2 * kTriBytes + kScalars * 4) + Hk * kC * Dk * 6;
}
int64_t all_slots(int64_t B, int64_t T) { return T / kC + B; }
int64_t pass_slots(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk) {
    return std::min(all_slots(B, T), std::max<int64_t>(kSegmentBytes / slot_bytes(Hk, Hv, Dk), 1));
}

}  // namespace

int64_t delta_chunk_workspace(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk) {
    return pass_slots(B, T, Hk, Hv, Dk) * slot_bytes(Hk, Hv, Dk);
}

int launch_delta_chunk(const DeltaArgs& d, int Hk, int Dk, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    ChunkArgs a;
    a.d = d;
    a.Hk = Hk;
    const int64_t total = all_slots(d.B, d.T), per = pass_slots(d.B, d.T, Hk, d.Hv, Dk), units = per * d.Hv;
    uint8_t* at = static_cast<uint8_t*>(workspace);
    auto take = [&](int64_t bytes) {
        uint8_t* was = at;
        at += bytes;
        return was;
    };
    a.T = reinterpret_cast<uint4*>(take(units * kTriBytes));
    a.P = reinterpret_cast<uint4*>(take(units * kTriBytes));
    a.sc = reinterpret_cast<float*>(take(units * kScalars * 4));
    a.Kt = reinterpret_cast<uint4*>(take(per * Hk * kC * Dk * 2));
    a.K = reinterpret_cast<uint4*>(take(per * Hk * kC * Dk * 2));
    a.Q = reinterpret_cast<uint4*>(take(per * Hk * kC * Dk * 2));
    if (at - static_cast<uint8_t*>(workspace) > workspace_bytes) return fail(MCV_ERR_INVALID_ARG, "delta_rule: workspace too small");
    const int64_t states = ceil_div(static_cast<int64_t>(d.B) * d.Hv, 8) * 8, tiles = d.Dv / 16;
    const int nt = tiles % 2 == 0 && states * (tiles / 2) >= 512 ? 2 : 1;
    for (int64_t s = 0; s < total; s += per) {
        a.slot0 = static_cast<int>(s);
        a.slots = static_cast<int>(std::min(per, total - s));
        hipLaunchKernelGGL((Dk == 64 ? delta_prepare_kernel<64> : delta_prepare_kernel<128>),
                           dim3(static_cast<unsigned>(a.slots * static_cast<int64_t>(d.Hv))), dim3(256), 0, stream, a);
        int rc = check_launch("delta_prepare_kernel");
        if (rc != MCV_OK) return rc;
        auto fn = Dk == 64 ? (nt == 1 ? delta_scan_kernel<64, 1> : delta_scan_kernel<64, 2>)
                           : (nt == 1 ? delta_scan_kernel<128, 1> : delta_scan_kernel<128, 2>);
        hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(states * (tiles / nt))), dim3(512), 0, stream, a);
        rc = check_launch("delta_scan_kernel");
        if (rc != MCV_OK) return rc;
    }
    return MCV_OK;
}

}  // namespace mcv
