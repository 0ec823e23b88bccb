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
// The scan takes K and V as they come and applies T: three products that wait for one another
// where T K and T V made ahead would leave two, but K is exact in fp16 where T K takes two
// parts, and less goes through memory (8192 tokens: 49 + 144 us, with T K and T V 70 + 147; before the order in
// time and the scales below were right, 47 + 148 since).
//
// The first is bound by memory (8192 tokens, 16 heads of 128: 250 MB in 47 us on MI355X).
// The second walks in series, 1.16 us a chunk; 1.12 before every chunk had a scale and a look
// at what is not finite, and then without its outputs 1.04, without the loads of the state's
// waves 0.85, without both 0.75, which is three times an LDS write, a barrier, an LDS read and
// a short chain of products; the loads are 76 KB a chunk and CU.
//
// Precision.  The state, G, L, T and all sums are fp32 (G's differences from a sum in 64
// bits; T by substitution, in fp32 products).  Operands of products are two fp16 parts,
// 22 bits, of which only lo x lo is left out; q, k and v are fp16 as they come.  fp16's
// range: turned k rows are scaled by the power of two next to their norm's factor, q's
// norm is taken out of P, and the scan works on states and values scaled, for each chunk, by
// a power of two that brings M to 8 .. 16, M = the largest |v| of it and the chunk before or
// what decay leaves of the M before: they may grow 4096-fold, and a part's last bit is 2^-25
// at worst, 2^-28 M.  (The state's own largest would be less where the rule takes from it
// without decay; found by the outputs' waves it cost 0.13 us a chunk.)
//
// Order in time.  The products T X and P U run over whole tiles, zeros above the diagonal included, and a zero times an
// infinity or NaN of a later token would be NaN.  So T holds no rows of tokens whose k or gates are not finite (X has
// NaN there instead), a product that comes out not finite is made again without what is not, NaN put in from the
// first such token of its column on, and the scale goes by finite values alone.
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
constexpr int kKeep = 320, kVmax = 321;          // e^(G_last), largest |v|
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

// The sequence whose slots include `slot`: the last b whose first slot is not past it, 64 probes at a time; its span.
__device__ __forceinline__ int seq_of_slot(const DeltaArgs& p, int slot, int& t0, int& t1) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int n = p.B;;) {                        // among b .. b + n - 1
        const int step = (n + 63) / 64, mine = b + lane * step;
        int from = 0, to = 0;
        if (lane * step < n) delta_span(p, mine, from, to);
        const unsigned long long on = __ballot(lane * step < n && first_slot(from, mine) <= slot);
        const int at = on ? 63 - __builtin_clzll(on) : 0;
        b += at * step;
        if (step == 1) {
            t0 = __builtin_amdgcn_readlane(from, at);
            t1 = __builtin_amdgcn_readlane(to, at);
            return b;
        }
        n = n - at * step < step ? n - at * step : step;
    }
}

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float float8_t __attribute__((ext_vector_type(8)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));

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
// Sum over the lanes up to this one: rows of 16 by one, two, four, eight; a row's last to the next; lane 31 to the upper half.
template <int CTRL, int ROWS>
__device__ __forceinline__ double lane_of(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
    v += lane_of<0x111, 0xf>(v);
    v += lane_of<0x112, 0xf>(v);
    v += lane_of<0x114, 0xf>(v);
    v += lane_of<0x118, 0xf>(v);
    v += lane_of<0x142, 0xa>(v);
    return v + lane_of<0x143, 0xc>(v);
}
// Lane r's value of each four lanes.
__device__ __forceinline__ float of_quad(float v, int r) {
    const int i = __float_as_int(v);
    return __int_as_float(r == 0   ? __builtin_amdgcn_update_dpp(0, i, 0x00, 0xf, 0xf, false)
                          : r == 1 ? __builtin_amdgcn_update_dpp(0, i, 0x55, 0xf, 0xf, false)
                          : r == 2 ? __builtin_amdgcn_update_dpp(0, i, 0xaa, 0xf, 0xf, false)
                                   : __builtin_amdgcn_update_dpp(0, i, 0xff, 0xf, 0xf, false));
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// LDS is ready for the other waves; global loads in flight stay there.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Global loads after this stay behind the LDS writes before it, which others wait for.
__device__ __forceinline__ void lds_first() { asm volatile("" ::: "memory"); }

// For the largest of two fp16 values' magnitudes, of finite ones: whole numbers from 0x400 on, where what is not finite
// has wrapped to less; and that number's value.
__device__ __forceinline__ ushort2_t finite_up(uint32_t x) { return __builtin_bit_cast(ushort2_t, ((x & 0x7fff7fffu) + 0x04000400u) & 0x7fff7fffu); }
__device__ __forceinline__ float largest_of(ushort2_t v) {
    const int top = v[0] > v[1] ? v[0] : v[1];
    return top < 0x400 ? 0.f : h2f(static_cast<uint16_t>(top - 0x400));
}

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
    int t0, t1;
    const int b = seq_of_slot(p, slot, t0, t1);
    const int chunk = slot - first_slot(t0, b);
    const int64_t start = t0 + static_cast<int64_t>(chunk) * kC;
    if (chunk < 0 || start >= t1 || t1 - t0 < p.short_below) return;
    const int n = t1 - start < kC ? static_cast<int>(t1 - start) : kC;
    const int64_t unit = static_cast<int64_t>(local) * p.Hv + h;

    // k and q as rows, 16-byte chunks moved so that operand reads do not conflict; then k turned and L, T
    constexpr int RC = DK / 8;                   // chunks of a row
    __shared__ __attribute__((aligned(16))) uint8_t space[2][kC * PT * 4];
    __shared__ __attribute__((aligned(16))) float gh[kC], gl[kC], bet[kC], rkn[kC], rqn[kC], kk[kC], qq[kC], lrow[kC], pcol[kC], fall[4][kC], vmax[2];
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
    constexpr int VT = 8;                        // 16-byte chunks of v a thread of waves 0 and 1 has: 128 columns at a time
    uint4 vx[VT];
    auto load_v = [&](int v0) {
        const int col = v0 + static_cast<int>(threadIdx.x) % 16 * 8;
        const uint16_t* at = vb + (col < p.Dv ? col : v0);
#pragma unroll
        for (int i = 0; i < VT; ++i) vx[i] = *reinterpret_cast<const uint4*>(at + row(static_cast<int>(threadIdx.x) / 16 + 8 * i) * p.v_row);
    };
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
    if (w < 2) load_v(0);
    lds_barrier();
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
        G = wave_scan(G);
        gh[lane] = static_cast<float>(G);
        gl[lane] = static_cast<float>(G - static_cast<double>(static_cast<float>(G)));
    } else if (w == 1) {
        bet[lane] = lane < n ? gate : 0.f;
    }
    if (w < 2) {                                 // the largest |v|, for the scan's scale; these have fewer products
        ushort2_t most = {0, 0};
        for (int from = 0;;) {
#pragma unroll
            for (int i = 0; i < VT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = e == 0 ? vx[i].x : e == 1 ? vx[i].y : e == 2 ? vx[i].z : vx[i].w;
                    most = __builtin_elementwise_max(most, finite_up(x));
                }
            from += 128;
            if (from >= p.Dv) break;
            load_v(from);
        }
        const float big = wave_butterfly(largest_of(most), [](float x, float y) { return fmaxf(x, y); });
        if (lane == 0) vmax[w] = big;
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
    // The first token whose k or gates (g's running sum) are not finite.
    const unsigned long long odd = __ballot(!(fabsf(kk[lane]) < INFINITY && fabsf(gh[lane]) < INFINITY && fabsf(bet[lane]) < INFINITY));
    const int clean = odd ? __builtin_ctzll(odd) : kC;
    {
        // Norm factors within a last bit: the same ones enter T, P and the scan's scalars.
        const float k2 = kk[lane], q2 = qq[lane], g_hi = gh[lane], g_lo = gl[lane];
        const float rk = p.normalize ? __builtin_amdgcn_rsqf(k2 + kDeltaEps) : 1.0f;
        const float rn = q2 > 0.f ? __builtin_amdgcn_rsqf(q2) : 0.f;
        // e^(G_i - G_j) of tiles below the diagonal is e^(G_i - G_r) e^(G_r - G_j), r the row tile's first token: neither is above one
        fall[w][lane] = exp2_of((gh[16 * w] - g_hi) + (gl[16 * w] - g_lo)) * rk;
        if (w == 0) {
            const float eg = exp2_of(g_hi + g_lo), to_end = exp2_of((gh[kC - 1] - g_hi) + (gl[kC - 1] - g_lo));
            const uint32_t bits = __float_as_uint(rk);           // pw: the power of two at or below it
            const float b = bet[lane];
            kpow[lane] = static_cast<_Float16>(p.normalize ? __uint_as_float(bits & 0x7f800000u) : 1.0f);
            rkn[lane] = rk;
            sc[kBet + lane] = lane < clean ? b : NAN;
            sc[kBr + lane] = b * rk * eg;
            sc[kEf + lane] = to_end * (p.normalize ? __uint_as_float((bits & 0x007fffffu) | 0x3f800000u) : 1.0f);
            if (lane == kC - 1) sc[kKeep] = eg;
            if (lane == 0) sc[kVmax] = fmaxf(vmax[0], vmax[1]);
        } else if (w == 1) {
            rqn[lane] = rn;
            sc[kEq + lane] = exp2_of(g_hi + g_lo) * rn;
            sc[kOsc + lane] = p.scale * (q2 * rn) * (p.normalize ? __builtin_amdgcn_rsqf(q2 + kDeltaEps) : 1.0f);
        } else if (w == 2) {
            const float ea = exp2_of((g_hi - gh[lane & 48]) + (g_lo - gl[lane & 48]));
            lrow[lane] = bet[lane] * ea * rk;
            pcol[lane] = ea * rn;
        }
    }
    __syncthreads();

    // L into LDS; P straight out: its tile pairs are operands
    float4_t pt[4];
    const float4_t lr = *reinterpret_cast<const float4_t*>(&lrow[16 * w + 4 * j]);
    const float pc = pcol[16 * w + c];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        pt[x] = float4_t{0, 0, 0, 0};
        if (x > w) {
            if (x == w + 1 && (w & 1) == 0)      // the other half of T's own step
#pragma unroll
                for (int r = 0; r < 4; ++r) tri[16 * w + 4 * j + r][16 * x + c] = 0.f;
        } else if (x < w) {
            const float fc = fall[w][16 * x + c];
            const float4_t fr = *reinterpret_cast<const float4_t*>(&fall[w][16 * x + 4 * j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                tri[16 * w + 4 * j + r][16 * x + c] = lr[r] * fc * kkt[x][r];        // L: row 16 w + 4 j + r, column 16 x + c
                pt[x][r] = fr[r] * pc * kqt[x][r];                                   // P: key 16 x + 4 j + r, query 16 w + c
            }
        } else {
            const float ghc = gh[16 * w + c], glc = gl[16 * w + c], rkc = rkn[16 * w + c], rqc = rqn[16 * w + c];
            const float4_t hr = *reinterpret_cast<const float4_t*>(&gh[16 * w + 4 * j]), lo = *reinterpret_cast<const float4_t*>(&gl[16 * w + 4 * j]);
            const float4_t rr = *reinterpret_cast<const float4_t*>(&rkn[16 * w + 4 * j]), br = *reinterpret_cast<const float4_t*>(&bet[16 * w + 4 * j]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float d = (hr[r] - ghc) + (lo[r] - glc);
                tri[16 * w + 4 * j + r][16 * w + c] = c < 4 * j + r ? br[r] * exp2_of(d) * rr[r] * rkc * kkt[x][r] : 0.f;
                pt[x][r] = 4 * j + r <= c ? exp2_of(-d) * rr[r] * rqc * kqt[x][r] : 0.f;
            }
        }
    }
    if (clean < kC)
        for (int x = 0; x <= w; ++x)
            for (int r = 0; r < 4; ++r)
                if (16 * w + 4 * j + r >= clean) tri[16 * w + 4 * j + r][16 * x + c] = 0.f;
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
    if (h % p.group == 0 && w < 2)
#pragma unroll
        for (int i = w; i < DK / 16; i += 2) {
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
    constexpr int PD = 2;                        // chunks whose operands are in flight
    constexpr int KS = DK / 32, MT = DK / 64;    // steps over dk; tiles of the state a wave carries
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
    if ((c0 >= c1 && !(chunks == 0 && starts)) || t1 - t0 < p.short_below) return;
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
    __shared__ float maxes[4], down_next;

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
                    big = fmaxf(big, fabsf(S[m][x][r]) < INFINITY ? fabsf(S[m][x][r]) : 0.f);
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
    float up, down, largest;                     // M, in true size
    auto scale_for = [](float most, float& up, float& down) {    // (2^126 at most: both are normal numbers)
        const int ex = min(3 + 127 - static_cast<int>(__float_as_uint(most) >> 23), 126);
        up = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
        down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
    };
    // Both kinds of waves call this once, with their first operands on the way.
    const float first_vmax = a.sc[unit0 * kScalars + kVmax];
    auto agree_on_scale = [&]() {
        float most = wave_butterfly(big, [](float x, float y) { return fmaxf(x, y); });
        if (lane == 0 && wave < 4) maxes[wave] = most;
        lds_barrier();
        most = first_vmax;
#pragma unroll
        for (int i = 0; i < 4; ++i) most = fmaxf(most, maxes[i]);
        largest = most;
        scale_for(most, up, down);
    };
    const int64_t first = t0 + static_cast<int64_t>(c0) * kC;
    const int n_last = t1 - (first + static_cast<int64_t>(count - 1) * kC) < kC
                           ? static_cast<int>(t1 - (first + static_cast<int64_t>(count - 1) * kC)) : kC;
    auto row = [&](int t, int n) { return static_cast<int64_t>(t < n ? t : n - 1); };

    // An operand of 64 tokens (two steps, two parts) and 16 columns: what is not finite becomes zero; the first such
    // token of the lane's column, kC if there is none.
    auto first_of_columns = [&](half8_t (&g)[2][2]) {
        int bad = kC;
#pragma unroll
        for (int k = 1; k >= 0; --k)
#pragma unroll
            for (int e = 7; e >= 0; --e)
                if (!(fabsf(static_cast<float>(g[0][k][e])) < INFINITY)) {
                    bad = 32 * k + (e < 4 ? 0 : 12) + 4 * j + e;
                    g[0][k][e] = g[1][k][e] = 0;
                }
        bad = min(bad, __shfl_xor(bad, 16));
        return min(bad, __shfl_xor(bad, 32));
    };

    if (wave < 4) {
        typedef _Float16 vrow __attribute__((ext_vector_type(NT)));
        struct Stage {
            half8_t k[KS], kt[MT][2], t[2][2];
            vrow v[4];
            float bet, br, ef, keep, vmax;       // of token 4 j + c % 4 of the wave's tile; e^(G_last); the next chunk's largest |v|
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
            const float* sc = a.sc + (unit0 + static_cast<int64_t>(i) * p.Hv) * kScalars;
            s.keep = sc[kKeep];
            s.vmax = sc[(i + 1 < count ? p.Hv * kScalars : 0) + kVmax];
            sc += 16 * w + 4 * j + c % 4;
            s.bet = sc[kBet];
            s.br = sc[kBr];
        };
        auto load_t = [&](Stage& s, int i) {
            const int64_t unit = unit0 + static_cast<int64_t>(i) * p.Hv;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int part = 0; part < 2; ++part)
                    s.t[q][part] = as_h8(a.T[((unit * 6 + tri_block(w, w < 2 ? 0 : q)) * 2 + part) * 64 + lane]);
            s.ef = a.sc[unit * kScalars + kEf + 16 * w + 4 * j + c % 4];
        };
        auto load_kt = [&](Stage& s, int i) {
            const uint4* at = a.Kt + (static_cast<int64_t>(slot + i) * a.Hk + hk) * (DK / 16) * 2 * 64 + lane;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q) s.kt[m][q] = as_h8(at[((MT * w + m) * 2 + q) * 64]);
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
        agree_on_scale();
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int x = 0; x < NT; ++x) S[m][x] *= up;
        put_state();
        float vmax = first_vmax;                 // of this chunk
        for (int i0 = 0; i0 < count; i0 += PD)
#pragma unroll
            for (int q = 0; q < PD; ++q) {
                const int i = i0 + q;
                if (i >= count) break;
                Stage &s = st[q], &before = st[(q + PD - 1) % PD];
                const int ahead = next(i + PD);
                const int live = i == count - 1 ? n_last : kC;
                lds_barrier();                   // S is there
                half8_t f[2][KS];
                auto read_state = [&](int x) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        f[0][k] = as_h8(*reinterpret_cast<const uint4*>(&sf[0][x][k][lane][0]));
                        f[1][k] = as_h8(*reinterpret_cast<const uint4*>(&sf[1][x][k][lane][0]));
                    }
                };
                // What a phase has used is loaded anew in the next, behind its LDS reads and while they take their time.
                read_state(0);
                lds_first();
                load_kt(before, next(i - 1 + PD));
                lds_first();
                const float bet_up = s.bet * up;
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    float4_t ks[4] = {};         // short chains: a product's result is late for the next
                    if (x) read_state(x);
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        ks[k % 2] = mfma16(s.k[k], f[0][k], ks[k % 2]);
                        ks[2 + k % 2] = mfma16(s.k[k], f[1][k], ks[2 + k % 2]);
                    }
                    ks[0] = (ks[0] + ks[1]) + (ks[2] + ks[3]);
                    float4_t v;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        v[r] = apart(fmaf(of_quad(bet_up, r), static_cast<float>(s.v[r][x]), -(of_quad(s.br, r) * ks[0][r])));
                    if (live < kC)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (16 * w + 4 * j + r >= live) v[r] = 0.f;
                    half4_t hi, lo;
                    split<4>(v, hi, lo);
                    xf[0][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, hi);
                    xf[1][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, lo);
                }
                lds_barrier();                   // X is there
                half8_t g[2][2];
                auto read_x = [&](int x) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int part = 0; part < 2; ++part) g[part][k] = as_h8(*reinterpret_cast<const uint4*>(&xf[part][x][k][lane][0]));
                };
                // U of column x's tokens before the first X that is not finite, NaN from it on, for the outputs.
                auto in_order = [&](int x) {
                    read_x(x);
                    const int bad = first_of_columns(g);
                    float4_t u = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (2 * k > w) continue;
                        u = mfma16(s.t[k][0], g[0][k], u);
                        u = mfma16(s.t[k][0], g[1][k], u);
                        u = mfma16(s.t[k][1], g[0][k], u);
                    }
                    half4_t hi, lo;
#pragma unroll
                    for (int r = 0; r < 4; ++r) u[r] = 16 * w + 4 * j + r >= bad ? NAN : apart(u[r]);
                    split<4>(u, hi, lo);
                    uf[0][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, hi);
                    uf[1][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, lo);
                };
                float all = 0.f;
                // The next chunk's scale (no step of it past 2^64); behind X's reads 1 us more over 8192 tokens.
                const float keep = s.keep;
                largest = fmaxf(fmaxf(largest * (keep < 0x1p60f ? keep : 1.f), 0x1p-60f * down), fmaxf(vmax, s.vmax));
                vmax = s.vmax;
                float up_next, down_to;
                scale_for(largest, up_next, down_to);
                const float rescale = up_next * down, keep_to = keep * rescale;
                down_next = down_to;             // (of every lane: a branch for one costs 0.06 us a chunk)
                read_x(0);
                lds_first();
                load_k(s, ahead);
                load_v(s, ahead);
                lds_first();
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    if (x) read_x(x);
                    float4_t u = {0, 0, 0, 0}, v = {0, 0, 0, 0}, z = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (2 * k > w) continue;
                        u = mfma16(s.t[k][0], g[0][k], u);
                        v = mfma16(s.t[k][0], g[1][k], v);
                        z = mfma16(s.t[k][1], g[0][k], z);
                    }
                    u += v + z;
                    all += (u[0] + u[1]) + (u[2] + u[3]);
                    const float ef = s.ef * rescale;
                    float4_t eu;
                    half4_t part[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) eu[r] = apart(of_quad(ef, r) * u[r]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) u[r] = apart(u[r]);
                    split<4>(eu, part[2], part[3]);
                    split<4>(u, part[0], part[1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) uf[e][x][w / 2][lane][w % 2] = __builtin_bit_cast(uint2, part[e]);
                }
                if (__any(!(fabsf(all) < INFINITY)))     // (the state's own parts stay: it has NaN of any token of the chunk)
                    for (int x = 0; x < NT; ++x) in_order(x);
                lds_barrier();                   // U is there, S has been read
                auto read_u = [&](int x) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int part = 0; part < 2; ++part) g[part][k] = as_h8(*reinterpret_cast<const uint4*>(&uf[2 + part][x][k][lane][0]));
                };
                read_u(0);
                lds_first();
                load_t(s, ahead);
                lds_first();
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    if (x) read_u(x);
                    float4_t low[MT] = {};
#pragma unroll
                    for (int m = 0; m < MT; ++m) S[m][x] *= keep_to;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            S[m][x] = mfma16(s.kt[m][k], g[0][k], S[m][x]);
                            low[m] = mfma16(s.kt[m][k], g[1][k], low[m]);
                        }
#pragma unroll
                    for (int m = 0; m < MT; ++m) S[m][x] += low[m];
                }
                up = up_next;
                down = down_to;
                put_state();
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
        agree_on_scale();
        float down_to = down;                    // the scales of the chunk to finish next, and of the one after
        float4_t o[NT], ol[NT];                  // e^G Q S of a chunk: rows dv, column token
        // P U of column x, U's first that is not finite and all after it NaN: rows dv, column token
        auto in_order = [&](const Stage& s, int x) {
            half8_t g[2][2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int part = 0; part < 2; ++part) g[part][k] = as_h8(*reinterpret_cast<const uint4*>(&uf[part][x][k][lane][0]));
            const int bad = first_of_columns(g);
            float4_t y = (o[x] + ol[x]) * s.eq;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (2 * k > w) continue;
                y = mfma16(g[0][k], s.pf[k][0], y);
                y = mfma16(g[1][k], s.pf[k][0], y);
                y = mfma16(g[0][k], s.pf[k][1], y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (16 * w + c >= __shfl(bad, 4 * j + e)) y[e] = NAN;
            return y;
        };
        auto finish = [&](const Stage& s, int i) {
            const int64_t t = first + static_cast<int64_t>(i) * kC + 16 * w + c;
            float4_t sum[NT];
            float all = 0.f;
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                float4_t y = (o[x] + ol[x]) * s.eq, z = {0, 0, 0, 0}, v = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (2 * k > w) continue;
                    const half8_t hi = as_h8(*reinterpret_cast<const uint4*>(&uf[0][x][k][lane][0]));
                    const half8_t lo = as_h8(*reinterpret_cast<const uint4*>(&uf[1][x][k][lane][0]));
                    y = mfma16(hi, s.pf[k][0], y);
                    z = mfma16(lo, s.pf[k][0], z);
                    v = mfma16(hi, s.pf[k][1], v);
                }
                sum[x] = y + (z + v);
                all += (sum[x][0] + sum[x][1]) + (sum[x][2] + sum[x][3]);
            }
            auto put = [&]() {
                const float osc = s.osc * down;
                uint16_t r[4 * NT];
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[NT * e + x] = f2h(sum[x][e] * osc);
                if (t < t1) {
                    uint2* at_out = reinterpret_cast<uint2*>(p.out + (t * p.Hv + h) * p.Dv + dv0 + 4 * NT * j);
#pragma unroll
                    for (int x = 0; x < NT; ++x)
                        at_out[x] = make_uint2(r[4 * x] | (static_cast<uint32_t>(r[4 * x + 1]) << 16),
                                               r[4 * x + 2] | (static_cast<uint32_t>(r[4 * x + 3]) << 16));
                }
            };
            put();                               // (looked at after it: before, 2.2 us more over 8192 tokens)
            if (__any(!(fabsf(all) < INFINITY))) {
#pragma unroll
                for (int x = 0; x < NT; ++x) sum[x] = in_order(s, x);
                put();
            }
        };
        for (int i0 = 0; i0 < count; i0 += PD)
#pragma unroll
            for (int q = 0; q < PD; ++q) {
                const int i = i0 + q;
                if (i >= count) break;
                Stage &s = st[q], &before = st[(q + PD - 1) % PD];
                lds_barrier();                   // S is there, and U of the chunk before until X is
                if (i > 0) finish(before, i - 1);
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
                lds_barrier();                   // U is there, S has been read
                load_p(before, next(i - 1 + PD));
                load_q(s, next(i + PD));
                down = down_to;
                down_to = down_next;
            }
#pragma unroll
        for (int q = 0; q < PD; ++q)
            if ((count - 1) % PD == q) finish(st[q], count - 1);
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
    // 32 columns a workgroup where that still leaves one for every CU.  MI355X, us a pass (Dk = Dv = 128), 16 and 32
    // columns: 32 states of 1000 tokens 41 49, 64 of 1000 76 76, 128 of 500 84 77, 288 of 100 74 60.
    const int nt = tiles % 2 == 0 && states * (tiles / 2) >= 256 ? 2 : 1;
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
