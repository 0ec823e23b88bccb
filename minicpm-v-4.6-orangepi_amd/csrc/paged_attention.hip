// paged_attention.hip -- attention of one new token over a paged cache, gfx950.
//
// One pass over the cache with the running maximum m and sum l of the softmax, in
// 32 bits and base 2:  w_t = 2^(s_t - m), o = sum w_t v_t / l.  The up to 16 query
// heads of one cache head share every byte of K and V (and are one side of the matrix
// products, however few they are: the matrix cores have time to spare here).
//
// A wave takes 32 tokens at a time:
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16, twice 16 tokens as rows; lane (c, j), c =
//                 lane % 16, j = lane / 16, then holds head c and tokens 4j .. 4j + 3 of each half
//   O^T += V^T P^T  the sum over tokens may run in any order, so lane (c, j)'s eight
//                 weights are the product's operand as they stand, and the lane loads V's
//                 same eight rows, 8 d of each, whose 8 x 8 values it turns in registers
// K as an operand has its 16 rows on 16 neighbouring lanes, and a load costs a cycle a
// line touched: K comes as whole rows instead and turns through LDS, each wave its own.
// What lies past the sequence's end, or in a page that is not there, has score -inf and
// its V is set to zero (it may hold NaN).
//
// Only the device knows the lengths: every workgroup adds them up, and each (sequence, cache
// head) is cut into parts of one size, about the work over the workgroups that the chip
// holds, so that none waits for the longest sequence.  Parts of one (sequence, cache head)
// meet through the workspace: each writes its 32-bit part with device-scope stores
// (written through; see w4a16_gemm_sk.hip) and counts itself in; the last of each kFan
// parts joins them in order, and where there are more than kFan the last of those joins
// the joined, so the bits do not depend on who is last and nobody waits.
//
// Long caches are bound by HBM: 8 heads on 2 of 256, 200000 tokens 69.0 us on MI355X, 5.9
// TB/s (a read-only stream reaches 6.3).  Short ones by round trips that wait for one
// another (lengths, page numbers, K and V, the part written through, its counter, the
// other parts: 1100 tokens 9.1 us).
#include <algorithm>

#include "mixers.h"

namespace mcv {
namespace {

constexpr int kTile = 32;                        // tokens a wave takes at a time
constexpr int kHeads = 16;                       // query heads of one matrix product
constexpr int kCus = 256;
constexpr int kFan = 16;                         // parts joined by one workgroup
constexpr int64_t kCounterBytes = 4096;
constexpr int64_t kMaxLen = int64_t(1) << 30;   // tokens of one sequence
// Non-temporal loads: K and V pass once.  MI355X, us a pass of inputs not in any cache, with and without: 1 x 200000 tokens
// 69.3 77.9, 41 x 4096 27.9 29.8, 1 x 30000 20.4 21.6, 1 x 1100 10.4 9.7 (9.0 both ways where they may be).
constexpr int kOnce = 2;
constexpr float kLog2e = 1.44269504088896340736f;
// The largest weight, of 2^(s - m) at most one.  As an operand a weight is two fp16 parts, the second what the first,
// cut off, leaves: off by 2^-21 of the weight, or 2^-39 of the largest.  (One part under a largest weight of one is
// nothing from 2^-25 on, while l counts it: one token far above 4096 others, its v zero, 25 % off.)  l and the sums
// of v carry the factor alike.  The second part is never of the other sign, nor zero beside a first that is not: an
// infinite v stays infinite.
constexpr float kTop = 32768.f;

struct AttnArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* lens;
    uint16_t* out;
    uint8_t* ws;
    int64_t q_row, q_head, k_page, k_head, v_page, v_head, table_row;
    int k_token, v_token, pages, page16, max_len, B, Hq, Hkv, group, htiles;
    uint32_t page16_inv;                         // ceil(2^32 / page16), page16 > 1
    float scale_log2;
    int split;                                   // workgroups to cut for; 0: every (sequence, cache head) whole
};

// Bytes of one part: [rows][D] sums, [rows][2] maximum and sum, whole 16-byte chunks.
__host__ __device__ constexpr int64_t part_bytes(int rows, int D) { return int64_t(rows) * D * 4 + ((rows * 8 + 15) & ~15); }

// Sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);       // rows of 16: one to the right, two, four, eight
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);       // a row's last lane to the next row
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);       // lane 31 to the upper half
    return v;
}
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max4(float v) {          // over the four lanes of one column
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <int D>
__device__ __forceinline__ void put_out(const AttnArgs& p, int64_t head0, int i, float4_t sum, float l) {
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);          // a row of nothing: zeros; NaN stays
    uint16_t r[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) r[x] = f2h(l == 0.f ? 0.f : sum[x] * inv);
    *reinterpret_cast<uint2*>(p.out + head0 * D + i * 4) =
        make_uint2(r[0] | (static_cast<uint32_t>(r[1]) << 16), r[2] | (static_cast<uint32_t>(r[3]) << 16));
}

// What no kernel in flight writes, at an address that a whole wave shares: read through the scalar cache, whose
// loads have a counter of their own (a wait for a page number must not be one for all the K and V in flight).
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ scalar_ints as_scalar(const int32_t* p) { return (scalar_ints)reinterpret_cast<uintptr_t>(p); }

// Counts this workgroup in; true in every thread of the one that is the last of n.
__device__ __forceinline__ bool last_in(unsigned* counter, int n, int* flag) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this thread's part is written through
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned old = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int last = old == static_cast<unsigned>(n - 1);
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = last;
    }
    __syncthreads();
    return *flag != 0;
}

template <int D, int W>
__global__ __launch_bounds__(64 * W, 2) void paged_attention_kernel(AttnArgs p) {
    constexpr int KS = D / 32;                   // steps of the score product
    constexpr int RC = D / 8;                    // 16-byte chunks of a row
    constexpr int VW = D / 16;                   // d of V a lane loads of one token
    constexpr int VC = VW < 8 ? VW : 8;          // ... in chunks of this many
    constexpr int VN = VW / VC;
    typedef uint32_t vchunk __attribute__((ext_vector_type(VC / 2)));
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];        // K [wave][32][D + 8]; then the waves' parts [wave][head][D]
    __shared__ float2 stat[W][kHeads];
    __shared__ int flag;
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_seq = p.Hkv * p.htiles;
    auto length = [&](int b) {
        const int n = b < p.B ? p.lens[b] : 0;
        return n < 0 ? 0 : n > p.max_len ? p.max_len : n;
    };
    auto tiles_of = [&](int b, int len) { return b >= p.B ? 0 : len <= kTile ? 1 : (len + kTile - 1) / kTile; };   // none: one, its zeros

    // Tiles of a part, and this workgroup's sequence b, whose first part has number w_first and whose first tile b_first.
    // A lane adds up `span` sequences; where that is more than one, the chosen lane's are then taken one a lane.
    const int me = blockIdx.x, span = (p.B + 63) / 64;
    int per = 0x3fffffff, b, len = 0, b_first = 0, w_first = 0;
    {
        int mine = length(lane);                 // (of span 1)
        auto sum_of = [&](auto f) {
            if (span == 1) return f(lane, mine);
            int sum = 0;
#pragma unroll 4
            for (int i = 0; i < span; ++i) sum += f(lane * span + i, length(lane * span + i));
            return sum;
        };
        if (p.split) {
            const int total = __builtin_amdgcn_readlane(wave_scan(sum_of(tiles_of)), 63) * per_seq;
            const auto whole_steps = [](int n) { return (n + W - 1) / W * W; };
            per = whole_steps((total + p.split - 1) / p.split);
            // Few (sequence, cache head)s: as many parts as CUs at most, so that none has two while others have one.
            // MI355X, us of 256, 512 and 768 workgroups: 1 x 200000 70 72 79, 1 x 25000 D 128 24 27 28; where there
            // are many, small parts even out better than one each: 41 x 4096 ragged 35 28 28, 8 x 20000 D 128 59 48 51.
            if (p.B * per_seq <= kCus / 8 && total > kCus * W) {
                per = whole_steps((total + kCus - 1) / kCus);
                for (int i = 0; i < 4; ++i) {
                    const int n = __builtin_amdgcn_readlane(wave_scan(sum_of([&](int b, int len) { return (tiles_of(b, len) + per - 1) / per; })), 63) * per_seq;
                    if (n <= kCus) break;
                    per = whole_steps(per + (per * (n - kCus) + kCus - 1) / kCus);
                }
            }
        }
        auto parts_of = [&](int b, int n) { return (tiles_of(b, n) + per - 1) / per; };
        int upto = wave_scan(sum_of(parts_of) * per_seq), tiles_upto = wave_scan(sum_of(tiles_of) * per_seq);
        unsigned long long past = __ballot(upto > me);           // lanes at and past this workgroup's
        if (!past) return;
        int at = __builtin_ctzll(past);
        auto go_to = [&]() {
            if (at) {
                w_first += __builtin_amdgcn_readlane(upto, at - 1);
                b_first += __builtin_amdgcn_readlane(tiles_upto, at - 1);
            }
        };
        go_to();
        b = at * span;
        while (span > 1) {
            mine = length(b + lane);
            upto = wave_scan(parts_of(b + lane, mine) * per_seq);
            tiles_upto = wave_scan(tiles_of(b + lane, mine) * per_seq);
            past = __ballot(w_first + upto > me);
            at = past ? __builtin_ctzll(past) : 64;
            go_to();
            b += at;
            if (past) break;
            if (b >= p.B) return;                // (lengths that changed meanwhile)
        }
        len = __builtin_amdgcn_readlane(mine, at);
    }
    per = __builtin_amdgcn_readfirstlane(per);
    const int tiles = len <= kTile ? 1 : (len + kTile - 1) / kTile, parts = (tiles + per - 1) / per;
    // (the cache heads of one part side by side: their rows lie together in memory)
    const int part = (me - w_first) / per_seq, in_seq = me - w_first - part * per_seq;
    const int s0 = part * per, hk = in_seq / p.htiles, ht = in_seq - hk * p.htiles;
    const int rows = p.group - ht * kHeads < kHeads ? p.group - ht * kHeads : kHeads;
    const int64_t head0 = static_cast<int64_t>(b) * p.Hq + hk * p.group + ht * kHeads;
    const int t1 = part < parts - 1 ? (s0 + per) * kTile : len;

    constexpr int RS = RC + 1;                   // chunks from row to row: 16 rows' same chunk are in 16 places of the banks
    half8_t* const kl = reinterpret_cast<half8_t*>(lds) + wave * kTile * RS;
    half8_t *const k_in = kl + lane / RC * RS + lane % RC, *const k_out = kl + c * RS + j;
    const int koff = 2 * (lane / RC * p.k_token + lane % RC * 8), voff = 2 * (4 * j * p.v_token + VC * c);

    half8_t q[KS];                           // lanes past the last head: the first again, never stored
#pragma unroll
    for (int s = 0; s < KS; ++s)
        q[s] = *reinterpret_cast<const half8_t*>(p.q + b * p.q_row + static_cast<int64_t>(hk * p.group + ht * kHeads + (c < rows ? c : 0)) * p.q_head +
                                                 32 * s + 8 * j);
    const scalar_ints table = as_scalar(p.table + b * p.table_row);
    const uint16_t* kh = p.k + hk * p.k_head;
    const uint16_t* vh = p.v + hk * p.v_head;

    // Rows of 16 tokens from t on: their page's number (-1: not there, or past the end) and first row in it.
    auto place = [&](int t, int& page, int& row) {
        const uint32_t t16 = static_cast<uint32_t>(t) >> 4;
        uint32_t at = t16;
        row = 0;
        if (p.page16 > 1) {
            at = __umulhi(t16, p.page16_inv);    // one too many at most
            int r = static_cast<int>(t16 - at * p.page16);
            if (r < 0) --at, r += p.page16;
            row = 16 * r;
        }
        page = t < t1 ? table[at] : -1;
        page = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(page) < static_cast<uint32_t>(p.pages) ? page : -1);
    };
    // Loads are unconditional, of no bytes where there is no page, so that a wait counts those in flight exactly.
    auto rows16 = [](const uint16_t* base, int page, int row, int64_t page_stride, int token_stride) {
        const uint16_t* at = base + (page < 0 ? 0 : page) * page_stride + static_cast<int64_t>(row) * token_stride;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(at), 0, page < 0 ? 0 : 2 * (15 * token_stride + D), 0x00020000);
    };
    int4_t kr[2][KS];
    vchunk vr[8][VN];
    auto load_k = [&](const int (&page)[2], const int (&row)[2]) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const __amdgpu_buffer_rsrc_t r = rows16(kh, page[x], row[x], p.k_page, p.k_token);
#pragma unroll
            for (int i = 0; i < KS; ++i) kr[x][i] = __builtin_amdgcn_raw_buffer_load_b128(r, koff, 2 * i * (64 / RC) * p.k_token, kOnce);
        }
    };
    auto load_v = [&](const int (&page)[2], const int (&row)[2]) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const __amdgpu_buffer_rsrc_t r = rows16(vh, page[x], row[x], p.v_page, p.v_token);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < VN; ++n) {
                    if constexpr (VC == 8)
                        vr[4 * x + i][n] = __builtin_bit_cast(vchunk, __builtin_amdgcn_raw_buffer_load_b128(r, voff + 256 * n, 2 * i * p.v_token, kOnce));
                    else
                        vr[4 * x + i][n] = __builtin_bit_cast(vchunk, __builtin_amdgcn_raw_buffer_load_b64(r, voff, 2 * i * p.v_token, kOnce));
                }
        }
    };

    float4_t acc[VN][VC] = {};
    float m = -INFINITY, l = 0.f;
    int t = (s0 + wave - W) * kTile;         // the tile in the registers: none yet
    int page[2] = {-1, -1};
    bool have = false;
    do {
        const int tn = t + W * kTile;
        int npage[2], nrow[2];
        place(tn, npage[0], nrow[0]);
        place(tn + 16, npage[1], nrow[1]);
        float4_t s[2] = {};
        if (have) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    k_in[(16 * x + i * (64 / RC)) * RS] = __builtin_bit_cast(half8_t, kr[x][i]);
        }
        load_k(npage, nrow);
        if (have) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    s[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k_out[16 * x * RS + 4 * i], q[i], s[x], 0, 0, 0);
            __builtin_amdgcn_wave_barrier();
            const bool whole = t + kTile <= t1 && page[0] >= 0 && page[1] >= 0;
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = s[x][r] * p.scale_log2;
                    if (!whole && (page[x] < 0 || t + 16 * x + 4 * j + r >= t1)) v = -INFINITY;
                    s[x][r] = v;
                    mx = fmaxf(mx, v);
                }
            mx = fmaxf(max4(mx), m);
            if (__any(mx > m)) {
                const float keep = m == -INFINITY ? 0.f : exp2_of(m - mx);
                l *= keep;
#pragma unroll
                for (int n = 0; n < VN; ++n)
#pragma unroll
                    for (int i = 0; i < VC; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[n][i][r] *= keep;
                m = mx;
            }
            const float base = m == -INFINITY ? 0.f : m;         // nothing so far: every weight 2^-inf
            float e[8];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    e[4 * x + r] = exp2_of(s[x][r] - base) * kTop;
                    l += e[4 * x + r];
                }
            uint4 w, w_lo;
            auto parts_of = [&](int i, uint32_t& hi, uint32_t& lo) {
                const auto h = __builtin_amdgcn_cvt_pkrtz(e[i], e[i + 1]);
                const half2_t r = {static_cast<_Float16>(e[i] - static_cast<float>(h[0])), static_cast<_Float16>(e[i + 1] - static_cast<float>(h[1]))};
                hi = __builtin_bit_cast(uint32_t, h);
                const ushort2_t least = __builtin_elementwise_min(__builtin_bit_cast(ushort2_t, h), ushort2_t{1, 1});
                lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, r), least));
            };
            parts_of(0, w.x, w_lo.x);
            parts_of(2, w.y, w_lo.y);
            parts_of(4, w.z, w_lo.z);
            parts_of(6, w.w, w_lo.w);
            if (!whole)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (page[x] < 0 || t + 16 * x + 4 * j + i >= t1)
#pragma unroll
                            for (int n = 0; n < VN; ++n) vr[4 * x + i][n] = vchunk(0);
#pragma unroll
            for (int n = 0; n < VN; ++n)
#pragma unroll
                for (int d = 0; d < VC; ++d) {
                    const uint32_t pick = d & 1 ? 0x07060302u : 0x05040100u;
                    uint4 a;
                    a.x = __builtin_amdgcn_perm(vr[1][n][d / 2], vr[0][n][d / 2], pick);
                    a.y = __builtin_amdgcn_perm(vr[3][n][d / 2], vr[2][n][d / 2], pick);
                    a.z = __builtin_amdgcn_perm(vr[5][n][d / 2], vr[4][n][d / 2], pick);
                    a.w = __builtin_amdgcn_perm(vr[7][n][d / 2], vr[6][n][d / 2], pick);
                    acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, w), acc[n][d], 0, 0, 0);
                    acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, w_lo), acc[n][d], 0, 0, 0);
                }
        }
        load_v(npage, nrow);
        t = tn;
        have = true;
#pragma unroll
        for (int x = 0; x < 2; ++x) page[x] = npage[x];
    } while (t < t1);
    l = sum4(l);

    // The waves' parts meet in LDS.
    const int slot = static_cast<int>(part_bytes(p.group < kHeads ? p.group : kHeads, D));     // sized for the widest head tile
    // Part i has the id w0 + i, w0 the part of an even cut of all tiles that the first tile falls into.  A part 0
    // has slot 2 id + 1, others 2 id: ids of one (sequence, cache head) are its own but for its last,
    // which may be the next one's first.
    const int w0 = (b_first + in_seq * tiles) / per;
    const int slots0 = static_cast<int>(kCounterBytes);
    auto part_at = [&](int i) { return slots0 + (i == 0 ? 2 * w0 + 1 : 2 * (w0 + i)) * slot; };
    const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc(p.ws, 0, 0x7fffffff, 0x00020000);
    auto put = [&](int at, int i, float4_t sum, float m2, float l2) {
        if (at < 0) {
            put_out<D>(p, head0, i, sum, l2);
            return;
        }
        const int4_t v = {__float_as_int(sum[0]), __float_as_int(sum[1]), __float_as_int(sum[2]), __float_as_int(sum[3])};
        __builtin_amdgcn_raw_buffer_store_b128(v, ws, at + i * 16, 0, 16);
        if (i % (D / 4) == 0) {
            typedef unsigned u2 __attribute__((ext_vector_type(2)));
            __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(m2), __float_as_uint(l2)}, ws, at + rows * D * 4 + i / (D / 4) * 8, 0, 16);
        }
    };
    int tid = threadIdx.x;                   // (opaque: addresses made from it would be kept through the loop above)
    asm volatile("" : "+v"(tid));
    const int tc = tid & 15, tj = (tid & 63) >> 4;
    float* const meet = reinterpret_cast<float*>(lds);
    __syncthreads();                         // K has been read
    if (tc < rows) {
        if (tj == 0) stat[wave][tc] = make_float2(m, l);
#pragma unroll
        for (int n = 0; n < VN; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // acc[n][i][r]: d = 128 n + VC (4 j + r) + i
                float* at = meet + (wave * rows + tc) * D + 128 * n + VC * (4 * tj + r);
#pragma unroll
                for (int i = 0; i < VC; i += 4)
                    *reinterpret_cast<float4_t*>(at + i) = float4_t{acc[n][i][r], acc[n][i + 1][r], acc[n][i + 2][r], acc[n][i + 3][r]};
            }
    }
    __syncthreads();
    for (int i = tid; i < rows * D / 4; i += 64 * W) {
        const int h = i / (D / 4);
        float4_t sum = {0, 0, 0, 0};
        float top = -INFINITY, tot = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w][h].x);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 st = stat[w][h];
            const float by = st.x == -INFINITY ? 0.f : exp2_of(st.x - top);
            const float4_t o = *reinterpret_cast<const float4_t*>(meet + w * rows * D + i * 4);
            tot = fmaf(st.y, by, tot);
#pragma unroll
            for (int x = 0; x < 4; ++x) sum[x] = fmaf(o[x], by, sum[x]);
        }
        put(parts == 1 ? -1 : part_at(part), i, sum, top, tot);
    }
    if (parts > 1) {
        // Counters: one by w0 (of those cut, each has its own); where there are several fans (then no other such begins
        // within kFan ids), one for the first and one for each of the others.
        unsigned* const counters = reinterpret_cast<unsigned*>(p.ws);
        const int ids = p.split + 2, of_fans = (ids + kFan - 1) / kFan;
        const int fan = part / kFan, fans = (parts + kFan - 1) / kFan;
        auto fan_id = [&](int f) { return f == 0 ? w0 / kFan : of_fans + (w0 + f * kFan) / kFan; };
        const int joined = slots0 + 2 * ids * slot;
        for (int level = fans == 1 ? 1 : 0; level < 2; ++level) {
            // level 0: this fan's parts into one; level 1: all there is into the output
            const int n = level == 0 ? (parts - fan * kFan < kFan ? parts - fan * kFan : kFan) : fans == 1 ? parts : fans;
            if (!last_in(level == 0 ? counters + ids + fan_id(fan) : counters + w0, n, &flag)) break;
            const bool of_parts = level == 0 || fans == 1;
            const int from0 = of_parts ? part_at(level == 0 ? fan * kFan : 0) : joined + fan_id(0) * slot;
            const int from1 = of_parts ? part_at((level == 0 ? fan * kFan : 0) + 1) : joined + fan_id(1) * slot;
            const int step = of_parts ? 2 * slot : slot;
            for (int i = tid; i < rows * D / 4; i += 64 * W) {
                const int h = i / (D / 4);
                float4_t sum = {0, 0, 0, 0};
                float top = -INFINITY, tot = 0.f;
                constexpr int kBatch = kFan;   // loads of a batch go out together
                for (int u0 = 0; u0 < n; u0 += kBatch) {
                    int4_t o[kBatch];
                    float2 st[kBatch];
                    float most = top;
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const int e = u0 + u < n ? u0 + u : n - 1;
                        const int at = e == 0 ? from0 : from1 + (e - 1) * step;
                        o[u] = __builtin_amdgcn_raw_buffer_load_b128(ws, i * 16, at, 16);
                        const auto x = __builtin_amdgcn_raw_buffer_load_b64(ws, rows * D * 4 + h * 8, at, 16);
                        st[u] = make_float2(__uint_as_float(x[0]), __uint_as_float(x[1]));
                    }
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) most = fmaxf(most, st[u].x);
                    const float keep = top == -INFINITY ? 0.f : exp2_of(top - most);
                    tot *= keep;
                    sum *= keep;
                    top = most;
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        if (u0 + u >= n) continue;
                        const float by = st[u].x == -INFINITY ? 0.f : exp2_of(st[u].x - top);
                        tot = fmaf(st[u].y, by, tot);
#pragma unroll
                        for (int x = 0; x < 4; ++x) sum[x] = fmaf(__int_as_float(o[u][x]), by, sum[x]);
                    }
                }
                put(level == 0 ? joined + fan_id(fan) * slot : -1, i, sum, top, tot);
            }
        }
    }
}

// Workgroups to cut the `groups` (sequence, cache head, head tile)s of up to `most` tokens for: what the chip
// holds at once with D = 256, two a CU.  With D = 128 it holds three; MI355X, us of 512, 640 and 768: 16 x 2000 ragged
// 15.7 15.6 16.2, 8 x 20000 48 51 51, 41 x 4096 (32 heads on 8) 55 49 51, 5 x 60000 48 53 50, 64 x 1000 25.9 25.9 26.4:
// no number is the best of all, 512 loses once.
// 0: nothing to cut.
int choose_workers(int64_t groups, int64_t most) {
    const int64_t tiles = ceil_div(most, kTile);
    if (most <= 4 * kTile) return 0;
    return static_cast<int>(std::min<int64_t>(512, groups * ceil_div(tiles, 4)));
}
int64_t split_bytes(int64_t workers, int64_t rows, int64_t D) {
    return workers == 0 ? 0 : kCounterBytes + (2 * (workers + 2) + 2 * ceil_div(workers + 2, kFan)) * part_bytes(static_cast<int>(rows), static_cast<int>(D));
}

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int64_t mcv_paged_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seq_len) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || B > 0x7fffffff / Hq || D <= 0 || max_seq_len < 0) return 0;
    const int64_t group = Hq / Hkv, groups = B * Hkv * ceil_div(group, kHeads);
    const int64_t most = max_seq_len < kMaxLen ? max_seq_len : kMaxLen;
    return split_bytes(choose_workers(groups, most), group < kHeads ? group : kHeads, D);
}

int mcv_paged_attention(const void* q, int64_t q_row, int64_t q_head, const void* k_cache, int64_t k_page,
                        int64_t k_token, int64_t k_head, const void* v_cache, int64_t v_page, int64_t v_token,
                        int64_t v_head, int64_t pages, int64_t page_size, const void* block_table,
                        int64_t table_row, int64_t table_width, const void* seq_lens, int64_t max_seq_len, int64_t B,
                        int64_t Hq, int64_t Hkv, int64_t D, double scale, void* out, void* workspace,
                        int64_t workspace_bytes, mcv_stream_t stream) {
    if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out)
        return fail(MCV_ERR_INVALID_ARG, "paged_attention: null pointer");
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || B > 0x7fffffff / Hq)
        return fail(MCV_ERR_SHAPE, "paged_attention: bad shape B=%lld Hq=%lld Hkv=%lld", (long long)B, (long long)Hq,
                    (long long)Hkv);
    if (D != 64 && D != 128 && D != 256)
        return fail(MCV_ERR_SHAPE, "paged_attention: D must be 64, 128 or 256 (D=%lld)", (long long)D);
    if (page_size <= 0 || page_size % 16 != 0 || page_size > (1 << 20))
        return fail(MCV_ERR_SHAPE, "paged_attention: page_size must be a multiple of 16 (page_size=%lld)", (long long)page_size);
    if (pages <= 0 || pages > 0x7fffffff || table_width <= 0 || max_seq_len < 0)
        return fail(MCV_ERR_SHAPE, "paged_attention: bad cache pages=%lld table_width=%lld max_seq_len=%lld", (long long)pages,
                    (long long)table_width, (long long)max_seq_len);
    if (q_row < 0 || q_head < 0 || k_page < 0 || k_token < 0 || k_head < 0 || v_page < 0 || v_token < 0 || v_head < 0 ||
        table_row < 0)
        return fail(MCV_ERR_SHAPE, "paged_attention: negative stride");
    if (!chunked16(q, {q_row, q_head}) || !chunked16(k_cache, {k_page, k_token, k_head}) ||
        !chunked16(v_cache, {v_page, v_token, v_head}) || !chunked16(out, {}))
        return fail(MCV_ERR_UNSUPPORTED, "paged_attention: pointers must be 16-byte aligned, strides multiples of 8 elements");
    int rc = require_device();
    if (rc != MCV_OK) return rc;
    if (k_token > (1 << 25) || v_token > (1 << 25))
        return fail(MCV_ERR_UNSUPPORTED, "paged_attention: tokens of one page too far apart");
    // (width counted in pages first: width * page_size could pass 64 bits)
    const int64_t held = table_width > kMaxLen / page_size ? kMaxLen : table_width * page_size;
    const int64_t most = max_seq_len < held ? max_seq_len : held;
    const int64_t group = Hq / Hkv, htiles = ceil_div(group, kHeads), groups = B * Hkv * htiles;
    const int64_t rows = group < kHeads ? group : kHeads;
    int workers = groups * ceil_div(most, kTile) <= 0x3fffffff ? choose_workers(groups, most) : 0;      // tiles are counted in 32 bits
    if (workers && (!workspace || workspace_bytes < split_bytes(workers, rows, D))) workers = 0;
    if (workers && reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return fail(MCV_ERR_INVALID_ARG, "paged_attention: workspace must be 256-byte aligned");
    const uint32_t page16 = static_cast<uint32_t>(page_size / 16);
    AttnArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache),
               static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(seq_lens), static_cast<uint16_t*>(out),
               static_cast<uint8_t*>(workspace), q_row, q_head, k_page, k_head, v_page, v_head, table_row,
               static_cast<int>(k_token), static_cast<int>(v_token), static_cast<int>(pages), static_cast<int>(page16),
               static_cast<int>(most), static_cast<int>(B), static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(group),
               static_cast<int>(htiles), page16 > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + page16 - 1) / page16) : 0,
               static_cast<float>(scale) * kLog2e, workers};
    auto fn = D == 64 ? paged_attention_kernel<64, 4> : D == 128 ? paged_attention_kernel<128, 4> : paged_attention_kernel<256, 4>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups + workers)), dim3(256),
                       static_cast<unsigned>(4 * std::max<int64_t>(kTile * 2 * (D + 8), rows * 4 * D)), static_cast<hipStream_t>(stream), a);
    return check_launch("paged_attention_kernel");
}

}  // extern "C"
