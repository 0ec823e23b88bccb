// paged_attention.hip -- attention of one new token over a paged cache, gfx950.
//
// One pass over the cache with the running maximum m and sum l of the softmax, in
// 32 bits and base 2:  w_t = 2^(s_t - m), o = sum w_t v_t / l.  The up to 16 query
// heads of one cache head share every byte of K and V (and are one side of the matrix
// products, however few they are: the matrix cores have time to spare here).
//
// A wave takes 32 tokens at a time, straight from memory into registers, no LDS:
//   S^T = K Q^T   v_mfma_f32_16x16x32_f16, twice 16 tokens as rows; lane (c, j), c =
//                 lane % 16, j = lane / 16, then holds head c and tokens 4j .. 4j + 3 of each half
//   O^T += V^T P^T  the sum over tokens may run in any order, so lane (c, j)'s eight
//                 weights are the product's operand as they stand, and the lane loads V's
//                 same eight rows, 8 d of each, whose 8 x 8 values it turns in registers
// What lies past the sequence's end, or in a page that is not there, has score -inf and
// its V is set to zero (it may hold NaN).
//
// A unit is `unit` tokens of one (sequence, cache head), shared by the four waves of a
// workgroup tile by tile.  Units of one sequence meet through the workspace: each
// writes its 32-bit part with device-scope stores (written through; see
// w4a16_gemm_sk.hip) and counts itself in; the last of each kFan units joins them in
// order, and where there are more than kFan the last of those joins the joined, so
// the bits do not depend on who is last and nobody waits.
#include "mixers.h"

namespace mcv {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;                        // tokens a wave takes at a time
constexpr int kStep = kWaves * kTile;            // units are whole multiples of this
constexpr int kHeads = 16;                       // query heads of one matrix product
constexpr int kFan = 16;                         // parts joined by one workgroup
constexpr int64_t kCounterBytes = 4096;
constexpr int64_t kMaxLen = int64_t(1) << 30;   // tokens of one sequence
constexpr float kLog2e = 1.44269504088896340736f;

struct AttnArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* lens;
    uint16_t* out;
    uint8_t* ws;
    int64_t q_row, q_head, k_page, k_head, v_page, v_head, table_row;
    int k_token, v_token, pages, page16, max_len, Hq, Hkv, group, htiles, unit, max_units;
    uint32_t page16_inv;                         // ceil(2^32 / page16), page16 > 1
    float scale_log2;
};

// Bytes of one part: [rows][D] sums, [rows][2] maximum and sum, whole 16-byte chunks.
__host__ __device__ constexpr int64_t part_bytes(int rows, int D) { return int64_t(rows) * D * 4 + ((rows * 8 + 15) & ~15); }

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

// Weights of two parts with maxima m and n against their common one (-inf: a part of nothing).
__device__ __forceinline__ void join_weights(float m, float n, float& top, float& wm, float& wn) {
    top = fmaxf(m, n);
    wm = m == -INFINITY ? 0.f : exp2_of(m - top);
    wn = n == -INFINITY ? 0.f : exp2_of(n - top);
}

// Joins parts 0 .. n - 1 at byte `from` of the workspace, in order.  Thread i has the
// float4s i, i + 256, ... of [rows][D]; `put` takes (float4 number, sum, m, l).
template <int D, class Put>
__device__ __forceinline__ void join_parts(const AttnArgs& p, int64_t from, int n, int rows, Put put) {
    const int64_t bytes = part_bytes(rows, D);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(p.ws + from, 0, static_cast<int>(n * bytes), 0x00020000);
    for (int i = threadIdx.x; i < rows * D / 4; i += 64 * kWaves) {
        const int row = i / (D / 4);
        float4_t sum = {0, 0, 0, 0};
        float m = -INFINITY, l = 0.f;
        constexpr int kBatch = 8;                // loads of a batch go out together
        for (int u0 = 0; u0 < n; u0 += kBatch) {
            int4_t o[kBatch];
            uint2 st[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int at = static_cast<int>((u0 + u < n ? u0 + u : n - 1) * bytes);
                o[u] = __builtin_amdgcn_raw_buffer_load_b128(r, at + i * 16, 0, 16);
                const auto s = __builtin_amdgcn_raw_buffer_load_b64(r, at + rows * D * 4 + row * 8, 0, 16);
                st[u] = make_uint2(s[0], s[1]);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (u0 + u >= n) break;
                float top, a, b;
                join_weights(m, __uint_as_float(st[u].x), top, a, b);
                m = top;
                l = l * a + __uint_as_float(st[u].y) * b;
#pragma unroll
                for (int x = 0; x < 4; ++x) sum[x] = sum[x] * a + __int_as_float(o[u][x]) * b;
            }
        }
        put(i, sum, m, l);
    }
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

template <int D>
__device__ __forceinline__ void put_part(const AttnArgs& p, int64_t at, int rows, int i, float4_t sum, float m, float l) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(p.ws + at, 0, static_cast<int>(part_bytes(rows, D)), 0x00020000);
    const int4_t v = {__float_as_int(sum[0]), __float_as_int(sum[1]), __float_as_int(sum[2]), __float_as_int(sum[3])};
    __builtin_amdgcn_raw_buffer_store_b128(v, r, i * 16, 0, 16);
    if (i % (D / 4) == 0) {
        typedef unsigned u2 __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(m), __float_as_uint(l)}, r, rows * D * 4 + i / (D / 4) * 8, 0, 16);
    }
}

template <int D>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_attention_kernel(AttnArgs p) {
    constexpr int KS = D / 32;                   // steps of the score product
    constexpr int VW = D / 16;                   // d of V a lane loads of one token
    constexpr int VC = VW < 8 ? VW : 8;          // ... in chunks of this many
    constexpr int VN = VW / VC;
    typedef uint32_t vchunk __attribute__((ext_vector_type(VC / 2)));
    const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bh = blockIdx.x;
    const int ht = bh % p.htiles, hk = bh / p.htiles % p.Hkv, b = bh / p.htiles / p.Hkv;
    const int rows = p.group - ht * kHeads < kHeads ? p.group - ht * kHeads : kHeads;
    const int64_t head0 = static_cast<int64_t>(b) * p.Hq + hk * p.group + ht * kHeads;
    int len = p.lens[b];
    len = len < 0 ? 0 : len > p.max_len ? p.max_len : len;
    const int unit = blockIdx.y, units = len == 0 ? 1 : (len - 1) / p.unit + 1;
    if (unit >= units) return;
    const int t1 = len - unit * p.unit < p.unit ? len : (unit + 1) * p.unit;

    half8_t q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (c < rows)
            w = *reinterpret_cast<const uint4*>(p.q + b * p.q_row + static_cast<int64_t>(hk * p.group + ht * kHeads + c) * p.q_head + 32 * s + 8 * j);
        q[s] = __builtin_bit_cast(half8_t, w);
    }
    const int32_t* __restrict__ table = p.table + b * p.table_row;
    const uint16_t* kh = p.k + hk * p.k_head;
    const uint16_t* vh = p.v + hk * p.v_head;
    const int koff = c * p.k_token + 8 * j, voff = 4 * j * p.v_token + VC * c;

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
        if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.pages)) page = -1;
    };
    half8_t kf[2][KS];
    vchunk vr[8][VN];
    auto load_k = [&](const int (&page)[2], const int (&row)[2]) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint16_t* at = kh + (page[x] < 0 ? 0 : page[x]) * p.k_page + static_cast<int64_t>(row[x]) * p.k_token;
#pragma unroll
            for (int s = 0; s < KS; ++s) kf[x][s] = *reinterpret_cast<const half8_t*>(at + koff + 32 * s);
        }
    };
    auto load_v = [&](const int (&page)[2], const int (&row)[2]) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint16_t* at = vh + (page[x] < 0 ? 0 : page[x]) * p.v_page + static_cast<int64_t>(row[x]) * p.v_token;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < VN; ++n)
                    vr[4 * x + i][n] = *reinterpret_cast<const vchunk*>(at + static_cast<int64_t>(i) * p.v_token + voff + 128 * n);
        }
    };

    float4_t acc[VN][VC] = {};
    float m = -INFINITY, l = 0.f;
    int t = unit * p.unit + wave * kTile;
    int page[2], row[2];
    if (t < t1) {
        place(t, page[0], row[0]);
        place(t + 16, page[1], row[1]);
        load_k(page, row);
        load_v(page, row);
    }
    while (t < t1) {
        const int tn = t + kStep;
        int npage[2] = {-1, -1}, nrow[2] = {0, 0};
        if (tn < t1) {
            place(tn, npage[0], nrow[0]);
            place(tn + 16, npage[1], nrow[1]);
        }
        float4_t s[2] = {};
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < KS; ++i) s[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[x][i], q[i], s[x], 0, 0, 0);
        if (tn < t1) load_k(npage, nrow);
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
        half8_t w;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = exp2_of(s[x][r] - base);
                l += e;
                w[4 * x + r] = static_cast<_Float16>(e);     // the product's operand: one rounding of each weight
            }
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
                acc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), w, acc[n][d], 0, 0, 0);
            }
        if (tn < t1) load_v(npage, nrow);
        t = tn;
#pragma unroll
        for (int x = 0; x < 2; ++x) page[x] = npage[x], row[x] = nrow[x];
    }
    l = sum4(l);

    // The waves' parts meet in LDS, up to 128 d at a time: [wave][head][DL].
    constexpr int DL = D < 128 ? D : 128;
    extern __shared__ float lds[];
    __shared__ float2 stat[kWaves][kHeads];
    __shared__ int flag;
    if (c < rows && j == 0) stat[wave][c] = make_float2(m, l);
    const int64_t bytes = part_bytes(rows, D);
    // this (sequence, cache head, head tile)'s parts: sized for the widest tile
    const int64_t all = part_bytes(p.group < kHeads ? p.group : kHeads, D);
    const int fans = (p.max_units + kFan - 1) / kFan;
    const int64_t mine = kCounterBytes + bh * p.max_units * all;
#pragma unroll
    for (int n = 0; n < VN; ++n) {
        if (n) __syncthreads();
        if (c < rows)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // acc[n][i][r]: d = 128 n + VC (4 j + r) + i
                float* at = lds + (wave * rows + c) * DL + VC * (4 * j + r);
#pragma unroll
                for (int i = 0; i < VC; i += 4)
                    *reinterpret_cast<float4_t*>(at + i) = float4_t{acc[n][i][r], acc[n][i + 1][r], acc[n][i + 2][r], acc[n][i + 3][r]};
            }
        __syncthreads();
        for (int e = threadIdx.x; e < rows * DL / 4; e += 64 * kWaves) {
            const int h = e / (DL / 4);
            float4_t sum = {0, 0, 0, 0};
            float top = -INFINITY, tot = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float4_t o = *reinterpret_cast<const float4_t*>(lds + w * rows * DL + e * 4);
                const float2 st = stat[w][h];
                float wa, wb, nt;
                join_weights(top, st.x, nt, wa, wb);
                top = nt;
                tot = tot * wa + st.y * wb;
#pragma unroll
                for (int x = 0; x < 4; ++x) sum[x] = sum[x] * wa + o[x] * wb;
            }
            const int i = h * (D / 4) + n * (DL / 4) + e % (DL / 4);
            if (units == 1) put_out<D>(p, head0, i, sum, tot);
            else put_part<D>(p, mine + unit * bytes, rows, i, sum, top, tot);
        }
    }
    if (units == 1) return;
    // counters: one per (.., head tile), then one for each of its fans
    unsigned* const counters = reinterpret_cast<unsigned*>(p.ws);
    const int fan = unit / kFan, nfan = (units + kFan - 1) / kFan;
    const int in_fan = units - fan * kFan < kFan ? units - fan * kFan : kFan;
    auto out = [&](int i, float4_t sum, float, float l2) { put_out<D>(p, head0, i, sum, l2); };
    if (nfan == 1) {
        if (last_in(counters + bh, units, &flag)) join_parts<D>(p, mine, units, rows, out);
        return;
    }
    if (!last_in(counters + gridDim.x + bh * fans + fan, in_fan, &flag)) return;
    const int64_t joined = kCounterBytes + (static_cast<int64_t>(gridDim.x) * p.max_units + bh * fans) * all;
    join_parts<D>(p, mine + fan * kFan * bytes, in_fan, rows,
                  [&](int i, float4_t sum, float m2, float l2) { put_part<D>(p, joined + fan * bytes, rows, i, sum, m2, l2); });
    if (last_in(counters + bh, nfan, &flag)) join_parts<D>(p, joined, nfan, rows, out);
}

// Tokens a unit takes and units of the longest sequence, for `most` tokens at most.
struct Split {
    int64_t unit, units, fans;
};
Split choose_split(int64_t groups, int64_t most) {
    constexpr int64_t kWant = 1024;              // workgroups
    Split s;
    s.unit = ceil_div(ceil_div(groups * most, kWant), kStep) * kStep;
    if (s.unit < kStep) s.unit = kStep;
    s.units = most > 0 ? ceil_div(most, s.unit) : 1;
    s.fans = ceil_div(s.units, kFan);
    return s;
}
int64_t split_bytes(const Split& s, int64_t groups, int64_t rows, int64_t D) {
    return s.units == 1 ? 0 : kCounterBytes + groups * (s.units + (s.fans > 1 ? s.fans : 0)) * part_bytes(static_cast<int>(rows), static_cast<int>(D));
}

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int64_t mcv_paged_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seq_len) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || B > 0x7fffffff / Hq || D <= 0 || max_seq_len < 0) return 0;
    const int64_t group = Hq / Hkv, groups = B * Hkv * ceil_div(group, kHeads);
    const int64_t most = max_seq_len < kMaxLen ? max_seq_len : kMaxLen;
    return split_bytes(choose_split(groups, most), groups, group < kHeads ? group : kHeads, D);
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
    if (k_token > (1 << 26) || v_token > (1 << 26))
        return fail(MCV_ERR_UNSUPPORTED, "paged_attention: tokens of one page too far apart");
    // (width counted in pages first: width * page_size could pass 64 bits)
    const int64_t held = table_width > kMaxLen / page_size ? kMaxLen : table_width * page_size;
    const int64_t most = max_seq_len < held ? max_seq_len : held;
    const int64_t group = Hq / Hkv, htiles = ceil_div(group, kHeads), groups = B * Hkv * htiles;
    const int64_t rows = group < kHeads ? group : kHeads;
    Split s = choose_split(groups, most);
    if (s.units > 1 && (!workspace || workspace_bytes < split_bytes(s, groups, rows, D))) s = {ceil_div(most, kStep) * kStep, 1, 1};
    if (s.units > 1 && reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return fail(MCV_ERR_INVALID_ARG, "paged_attention: workspace must be 256-byte aligned");
    const uint32_t page16 = static_cast<uint32_t>(page_size / 16);
    AttnArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache),
               static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(seq_lens), static_cast<uint16_t*>(out),
               static_cast<uint8_t*>(workspace), q_row, q_head, k_page, k_head, v_page, v_head, table_row,
               static_cast<int>(k_token), static_cast<int>(v_token), static_cast<int>(pages), static_cast<int>(page16),
               static_cast<int>(most), static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(group),
               static_cast<int>(htiles), static_cast<int>(s.unit > 0 ? s.unit : kStep), static_cast<int>(s.units),
               page16 > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + page16 - 1) / page16) : 0,
               static_cast<float>(scale) * kLog2e};
    auto fn = D == 64 ? paged_attention_kernel<64> : D == 128 ? paged_attention_kernel<128> : paged_attention_kernel<256>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(groups), static_cast<unsigned>(s.units)), dim3(64 * kWaves),
                       static_cast<unsigned>(kWaves * rows * (D < 128 ? D : 128) * 4), static_cast<hipStream_t>(stream), a);
    return check_launch("paged_attention_kernel");
}

}  // extern "C"
