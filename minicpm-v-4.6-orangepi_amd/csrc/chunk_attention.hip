// chunk_attention.hip -- attention of chunks of new tokens over a paged cache, gfx950.
#include <algorithm>

#include "mixers.h"

namespace mcv {
namespace {

constexpr int kTile = 64;                        // tokens that are staged and taken at a time
constexpr int kWaves = 4;
constexpr int kRowsWave = 32;
constexpr int kRows = kWaves * kRowsWave;        // (token, head) rows of a workgroup
constexpr int kLeast = 4 * kTile;                // tokens of a part, at least
constexpr int kJoinRows = 16;                    // rows that a workgroup joins
constexpr int64_t kMaxLen = int64_t(1) << 30;    // tokens of one sequence
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kTopLog2 = 15.f;

struct ChunkArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    uint16_t* out;
    uint8_t* ws;
    int64_t q_row, q_head, k_page, k_head, v_page, v_head, table_row;
    int k_token, v_token, pages, page16, max_len, B, T, Hq, Hkv, group;
    uint32_t page16_inv;                         // ceil(2^32 / page16), page16 > 1
    float scale_log2;
    int slots;                                   // parts to cut for; 0: every tile of rows whole
    int64_t slot_bytes;
};

__host__ __device__ constexpr int64_t part_bytes(int64_t rows, int64_t D) { return rows * (D * 4 + 8); }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max2(float v) {          // over the two lanes of one column
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum2(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// What no kernel in flight writes, at an address that a whole wave shares: read through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
__device__ __forceinline__ scalar_ints as_scalar(const int32_t* p) { return (scalar_ints)reinterpret_cast<uintptr_t>(p); }

// ---------------------------------------------------------------- who does what --
struct Seq {
    int first, n, len;                           // first new row, new tokens, tokens in the cache
};
__device__ __forceinline__ Seq seq_of(const ChunkArgs& p, int b) {
    if (b >= p.B) return {0, 0, 0};
    auto row = [&](int i) {
        const int at = p.cu ? p.cu[i] : i * (p.T / p.B);
        return at < 0 ? 0 : at > p.T ? p.T : at;
    };
    const int first = row(b), n = row(b + 1) - first, len = p.lens[b];
    return {first, n < 0 ? 0 : n, len < 0 ? 0 : len > p.max_len ? p.max_len : len};
}
__device__ __forceinline__ int tiles_of(const ChunkArgs& p, const Seq& s) {
    return static_cast<int>((static_cast<int64_t>(s.n) * p.group + kRows - 1) / kRows);
}
// Tokens that the first i tiles of rows read, at most (of one cache head), and that tile i reads.
__device__ __forceinline__ int64_t reads_below(const ChunkArgs& p, const Seq& s, int64_t i) {
    const int64_t base = s.len > s.n ? s.len - s.n : 0, step = (kRows + p.group - 1) / p.group;
    return i * (base + kTile) + step * (i * (i + 1) / 2);
}
// Tiles of rows that have a part p > 0, which begins at token p S: the last ones.
__device__ __forceinline__ int tiles_with(const ChunkArgs& p, const Seq& s, int tiles, int64_t begin) {
    const int64_t x = begin - (s.len - s.n);     // the first new token that sees it
    return x <= 0 ? tiles : x >= s.n ? 0 : tiles - static_cast<int>(x * p.group / kRows);
}

__device__ __forceinline__ int wave_scan(int v) {
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const int u = __shfl_up(v, off, 64);
        v += static_cast<int>(threadIdx.x & 63) >= off ? u : 0;
    }
    return v;
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const int64_t u = __shfl_up(v, off, 64);
        v += static_cast<int>(threadIdx.x & 63) >= off ? u : 0;
    }
    return v;
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// The sequence that has this kernel's unit `me`, where sequence s has count(s, S) of them.
struct Place {
    Seq s;
    int b, unit;                                 // the unit's number in it
    int64_t read;                                // reads_below of all sequences before it
    int S;                                       // tokens of a part
};
template <class Count>
__device__ __forceinline__ bool find(const ChunkArgs& p, int me, Place& at, Count count) {
    const int lane = threadIdx.x & 63, span = (p.B + 63) / 64;
    Seq s = seq_of(p, lane);                     // (of span 1)
    auto reads = [&](const Seq& s) { return p.Hkv * reads_below(p, s, tiles_of(p, s)); };
    int64_t read = 0;
    if (span == 1) read = reads(s);
    else
        for (int i = 0; i < span; ++i) read += reads(seq_of(p, lane * span + i));
    int64_t read_upto = wave_scan(read);
    const int64_t total = lane_of(read_upto, 63);
    at.S = 0x40000000;
    if (p.slots) {
        const int64_t S = ((total + p.slots - 1) / p.slots + kTile - 1) / kTile * kTile;
        at.S = static_cast<int>(S < kLeast ? kLeast : S < 0x40000000 ? S : 0x40000000);
    }
    int units = 0;
    if (span == 1) units = count(s, at.S);
    else
        for (int i = 0; i < span; ++i) units += count(seq_of(p, lane * span + i), at.S);
    int upto = wave_scan(units);
    unsigned long long past = __ballot(upto > me);
    if (!past) return false;
    int l = __builtin_ctzll(past), before = 0;
    at.read = 0;
    auto go_to = [&]() {
        if (l) {
            before += __builtin_amdgcn_readlane(upto, l - 1);
            at.read += lane_of(read_upto, l - 1);
        }
    };
    go_to();
    at.b = l * span;
    while (span > 1) {                           // the chosen lane's sequences, 64 at a time
        s = seq_of(p, at.b + lane);
        upto = wave_scan(count(s, at.S));
        read_upto = wave_scan(reads(s));
        past = __ballot(before + upto > me);
        l = past ? __builtin_ctzll(past) : 64;
        go_to();
        at.b += l;
        if (past) break;
        if (at.b >= p.B) return false;           // (lengths that changed meanwhile)
    }
    at.s = {__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.len, l)};
    at.unit = me - before;
    return true;
}

// Where part i of a tile lies in the workspace. `read`: reads_below of all tiles before it. Part i has the id w0 + i, w0
// the part of an even cut of all reads that the tile's first falls into; a part 0 has slot 2 id + 1, others 2 id: ids of
// one tile are its own but for its last, which may be the next tile's first.
__device__ __forceinline__ int64_t slot_of(int64_t read, int S, int i) {
    const int64_t id = read / S + i;
    return i == 0 ? 2 * id + 1 : 2 * id;
}

__device__ __forceinline__ uint2 halves(const float4_t& v, float by, bool none) {
    uint16_t r[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) r[x] = f2h(none ? 0.f : v[x] * by);
    return make_uint2(r[0] | (static_cast<uint32_t>(r[1]) << 16), r[2] | (static_cast<uint32_t>(r[3]) << 16));
}

// ---------------------------------------------------------------------- a part --
template <int D>
__global__ __launch_bounds__(64 * kWaves, 1) void chunk_attention_kernel(ChunkArgs p) {
    constexpr int KS = D / 16;                   // steps of the score product
    constexpr int MB = D / 32;                   // blocks of 32 d
    constexpr int RC = D / 8;                    // 16-byte chunks of a row
    constexpr int RPI = 64 / RC;                 // rows that a wave's copy takes
    constexpr int CP = 16 / RPI;                 // copies of 16 rows
    constexpr int ROW = 2 * D;                   // bytes
    constexpr int KM = RC < 16 ? RC - 1 : 15;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];      // [2][K, V][kTile][D]
    const int lane = threadIdx.x & 63, c = lane & 31, j = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Place at;
    auto units = [&](const Seq& s, int S) {
        const int tiles = tiles_of(p, s), base = s.len - s.n, parts = (s.len + S - 1) / S;
        const int whole = base > 0 ? base / S : 0;
        int64_t sum = static_cast<int64_t>(tiles) * (1 + whole);
        for (int i = whole + 1; i < parts; ++i) sum += tiles_with(p, s, tiles, static_cast<int64_t>(i) * S);
        return static_cast<int>(sum) * p.Hkv;
    };
    if (!find(p, blockIdx.x, at, units)) return;
    const int rows = at.s.n * p.group, tiles = tiles_of(p, at.s), base = at.s.len - at.s.n;
    const int hk = at.unit % p.Hkv;
    int part, tile;
    {
        const int v = at.unit / p.Hkv, whole = base > 0 ? base / at.S : 0;
        part = v / tiles;
        int i = v - part * tiles;
        if (part > whole) {
            part = whole + 1;
            i = v - tiles * (1 + whole);
            for (;;) {
                const int have = tiles_with(p, at.s, tiles, static_cast<int64_t>(part) * at.S);
                if (have == 0) return;           // (lengths that changed meanwhile)
                if (i < have) break;
                i -= have;
                ++part;
            }
        }
        tile = tiles - 1 - i;                    // (the ones that read most first)
    }
    const int row0 = tile * kRows, last_row = (row0 + kRows < rows ? row0 + kRows : rows) - 1;
    auto seen_by = [&](int row) {                // tokens that a row sees
        const int n = base + row / p.group + 1;
        return n < 0 ? 0 : n;
    };
    const int end = seen_by(last_row), parts = end <= at.S ? 1 : (end + at.S - 1) / at.S;
    const int t_begin = part * at.S, t_end = part < parts - 1 ? t_begin + at.S : end;

    const int wrow = row0 + wave * kRowsWave;
    const bool mine = wrow < rows;               // this wave has rows
    const int row = wrow + c < rows ? wrow + c : rows - 1;
    const int seen = seen_by(row), least = mine ? seen_by(wrow) : 0;
    const int most = mine ? seen_by(wrow + kRowsWave - 1 < rows ? wrow + kRowsWave - 1 : rows - 1) : 0;
    const int token = row / p.group, head = hk * p.group + row - token * p.group;
    const uint16_t* qr = p.q + static_cast<int64_t>(at.s.first + token) * p.q_row + head * p.q_head;
    half8_t q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const half8_t*>(qr + 16 * s + 8 * j);

    const scalar_ints table = as_scalar(p.table + at.b * p.table_row);
    const uint16_t* kh = p.k + hk * p.k_head;
    const uint16_t* vh = p.v + hk * p.v_head;
    // Rows of 16 tokens from t on: their page's number (-1: not there, or past the end) and first row in it.
    auto place = [&](int t, int& page, int& prow) {
        const uint32_t t16 = static_cast<uint32_t>(t) >> 4;
        uint32_t i = t16;
        prow = 0;
        if (p.page16 > 1) {
            i = __umulhi(t16, p.page16_inv);     // one too many at most
            int r = static_cast<int>(t16 - i * p.page16);
            if (r < 0) --i, r += p.page16;
            prow = 16 * r;
        }
        page = t < t_end ? table[i] : -1;
        page = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(page) < static_cast<uint32_t>(p.pages) ? page : -1);
    };
    // 16 rows of K or V: as they lie, but a row's chunks in an order of its own, so that reads of a column meet other banks.
    const int lr = lane / RC, lc = lane % RC;
    auto copy16 = [&](const uint16_t* base, int64_t page_stride, int token_stride, int page, int prow, uint8_t* to, bool of_v) {
        const uint16_t* from = base + (page < 0 ? 0 : page) * page_stride + static_cast<int64_t>(page < 0 ? 0 : prow) * token_stride;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(from), 0, 2 * (15 * token_stride + D), 0x00020000);
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int at_row = i * RPI + lr;
            const int turn = of_v ? (RC < 16 ? 4 * ((at_row >> 1) & 1) : 4 * (at_row & 3)) : at_row & KM;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + i * 1024), 16, 2 * lr * token_stride + 16 * (lc ^ turn),
                                                     2 * i * RPI * token_stride, 0, 0);
        }
    };
    uint32_t gone[2] = {0, 0};                   // groups of 16 tokens that are not there, of the tiles in the two buffers
    auto stage = [&](int t, int buf) {
        uint8_t* to = lds + buf * 2 * kTile * ROW + wave * 16 * ROW;
        uint32_t none = 0;
        int page = -1, prow = 0;
#pragma unroll
        for (int x = 0; x < kTile / 16; ++x) {
            int pg, pr;
            place(t + 16 * x, pg, pr);
            none |= (pg < 0 ? 1u : 0u) << x;
            if (x == wave) page = pg, prow = pr;
        }
        gone[buf] = none;
        copy16(kh, p.k_page, p.k_token, page, prow, to, false);
        copy16(vh, p.v_page, p.v_token, page, prow, to + kTile * ROW, true);
    };

    float4_t zero4 = {0, 0, 0, 0};
    float16_t acc[MB] = {};
    float m = -INFINITY, l = 0.f;
    if (t_begin < t_end) stage(t_begin, 0);
    int buf = 0;
    for (int t = t_begin; t < t_end; t += kTile, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint8_t* const kl = lds + buf * 2 * kTile * ROW;
        uint8_t* const vl = kl + kTile * ROW;
        if (t + kTile > t_end || gone[buf]) {
            // what lies past the end or is not there may be NaN, whose product with a weight of zero is no zero
            for (int i = lane; i < 16 * RC; i += 64) {
                const int r = 16 * wave + i / RC;
                if (t + r >= t_end || (gone[buf] >> wave & 1)) *reinterpret_cast<float4_t*>(vl + r * ROW + 16 * (i % RC)) = zero4;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (t + kTile < t_end) stage(t + kTile, buf ^ 1);
        if (!mine || t >= most) continue;
        float16_t s[2] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const half8_t k = *reinterpret_cast<const half8_t*>(kl + (32 * h + c) * ROW + 16 * ((2 * x + j) ^ (c & KM)));
                s[h] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[x], s[h], 0, 0, 0);
            }
        const bool all = t + kTile <= least && gone[buf] == 0;
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float v = s[h][i] * p.scale_log2;
                if (!all && (t + 32 * h + 8 * (i / 4) + 4 * j + i % 4 >= seen || (gone[buf] >> (2 * h + i / 8) & 1))) v = -INFINITY;
                s[h][i] = v;
                mx = fmaxf(mx, v);
            }
        mx = fmaxf(max2(mx), m);
        if (__any(mx > m)) {
            const float keep = m == -INFINITY ? 0.f : exp2_of(m - mx);
            l *= keep;
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b][i] *= keep;
            m = mx;
        }
        const float from = m == -INFINITY ? 0.f : m - kTopLog2;
        half8_t w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = exp2_of(s[x / 2][8 * (x & 1) + i] - from);
                l += e;
                w[x][i] = static_cast<_Float16>(e);
            }
        const int vrow = 4 * j + ((lane & 15) >> 2);
        const int vturn = RC < 16 ? 4 * ((vrow >> 1) & 1) : 4 * (vrow & 3);
        const int vcol = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        typedef __fp16 half4_b __attribute__((ext_vector_type(4)));
        typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                half8_t a;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint8_t* from = vl + (16 * x + 8 * y + vrow) * ROW + 16 * ((4 * b + vcol) ^ vturn) + 8 * (lane & 1);
                    const auto r = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) half4_b*)(from)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[4 * y + e] = r[e];
                }
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, w[x], acc[b], 0, 0, 0);
            }
    }
    if (!mine) return;
    l = sum2(l);

    // acc[b][i]: d = 32 b + 8 (i / 4) + 4 j + i % 4 of this lane's row
    bool odd = !(fabsf(l) < INFINITY);
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd |= !(fabsf(acc[b][i]) < INFINITY);
    const unsigned long long odds = __ballot(odd);
    const uint32_t bad = static_cast<uint32_t>(odds) | static_cast<uint32_t>(odds >> 32);
    float* slot = nullptr;
    const int64_t read = at.read + p.Hkv * reads_below(p, at.s, tile) + hk * (reads_below(p, at.s, tile + 1) - reads_below(p, at.s, tile));
    if (parts > 1) slot = reinterpret_cast<float*>(p.ws + slot_of(read, at.S, part) * p.slot_bytes);
    const int slot_rows = static_cast<int>(p.slot_bytes / (D * 4 + 8));
    auto out_row = [&](int r) {
        const int tk = r / p.group;
        return p.out + (static_cast<int64_t>(at.s.first + tk) * p.Hq + hk * p.group + r - tk * p.group) * D;
    };
    if (wrow + c < rows && !(bad >> c & 1)) {
        if (slot) {
            float* to = slot + static_cast<int64_t>(wave * kRowsWave + c) * D;
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4_t*>(to + 32 * b + 8 * i + 4 * j) = float4_t{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]};
            if (j == 0) *reinterpret_cast<float2*>(slot + static_cast<int64_t>(slot_rows) * D + 2 * (wave * kRowsWave + c)) = make_float2(m, l);
        } else {
            const float by = l > 0.f ? 1.0f / l : 0.f;
            uint16_t* to = out_row(wrow + c);
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint2*>(to + 32 * b + 8 * i + 4 * j) =
                        halves(float4_t{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]}, by, l == 0.f);
        }
    }
    // Rows that are not finite, one at a time and token by token: an infinity or NaN in V reaches the rows that see its
    // token, where above it reaches every row of its tile (zero weights times it are NaN).
    for (uint32_t left = bad; left; left &= left - 1) {
        const int r = __builtin_ctz(left), rr = wrow + r;
        if (rr >= rows) break;
        constexpr int E = D / 64;
        const int tk = rr / p.group;
        const uint16_t* from = p.q + static_cast<int64_t>(at.s.first + tk) * p.q_row + (hk * p.group + rr - tk * p.group) * p.q_head + E * lane;
        float qv[E], sum[E];
#pragma unroll
        for (int e = 0; e < E; ++e) qv[e] = h2f(from[e]), sum[e] = 0.f;
        const int upto = seen_by(rr) < t_end ? seen_by(rr) : t_end;
        float top = -INFINITY, tot = 0.f;
        auto tokens = [&](auto use) {
            for (int t16 = t_begin; t16 < upto; t16 += 16) {
                int page, prow;
                place(t16, page, prow);
                for (int x = 0; page >= 0 && x < 16 && t16 + x < upto; ++x) {
                    const uint16_t* k = kh + page * p.k_page + static_cast<int64_t>(prow + x) * p.k_token + E * lane;
                    float dot = 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) dot = fmaf(qv[e], h2f(k[e]), dot);
                    use(wave_butterfly(dot, [](float a, float b) { return a + b; }) * p.scale_log2,
                        vh + page * p.v_page + static_cast<int64_t>(prow + x) * p.v_token + E * lane);
                }
            }
        };
        tokens([&](float s, const uint16_t*) { top = fmaxf(top, s); });
        const float less = top == -INFINITY ? 0.f : top - kTopLog2;
        tokens([&](float s, const uint16_t* v) {
            const float w = exp2_of(s - less);
            tot += w;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] = fmaf(w, h2f(v[e]), sum[e]);
        });
        const float by = tot > 0.f ? 1.0f / tot : (tot == 0.f ? 0.f : tot);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (slot) slot[static_cast<int64_t>(wave * kRowsWave + r) * D + E * lane + e] = sum[e];
            else out_row(rr)[E * lane + e] = f2h(tot == 0.f ? 0.f : sum[e] * by);
        }
        if (slot && lane == 0) *reinterpret_cast<float2*>(slot + static_cast<int64_t>(slot_rows) * D + 2 * (wave * kRowsWave + r)) = make_float2(top, tot);
    }
}

// ------------------------------------------------------------------- the parts' sum --
template <int D>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs p) {
    Place at;
    auto cut = [&](const Seq& s, int S) { return s.len > S ? tiles_with(p, s, tiles_of(p, s), S) * p.Hkv : 0; };
    if (!find(p, blockIdx.x, at, cut)) return;
    const int rows = at.s.n * p.group, tiles = tiles_of(p, at.s), base = at.s.len - at.s.n;
    const int hk = at.unit % p.Hkv, tile = tiles - 1 - at.unit / p.Hkv;
    const int row0 = tile * kRows, last_row = (row0 + kRows < rows ? row0 + kRows : rows) - 1;
    const int end = base + last_row / p.group + 1, parts = (end + at.S - 1) / at.S;
    const int64_t read = at.read + p.Hkv * reads_below(p, at.s, tile) + hk * (reads_below(p, at.s, tile + 1) - reads_below(p, at.s, tile));
    const int slot_rows = static_cast<int>(p.slot_bytes / (D * 4 + 8));
    for (int i = threadIdx.x; i < kJoinRows * D / 4; i += 256) {
        const int r = blockIdx.y * kJoinRows + i / (D / 4), d = i % (D / 4) * 4, rr = row0 + r;
        if (rr > last_row) break;
        float4_t sum = {0, 0, 0, 0};
        float top = -INFINITY, tot = 0.f;
        constexpr int kBatch = 8;                // loads of a batch go out together
        for (int u0 = 0; u0 < parts; u0 += kBatch) {
            float4_t o[kBatch];
            float2 st[kBatch];
            float most = top;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const float* slot = reinterpret_cast<const float*>(p.ws + slot_of(read, at.S, u0 + u < parts ? u0 + u : parts - 1) * p.slot_bytes);
                o[u] = *reinterpret_cast<const float4_t*>(slot + static_cast<int64_t>(r) * D + d);
                st[u] = *reinterpret_cast<const float2*>(slot + static_cast<int64_t>(slot_rows) * D + 2 * r);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) most = fmaxf(most, st[u].x);
            const float keep = top == -INFINITY ? 0.f : exp2_of(top - most);
            tot *= keep;
            sum *= keep;
            top = most;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (u0 + u >= parts) continue;
                const float by = st[u].x == -INFINITY ? 0.f : exp2_of(st[u].x - top);
                tot = fmaf(st[u].y, by, tot);
#pragma unroll
                for (int x = 0; x < 4; ++x) sum[x] = fmaf(o[u][x], by, sum[x]);
            }
        }
        const int tk = rr / p.group;
        const float by = tot > 0.f ? 1.0f / tot : (tot == 0.f ? 0.f : tot);
        *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(at.s.first + tk) * p.Hq + hk * p.group + rr - tk * p.group) * D + d) = halves(sum, by, tot == 0.f);
    }
}

// Parts to cut for, of rows that read up to `most` tokens: what the chip holds at once.  0: nothing to cut.
int choose_slots(int64_t most, int64_t D) { return most <= kLeast ? 0 : D == 256 ? 256 : 512; }
int64_t slot_rows_of(int64_t T, int64_t group) { return std::min<int64_t>(kRows, T * group); }
int64_t split_bytes(int64_t slots, int64_t rows, int64_t D) { return slots == 0 ? 0 : 2 * (slots + 2) * part_bytes(rows, D); }

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int64_t mcv_paged_attention_chunk_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seq_len) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || T > 0x7fffffff / Hq || D <= 0 || max_seq_len < 0) return 0;
    return split_bytes(choose_slots(std::min(max_seq_len, kMaxLen), D), slot_rows_of(T, Hq / Hkv), D);
}

int mcv_paged_attention_chunk(const void* q, int64_t q_row, int64_t q_head, const void* k_cache, int64_t k_page,
                              int64_t k_token, int64_t k_head, const void* v_cache, int64_t v_page, int64_t v_token,
                              int64_t v_head, int64_t pages, int64_t page_size, const void* block_table,
                              int64_t table_row, int64_t table_width, const void* seq_lens, int64_t max_seq_len,
                              const void* cu_seqlens, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, double scale,
                              void* out, void* workspace, int64_t workspace_bytes, mcv_stream_t stream) {
    const char* who = "paged_attention_chunk";
    if (!q || !k_cache || !v_cache || !block_table || !seq_lens || !out) return fail(MCV_ERR_INVALID_ARG, "%s: null pointer", who);
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || T > 0x7fffffff / Hq || B > 0x7fffffff / Hq || (!cu_seqlens && T % B != 0))
        return fail(MCV_ERR_SHAPE, "%s: bad shape B=%lld T=%lld Hq=%lld Hkv=%lld", who, (long long)B, (long long)T, (long long)Hq, (long long)Hkv);
    if (D != 64 && D != 128 && D != 256) return fail(MCV_ERR_SHAPE, "%s: D must be 64, 128 or 256 (D=%lld)", who, (long long)D);
    if (page_size <= 0 || page_size % 16 != 0 || page_size > (1 << 20))
        return fail(MCV_ERR_SHAPE, "%s: page_size must be a multiple of 16 (page_size=%lld)", who, (long long)page_size);
    if (pages <= 0 || pages > 0x7fffffff || table_width <= 0 || max_seq_len < 0)
        return fail(MCV_ERR_SHAPE, "%s: bad cache pages=%lld table_width=%lld max_seq_len=%lld", who, (long long)pages, (long long)table_width,
                    (long long)max_seq_len);
    for (int64_t s : {q_row, q_head, k_page, k_token, k_head, v_page, v_token, v_head, table_row})
        if (s < 0) return fail(MCV_ERR_SHAPE, "%s: negative stride", who);
    if (!chunked16(q, {q_row, q_head}) || !chunked16(k_cache, {k_page, k_token, k_head}) || !chunked16(v_cache, {v_page, v_token, v_head}) ||
        !chunked16(out, {}))
        return fail(MCV_ERR_UNSUPPORTED, "%s: pointers must be 16-byte aligned, strides multiples of 8 elements", who);
    if (k_token > (1 << 25) || v_token > (1 << 25)) return fail(MCV_ERR_UNSUPPORTED, "%s: tokens of one page too far apart", who);
    int rc = require_device();
    if (rc != MCV_OK) return rc;
    // (width counted in pages first: width * page_size could pass 64 bits)
    const int64_t held = table_width > kMaxLen / page_size ? kMaxLen : table_width * page_size;
    const int64_t most = max_seq_len < held ? max_seq_len : held;
    const int64_t group = Hq / Hkv, rows = slot_rows_of(T, group);
    const int64_t tiles = std::min(T * group / kRows + B, T * group);
    int slots = choose_slots(most, D);
    if (slots && (!workspace || workspace_bytes < split_bytes(slots, rows, D))) slots = 0;
    if (slots && reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return fail(MCV_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", who);
    if (tiles * Hkv + slots > 0x7fffffff) return fail(MCV_ERR_SHAPE, "%s: too many rows B=%lld T=%lld Hq=%lld", who, (long long)B, (long long)T, (long long)Hq);
    const uint32_t page16 = static_cast<uint32_t>(page_size / 16);
    const ChunkArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache),
                      static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(seq_lens), static_cast<const int32_t*>(cu_seqlens),
                      static_cast<uint16_t*>(out), static_cast<uint8_t*>(workspace), q_row, q_head, k_page, k_head, v_page, v_head, table_row,
                      static_cast<int>(k_token), static_cast<int>(v_token), static_cast<int>(pages), static_cast<int>(page16), static_cast<int>(most),
                      static_cast<int>(B), static_cast<int>(T), static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(group),
                      page16 > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + page16 - 1) / page16) : 0, static_cast<float>(scale) * kLog2e,
                      slots, part_bytes(rows, D)};
    const auto s = static_cast<hipStream_t>(stream);
    auto fn = D == 64 ? chunk_attention_kernel<64> : D == 128 ? chunk_attention_kernel<128> : chunk_attention_kernel<256>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(tiles * Hkv + slots)), dim3(64 * kWaves), static_cast<unsigned>(4 * kTile * 2 * D), s, a);
    rc = check_launch("chunk_attention_kernel");
    if (rc != MCV_OK || !slots) return rc;
    auto join = D == 64 ? chunk_join_kernel<64> : D == 128 ? chunk_join_kernel<128> : chunk_join_kernel<256>;
    hipLaunchKernelGGL(join, dim3(static_cast<unsigned>(std::min<int64_t>(tiles * Hkv, slots)), static_cast<unsigned>(ceil_div(rows, kJoinRows))), dim3(256), 0, s, a);
    return check_launch("chunk_join_kernel");
}

}  // extern "C"
