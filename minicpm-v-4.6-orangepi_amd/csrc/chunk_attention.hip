// chunk_attention.hip -- attention of chunks of new tokens over a paged cache, gfx950.
//
//   out[row][h] = sum_t w_t V[t] / sum_t w_t,  w_t = exp(scale q[row][h] . K[t] - max),  t up to the row's own place
//
// Rows and heads. The heads of a group read the same K and V: a sequence's (token, head) pairs of one cache head, token by
// token, are the rows of one matrix, of which a workgroup has a tile of 128, a wave 32. So 8 heads over 2 and 32 over 8 fill
// the matrix cores from 8 or 32 tokens on, and one token's heads share one read of the cache.
//
// A wave's step, 32 tokens: S^T = K q^T on 32x32x16 matrix instructions, q in registers from the start, K from LDS; a lane then
// has 16 scores of one row, so that a row's maximum and sum are in two lanes and the weights, rounded, are where the second
// product wants them: out^T += V^T w^T, V read from LDS transposed. Weights are fp16, the operand type of the matrix cores:
// half a step of 2^-11 each, and the sum that divides them is of the rounded ones. Scores, maxima and sums are in 32 bits. The
// reference that weights are taken against is a whole power of two and moves only when a row's largest grows past 2^6 times
// what it was set for: few rows ever scale what they have.
//
// K and V come to LDS by copies that pass no register, 32 tokens (heads of 256) or 64 at a time, in two buffers: the next
// tile's are on their way while one is taken. Rows of LDS have their chunks in orders of their own, so that reads meet
// other banks (counted: conflicts in 0.7% of LDS cycles). Operands of the products are read three ahead.
//
// Parts. All reads of a call are cut evenly, on the device and from the lengths alone, into as many parts as workgroups that
// the chip holds at once (two a CU); a unit is a tile's part. Up to four parts are joined by the last of them to arrive, more
// by a launch that follows. Partial sums are 128 KiB a tile of 128 rows of 256, what 128 tokens of cache are: but for few tiles
// no part is smaller than that.
//
// What bounds it, heads 8/2 of 256. 8192 new tokens 278 to 303 us by the card's clock, 0.91 to 0.99 PFLOP/s (a large matrix
// product 1.14 to 1.31): the matrix cores are busy in 51 to 58% of cycles, LDS in 28 to 32%, and the clock falls to 1.7 GHz; what is left
// is the softmax between the products, which two waves a SIMD hide by half. 512 over 100000 412 to 450 us: 61% at 1.5 GHz, the
// copies cost a fifth of it. 32 sequences' 5 over up to 9000 46.3 us, 3.1 TB/s: 33 of them at the cache's 145 MB, then the
// join. Small calls are latencies: 24 over 1100 14.7 us, 1100 over none 27.5: the lengths, the table and the first tile, three
// loads that wait for one another, 4 us; 1.3 us a step of 32 tokens; a part written and read 2 and 4 us.
//
// Tried and not better: 64 rows a wave (halves what LDS reads; registers spill), two waves on the same rows, 64 tokens of 256 at
// a time with one workgroup a CU (8192: 394 us), 256 rows and one workgroup a CU (1% better here, 10% worse for mixed lengths), copies spread over the products
// (307), longest parts first (303), four reads ahead (the same), the tile after the next fetched into L2 (321), workgroups of the
// join over several tiles (the same).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "mixers.h"

namespace mcv {
namespace {

constexpr int kTile = 64;                        // a part has whole ones of so many tokens
constexpr int kLeast = 2 * kTile;                // tokens of a part, at least, but for few tiles
constexpr int kNearLog2 = 2;                     // 1 << kNearLog2 units side by side on one XCD
constexpr int64_t kMaxLen = int64_t(1) << 30;    // tokens of one sequence
constexpr float kLog2e = 1.44269504088896340736f;
// A row's weights are 2^(s - m). m is a whole number, so that what it once stood for is brought to another by an exact product; it
// begins kTop below a row's largest score and moves only when one passes it by kMost: the weights end at 2^15, below fp16's
// 65504, and the row's largest begins above 2^8: those that are lost, below 2^-25, are less than 2^-33 of it. From kFar on,
// where 32 bits end to hold every whole number, scores are rounded to 32 bits before m is taken from them, and m is the largest.
constexpr float kMost = 15.f, kTop = 9.f, kFar = 8388608.f;

struct ChunkArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* cu;
    const int32_t* positions;                    // int64 [T], or null
    uint16_t* out;
    uint8_t* ws;
    int64_t q_row, q_head, k_page, k_head, v_page, v_head, table_row;
    int k_token, v_token, pages, page16, max_len, B, T, Hq, Hkv, group;
    uint32_t page16_inv, group_inv;              // ceil(2^32 / n), n > 1
    float scale_log2;                            // above zero: a score of -inf stays one
    float q_by;                                  // 1, -1 or 0: the scale's sign
    int slots_log2;                              // parts to cut for; -1: every tile of rows whole
    int least;                                   // tokens of a part, at least
    int64_t slot_bytes;
};

constexpr int kFan = 4;                          // parts of a tile that the last of them to arrive joins; where there are more, a launch of its own does
constexpr int64_t kCounterBytes = 8192;          // a counter for each part

// Bytes of a wave's part: a lane's sums, and its reference exponent and sum of weights, as they are in registers.
__host__ __device__ constexpr int64_t part_bytes(int64_t D) { return 64 * (2 * D + 8); }

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
    int first, n, len, base;                     // first new row, new tokens (below zero: cu_seqlens falls), tokens in the cache, of them before the first new one
};
template <class Ints>
__device__ __forceinline__ Seq seq_of(const ChunkArgs& p, int b, Ints lens, Ints cu, Ints positions) {
    const int at = b < p.B ? b : p.B - 1;        // (no branch: several are loaded at once)
    int first, next;
    const int held = lens[at];
    if (cu) first = cu[at], next = cu[at + 1];
    else first = at * (p.T / p.B), next = first + p.T / p.B;
    auto inside = [](int v, int most) { return v < 0 ? 0 : v > most ? most : v; };
    first = inside(first, p.T);
    next = inside(next, p.T);
    Seq s{first, b < p.B ? next - first : 0, inside(held, p.max_len), 0};
    s.base = s.len - s.n;
    if (positions) {                             // (the first new token sees the last there is, at most)
        const int64_t row = 2 * static_cast<int64_t>(first < p.T ? first : p.T - 1);
        const int lo = positions[row], hi = positions[row + 1], most = s.len > 0 ? s.len - 1 : 0;
        s.base = hi < 0 ? 0 : hi > 0 || static_cast<uint32_t>(lo) > static_cast<uint32_t>(most) ? most : lo;
    }
    return s;
}
__device__ __forceinline__ Seq seq_of(const ChunkArgs& p, int b) { return seq_of(p, b, p.lens, p.cu, p.positions); }
__device__ __forceinline__ int token_of(const ChunkArgs& p, int row) {         // row / group
    if (p.group == 1) return row;
    int t = static_cast<int>(__umulhi(static_cast<uint32_t>(row), p.group_inv));      // one too many at most
    if (t * static_cast<int64_t>(p.group) > row) --t;
    return t;
}
// Tokens that a new one sees.
__device__ __forceinline__ int sees(const Seq& s, int token) {
    if (token >= s.len - s.base) return s.len;
    const int n = s.base + token + 1;
    return n < 0 ? 0 : n;
}
// R: rows of a tile.
template <int R>
__device__ __forceinline__ int tiles_of(const ChunkArgs& p, const Seq& s) {
    return s.n < 0 ? 0 : static_cast<int>((static_cast<int64_t>(s.n) * p.group + R - 1) / R);
}
// Tokens that the first i tiles of rows read, at most (of one cache head).
template <int R>
__device__ __forceinline__ int64_t reads_below(const ChunkArgs& p, const Seq& s, int i) {
    const int base = s.base > 0 ? s.base : 0, step = token_of(p, R + p.group - 1);
    return static_cast<int64_t>(i) * (base + kTile) + step * (static_cast<int64_t>(i) * (i + 1) / 2);
}
// Tiles of rows that have a part p > 0, which begins at token p S: the last ones.
template <int R>
__device__ __forceinline__ int tiles_with(const ChunkArgs& p, const Seq& s, int tiles, int64_t begin) {
    const int64_t x = begin - s.base;            // the first new token that sees it
    return x <= 0 ? tiles : x >= s.n ? 0 : tiles - static_cast<int>(x * p.group / R);
}

__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);       // rows of 16: one to the right, two, four, eight
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);       // a row's last lane to the next row
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);       // lane 31 to the upper half
    return v;
}
// Of values below 2^50: 25 bits at a time, whose sums of 64 lanes fit in 32.
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    const int lo = wave_scan(static_cast<int>(v & 0x1ffffff)), hi = wave_scan(static_cast<int>(v >> 25));
    return (static_cast<int64_t>(hi) << 25) + static_cast<uint32_t>(lo);
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

// The sequence that has this kernel's unit `me`, where sequence s has count(s, S) of them. A lane has a sequence, or, where
// there are more than 64, a thread of the workgroup several, which then meet in LDS (4096 sequences' tokens over 200 each, heads
// 8/2 of 256: 520 us, 933 with a wave's lanes alone). False in every thread: there is no such unit. Nor is there any where
// cu_seqlens falls: rows would have two sequences, and more units than workgroups.
struct Place {
    Seq s;
    int b, unit;                                 // the unit's number in it
    int64_t read;                                // reads_below of all sequences before it
    int S;                                       // tokens of a part
};
template <int R, class Count>
__device__ __forceinline__ bool search(const ChunkArgs& p, int me, Place& at, Count count) {
    auto part_of = [&](int64_t total) {
        if (p.slots_log2 < 0) return 0x40000000;
        const int64_t S = (((total - 1) >> p.slots_log2) + kTile) / kTile * kTile;
        return static_cast<int>(S < p.least ? p.least : S < 0x40000000 ? S : 0x40000000);
    };
    auto reads = [&](const Seq& s) { return p.Hkv * reads_below<R>(p, s, tiles_of<R>(p, s)); };
    at.read = 0;
    at.b = 0;
    if (p.B == 1) {                              // (nothing to look for)
        at.s = seq_of(p, 0, as_scalar(p.lens), as_scalar(p.cu), as_scalar(p.positions));
        at.unit = me;
        at.S = part_of(reads(at.s));
        return me < count(at.s, at.S);
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    // of the 64 sequences from at.b on, whose units begin at `before`; false: it is none of theirs
    auto look = [&](const Seq& s, int upto, int64_t read_upto) {
        const unsigned long long past = __ballot(before + upto > me);
        const int l = past ? __builtin_ctzll(past) : 64;
        if (l) {
            before += __builtin_amdgcn_readlane(upto, l - 1);
            at.read += lane_of(read_upto, l - 1);
        }
        at.b += l;
        if (!past) return false;
        at.s = {__builtin_amdgcn_readlane(s.first, l), __builtin_amdgcn_readlane(s.n, l), __builtin_amdgcn_readlane(s.len, l),
                __builtin_amdgcn_readlane(s.base, l)};
        at.unit = me - before;
        return true;
    };
    if (p.B <= 64) {
        const Seq s = seq_of(p, lane);
        if (__any(s.n < 0)) return false;
        const int64_t read_upto = wave_scan(reads(s));
        at.S = part_of(lane_of(read_upto, 63));
        return look(s, wave_scan(count(s, at.S)), read_upto);
    }
    constexpr int kWaves = 4;
    __shared__ int64_t wave_reads[kWaves];
    __shared__ int wave_units[kWaves], falls[kWaves], owner[2];
    __shared__ int64_t owner_read;
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), span = (p.B + 64 * kWaves - 1) / (64 * kWaves);
    int64_t read = 0;
    bool fall = false;
#pragma unroll 1
    for (int i = 0; i < span; ++i) {
        const Seq s = seq_of(p, t * span + i);
        read += reads(s);
        fall |= s.n < 0;
    }
    const int64_t read_upto = wave_scan(read);
    const bool falling = __any(fall);
    if (lane == 63) wave_reads[wave] = read_upto, falls[wave] = falling;
    __syncthreads();
    int64_t total = 0;
    int any = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += wave_reads[w], any |= falls[w];
    at.S = part_of(lane_of(total, 0));
    int units = 0;
#pragma unroll 1
    for (int i = 0; i < span; ++i) units += count(seq_of(p, t * span + i), at.S);
    const int upto = wave_scan(units);
    if (lane == 63) wave_units[wave] = upto;
    __syncthreads();
    int w = 0;                                   // the wave that has it
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
        const int its = __builtin_amdgcn_readfirstlane(wave_units[x]);
        if (w == x && before + its <= me) {
            before += its;
            at.read += lane_of(wave_reads[x], 0);
            ++w;
        }
    }
    if (__builtin_amdgcn_readfirstlane(any) || w == kWaves) return false;
    if (w == wave) {
        const int l = __builtin_ctzll(__ballot(before + upto > me));
        const int its = l ? __builtin_amdgcn_readlane(upto, l - 1) : 0;
        const int64_t below = l ? lane_of(read_upto, l - 1) : 0;
        owner[0] = (64 * w + l) * span;
        owner[1] = before + its;
        owner_read = at.read + below;
    }
    __syncthreads();
    at.b = __builtin_amdgcn_readfirstlane(owner[0]);
    before = __builtin_amdgcn_readfirstlane(owner[1]);
    at.read = lane_of(owner_read, 0);
    while (at.b < p.B) {                         // the chosen thread's sequences, 64 at a time
        const Seq s = seq_of(p, at.b + lane);
        if (look(s, wave_scan(count(s, at.S)), wave_scan(reads(s)))) return true;
    }
    return false;                                // (lengths that changed meanwhile)
}

template <int R, class Count>
__device__ __forceinline__ bool find(const ChunkArgs& p, int me, Place& at, Count count) {
    if (!__builtin_amdgcn_readfirstlane(search<R>(p, me, at, count))) return false;
    auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    at = {{one(at.s.first), one(at.s.n), one(at.s.len), one(at.s.base)}, one(at.b), one(at.unit), lane_of(at.read, 0), one(at.S)};
    return true;
}

// The number of the unit that workgroup b takes. Workgroup b runs on XCD b % 8: runs of `near` units, which read the same K
// and V, go to one XCD, whose L2 they share; every other round of eight runs goes to them in reverse, as the first of a
// sequence read most. Runs of four against single units, 8192 new tokens 300, 310 us (mixed lengths of 128 86.9, 85.4).
__device__ __forceinline__ int unit_of(int b) {
    const int x = b & 7, i = (b >> 3) & ((1 << kNearLog2) - 1), round = b >> (3 + kNearLog2);
    return (((round << 3) + (round & 1 ? 7 - x : x)) << kNearLog2) + i;
}

// Where part i of a tile lies in the workspace. `read`: reads_below of all tiles before it. Part i has the id w0 + i, w0
// the part of an even cut of all reads that the tile's first falls into; a part 0 has slot 2 id + 1, others 2 id: ids of
// one tile are its own but for its last, which may be the next tile's first. (The quotient in 64-bit floating point, which
// finds the whole number of any that the workspace is large enough for, and in a tenth of an integer division's time.)
template <int R>
__device__ __forceinline__ int first_id(const ChunkArgs& p, const Place& at, int tile, int hk) {
    const int64_t here = reads_below<R>(p, at.s, tile), read = at.read + p.Hkv * here + hk * (reads_below<R>(p, at.s, tile + 1) - here);
    return __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<double>(read) / static_cast<double>(at.S)));
}
__device__ __forceinline__ uint8_t* slot_of(const ChunkArgs& p, int w0, int i) { return p.ws + kCounterBytes + (2 * (w0 + i) + (i == 0)) * p.slot_bytes; }

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

// The page of the 16 tokens from 16 t16 on (-1: not there, or from `upto` on) and their first row in it.
__device__ __forceinline__ void page_of(const ChunkArgs& p, const int32_t* table, int t16, int upto, int& page, int& row) {
    uint32_t i = static_cast<uint32_t>(t16);
    row = 0;
    if (p.page16 > 1) {
        i = __umulhi(static_cast<uint32_t>(t16), p.page16_inv);  // one too many at most
        int r = t16 - static_cast<int>(i * p.page16);
        if (r < 0) --i, r += p.page16;
        row = 16 * r;
    }
    page = 16 * t16 < upto ? table[i] : -1;
    page = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.pages) ? page : -1;
}
__device__ __forceinline__ uint16_t* out_row(const ChunkArgs& p, const Place& at, int hk, int row, int D) {
    const int token = token_of(p, row);
    return p.out + (static_cast<int64_t>(at.s.first + token) * p.Hq + hk * p.group + row - token * p.group) * D;
}

__device__ __forceinline__ uint2 halves(const float4_t& v, float by) {
    const half2_t a = {static_cast<_Float16>(v[0] * by), static_cast<_Float16>(v[1] * by)}, b = {static_cast<_Float16>(v[2] * by), static_cast<_Float16>(v[3] * by)};
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

// ---------------------------------------------------------------------- a part --
// W: waves, each with 32 rows. KT: tokens that are staged and taken at a time. True, in every thread: V is not finite
// somewhere, and the part has to be taken `again`. On the matrix cores such an element reaches every row of its tile, as zero
// weights times it are NaN; the second time it is taken out of V, and its d's first token that has it is kept: the rows that see
// that one get in the end what it makes of them. 8192 new tokens, heads 8/2 of 256: 287 us, with one infinity in the first page
// 607, in every 16th token 717; 512 over 100000 487, 877, 1058.
template <int D, int W, int KT>
__device__ __forceinline__ bool take_part(const ChunkArgs& p, uint8_t* lds, bool again, unsigned block, unsigned thread) {
    constexpr int R = 32 * W;                    // (token, head) rows of a workgroup
    constexpr int KS = D / 16;                   // steps of the score product
    constexpr int MB = D / 32;                   // blocks of 32 d
    constexpr int RC = D / 8;                    // 16-byte chunks of a row
    constexpr int RPI = 64 / RC;                 // rows that a copy takes
    constexpr int CR = KT / W;                   // rows of K and of V that a wave copies
    constexpr int ROW = 2 * D;                   // bytes
    constexpr int KM = RC < 16 ? RC - 1 : 15;
    constexpr int QL = D == 256 ? 3 : 0;         // of q's operands, those that lie in LDS: the registers are one or two short
    constexpr int kAhead = 3;                    // operands on their way from LDS while a product runs
    __shared__ int flag, odd_of[W], odd_from[2][D];
    constexpr int kThrough = 16;                 // accesses that all XCDs see
    const int lane = thread & 63, c = lane & 31, j = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);

    Place at;
    auto units = [&](const Seq& s, int S) {
        const int tiles = tiles_of<R>(p, s), parts = (s.len + S - 1) / S;
        const int whole = s.base > 0 ? s.base / S : 0;
        int sum = tiles * (1 + whole);
        for (int i = whole + 1; i < parts; ++i) sum += tiles_with<R>(p, s, tiles, static_cast<int64_t>(i) * S);
        return sum * p.Hkv;
    };
    if (!find<R>(p, unit_of(block), at, units)) return false;
    const int rows = at.s.n * p.group, tiles = tiles_of<R>(p, at.s), base = at.s.base;
    // Part by part; in one, `near` tiles of a cache head after another, those that read most first.
    int part, tile, hk;
    {
        const int whole = base > 0 ? base / at.S : 0;
        int i = at.unit, have = tiles;
        part = i / (tiles * p.Hkv);
        if (part <= whole) i -= part * tiles * p.Hkv;
        else {
            part = whole + 1;
            i -= part * tiles * p.Hkv;
            for (;;) {
                have = tiles_with<R>(p, at.s, tiles, static_cast<int64_t>(part) * at.S);
                if (have == 0) return false;     // (lengths that changed meanwhile)
                if (i < have * p.Hkv) break;
                i -= have * p.Hkv;
                ++part;
            }
        }
        const int near = 1 << kNearLog2, first = i / (near * p.Hkv) * near, of = have - first < near ? have - first : near;
        i -= first * p.Hkv;
        hk = i / of;
        tile = tiles - 1 - first - (i - hk * of);
    }
    part = __builtin_amdgcn_readfirstlane(part);         // (the same in all lanes, which the compiler does not see)
    tile = __builtin_amdgcn_readfirstlane(tile);
    hk = __builtin_amdgcn_readfirstlane(hk);
    const int row0 = tile * R, last_row = (row0 + R < rows ? row0 + R : rows) - 1;
    auto seen_by = [&](int row) { return sees(at.s, token_of(p, row)); };
    const int end = seen_by(last_row), parts = end <= at.S ? 1 : (end + at.S - 1) / at.S;
    const int t_begin = part * at.S, t_end = part < parts - 1 ? t_begin + at.S : end;

    const int wrow = row0 + wave * 32;
    const bool mine = wrow < rows;               // this wave has rows
    const int least = mine ? seen_by(wrow) : 0, most = mine ? seen_by(wrow + 31 < rows ? wrow + 31 : rows - 1) : 0;
    const int row = wrow + c < rows ? wrow + c : rows - 1, token = token_of(p, row);      // past the last one: that one again, never stored
    const int seen = seen_by(row);

    const int32_t* table = p.table + at.b * p.table_row;
    const uint16_t* kh = p.k + hk * p.k_head;
    const uint16_t* vh = p.v + hk * p.v_head;
    // A lane holds where K and V of one of the 64 groups of 16 tokens from token `known` on begin; above all addresses: nowhere.
    uint64_t my_k, my_v;
    int known = t_begin;
    auto know = [&]() {
        int page, row;
        page_of(p, table, known / 16 + lane, t_end, page, row);
        const uint64_t none = page < 0 ? uint64_t(1) << 63 : 0;
        my_k = reinterpret_cast<uintptr_t>(kh + (page < 0 ? 0 : page) * p.k_page + static_cast<int64_t>(row) * p.k_token) | none;
        my_v = reinterpret_cast<uintptr_t>(vh + (page < 0 ? 0 : page) * p.v_page + static_cast<int64_t>(row) * p.v_token) | none;
    };
    know();
    half8_t all[KS];
    if (mine) {
        const uint16_t* qr = p.q + static_cast<int64_t>(at.s.first + token) * p.q_row + static_cast<int64_t>(hk * p.group + row - token * p.group) * p.q_head;
#pragma unroll
        for (int s = 0; s < KS; ++s) all[s] = *reinterpret_cast<const half8_t*>(qr + 16 * s + 8 * j);
    }
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
    // A tile's copies. Rows lie in LDS as they do in memory, but a row's chunks in an order of its own, so that reads of a
    // column meet other banks. Each wave has CP copies of K and CP of V to make, spread over the products of the tile before:
    // in one go they would hold all waves up, and with them the matrix cores.
    auto turn_of_v = [](uint32_t row) { return RC < 16 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); };
    constexpr int CP = CR / RPI;
    const int first_row = wave * CR % 16;        // of its 16 rows
    int4_t k_from, v_from;                       // buffer descriptors
    uint32_t copy_to;
    // Groups of 16 tokens that are not there, of the tile that is being taken, of the one that is on its way and
    // of the one after it.
    constexpr uint32_t kAgain = 1u << 31;        // (among them, as the loop has no register for it)
    uint32_t gone = 0, gone_next = 0, gone_then = again ? kAgain : 0;
    auto aim = [&](int t, int buf) {
        copy_to = lds_at + buf * 2 * KT * ROW + wave * CR * ROW;
        const int g = (t - known) / 16, own = g + wave * CR / 16;
        gone_then = (gone_then & kAgain) | (static_cast<uint32_t>(__ballot(static_cast<int64_t>(my_k) < 0) >> g) & (KT == 64 ? 15u : 3u));
        auto rows16 = [&](uint64_t at, int token_stride) {
            const int lo = __builtin_amdgcn_readlane(static_cast<int>(at), own), hi = __builtin_amdgcn_readlane(static_cast<int>(at >> 32), own);
            return int4_t{lo, hi & 0xffff, hi < 0 ? 0 : 2 * (15 * token_stride + D), 0x00020000};
        };
        k_from = rows16(my_k, p.k_token);
        v_from = rows16(my_v, p.v_token);
        asm volatile("s_nop 4" : "+s"(k_from), "+s"(v_from));     // from a readlane to a copy, whose operands the compiler does not watch
    };
    const uint32_t lr = static_cast<uint32_t>(lane) / RC, lc = static_cast<uint32_t>(lane) % RC;
    const uint32_t k_row = 2 * lr * p.k_token, v_row = 2 * lr * p.v_token, k_chunk = 16 * (lc ^ (lr & KM)), v_chunk = 16 * (lc ^ turn_of_v(lr));
    // (Written out: the compiler would have every read of V in LDS wait for all copies on their way, whatever buffer they go
    // to. The loop waits for them where it takes the tile.)
    auto copy = [&](int i) {                     // 0 .. CP - 1: of K, then of V
        const bool of_v = i >= CP;
        const int row = first_row + (of_v ? i - CP : i) * RPI;
        uint32_t chunk = of_v ? v_chunk : k_chunk;       // (opaque: what is made from it would be kept through the loop)
        asm volatile("" : "+v"(chunk));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"            // (m0 is reserved: it is set anew wherever it is used, unless an older value is known to stand)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(copy_to + (of_v ? KT * ROW + (i - CP) * 1024 : i * 1024)),
                     "v"((chunk ^ (16 * (of_v ? turn_of_v(row) : row & KM))) + (of_v ? v_row : k_row)), "s"(of_v ? v_from : k_from), "s"(2 * row * (of_v ? p.v_token : p.k_token)) : "m0", "memory");
#pragma clang diagnostic pop
    };
    if (t_begin < t_end) {
        aim(t_begin, 0);
        gone_next = gone_then;
#pragma unroll
        for (int i = 0; i < 2 * CP; ++i) copy(i);
        aim(t_begin + KT, 1);                    // (past the end: copies of nothing)
    }
    half8_t q[KS - QL], *const q_held = reinterpret_cast<half8_t*>(lds + 4 * KT * ROW) + thread;
    if (mine) {
        if (p.q_by != 1.f)
#pragma unroll
            for (int s = 0; s < KS; ++s) all[s] *= static_cast<_Float16>(p.q_by);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            asm volatile("" : "+v"(all[s]));     // (waited for here: a wait in the loop would be one for its copies too)
            if (s < KS - QL) q[s] = all[s];
            else q_held[(s - KS + QL) * 64 * W] = all[s];
        }
    }
    float16_t acc[MB] = {};
    float m = -INFINITY, l = 0.f;
    // Operands lie in LDS where a lane's place of the first turns by whole chunks: an exclusive or on the address.
    const int vrow = 4 * j + ((lane & 15) >> 2);
    const uint32_t k_at = c * ROW + 16 * (j ^ (c & KM));
    const uint32_t v_at = (KT + vrow) * ROW + 16 * (turn_of_v(vrow) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + 8 * (lane & 1);
    typedef __fp16 half4_b __attribute__((ext_vector_type(4)));
    typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
    typedef const __attribute__((address_space(3))) half8_t* lds_half8;
    typedef __attribute__((address_space(3))) half4_b* lds_half4;
    typedef uint32_t uint2_v __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) uint2_v* lds_uint2;

    // Of a SIMD's two waves the one in the odd slot goes first: alike, they share the matrix cores and come to their softmaxes at
    // one time. 9 prompts of 1 to 1501 tokens, heads 32/8 of 128: 81.6 us, 86.9 without; with heads of 256 within 3% either way.
    if (D < 256 && (__builtin_amdgcn_s_getreg((3 << 11) | 4) & 1)) __builtin_amdgcn_s_setprio(2);
    if (again) {
        for (int i = threadIdx.x; i < 2 * D; i += 64 * W) odd_from[i / D][i % D] = 0x7fffffff;
        __syncthreads();
    }
    int buf = 0;
    for (int t = t_begin; t < t_end; t += KT, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint8_t* const vl = lds + (2 * buf + 1) * KT * ROW;
        const uint32_t k_now = lds_at + buf * 2 * KT * ROW + k_at, v_now = lds_at + buf * 2 * KT * ROW + v_at;
        gone = gone_next;
        gone_next = gone_then;
        if (t + KT > t_end || gone) {
            // what lies past the end or is not there may be NaN, whose product with a weight of zero is no zero
            int first = lane;                    // (opaque, as the chunk of a copy)
            asm volatile("" : "+v"(first));
#pragma unroll 1
            for (int i = first; i < CR * RC; i += 64) {
                const int r = CR * wave + i / RC;
                uint4* const chunk = reinterpret_cast<uint4*>(vl + r * ROW + 16 * (i % RC));
                if (t + r >= t_end || (gone >> (CR * wave / 16) & 1)) *chunk = make_uint4(0, 0, 0, 0);
                else if (gone & kAgain) {
                    uint4 v = *chunk;
                    uint32_t* const w = &v.x;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t h = w[e / 2] >> (16 * (e % 2)) & 0xffff;
                        if ((h & 0x7c00) != 0x7c00) continue;
                        const int d = 8 * (i % RC ^ turn_of_v(r)) + e;
                        if (h != 0xfc00) atomicMin(&odd_from[0][d], t + r);      // a NaN is both infinities
                        if (h != 0x7c00) atomicMin(&odd_from[1][d], t + r);
                        w[e / 2] &= e % 2 ? 0xffffu : 0xffff0000u;
                    }
                    *chunk = v;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        if (t + 2 * KT - known >= 1024) {        // (before the copies: it is waited for)
            known += 1024;
            know();
        }
        // (Copies and what aims the next ones go out before the products: between them they cost more than they hide, 8192 new
        // tokens 307 us against 286.)
#pragma unroll
        for (int i = 0; i < 2 * CP; ++i) copy(i);
        aim(t + 2 * KT, buf);
        if (!mine || t >= most) continue;
        const bool all = t + KT <= least && gone == 0;
        // Scores of 32 tokens; the reference exponent of what follows, and its rare change; weights; their products
        auto k_read = [&](int h, int x) {
            return *reinterpret_cast<lds_half8>((k_now ^ (32 * x % (16 * (KM + 1)))) + 32 * h * ROW + 32 * x / (16 * (KM + 1)) * (16 * (KM + 1)));
        };
        auto scores = [&](int h, float16_t& s) {
            half8_t k[kAhead];
#pragma unroll
            for (int x = 0; x < kAhead; ++x) k[x] = k_read(h, x);
            s = float16_t{};
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const half8_t qx = x < KS - QL ? q[x < KS - QL ? x : 0] : q_held[(x - KS + QL) * 64 * W];
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[x % kAhead], qx, s, 0, 0, 0);
                if (x + kAhead < KS) k[x % kAhead] = k_read(h, x + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto refer = [&](int h, float16_t& s) {
            if (!all) {
                const int left = seen - t - 32 * h - 4 * j;
                const uint32_t none = gone >> (2 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i / 4) + i % 4 >= left || (none >> (i / 8) & 1)) s[i] = -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
            mx = max2(mx);
            if (__any(fmaf(mx, p.scale_log2, -m) > kMost || fabsf(m) >= kFar)) {
                const float top = mx * p.scale_log2, to = fmaxf(m, fabsf(top) < kFar ? ceilf(top) - kTop : top), keep = m == -INFINITY ? 0.f : exp2_of(m - to);
                m = to;
                l *= keep;
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[b][i] *= keep;
                const bool far = fabsf(m) >= kFar && fabsf(m) < INFINITY;
                if (__any(far)) {
                    float by = p.scale_log2;     // (opaque: its reciprocal would be kept through the loop)
                    asm volatile("" : "+s"(by));
                    const float back = __builtin_amdgcn_rcpf(by);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = far ? (s[i] * p.scale_log2 - m) * back : s[i];
                }
            }
        };
        auto weigh = [&](const float16_t& s, half8_t (&w)[2]) {
            const float from = fabsf(m) < kFar ? m : 0.f;        // (-inf: nothing seen; past kFar: taken off already)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const half2_t e = {static_cast<_Float16>(exp2_of(fmaf(s[i], p.scale_log2, -from))),
                                   static_cast<_Float16>(exp2_of(fmaf(s[i + 1], p.scale_log2, -from)))};
                l = __builtin_amdgcn_fdot2(e, half2_t{1, 1}, l, false);
                w[i / 8][i % 8] = e[0];
                w[i / 8][i % 8 + 1] = e[1];
            }
        };
        auto v_read = [&](int h, int y) {        // product y: block y % MB of d, 16 tokens
            half8_t a;
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                constexpr int TM = RC < 16 ? 2 : 4;      // blocks that turn into one another
                const int b = y % MB;
                const uint32_t from = (v_now ^ (64 * (b % TM))) + (32 * h + 16 * (y / MB) + 8 * z) * ROW + 64 * TM * (b / TM);
                const auto r = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16(reinterpret_cast<lds_half4>(from)));
#pragma unroll
                for (int e = 0; e < 4; ++e) a[4 * z + e] = r[e];
            }
            return a;
        };
        auto add = [&](int h, const half8_t (&w)[2], half8_t (&v)[kAhead]) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int y = 0; y < 2 * MB; ++y) {
                acc[y % MB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[y % kAhead], w[y / MB], acc[y % MB], 0, 0, 0);
                if (y + kAhead < 2 * MB) v[y % kAhead] = v_read(h, y + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
#pragma unroll
        for (int h = 0; h < KT / 32; ++h) {
            float16_t s;
            half8_t w[2], v[kAhead];
            scores(h, s);
            auto v_first = [&]() {
#pragma unroll
                for (int y = 0; y < kAhead; ++y) v[y] = v_read(h, y);
            };
            if (D < 256) v_first();              // (before the softmax where there are registers)
            refer(h, s);
            weigh(s, w);
            if (D == 256) {
                __builtin_amdgcn_sched_barrier(0);
                v_first();
            }
            add(h, w, v);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // no copy is on its way
    if (again)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int d = 32 * b + 8 * (i / 4) + 4 * j + i % 4;
                const bool up = odd_from[0][d] < seen, down = odd_from[1][d] < seen;
                acc[b][i] = up ? down ? NAN : INFINITY : down ? -INFINITY : acc[b][i];
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
    int w0 = 0;
    const int mine_at = wave * static_cast<int>(part_bytes(D)) + 16 * lane, stat_at = wave * static_cast<int>(part_bytes(D)) + 128 * D + 8 * lane;
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    auto slot = [&](int i) {                     // of nothing where there is no such part
        return __builtin_amdgcn_make_buffer_rsrc(slot_of(p, w0, i), 0, i < parts ? static_cast<int>(p.slot_bytes) : 0, 0x00020000);
    };
    if (parts > 1) {
        w0 = first_id<R>(p, at, tile, hk);
        if (mine) {
            const auto to = slot(part);
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    __builtin_amdgcn_raw_buffer_store_b128(int4_t{__float_as_int(acc[b][4 * i]), __float_as_int(acc[b][4 * i + 1]), __float_as_int(acc[b][4 * i + 2]),
                                                                  __float_as_int(acc[b][4 * i + 3])},
                                                           to, mine_at + 1024 * (4 * b + i), 0, kThrough);
            __builtin_amdgcn_raw_buffer_store_b64(u2{__float_as_uint(m), __float_as_uint(l)}, to, stat_at, 0, kThrough);
        }
    }
    if (!again) {                                // while the part is on its way out, which another pass replaces
        float4_t some = {};                      // (the sums' products two by two pass no 2^127: a sum is below 2^62)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) some[i / 2 % 4] = fmaf(acc[b][i], acc[b][i + 1], some[i / 2 % 4]);
        const float none = (some[0] + some[1]) + (some[2] + some[3]);
        const float sum = sum2(l);               // not finite itself: nor are the row's values, and rightly
        odd_of[wave] = __any(mine && !(fabsf(none) < INFINITY) && fabsf(sum) < INFINITY);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                // K and V have been read
    asm volatile("" ::: "memory");
    if (!again) {
        int odd = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) odd |= odd_of[w];
        if (__builtin_amdgcn_readfirstlane(odd)) return true;
    }

    // Up to four parts meet in the last of them to arrive; always (0 + 1) + (2 + 3), so that the bits do not depend on who is
    // last: scaling by powers of two is exact, and a sum of two has one value.
    if (parts > 1) {
        if (parts > kFan) return false;
        if (!last_in(reinterpret_cast<unsigned*>(p.ws) + w0, parts, &flag) || !mine) return false;
        const int others = (part ^ 2) & ~1, with[3] = {part ^ 1, others, others + 1};
        __amdgpu_buffer_rsrc_t from[3];
        float om[3], ol[3], by[3], top = m;
        u2 st[3];
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            from[x] = slot(with[x]);
            st[x] = __builtin_amdgcn_raw_buffer_load_b64(from[x], stat_at, 0, kThrough);
        }
        int4_t o[2][3][4];                       // a block's sums are on their way while those before are added
        auto load = [&](int b) {
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[b % 2][x][i] = __builtin_amdgcn_raw_buffer_load_b128(from[x], mine_at + 1024 * (4 * b + i), 0, kThrough);
        };
        load(0);
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            om[x] = with[x] < parts ? __uint_as_float(st[x][0]) : -INFINITY;
            ol[x] = __uint_as_float(st[x][1]);
            top = fmaxf(top, om[x]);
        }
#pragma unroll
        for (int x = 0; x < 3; ++x) by[x] = om[x] == -INFINITY ? 0.f : exp2_of(om[x] - top);
        const float keep = m == -INFINITY ? 0.f : exp2_of(m - top);
        m = top;
        l = (l * keep + ol[0] * by[0]) + (ol[1] * by[1] + ol[2] * by[2]);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            if (b + 1 < MB) load(b + 1);
            __builtin_amdgcn_sched_barrier(0);
            const auto& now = o[b % 2];
#pragma unroll
            for (int i = 0; i < 16; ++i)
                acc[b][i] = (acc[b][i] * keep + __int_as_float(now[0][i / 4][i % 4]) * by[0]) +
                            (__int_as_float(now[1][i / 4][i % 4]) * by[1] + __int_as_float(now[2][i / 4][i % 4]) * by[2]);
        }
    }
    if (!mine) return false;

    l = sum2(l);
    // acc[b][i]: d = 32 b + 8 (i / 4) + 4 j + i % 4 of this lane's row
    if (__any(l == 0.f))                         // no weight but zeros: nothing, whatever V holds
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][i] = l == 0.f ? 0.f : acc[b][i];
    // Whole rows go out, turned in LDS, a wave in its own part of it: a row's 16-byte chunks in an order of its own, so that
    // what a lane has of its row meets other banks; and each row's place in `out`, worked out once by the lanes that have it.
    {
        constexpr int CH = D / 8, CM = CH < 16 ? CH - 1 : 15, N = CH / 2 < 8 ? CH / 2 : 8;       // N: stores of a lane in a go
        typedef __attribute__((address_space(3))) uint64_t* lds_uint64;
        typedef uint32_t uint4_v __attribute__((ext_vector_type(4)));
        typedef const __attribute__((address_space(3))) uint4_v* lds_uint4;
        const float by = l > 0.f ? 1.0f / l : 0.f;
        const uint32_t mine_at = lds_at + wave * 64 * D, rows_at = lds_at + 64 * D * W + 256 * wave, to = mine_at + 16 * (c * CH + (c & CM)) + 8 * j;
        *reinterpret_cast<lds_uint64>(rows_at + 8 * c) =
            wrow + c < rows ? reinterpret_cast<uintptr_t>(p.out + (static_cast<int64_t>(at.s.first + token) * p.Hq + hk * p.group + row - token * p.group) * D) : 0;
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint2 h = halves(float4_t{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]}, by);
                *reinterpret_cast<lds_uint2>((to ^ (64 * (b % ((CM + 1) / 4)) + 16 * i)) + 16 * (CM + 1) * (b / ((CM + 1) / 4))) = uint2_v{h.x, h.y};
            }
        const int r0 = lane / CH, ch = lane % CH;
#pragma unroll 1
        for (int r = r0; r < 32; r += 64 / CH * N) {
            uint64_t place[N];
            uint4_v v[N];
#pragma unroll
            for (int x = 0; x < N; ++x) {
                const int rx = r + 64 / CH * x;
                place[x] = *reinterpret_cast<lds_uint64>(rows_at + 8 * rx);
                v[x] = *reinterpret_cast<lds_uint4>(mine_at + 16 * (rx * CH + (ch ^ (rx & CM))));
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < N; ++x) asm volatile("" : "+v"(v[x]), "+v"(place[x]));       // (read before the first is stored)
#pragma unroll
            for (int x = 0; x < N; ++x)
                if (place[x]) *reinterpret_cast<__attribute__((address_space(1))) uint4_v*>(place[x] + 16 * ch) = v[x];
        }
    }
    return false;
}

template <int D, int W, int KT>
__global__ __launch_bounds__(64 * W, 2) void chunk_attention_kernel(ChunkArgs p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];      // [2][K, V][KT][D]; the last of q's operands
    bool again = false;
#pragma unroll 1
    for (;;) {
        unsigned block = blockIdx.x, thread = threadIdx.x;
        auto args = (const __attribute__((address_space(4))) ChunkArgs*)(uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(block), "+v"(thread), "+s"(args));    // (opaque: what is made from them would be kept for a second time, in registers that the loop needs)
        p = *(const ChunkArgs*)args;
        if (!take_part<D, W, KT>(p, lds, again, block, thread)) return;
        again = true;
    }
}

// ------------------------------------------------------------------- many parts' sum --
// Of the tiles that are in more than kFan parts: a workgroup has 32 rows and 32 d, as their parts have them in a wave's
// registers, each of its waves a quarter of the parts. Bound by the partial sums' bytes and by its own start: 4 us for 24 new
// tokens over 1100 (3.5 MB), 15 for 512 over 100000 (67 MB, 4.4 TB/s), 5 where it finds nothing to do.
template <int D, int R>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs p) {
    constexpr int MB = D / 32;
    Place at;
    auto many = [&](const Seq& s, int S) { return s.len > kFan * static_cast<int64_t>(S) ? tiles_with<R>(p, s, tiles_of<R>(p, s), kFan * static_cast<int64_t>(S)) * p.Hkv : 0; };
    if (!find<R>(p, blockIdx.x, at, many)) return;
    const int rows = at.s.n * p.group, tiles = tiles_of<R>(p, at.s);
    const int hk = at.unit % p.Hkv, tile = tiles - 1 - at.unit / p.Hkv;
    const int lane = threadIdx.x & 63, c = lane & 31, j = lane >> 5, quarter = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = blockIdx.y / MB, b = blockIdx.y % MB;
    const int row0 = tile * R, last_row = (row0 + R < rows ? row0 + R : rows) - 1, wrow = row0 + 32 * wave;
    if (wrow > last_row) return;
    const int parts = (sees(at.s, token_of(p, last_row)) + at.S - 1) / at.S;
    const int w0 = first_id<R>(p, at, tile, hk), per = (parts + 3) / 4, end = (quarter + 1) * per < parts ? (quarter + 1) * per : parts;
    float4_t sum[4] = {};
    float top = -INFINITY, l = 0.f;
    constexpr int kBatch = 6;                    // parts whose loads go out together (24 over 1100, 18 parts: 14.6 us, 15.4 with four)
    for (int u0 = quarter * per; u0 < end; u0 += kBatch) {
        float4_t o[kBatch][4];
        float2 st[kBatch];
        float most = top;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint8_t* slot = slot_of(p, w0, u0 + u < end ? u0 + u : end - 1) + wave * part_bytes(D);
            st[u] = *reinterpret_cast<const float2*>(slot + 128 * D + 8 * lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[u][i] = *reinterpret_cast<const float4_t*>(slot + 1024 * (4 * b + i) + 16 * lane);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) most = fmaxf(most, st[u].x);
        const float keep = top == -INFINITY ? 0.f : exp2_of(top - most);
        l *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] *= keep;
        top = most;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (u0 + u >= end) continue;
            const float by = st[u].x == -INFINITY ? 0.f : exp2_of(st[u].x - top);
            l = fmaf(st[u].y, by, l);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[i][e] = fmaf(o[u][i][e], by, sum[i][e]);
        }
    }
    // the quarters' sums meet in the first wave
    __shared__ float4_t meet[3][4][64];
    __shared__ float2 stat[3][64];
    if (quarter) {
        stat[quarter - 1][lane] = make_float2(top, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) meet[quarter - 1][i][lane] = sum[i];
    }
    __syncthreads();
    if (quarter) return;
    {
        const float own = top;
        float2 st[3];
#pragma unroll
        for (int u = 0; u < 3; ++u) {
            st[u] = stat[u][lane];
            top = fmaxf(top, st[u].x);
        }
        const float keep = own == -INFINITY ? 0.f : exp2_of(own - top);
        l *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] *= keep;
#pragma unroll
        for (int u = 0; u < 3; ++u) {
            const float by = st[u].x == -INFINITY ? 0.f : exp2_of(st[u].x - top);
            l = fmaf(st[u].y, by, l);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4_t o = meet[u][i][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[i][e] = fmaf(o[e], by, sum[i][e]);
            }
        }
    }
    l = sum2(l);
    if (wrow + c <= last_row) {
        uint16_t* to = out_row(p, at, hk, wrow + c, D) + 32 * b + 4 * j;
        const float by = l > 0.f ? 1.0f / l : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint2*>(to + 8 * i) = halves(l == 0.f ? float4_t{0, 0, 0, 0} : sum[i], by);
    }
}

// Rows of a workgroup, and tokens that it takes at a time.
constexpr int kRows = 128;
constexpr int tokens_of(int64_t D) { return D == 256 ? 32 : 64; }
// Parts to cut for, of rows that read up to `most` tokens: what the chip holds at once.  -1: nothing to cut. (Two parts of 128
// tokens are joined in more time than they save: 200 new tokens, heads 8/2 of 256, 16.5 us in one, 18.4 in two.)
int choose_slots_log2(int64_t most, int64_t D) { return most <= 2 * kLeast ? -1 : D == 64 ? 10 : 9; }
// Tokens of a part, at least. Where there are tiles enough for the chip, a quarter of the longest sequence's: no tile is then in
// more parts than the last of them joins, and no launch follows for those that are. Measured with a quarter and with kLeast, us:
// 1100 new tokens, heads 8/2 of 256 (70 tiles) 31.2, 37.0; 2048 47.6, 54.1; 3000 70.0, 78.3; 16 x 32 over 1000, heads 32/8 of
// 128 (128 tiles) 15.1, 18.8. Otherwise 300 over 800 (20 tiles) 30.0, 25.2; 16 x 32 over 2000 (32 tiles) 30.7, 22.6; 1000 over
// 3000 (64 tiles) 61.2, 57.3. A few tiles of 256, whose tokens take longest, are cut down to kTile: 24 over 1100 (2 tiles) 15.4
// us, 16.8 with kLeast; 2 x 16 over 700 (4) 13.7, 19.5; otherwise 8 over 4000 18.1, 17.0, 8 x 4 over 500 (16 tiles) 16.5, 14.6.
int choose_least(int64_t most, int64_t tiles, int64_t D) {
    if (D == 256 && tiles <= 8 && most <= 2048) return kTile;
    if (tiles < 40 || most > std::min<int64_t>(50 * tiles, 4096)) return kLeast;
    return static_cast<int>(std::max<int64_t>(ceil_div(most, kFan * kTile) * kTile, kLeast));
}
int64_t slot_bytes_of(int64_t T, int64_t group, int64_t D) { return ceil_div(std::min<int64_t>(kRows, T * group), 32) * part_bytes(D); }
// A workgroup reads its rows of q before it writes them and nobody else's, so that out may be q; but no rows otherwise placed.
bool meets(const void* q, int64_t row, int64_t head, const void* out, int64_t T, int64_t Hq, int64_t D) {
    if (q == out && (T == 1 || row == Hq * D) && (Hq == 1 || head == D)) return false;
    const int64_t begin = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(q)) / 2, end = begin + T * Hq * D;      // elements from q on
    for (int64_t h = 0; h < Hq; ++h) {
        const int64_t past = begin - D - h * head;       // the first token whose head ends behind out's first element
        const int64_t t = past < 0 ? 0 : row > 0 ? past / row + 1 : T;
        if (t < T && t * row + h * head < end) return true;
    }
    return false;
}
int64_t split_bytes(int slots_log2, int64_t slot_bytes) { return slots_log2 < 0 ? 0 : kCounterBytes + 2 * ((int64_t(1) << slots_log2) + 2) * slot_bytes; }

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int64_t mcv_paged_attention_chunk_workspace_bytes(int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seq_len) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || T > 0x7fffffff / Hq || D <= 0 || max_seq_len < 0) return 0;
    return split_bytes(choose_slots_log2(std::min(max_seq_len, kMaxLen), D), slot_bytes_of(T, Hq / Hkv, D));
}

int mcv_paged_attention_chunk(const void* q, int64_t q_row, int64_t q_head, const void* k_cache, int64_t k_page,
                              int64_t k_token, int64_t k_head, const void* v_cache, int64_t v_page, int64_t v_token,
                              int64_t v_head, int64_t pages, int64_t page_size, const void* block_table,
                              int64_t table_row, int64_t table_width, const void* seq_lens, int64_t max_seq_len,
                              const void* cu_seqlens, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, double scale,
                              void* out, void* workspace, int64_t workspace_bytes, mcv_stream_t stream) {
    return mcv_paged_attention_chunk_at(q, q_row, q_head, k_cache, k_page, k_token, k_head, v_cache, v_page, v_token, v_head, pages, page_size,
                                        block_table, table_row, table_width, seq_lens, max_seq_len, cu_seqlens, nullptr, B, T, Hq, Hkv, D, scale,
                                        out, workspace, workspace_bytes, stream);
}

int mcv_paged_attention_chunk_at(const void* q, int64_t q_row, int64_t q_head, const void* k_cache, int64_t k_page,
                                 int64_t k_token, int64_t k_head, const void* v_cache, int64_t v_page, int64_t v_token,
                                 int64_t v_head, int64_t pages, int64_t page_size, const void* block_table,
                                 int64_t table_row, int64_t table_width, const void* seq_lens, int64_t max_seq_len,
                                 const void* cu_seqlens, const void* positions, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                 double scale, void* out, void* workspace, int64_t workspace_bytes, mcv_stream_t stream) {
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
    if (meets(q, q_row, q_head, out, T, Hq, D)) return fail(MCV_ERR_INVALID_ARG, "%s: out overlaps q without being it", who);
    int rc = require_device();
    if (rc != MCV_OK) return rc;
    // (width counted in pages first: width * page_size could pass 64 bits)
    const int64_t held = table_width > kMaxLen / page_size ? kMaxLen : table_width * page_size;
    const int64_t most = max_seq_len < held ? max_seq_len : held;
    const int64_t group = Hq / Hkv;
    const int64_t slot_bytes = slot_bytes_of(T, group, D), tiles = std::min(T * group / kRows + B, T * group);
    int slots_log2 = choose_slots_log2(most, D);
    if (slots_log2 >= 0 && (!workspace || workspace_bytes < split_bytes(slots_log2, slot_bytes))) slots_log2 = -1;
    if (slots_log2 >= 0 && reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
        return fail(MCV_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", who);
    const int least = choose_least(most, tiles * Hkv, D);
    const int64_t slots = slots_log2 < 0 ? 0 : int64_t(1) << slots_log2;
    if (tiles * Hkv + slots > 0x7fffff00) return fail(MCV_ERR_SHAPE, "%s: too many rows B=%lld T=%lld Hq=%lld", who, (long long)B, (long long)T, (long long)Hq);
    const uint32_t page16 = static_cast<uint32_t>(page_size / 16);
    auto inverse = [](uint64_t n) { return n > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + n - 1) / n) : 0; };
    // (A scale that 32 bits do not hold weighs all tokens alike, as the least that they do; the product with zero would not leave -inf what it is.)
    const float scale_log2 = scale == 0.0 ? 1.f : std::max(std::fabs(static_cast<float>(scale) * kLog2e), FLT_MIN);
    const ChunkArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache),
                      static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(seq_lens), static_cast<const int32_t*>(cu_seqlens),
                      static_cast<const int32_t*>(positions), static_cast<uint16_t*>(out), static_cast<uint8_t*>(workspace), q_row, q_head, k_page, k_head, v_page, v_head, table_row,
                      static_cast<int>(k_token), static_cast<int>(v_token), static_cast<int>(pages), static_cast<int>(page16), static_cast<int>(most),
                      static_cast<int>(B), static_cast<int>(T), static_cast<int>(Hq), static_cast<int>(Hkv), static_cast<int>(group),
                      inverse(page16), inverse(group), scale_log2, scale < 0.0 ? -1.f : scale == 0.0 ? 0.f : 1.f,
                      slots_log2, least, slot_bytes};
    const auto s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(ceil_div(tiles * Hkv + slots, 8 << kNearLog2) * (8 << kNearLog2)));
    auto fn = D == 64 ? chunk_attention_kernel<64, 4, tokens_of(64)> : D == 128 ? chunk_attention_kernel<128, 4, tokens_of(128)> : chunk_attention_kernel<256, 4, tokens_of(256)>;
    hipLaunchKernelGGL(fn, grid, dim3(2 * kRows), static_cast<unsigned>(8 * tokens_of(D) * D + (D == 256 ? 3 * 32 * kRows : 0)), s, a);
    rc = check_launch("chunk_attention_kernel");
    if (rc != MCV_OK || most <= kFan * least || !slots) return rc;
    const dim3 joins(static_cast<unsigned>(std::min(tiles * Hkv, slots / kFan)), static_cast<unsigned>(ceil_div(std::min<int64_t>(kRows, T * group), 32) * D / 32));
    auto join = D == 64 ? chunk_join_kernel<64, kRows> : D == 128 ? chunk_join_kernel<128, kRows> : chunk_join_kernel<256, kRows>;
    hipLaunchKernelGGL(join, joins, dim3(256), 0, s, a);
    return check_launch("chunk_join_kernel");
}

}  // extern "C"
