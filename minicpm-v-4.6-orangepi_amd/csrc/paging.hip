// paging.hip -- pages of a paged cache dealt out to growing sequences and taken back, gfx950.
//
// A sequence of n tokens has ceil(n / page_size) pages. The free list is a stack: its first `count` entries are free pages, and
// the page that is dealt out as number i of a call is entry count - 1 - i, sequence by sequence, so that every workgroup finds
// every page by a sum over the sequences before and no two of them have to talk. A thread adds up `span` sequences, the
// workgroup scans the threads' sums; a token then finds its thread by bisection in LDS and walks that thread's sequences.
//
// A few kilobytes are read and written: what counts is the launch and a chain of four loads (lengths, token's sequence, its
// page, the store).
#include <algorithm>

#include "common.h"
#include "mcv_mixers.h"

namespace mcv {
namespace {

constexpr int kThreads = 1024;

struct PageArgs {
    int32_t* table;
    const int32_t* lens;
    const int32_t* cu;                           // append: first rows; truncate: tokens kept
    int32_t* list;
    const int32_t* count;
    int64_t* slots;
    int64_t* positions;
    int32_t* lens_out;
    int32_t* count_out;
    int64_t table_row, capacity;
    int width, page, B, T;
    int what;                                    // kPages, kState or both
};
constexpr int kPages = 1, kState = 2;

__device__ __forceinline__ int pages_of(int tokens, int page) { return tokens / page + (tokens % page != 0); }

struct Growth {
    int first, next, held, old, need, want;      // rows, tokens, pages before, pages to come, tokens wanted
};
__device__ __forceinline__ int first_row(const PageArgs& p, int b) {
    const int at = p.cu ? p.cu[b] : b * (p.T / p.B);
    return at < 0 ? 0 : at > p.T ? p.T : at;
}
// Tokens that a table row has room for.
__device__ __forceinline__ int room_of(const PageArgs& p) {
    const int64_t room = static_cast<int64_t>(p.width) * p.page;
    return room < 0x7fffffff ? static_cast<int>(room) : 0x7fffffff;
}
__device__ __forceinline__ int held_by(const PageArgs& p, int b) {
    const int n = p.lens[b], room = room_of(p);
    return n < 0 ? 0 : n > room ? room : n;
}
__device__ __forceinline__ Growth growth_of(const PageArgs& p, int b) {
    Growth g;
    g.first = first_row(p, b);
    g.next = first_row(p, b + 1);
    g.held = held_by(p, b);
    const int n = g.next > g.first ? g.next - g.first : 0, room = room_of(p);
    g.want = n < room - g.held ? g.held + n : room;
    g.old = pages_of(g.held, p.page);
    g.need = p.list ? pages_of(g.want, p.page) - g.old : 0;
    return g;
}

// Exclusive scan over the workgroup's threads; the last entry of `upto` has the sum of all.
__device__ __forceinline__ void block_scan(int mine, int* upto, int* waves) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int v = mine;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const int u = __shfl_up(v, off, 64);
        v += lane >= off ? u : 0;
    }
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; ++w) before += waves[w];
    upto[t] = before + v - mine;
    if (t == static_cast<int>(blockDim.x) - 1) upto[kThreads] = before + v;
    __syncthreads();
}

__global__ __launch_bounds__(kThreads) void append_kernel(PageArgs p) {
    __shared__ int upto[kThreads + 1], begin[kThreads], waves[kThreads / 64];
    const int t = threadIdx.x, threads = blockDim.x, span = (p.B + threads - 1) / threads;
    const int b0 = t * span < p.B ? t * span : p.B, b1 = b0 + span < p.B ? b0 + span : p.B;
    int need = 0, first = 0x7fffffff;
    for (int b = b0; b < b1; ++b) {
        const Growth g = growth_of(p, b);
        need += g.need;
        if (b == b0) first = g.first;
    }
    begin[t] = first;
    block_scan(need, upto, waves);
    const int64_t listed = p.list ? *p.count : 0;
    const int64_t count = listed < 0 ? 0 : listed < p.capacity ? listed : p.capacity;
    if (p.what & kPages)
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + t; i < p.T; i += static_cast<int64_t>(gridDim.x) * threads) {
            const int row = static_cast<int>(i);
            int lo = 0, hi = threads;            // the last thread whose sequences begin at or before this row
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (begin[mid] <= row) lo = mid;
                else hi = mid;
            }
            int b = lo * span, given = upto[lo];
            Growth g = growth_of(p, b);
            for (; b + 1 < p.B && b + 1 < (lo + 1) * span && g.next <= row; g = growth_of(p, ++b)) given += g.need;
            int64_t slot = -1, position = 0;
            if (row >= g.first && row < g.next) {
                position = static_cast<int64_t>(g.held) + (row - g.first);
                if (position < g.want) {
                    const int at = static_cast<int>(position) / p.page, in = static_cast<int>(position) - at * p.page;
                    int32_t* entry = p.table + b * p.table_row + at;
                    int page = -1;
                    if (!p.list || at < g.old) page = *entry;
                    else {
                        const int64_t from = count - 1 - given - (at - g.old);
                        if (from >= 0) {
                            page = p.list[from];
                            if (in == 0) *entry = page;
                        }
                    }
                    if (page >= 0) slot = static_cast<int64_t>(page) * p.page + in;
                }
            }
            p.slots[i] = slot;
            p.positions[i] = position;
        }
    if ((p.what & kState) && blockIdx.x == 0) {
        __syncthreads();                         // all have read: lens_out may be lens, count_out count
        int given = upto[t];
        for (int b = b0; b < b1; ++b) {
            const Growth g = growth_of(p, b);
            const int64_t have = count - given;
            const int got = have < 0 ? 0 : have < g.need ? static_cast<int>(have) : g.need;
            given += g.need;
            p.lens_out[b] = got == g.need ? g.want : (g.old + got) * p.page < g.want ? (g.old + got) * p.page : g.want;
        }
        if (p.list && t == 0) *p.count_out = static_cast<int32_t>(count - upto[kThreads]);
    }
}

__device__ __forceinline__ int kept_by(const PageArgs& p, int b) {
    const int held = held_by(p, b), keep = p.cu ? p.cu[b] : 0;
    return keep < 0 ? 0 : keep < held ? keep : held;
}

__global__ __launch_bounds__(kThreads) void truncate_kernel(PageArgs p) {
    __shared__ int upto[kThreads + 1], waves[kThreads / 64];
    const int t = threadIdx.x, threads = blockDim.x, span = (p.B + threads - 1) / threads;
    const int b0 = t * span < p.B ? t * span : p.B, b1 = b0 + span < p.B ? b0 + span : p.B;
    auto leaving = [&](int b) { return pages_of(held_by(p, b), p.page) - pages_of(kept_by(p, b), p.page); };
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += leaving(b);
    block_scan(sum, upto, waves);
    const int64_t listed = *p.count;
    const int64_t count = listed < 0 ? 0 : listed < p.capacity ? listed : p.capacity;
    if (p.what & kPages) {                       // a wave takes a sequence
        const int lane = t & 63, per = threads / 64;
        for (int b = blockIdx.x * per + (t >> 6); b < p.B; b += gridDim.x * per) {
            const int owner = b / span;
            int64_t to = count + upto[owner];
            for (int i = owner * span; i < b; ++i) to += leaving(i);
            const int from = pages_of(kept_by(p, b), p.page), n = leaving(b);
            for (int i = lane; i < n; i += 64)
                if (to + i < p.capacity) p.list[to + i] = p.table[b * p.table_row + from + i];
        }
    }
    if ((p.what & kState) && blockIdx.x == 0) {
        __syncthreads();                         // all have read: lens_out may be lens, count_out count
        for (int b = b0; b < b1; ++b) p.lens_out[b] = kept_by(p, b);
        if (t == 0) *p.count_out = static_cast<int32_t>(count + upto[kThreads]);
    }
}

bool meet(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

// other_state: append none, truncate seq_lens_out, which may be `keep` too.
int check_pages(const char* who, const PageArgs& a, int64_t page, int64_t width, int64_t B, int64_t capacity, const void* other_state) {
    if (page <= 0 || page > (1 << 20) || width <= 0 || width > 0x7fffffff || a.table_row < 0 || B <= 0 || B > (1 << 28) || capacity < 0 ||
        capacity > 0x7fffffff)
        return fail(MCV_ERR_SHAPE, "%s: bad shape B=%lld page_size=%lld table_width=%lld or free list", who, (long long)B, (long long)page, (long long)width);
    // what one workgroup writes while others read it: only in place as a whole
    if (a.lens_out != a.lens && meet(a.lens_out, 4 * B, a.lens, 4 * B))
        return fail(MCV_ERR_INVALID_ARG, "%s: seq_lens_out overlaps seq_lens without being it", who);
    if (a.cu && a.cu != other_state && meet(a.lens_out, 4 * B, a.cu, other_state ? 4 * B : 4 * B + 4))
        return fail(MCV_ERR_INVALID_ARG, "%s: seq_lens_out overlaps %s", who, other_state ? "keep without being it" : "cu_seqlens");
    return require_device();
}

// `items`, which a workgroup of 256 threads has `per` of in a pass. In place, what some workgroups read others may not write:
// then the state has a launch of its own, unless one workgroup does it all, which is faster up to `alone` items (apart: up to
// alone / 4). Append, us, one workgroup / several: 512 tokens apart 4.9, 4.5, in place 5.0, 7.6; 2048 7.3, 4.6, in place 7.5,
// 7.8; 4096 in place 11.4, 7.8. Over 512 sequences a thread has several to add up, and workgroups are of 1024 threads: 4000
// tokens of 1000 sequences apart 6.5, 7.6 with 256; 65536 of 300 5.9, 5.4. Truncate, in place: 32 sequences 4.9, 6.7; 64 7.0, 6.6.
int launch_pages(const char* who, void (*fn)(PageArgs), PageArgs& a, int64_t items, int64_t per, int64_t alone, mcv_stream_t stream) {
    const bool in_place = a.lens_out == a.lens || a.lens_out == a.cu || a.count_out == a.count;
    const bool one = items <= (in_place ? alone : alone / 4);
    const int threads = one || a.B > 512 ? kThreads : 256;
    a.what = !one && in_place ? kPages : kPages | kState;
    hipLaunchKernelGGL(fn, dim3(one ? 1 : static_cast<unsigned>(std::min<int64_t>(ceil_div(items, per * (threads / 256)), 1024))), dim3(threads), 0,
                       static_cast<hipStream_t>(stream), a);
    int rc = check_launch(who);
    if (rc != MCV_OK || (a.what & kState)) return rc;
    a.what = kState;
    hipLaunchKernelGGL(fn, dim3(1), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
    return check_launch(who);
}

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int mcv_paged_append(void* block_table, int64_t table_row, int64_t table_width, const void* seq_lens, const void* cu_seqlens,
                     int64_t B, int64_t T, int64_t page_size, const void* free_pages, int64_t free_capacity, const void* free_count,
                     void* slots, void* positions, void* seq_lens_out, void* free_count_out, mcv_stream_t stream) {
    const char* who = "paged_append";
    if (!block_table || !seq_lens || !seq_lens_out || (T > 0 && (!slots || !positions)) || (free_pages && (!free_count || !free_count_out)))
        return fail(MCV_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!free_pages && free_count_out) return fail(MCV_ERR_INVALID_ARG, "%s: free_count_out without free_pages", who);
    if (T < 0 || T > 0x7fffffff || (!cu_seqlens && B > 0 && T % B != 0)) return fail(MCV_ERR_SHAPE, "%s: bad shape B=%lld T=%lld", who, (long long)B, (long long)T);
    PageArgs a{static_cast<int32_t*>(block_table), static_cast<const int32_t*>(seq_lens), static_cast<const int32_t*>(cu_seqlens),
               static_cast<int32_t*>(const_cast<void*>(free_pages)), static_cast<const int32_t*>(free_count), static_cast<int64_t*>(slots),
               static_cast<int64_t*>(positions), static_cast<int32_t*>(seq_lens_out), static_cast<int32_t*>(free_count_out), table_row,
               free_capacity, static_cast<int>(table_width), static_cast<int>(page_size), static_cast<int>(B), static_cast<int>(T), 0};
    if (free_pages && B > 1 && table_row < table_width) return fail(MCV_ERR_SHAPE, "%s: rows of block_table overlap", who);
    int rc = check_pages(who, a, page_size, table_width, B, free_capacity, nullptr);
    if (rc != MCV_OK) return rc;
    return launch_pages("append_kernel", append_kernel, a, T, 256, 2 * kThreads, stream);
}

int mcv_paged_truncate(const void* block_table, int64_t table_row, int64_t table_width, const void* seq_lens, const void* keep,
                       int64_t B, int64_t page_size, void* free_pages, int64_t free_capacity, const void* free_count,
                       void* seq_lens_out, void* free_count_out, mcv_stream_t stream) {
    const char* who = "paged_truncate";
    if (!block_table || !seq_lens || !seq_lens_out || !free_pages || !free_count || !free_count_out) return fail(MCV_ERR_INVALID_ARG, "%s: null pointer", who);
    PageArgs a{static_cast<int32_t*>(const_cast<void*>(block_table)), static_cast<const int32_t*>(seq_lens), static_cast<const int32_t*>(keep),
               static_cast<int32_t*>(free_pages), static_cast<const int32_t*>(free_count), nullptr, nullptr, static_cast<int32_t*>(seq_lens_out),
               static_cast<int32_t*>(free_count_out), table_row, free_capacity, static_cast<int>(table_width), static_cast<int>(page_size),
               static_cast<int>(B), 0, 0};
    int rc = check_pages(who, a, page_size, table_width, B, free_capacity, seq_lens_out);
    if (rc != MCV_OK) return rc;
    return launch_pages("truncate_kernel", truncate_kernel, a, B, 4, 48, stream);
}

}  // extern "C"
