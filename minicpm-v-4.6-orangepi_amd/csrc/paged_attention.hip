// paged_attention.hip -- attention of one new token over a paged cache, gfx950.
#include "mixers.h"

namespace mcv {
namespace {

struct AttnArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;
    const int32_t* lens;
    uint16_t* out;
    int64_t q_row, q_head, k_page, k_token, k_head, v_page, v_token, v_head, table_row;
    int pages, page_size, max_len, Hq, group;
    float scale;
};

// One wave per (sequence, q head): its lanes share out the elements of a head,
// tokens one after the other with the running maximum and sum of the softmax.
template <int D>
__global__ __launch_bounds__(64) void attn_simple_kernel(AttnArgs p) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x, h = blockIdx.x % p.Hq, b = blockIdx.x / p.Hq, hk = h / p.group;
    int len = p.lens[b];
    len = len > p.max_len ? p.max_len : len;
    float q[E], acc[E] = {}, m = -INFINITY, sum = 0.f;
    for (int e = 0; e < E; ++e) q[e] = h2f(p.q[b * p.q_row + h * p.q_head + lane * E + e]) * p.scale;
    for (int t = 0; t < len; ++t) {
        const int page = p.table[b * p.table_row + t / p.page_size];
        if (page < 0 || page >= p.pages) continue;
        const uint16_t* kp = p.k + page * p.k_page + (t % p.page_size) * p.k_token + hk * p.k_head + lane * E;
        const uint16_t* vp = p.v + page * p.v_page + (t % p.page_size) * p.v_token + hk * p.v_head + lane * E;
        float s = 0.f;
        for (int e = 0; e < E; ++e) s = fmaf(q[e], h2f(kp[e]), s);
        s = wave_butterfly(s, [](float x, float y) { return x + y; });
        const float top = fmaxf(m, s);
        if (top == -INFINITY) continue;
        const float keep = expf(m - top), w = expf(s - top);
        sum = sum * keep + w;
        for (int e = 0; e < E; ++e) acc[e] = acc[e] * keep + w * h2f(vp[e]);
        m = top;
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    for (int e = 0; e < E; ++e) p.out[(static_cast<int64_t>(b) * p.Hq + h) * D + lane * E + e] = f2h(sum > 0.f ? acc[e] * inv : 0.f);
}

}  // namespace
}  // namespace mcv

using namespace mcv;

extern "C" {

int64_t mcv_paged_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seq_len) {
    (void)B, (void)Hq, (void)Hkv, (void)D, (void)max_seq_len;
    return 0;
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
    // (width counted in pages first: width * page_size could pass 64 bits)
    const int64_t held = table_width > (int64_t(1) << 30) / page_size ? int64_t(1) << 30 : table_width * page_size;
    const int64_t most = max_seq_len < held ? max_seq_len : held;
    AttnArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache),
               static_cast<const int32_t*>(block_table), static_cast<const int32_t*>(seq_lens), static_cast<uint16_t*>(out),
               q_row, q_head, k_page, k_token, k_head, v_page, v_token, v_head, table_row, static_cast<int>(pages),
               static_cast<int>(page_size), static_cast<int>(most), static_cast<int>(Hq), static_cast<int>(Hq / Hkv),
               static_cast<float>(scale)};
    auto fn = D == 64 ? attn_simple_kernel<64> : D == 128 ? attn_simple_kernel<128> : attn_simple_kernel<256>;
    hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(B * Hq)), dim3(64), 0, static_cast<hipStream_t>(stream), a);
    return check_launch("attn_simple_kernel");
}

}  // extern "C"
