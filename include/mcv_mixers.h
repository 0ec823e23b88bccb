/*
 * mcv_mixers.h -- C-ABI of the token mixers that stand between a decoder layer's
 * quantised projections (mcv_quant.h, whose conventions hold here: device
 * pointers, fp16 as raw bits, stream-ordered calls that never allocate or
 * synchronise, shapes checked on the host before any launch).
 *
 * Strides are counted in elements.  fp16 operands are read 16 bytes at a time:
 * their pointers must be 16-byte aligned and their strides multiples of 8, with
 * the elements of one head contiguous (MCV_ERR_UNSUPPORTED otherwise).
 */
#ifndef MCV_MIXERS_H
#define MCV_MIXERS_H

#include "mcv_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------ gated delta rule -- */
/* The linear-attention layers' recurrence.  For every token t of a sequence and
 * every value head h (key head h / (Hv / Hk)), with S fp32 [Dk][Dv]:
 *   S <- exp(g_t) S;  u = beta_t (v_t - S^T k_t);  S <- S + k_t u^T;
 *   out_t = scale S^T q_t
 * normalize: q_t and k_t are divided by sqrt(|.|^2 + 1e-6) first.
 *
 *   q, k   fp16 [T][Hk][Dk]  (row and head strides)    out  fp16 [T][Hv][Dv]
 *   v      fp16 [T][Hv][Dv]  (row and head strides)
 *   g, beta  fp32 [T][Hv]    (row strides)
 *   state, state_out  fp32 [n_states][Hv][Dk][Dv]; state NULL: zeros.
 *          state_out may be state (in place).
 *   state_index  int32 [B]: the state of each sequence, NULL: its own number.
 *          A sequence whose index is outside [0, n_states) is skipped: its out
 *          rows are zero.  Two sequences must not share an index.
 *   cu_seqlens  int32 [B + 1]: sequence b is tokens cu[b] .. cu[b + 1] - 1 (none:
 *          its state is copied).  Values are clamped to [0, T]; tokens that no
 *          sequence holds leave their out rows as they are.  NULL: B sequences
 *          of T / B tokens each (T % B == 0).
 * Hv % Hk == 0, Dk 64 or 128, Dv a multiple of 16 up to 256.
 *
 * Sequences of a few tokens run the recurrence; long sequences run in
 * chunks of 64 tokens on the matrix cores, for which the call needs a workspace
 * of mcv_delta_rule_workspace_bytes(B, T, Hk, Hv, Dk, Dv) bytes, 256-byte aligned,
 * of any content (NULL or too small: the recurrence, however long).  Chunks hold
 * values and the state in two fp16 parts scaled by M, the largest |v| of the chunk
 * and the one before or what decay leaves of the M before (the first: the state's
 * largest): they are off by 2^-28 M at worst, and overflow where they grow past
 * 4096 M, which a stable rule (beta |k|^2 <= 2) does not do.  An infinity or NaN
 * in q, k, v, a gate or a state reaches what it reaches by the formulas, of its own
 * token and later ones; from there on the chunks may have NaN where the formulas
 * have an infinity.  The call's second launch reads what its first wrote into the
 * workspace: no other call may use it between them. */
int mcv_delta_rule(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                   const void* v, int64_t v_row, int64_t v_head, const void* g, int64_t g_row, const void* beta,
                   int64_t beta_row, const void* state, void* state_out, const void* state_index, int64_t n_states,
                   const void* cu_seqlens, int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv,
                   double scale, int normalize, void* out, void* workspace, int64_t workspace_bytes,
                   mcv_stream_t stream);
int64_t mcv_delta_rule_workspace_bytes(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk, int64_t Dv);

/* -------------------------------------------------------- paged attention -- */
/* Attention of one new token per sequence over a paged key-value cache:
 *   out[b][h] = sum_t softmax_t(scale q[b][h] . K[t][h / (Hq / Hkv)]) V[t][..]
 * over the t < seq_lens[b] that its pages hold.
 *   q, out  fp16 [B][Hq][D] (q: row and head strides; out contiguous)
 *   k_cache, v_cache  fp16 [pages][page_size][Hkv][D], page, token and head strides
 *   block_table  int32 [B][width] (row stride, 0 for one table of all): token t is
 *           row t % page_size of page block_table[b][t / page_size]
 *   seq_lens  int32 [B], clamped to [0, min(width * page_size, max_seq_len)]; a
 *           sequence of length 0 gives zeros
 * A page number outside [0, pages) is a page that is not there: its tokens are
 * left out, as masked ones.  What lies past a sequence's end is never used.
 * D is 64, 128 or 256; page_size a multiple of 16; Hq % Hkv == 0.
 * Long caches are split over workgroups, whose parts the last of them joins in
 * order (deterministic): workspace of mcv_paged_attention_workspace_bytes bytes,
 * 256-byte aligned, its first 4 KiB zero before its first use (every call leaves
 * them zero), for one call at a time; NULL or too small: no split.  The bytes for
 * a max_seq_len are enough for any shorter one. */
int mcv_paged_attention(const void* q, int64_t q_row, int64_t q_head, const void* k_cache, int64_t k_page,
                        int64_t k_token, int64_t k_head, const void* v_cache, int64_t v_page, int64_t v_token,
                        int64_t v_head, int64_t pages, int64_t page_size, const void* block_table,
                        int64_t table_row, int64_t table_width, const void* seq_lens, int64_t max_seq_len, int64_t B,
                        int64_t Hq, int64_t Hkv, int64_t D, double scale, void* out, void* workspace,
                        int64_t workspace_bytes, mcv_stream_t stream);
int64_t mcv_paged_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_seq_len);

/* ------------------------------------------------------- rotary positions -- */
/* Rotary positions with several axes (time, height, width): the pair (x[i],
 * x[i + rot / 2]) of a head's first `rot` elements turns by
 *   angle(t, i) = positions[axis[i]][t] freq[i]
 * computed in 64 bits; the elements from `rot` on are copied.
 *   q  fp16 [T][Hq][D], k fp16 [T][Hkv][D] (row and head strides); q_out, k_out the
 *      same with strides of their own; in place (q_out = q, k_out = k) is allowed
 *   positions  int64 [axes][T] (axis and token strides); freq  fp64 [rot / 2];
 *   axis  int32 [rot / 2], values clamped to [0, axes)
 * rot even, 2 <= rot <= D, D a multiple of 8 up to 512.
 * With k_cache: the rotated k and v (fp16 [T][Hkv][D]) go to row slots[t] %
 * page_size of page slots[t] / page_size of the caches (int64 slots; one outside
 * [0, pages * page_size) is written nowhere; no two tokens may share one), and
 * k_out is not used. */
int mcv_rotary_axes(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                    const void* positions, int64_t pos_axis, int64_t pos_token, int64_t axes, const void* freq,
                    const void* axis, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, int64_t rot, void* q_out,
                    int64_t qo_row, int64_t qo_head, void* k_out, int64_t ko_row, int64_t ko_head,
                    mcv_stream_t stream);
int mcv_rotary_axes_cached(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row, int64_t k_head,
                           const void* v, int64_t v_row, int64_t v_head, const void* positions, int64_t pos_axis,
                           int64_t pos_token, int64_t axes, const void* freq, const void* axis, int64_t T, int64_t Hq,
                           int64_t Hkv, int64_t D, int64_t rot, void* q_out, int64_t qo_row, int64_t qo_head,
                           void* k_cache, int64_t k_page, int64_t k_token, int64_t kc_head, void* v_cache,
                           int64_t v_page, int64_t v_token, int64_t vc_head, int64_t pages, int64_t page_size,
                           const void* slots, mcv_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif
