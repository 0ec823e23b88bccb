// delta_rule.h -- what the gated delta rule's two forms share.
#pragma once

#include "mixers.h"

namespace mcv {

constexpr float kDeltaEps = 1e-6f;               // of the norms of q and k

struct DeltaArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const float* g;
    const float* beta;
    const float* state;
    float* state_out;
    const int32_t* state_index;
    const int32_t* cu;
    uint16_t* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, beta_row, n_states;
    int T, B, per_seq, Hv, group, Dv;            // per_seq: tokens of every sequence where cu is null
    float scale;
    int normalize;
    int short_below;                             // sequences of fewer tokens are the recurrence's, the others the chunks'; 0: all one's
};

// First token and one past the last of sequence b, whatever cu holds.
__device__ __forceinline__ void delta_span(const DeltaArgs& p, int b, int& t0, int& t1) {
    t0 = p.cu ? p.cu[b] : b * p.per_seq;
    t1 = p.cu ? p.cu[b + 1] : t0 + p.per_seq;
    t0 = t0 < 0 ? 0 : t0 > p.T ? p.T : t0;
    t1 = t1 < t0 ? t0 : t1 > p.T ? p.T : t1;
}

// The chunked form (delta_chunk.hip).
int64_t delta_chunk_workspace(int64_t B, int64_t T, int64_t Hk, int64_t Hv, int64_t Dk);
int launch_delta_chunk(const DeltaArgs& a, int Hk, int Dk, void* workspace, int64_t workspace_bytes, hipStream_t stream);

}  // namespace mcv
