// Arguments and launch plan of attention over the 4-bit key/value cache.
#pragma once

#include "../../include/w4a16_b200.h"
#include "kv4.cuh"

namespace w4 {

struct Kv4AttentionArgs {
    Kv4View c;
    const __half* q;
    void* out;
    float* lse;              // may be null
    float* part_o;           // parts: unnormalised sums [CTA][first, last][row][128] ...
    float2* part_ml;         // ... and maximum (base 2) and sum of weights
    float scale;
    int group, q_stride;
};
struct Kv4WeightArgs {
    Kv4View c;
    const __half* q;
    const float* lse;
    float scale;
    int group, q_stride;
    int positions;           // of a CTA; the launch chooses
};
// How a call is cut; a function of its sizes alone, so that the workspace can be sized without a device.
struct Kv4AttentionPlan {
    int nt, ctas;
    long long tile_heads, ml_offset, bytes;
};
Kv4AttentionPlan kv4_attention_plan(int num_tokens, int num_seqs, int q_heads, int kv_heads);
int kv4_attention(Kv4AttentionArgs a, int q_heads, bool f32, void* workspace, cudaStream_t stream);
// The form for many query rows and an fp16 result (kv4_attention_tc.cu).
struct Kv4ChunkArgs {
    Kv4View c;
    const __half* q;
    __half* out;
    float* lse;              // may be null
    float* part_o;           // splits: unnormalised sums [tile][head][split][row][128] ...
    float2* part_ml;         // ... and maximum (base 2) and sum of weights
    float scale;
    int group, q_stride, splits;
};
struct Kv4ChunkPlan {
    int splits;
    long long tile_heads, ml_offset, bytes;
};
Kv4ChunkPlan kv4_chunk_plan(int num_tokens, int num_seqs, int q_heads, int kv_heads);
int kv4_chunk_attention(Kv4ChunkArgs a, int q_heads, void* workspace, cudaStream_t stream);
int kv4_chunk_set_attributes();
int kv4_chunk_timeouts(unsigned int* out);
// Which form a call takes: the tensor-memory kernel for fp16 results of at least 64 query rows a sequence and head.
inline bool kv4_takes_chunk(int num_tokens, int num_seqs, int q_heads, int kv_heads, bool f32) {
    return !f32 && static_cast<long long>(q_heads / kv_heads) * num_tokens >= 64ll * num_seqs;
}
int kv4_check_step(const w4a16_kv4_cache* cache, const w4a16_kv4_batch* batch, int num_q_heads, float softmax_scale, const int32_t* position,
                   const float* inv_freq, const w4a16_qwenbin_biases* biases, Kv4View* view);
int kv4_add_key_weights(Kv4WeightArgs a, cudaStream_t stream);

struct Kv4AppendArgs {
    const __half *q, *k, *v, *q_bias, *k_bias, *v_bias;
    __half* q_out;
    const int32_t* positions;
    const float* inv_freq;
    int q_heads, q_stride, kv_stride;
};
struct Kv4EvictArgs {
    const int32_t* dst_table;
    int32_t *new_lens, *kept;
    int dst_pages, budget, sink, recent;
};
int kv4_append(const Kv4View& c, const Kv4AppendArgs& x, cudaStream_t stream);
int kv4_read(const Kv4View& c, __half* k_out, __half* v_out, cudaStream_t stream);
int kv4_set_attributes();
int kv4_evict(const Kv4View& c, const Kv4EvictArgs& x, cudaStream_t stream);

}  // namespace w4
