// The operators that serve a decoder token by token: launch parameters of the kernels in kern/cache_kernels.hip,
// kern/masked_attention_kernels.hip and kern/sample_kernels.hip. The arguments have been checked by serving.cpp, which holds the
// entry points of the C ABI.
#pragma once

#include <cstddef>
#include <cstdint>

struct ihipStream_t;

namespace kn {

// n / d for 0 <= n < 2^31 as a multiplication: with 2^(l - 1) < d <= 2^l the multiplier m = floor(2^(31 + l) / d) + 1 exceeds
// 2^(31 + l) / d by e / d, e <= d <= 2^l, so that n m / 2^(31 + l) exceeds n / d by less than 1 / d.
struct FastDiv {
    uint32_t d = 1, m = 0x80000001u, shift = 31;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor) {
        uint32_t l = 0;
        while ((1ull << l) < divisor) l++;
        shift = 31 + l;
        m = (uint32_t) ((1ull << shift) / divisor + 1);
    }
#ifdef __HIPCC__
    __host__ __device__
#endif
    uint32_t div(uint32_t n) const { return (uint32_t) (((uint64_t) n * m) >> shift); }
};

struct CacheParams {
    bool quantised;
    void *k, *v;
    float *k_scales, *v_scales;
    long long page_stride, head_stride, token_stride;
    int slots;  // pages * page_tokens
    int heads, width, tokens;
    FastDiv page_tokens, heads_div;
    bool rows_f32;
    void *rows_k, *rows_v;
    long long k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    const int32_t *row_slots;
};
int launch_cache_write(const CacheParams &p, ihipStream_t *stream);
int launch_cache_read(const CacheParams &p, ihipStream_t *stream);

// Both attentions. A sequence has up to two stretches of keys, the shared prefix and its own; keys of a prompt lie in
// one stretch without pages.
struct ServingAttentionParams {
    const void *q;
    void *out;
    long long q_batch, q_token, q_head, o_batch, o_token, o_head;
    const void *k, *v;
    long long k_batch, k_page, k_head, k_token, v_batch, v_page, v_head, v_token;  // (batch: prompts only, page: caches only)
    const float *k_scales, *v_scales;  // null: f16 keys and values
    int batch, queries, heads, kv_heads, width;
    int paged;  // 0: prompts
    int pages;  // of the cache
    FastDiv page_tokens;
    const int32_t *lengths, *tables, *prefix_table;
    long long table_stride;
    int table_tokens;   // table_pages * page_tokens, below 2^30
    int prefix_tokens;
    int keys;           // prompts: keys per batch entry
    float scale, cap;
    const float *slopes;
    int causal, window;
    const int32_t *spans, *prefix;  // prompts only
    // set by the launcher: rows that share a head of keys, partial results (in rows of the padded width) and where they lie
    FastDiv group_div, queries_div;
    float *part_values, *part_stats;  // [row][width], [row][reference, sum]
    int32_t *part_items;  // [stretch][first item, items], the prefix first
    int32_t *item_list;   // [item]: its sequence; null: looked up in the lengths (without a prefix among the stretches)
    long long row_prefix_part, row_own_part;
    int prefix_splits, own_splits;
    int prefix_inside;  // the workgroups of a sequence's own keys take the prefix as well
};
int launch_serving_attention(const ServingAttentionParams &p, void *workspace, ihipStream_t *stream);
size_t serving_attention_workspace(const ServingAttentionParams &p);

constexpr int SAMPLE_MAX_VOCAB = 1 << 20;
struct SampleParams {
    bool f16;
    int rows, vocab;
    const void *logits;
    long long row_stride;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *tokens;
    float *probabilities;
    int bits;  // set by the launcher: of the fixed point weights
};
int launch_sample(const SampleParams &p, void *workspace, ihipStream_t *stream);
size_t sample_workspace(const SampleParams &p);

}  // namespace kn
