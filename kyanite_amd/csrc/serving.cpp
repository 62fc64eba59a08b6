// Entry points of the operators that serve a decoder token by token (include/knhip.h): checks of the arguments, and the
// launch parameters of the kernels declared in serving_kernels.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdlib>

#include "../../include/knhip.h"
#include "executor.h"
#include "matmul_api.h"
#include "serving_kernels.h"

using namespace kn;

namespace {

template <typename F>
int guarded(F f) {
    try {
        f();
        return KNHIP_OK;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return KNHIP_ERROR;
    } catch (...) {
        set_last_error("unknown failure");
        return KNHIP_ERROR;
    }
}

void select_device(int device) {
    HipDevice::check(device);
    hip_check(hipSetDevice(device), "hipSetDevice");
    (void) hipGetLastError();  // (what an earlier call left, an allocation that failed for one, would be taken for the launch's)
}

void require_aligned(const char *what, const char *name, const void *ptr, size_t bytes) {
    if ((uintptr_t) ptr % bytes != 0) fail(what, ": ", name, " must be ", bytes, " byte aligned");
}

void require_address(const char *what, const char *name, const void *ptr, size_t alignment) {
    if (ptr == nullptr) fail(what, ": ", name, " is null");
    require_aligned(what, name, ptr, alignment);
}

void check_workspace(const char *what, size_t need, const void *workspace, size_t workspace_bytes) {
    if (need == 0) return;
    if (workspace == nullptr || workspace_bytes < need) fail(what, ": needs ", need, " bytes of workspace, got ", workspace == nullptr ? 0 : workspace_bytes);
    require_aligned(what, "the workspace", workspace, 256);
}

// Whether rows of `width` elements at these strides may share memory: going from the smallest stride to the largest, each has to
// step over all that lies below it.
template <size_t N>
bool rows_overlap(const int64_t (&strides)[N], const int (&counts)[N], int width) {
    size_t order[N], axes = 0;
    for (size_t i = 0; i < N; i++)
        if (counts[i] > 1) order[axes++] = i;
    std::sort(order, order + axes, [&](size_t a, size_t b) { return std::llabs(strides[a]) < std::llabs(strides[b]); });
    int64_t reach = width;
    for (size_t i = 0; i < axes; i++) {
        const int64_t stride = std::llabs(strides[order[i]]);
        if (stride < reach) return true;
        if (stride > INT64_MAX / 4 / counts[order[i]]) return false;  // (no memory is that large)
        reach += stride * (counts[order[i]] - 1);
    }
    return false;
}

// (sizes first: an empty cache or call has no addresses to check)
void check_cache_sizes(const char *what, const knhip_kv_cache &c) {
    if (c.dtype != KNHIP_F16 && c.dtype != KNHIP_I8) fail(what, ": a cache holds f16 or i8, got dtype code ", c.dtype);
    if (c.pages < 0 || c.heads < 0 || c.page_tokens < 1) fail(what, ": a cache of ", c.pages, " pages of ", c.page_tokens, " tokens and ", c.heads, " heads");
    if (c.width < 16 || c.width > 256 || c.width % 16 != 0) fail(what, ": the width must be a multiple of 16 up to 256, got ", c.width);
    if ((long long) c.pages * c.page_tokens > INT_MAX) fail(what, ": pages * page_tokens must stay below 2^31");
}

void check_cache_addresses(const char *what, const knhip_kv_cache &c) {
    const int64_t elem = c.dtype == KNHIP_F16 ? 2 : 1;
    require_address(what, "the cache's k", c.k, 16);
    require_address(what, "the cache's v", c.v, 16);
    // rows that overlap could not hold what is written into them
    const int64_t strides[3] = {c.page_stride, c.head_stride, c.token_stride};
    const int counts[3] = {c.pages, c.heads, c.page_tokens};
    const char *names[3] = {"page", "head", "token"};
    for (int i = 0; i < 3; i++) {
        if (counts[i] <= 1) continue;
        if (strides[i] < c.width) fail(what, ": the cache's ", names[i], " stride ", strides[i], " is less than a row of ", c.width);
        if (strides[i] * elem % 16 != 0) fail(what, ": the cache's ", names[i], " stride must be a multiple of 16 bytes, got ", strides[i], " elements");
        if (strides[i] > (int64_t) 1 << 46) fail(what, ": the cache's ", names[i], " stride is out of range");
    }
    if (rows_overlap(strides, counts, c.width)) fail(what, ": rows of the cache may not overlap, got strides of ", strides[0], ", ", strides[1], ", ", strides[2]);
    if (c.dtype == KNHIP_I8) {
        require_address(what, "k_scales", c.k_scales, 4);
        require_address(what, "v_scales", c.v_scales, 4);
    }
}

// true when there is nothing to do
bool check_rows(const char *what, const knhip_kv_cache *cache, const knhip_cache_rows *rows, bool write, CacheParams &p) {
    if (cache == nullptr || rows == nullptr) fail(what, ": null argument");
    check_cache_sizes(what, *cache);
    if (rows->dtype != KNHIP_F16 && rows->dtype != KNHIP_F32) fail(what, ": rows are f16 or f32, got dtype code ", rows->dtype);
    if (rows->tokens < 0) fail(what, ": negative size");
    // (a launch has less than 2^32 threads, in workgroups of 8 rows or more with up to 32 lanes each)
    if ((long long) rows->tokens * cache->heads > (1 << 27) - 8) fail(what, ": tokens * heads must stay below 2^27 - 7");
    if (rows->tokens == 0 || cache->heads == 0) return true;
    if (cache->pages > 0) check_cache_addresses(what, *cache);
    const size_t elem = rows->dtype == KNHIP_F16 ? 2 : 4;
    require_address(what, "the rows' k", rows->k, elem);
    require_address(what, "the rows' v", rows->v, elem);
    require_address(what, "slots", rows->slots, 4);
    if (!write) {
        const int64_t k_strides[2] = {rows->k_token_stride, rows->k_head_stride}, v_strides[2] = {rows->v_token_stride, rows->v_head_stride};
        const int counts[2] = {rows->tokens, cache->heads};
        if (rows_overlap(k_strides, counts, cache->width) || rows_overlap(v_strides, counts, cache->width))
            fail(what, ": rows that are written may not overlap, got strides of ", k_strides[0], ", ", k_strides[1], " and ", v_strides[0], ", ", v_strides[1],
                 " for rows of ", cache->width);
    }
    p.quantised = cache->dtype == KNHIP_I8;
    p.k = cache->k;
    p.v = cache->v;
    p.k_scales = cache->k_scales;
    p.v_scales = cache->v_scales;
    p.page_stride = cache->page_stride;
    p.head_stride = cache->head_stride;
    p.token_stride = cache->token_stride;
    p.slots = cache->pages * cache->page_tokens;
    p.heads = cache->heads;
    p.width = cache->width;
    p.tokens = rows->tokens;
    p.page_tokens = FastDiv((uint32_t) cache->page_tokens);
    p.heads_div = FastDiv((uint32_t) cache->heads);
    p.rows_f32 = rows->dtype == KNHIP_F32;
    p.rows_k = rows->k;
    p.rows_v = rows->v;
    p.k_token_stride = rows->k_token_stride;
    p.k_head_stride = rows->k_head_stride;
    p.v_token_stride = rows->v_token_stride;
    p.v_head_stride = rows->v_head_stride;
    p.row_slots = rows->slots;
    return write && p.slots == 0;  // (a read of a cache without pages gives zeros)
}

void check_scores(const char *what, float scale, float cap, int window, const float *slopes) {
    // (in units of log2 too)
    if (!std::isfinite(scale * 1.5f)) fail(what, ": the scale must be finite");
    if (!(cap >= 0.0f) || !std::isfinite(cap * 1.5f)) fail(what, ": the cap must be finite and not negative");
    if (cap > 0.0f && !std::isfinite(std::max(std::fabs(scale), 1.0f) * 1.5f / cap)) fail(what, ": the cap is too small for the scale");
    if (window < 0) fail(what, ": the window must not be negative");
    if (slopes != nullptr) require_aligned(what, "slopes", slopes, 4);
}

void check_result_strides(const char *what, int64_t batch_stride, int64_t token_stride, int64_t head_stride, int batch, int tokens, int heads, int width) {
    const int64_t strides[3] = {batch_stride, token_stride, head_stride};
    const int counts[3] = {batch, tokens, heads};
    if (rows_overlap(strides, counts, width))
        fail(what, ": rows of out may not overlap, got strides of ", strides[0], ", ", strides[1], ", ", strides[2], " for rows of ", width);
}

// true when there is nothing to do
bool plan_cached_attention(const knhip_cached_attention_args *args, ServingAttentionParams &p) {
    const char *what = "cached_attention";
    if (args == nullptr) fail(what, ": null argument");
    const knhip_cached_attention_args &a = *args;
    const knhip_kv_cache &c = a.cache;
    check_cache_sizes(what, c);
    if (c.width > 128) fail(what, ": the width must be at most 128, got ", c.width);
    if (a.batch < 0 || a.queries < 0 || a.heads < 0 || a.table_pages < 0 || a.prefix_tokens < 0) fail(what, ": negative size");
    check_scores(what, a.scale, a.cap, a.window, a.slopes);
    if (a.batch == 0 || a.queries == 0 || a.heads == 0) return true;
    if (c.heads < 1 || a.heads % c.heads != 0) fail(what, ": ", a.heads, " heads cannot share ", c.heads, " heads of the cache evenly");
    if ((long long) a.batch * c.heads >= 1 << 22) fail(what, ": batch * heads of the cache must stay below 2^22");
    if ((long long) a.batch * a.queries * a.heads > INT_MAX / 128) fail(what, ": batch * queries * heads must stay below 2^24");
    // (pages may occur in several tables, so that the places of a sequence may outnumber the slots of the cache)
    const long long table_tokens = (long long) a.table_pages * c.page_tokens;
    if (table_tokens + a.prefix_tokens > INT_MAX / 2) fail(what, ": prefix_tokens + table_pages * page_tokens must stay below 2^30");
    if (c.pages > 0) check_cache_addresses(what, c);
    require_address(what, "q", a.q, 2);
    require_address(what, "out", a.out, 2);
    require_address(what, "lengths", a.lengths, 4);
    if (a.table_pages > 0) require_address(what, "tables", a.tables, 4);
    if (a.prefix_tokens > 0) require_address(what, "prefix_table", a.prefix_table, 4);
    check_result_strides(what, a.out_batch_stride, a.out_token_stride, a.out_head_stride, a.batch, a.queries, a.heads, c.width);
    p = ServingAttentionParams();
    p.q = a.q;
    p.out = a.out;
    p.q_batch = a.q_batch_stride; p.q_token = a.q_token_stride; p.q_head = a.q_head_stride;
    p.o_batch = a.out_batch_stride; p.o_token = a.out_token_stride; p.o_head = a.out_head_stride;
    p.k = c.k;
    p.v = c.v;
    p.k_page = p.v_page = c.page_stride;
    p.k_head = p.v_head = c.head_stride;
    p.k_token = p.v_token = c.token_stride;
    if (c.dtype == KNHIP_I8) {
        p.k_scales = c.k_scales;
        p.v_scales = c.v_scales;
    }
    p.batch = a.batch;
    p.queries = a.queries;
    p.heads = a.heads;
    p.kv_heads = c.heads;
    p.width = c.width;
    p.paged = 1;
    p.pages = c.pages;
    p.page_tokens = FastDiv((uint32_t) c.page_tokens);
    p.lengths = a.lengths;
    p.tables = a.tables;
    p.prefix_table = a.prefix_table;
    p.table_stride = a.table_stride;
    p.table_tokens = (int) table_tokens;
    p.prefix_tokens = a.prefix_tokens;
    p.scale = a.scale;
    p.cap = a.cap;
    p.slopes = a.slopes;
    p.causal = 1;
    p.window = std::min(a.window, 1 << 30);  // (no place is further away; keeps differences of places inside 32 bits)
    return false;
}

bool plan_attention(const knhip_attention_args *args, ServingAttentionParams &p) {
    const char *what = "attention";
    if (args == nullptr) fail(what, ": null argument");
    const knhip_attention_args &a = *args;
    if (a.batch < 0 || a.queries < 0 || a.keys < 0 || a.heads < 0) fail(what, ": negative size");
    if (a.width < 8 || a.width > 128 || a.width % 8 != 0) fail(what, ": the width must be a multiple of 8 up to 128, got ", a.width);
    check_scores(what, a.scale, a.cap, a.window, a.slopes);
    if (a.batch == 0 || a.queries == 0 || a.heads == 0) return true;
    if (a.kv_heads < 1 || a.heads % a.kv_heads != 0) fail(what, ": ", a.heads, " heads cannot share ", a.kv_heads, " heads of keys evenly");
    if ((long long) a.batch * a.kv_heads >= 1 << 22) fail(what, ": batch * kv_heads must stay below 2^22");
    if ((long long) a.batch * a.queries * a.heads > INT_MAX / 16) fail(what, ": batch * queries * heads must stay below 2^27");
    if (a.keys > INT_MAX / 2 || a.queries > INT_MAX / 2) fail(what, ": queries and keys must stay below 2^30");
    require_address(what, "q", a.q, 2);
    require_address(what, "out", a.out, 2);
    if (a.keys > 0) {
        require_address(what, "k", a.k, 2);
        require_address(what, "v", a.v, 2);
    }
    if (a.spans != nullptr) require_aligned(what, "spans", a.spans, 4);
    if (a.prefix != nullptr) require_aligned(what, "prefix", a.prefix, 4);
    check_result_strides(what, a.out_batch_stride, a.out_token_stride, a.out_head_stride, a.batch, a.queries, a.heads, a.width);
    p = ServingAttentionParams();
    p.q = a.q;
    p.out = a.out;
    p.q_batch = a.q_batch_stride; p.q_token = a.q_token_stride; p.q_head = a.q_head_stride;
    p.o_batch = a.out_batch_stride; p.o_token = a.out_token_stride; p.o_head = a.out_head_stride;
    p.k = a.k;
    p.v = a.v;
    p.k_batch = a.k_batch_stride; p.k_token = a.k_token_stride; p.k_head = a.k_head_stride;
    p.v_batch = a.v_batch_stride; p.v_token = a.v_token_stride; p.v_head = a.v_head_stride;
    p.batch = a.batch;
    p.queries = a.queries;
    p.heads = a.heads;
    p.kv_heads = a.kv_heads;
    p.width = a.width;
    p.keys = a.keys;
    p.scale = a.scale;
    p.cap = a.cap;
    p.slopes = a.slopes;
    p.causal = a.causal != 0;
    p.window = std::min(a.window, 1 << 30);  // (no place is further away; keeps differences of places inside 32 bits)
    p.spans = a.spans;
    p.prefix = a.prefix;
    return false;
}

bool plan_sample(const knhip_sample_args *args, SampleParams &p) {
    const char *what = "sample";
    if (args == nullptr) fail(what, ": null argument");
    const knhip_sample_args &a = *args;
    if (a.dtype != KNHIP_F16 && a.dtype != KNHIP_F32) fail(what, ": logits are f16 or f32, got dtype code ", a.dtype);
    if (a.rows < 0 || a.vocab < 0) fail(what, ": negative size");
    if (a.vocab > SAMPLE_MAX_VOCAB) fail(what, ": at most ", SAMPLE_MAX_VOCAB, " logits per row, got ", a.vocab);
    if (a.rows > (1 << 20)) fail(what, ": at most 2^20 rows, got ", a.rows);
    if (a.rows == 0) return true;
    if (a.vocab > 0) require_address(what, "logits", a.logits, a.dtype == KNHIP_F16 ? 2 : 4);
    require_address(what, "uniform", a.uniform, 4);
    require_address(what, "tokens", a.tokens, 4);
    const void *optional[5] = {a.temperature, a.top_k, a.top_p, a.min_p, a.probabilities};
    for (const void *ptr : optional)
        if (ptr != nullptr) require_aligned(what, "an array with an entry per row", ptr, 4);
    p = SampleParams();
    p.f16 = a.dtype == KNHIP_F16;
    p.rows = a.rows;
    p.vocab = a.vocab;
    p.logits = a.logits;
    p.row_stride = a.row_stride;
    p.temperature = a.temperature;
    p.top_k = a.top_k;
    p.top_p = a.top_p;
    p.min_p = a.min_p;
    p.uniform = a.uniform;
    p.tokens = a.tokens;
    p.probabilities = a.probabilities;
    return false;
}

}  // namespace

extern "C" {

int knhip_cache_write(int device, void *stream, const knhip_kv_cache *cache, const knhip_cache_rows *rows) {
    return guarded([&] {
        CacheParams p;
        if (check_rows("cache_write", cache, rows, true, p)) return;
        select_device(device);
        hip_check((hipError_t) launch_cache_write(p, (ihipStream_t *) stream), "cache_write launch");
    });
}

int knhip_cache_read(int device, void *stream, const knhip_kv_cache *cache, const knhip_cache_rows *rows) {
    return guarded([&] {
        CacheParams p;
        if (check_rows("cache_read", cache, rows, false, p)) return;
        select_device(device);
        hip_check((hipError_t) launch_cache_read(p, (ihipStream_t *) stream), "cache_read launch");
    });
}

int knhip_cached_attention_workspace_bytes(const knhip_cached_attention_args *args, size_t *bytes) {
    return guarded([&] {
        if (bytes == nullptr) fail("cached_attention: null argument");
        ServingAttentionParams p;
        *bytes = plan_cached_attention(args, p) ? 0 : serving_attention_workspace(p);
    });
}

int knhip_cached_attention(int device, void *stream, const knhip_cached_attention_args *args, void *workspace, size_t workspace_bytes) {
    return guarded([&] {
        ServingAttentionParams p;
        if (plan_cached_attention(args, p)) return;
        check_workspace("cached_attention", serving_attention_workspace(p), workspace, workspace_bytes);
        select_device(device);
        hip_check((hipError_t) launch_serving_attention(p, workspace, (ihipStream_t *) stream), "cached_attention launch");
    });
}

int knhip_attention_workspace_bytes(const knhip_attention_args *args, size_t *bytes) {
    return guarded([&] {
        if (bytes == nullptr) fail("attention: null argument");
        ServingAttentionParams p;
        *bytes = plan_attention(args, p) ? 0 : serving_attention_workspace(p);
    });
}

int knhip_attention(int device, void *stream, const knhip_attention_args *args, void *workspace, size_t workspace_bytes) {
    return guarded([&] {
        ServingAttentionParams p;
        if (plan_attention(args, p)) return;
        check_workspace("attention", serving_attention_workspace(p), workspace, workspace_bytes);
        select_device(device);
        hip_check((hipError_t) launch_serving_attention(p, workspace, (ihipStream_t *) stream), "attention launch");
    });
}

int knhip_sample_workspace_bytes(const knhip_sample_args *args, size_t *bytes) {
    return guarded([&] {
        if (bytes == nullptr) fail("sample: null argument");
        SampleParams p;
        *bytes = plan_sample(args, p) ? 0 : sample_workspace(p);
    });
}

int knhip_sample(int device, void *stream, const knhip_sample_args *args, void *workspace, size_t workspace_bytes) {
    return guarded([&] {
        SampleParams p;
        if (plan_sample(args, p)) return;
        check_workspace("sample", sample_workspace(p), workspace, workspace_bytes);
        select_device(device);
        hip_check((hipError_t) launch_sample(p, workspace, (ihipStream_t *) stream), "sample launch");
    });
}

}  // extern "C"
