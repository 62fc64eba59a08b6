// Attention over a paged cache and of whole prompts under caps, distance bias and masks (knhip_cached_attention,
// knhip_attention).
//
// Every mask of either operator is an interval of places per query, [lo, hi): causal and prefix mask end it, window and
// document begin it (serving_kernels.h). The softmax runs with a running maximum and sum in f32.
#include <hip/hip_runtime.h>

#include "../serving_kernels.h"

namespace kn {

namespace {

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8_any __attribute__((ext_vector_type(8), aligned(2)));

constexpr int WAVES = 4;
constexpr float LOG2E = 1.44269504088896340736f;

// One wave per query and head: lanes are keys for the scores and dims for the weighted sum.
__global__ __launch_bounds__(64 * WAVES) void masked_attention_kernel(ServingAttentionParams p) {
    __shared__ float qs[WAVES][128], ps[WAVES][64];
    __shared__ long long vo[WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long) blockIdx.x * WAVES + wave;
    const bool live_row = row < (long long) p.batch * p.queries * p.heads;
    const long long r = live_row ? row : 0;
    const int head = (int) (r % p.heads), t = (int) (r / p.heads % p.queries), b = (int) (r / p.heads / p.queries);
    const int kv_head = head / (p.heads / p.kv_heads);
    const _Float16 *q = (const _Float16 *) p.q + b * p.q_batch + t * p.q_token + head * p.q_head;
    for (int d = lane; d < p.width; d += 64) qs[wave][d] = (float) q[d];
    __syncthreads();

    int lo = 0, hi, at, keys[2] = {0, 0};
    if (p.paged) {
        const int length = min(max(p.lengths[b], 0), p.table_tokens);
        const int own = length - p.queries + t;
        at = p.prefix_tokens + own;
        keys[0] = p.prefix_tokens;
        keys[1] = length;
        hi = own < 0 ? 0 : at + 1;
        if (p.window) lo = max(lo, at - p.window + 1);
    } else {
        at = t + p.keys - p.queries;
        keys[1] = hi = p.keys;
        if (p.causal) hi = min(hi, max(at + 1, p.prefix ? p.prefix[b] : 0));
        if (p.window) lo = max(lo, at - p.window + 1);
        if (p.spans) {
            lo = max(lo, p.spans[2 * ((long long) b * p.queries + t)]);
            hi = min(hi, p.spans[2 * ((long long) b * p.queries + t) + 1]);
        }
    }
    const float slope = p.slopes ? p.slopes[head] : 0.0f;
    float top = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int part = 0; part < 2; part++) {
        const int base = part ? keys[0] : 0;  // place of the stretch's first key
        const int first = max(lo - base, 0), end = min(hi - base, keys[part]);
        for (int j0 = first; j0 < end; j0 += 64) {
            const int j = j0 + lane;
            float s = -INFINITY;
            long long v_at = -1;
            if (j < end) {
                long long k_at, scale_at = 0;
                bool there = true;
                if (p.paged) {
                    const unsigned n = p.page_tokens.div((unsigned) j), in = (unsigned) j - n * p.page_tokens.d;
                    const int page = part ? p.tables[b * p.table_stride + n] : p.prefix_table[n];
                    there = (unsigned) page < (unsigned) p.pages;
                    k_at = page * p.k_page + kv_head * p.k_head + in * p.k_token;
                    v_at = page * p.v_page + kv_head * p.v_head + in * p.v_token;
                    scale_at = ((long long) page * p.kv_heads + kv_head) * p.page_tokens.d + in;
                } else {
                    k_at = b * p.k_batch + kv_head * p.k_head + j * p.k_token;
                    v_at = b * p.v_batch + kv_head * p.v_head + j * p.v_token;
                }
                if (there) {
                    float dot = 0.0f;
                    if (p.k_scales) {
                        for (int d = 0; d < p.width; d++) dot += qs[wave][d] * (float) ((const signed char *) p.k)[k_at + d];
                        dot *= p.k_scales[scale_at];
                    } else {
                        for (int d = 0; d < p.width; d += 8) {
                            const halfx8 x = *(const halfx8_any *) ((const _Float16 *) p.k + k_at + d);
                            for (int i = 0; i < 8; i++) dot += qs[wave][d + i] * (float) x[i];
                        }
                    }
                    s = dot * p.scale;
                    if (p.cap > 0.0f) s = p.cap * tanhf(s / p.cap);
                    s -= slope * fabsf((float) (at - (base + j)));
                } else {
                    v_at = -1;
                }
            }
            float block_top = s;
            for (int m = 32; m; m >>= 1) block_top = fmaxf(block_top, __shfl_xor(block_top, m));
            const float new_top = fmaxf(top, block_top), ref = new_top == -INFINITY ? 0.0f : new_top;
            const float alpha = exp2f((top - ref) * LOG2E);
            float e = exp2f((s - ref) * LOG2E);
            top = new_top;
            float block_sum = e;
            for (int m = 32; m; m >>= 1) block_sum += __shfl_xor(block_sum, m);
            sum = sum * alpha + block_sum;
            if (v_at >= 0 && p.v_scales) {
                const unsigned n = p.page_tokens.div((unsigned) j), in = (unsigned) j - n * p.page_tokens.d;
                const int page = part ? p.tables[b * p.table_stride + n] : p.prefix_table[n];
                e *= p.v_scales[((long long) page * p.kv_heads + kv_head) * p.page_tokens.d + in];
            }
            ps[wave][lane] = e;
            vo[wave][lane] = v_at;
            __builtin_amdgcn_wave_barrier();
            for (int i = 0; i < 2; i++) {
                const int d = lane + 64 * i;
                acc[i] *= alpha;
                if (d >= p.width) continue;
                for (int u = 0; u < min(64, end - j0); u++)
                    if (vo[wave][u] >= 0)
                        acc[i] += ps[wave][u] * (p.v_scales ? (float) ((const signed char *) p.v)[vo[wave][u] + d] : (float) ((const _Float16 *) p.v)[vo[wave][u] + d]);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
    if (!live_row) return;
    _Float16 *o = (_Float16 *) p.out + b * p.o_batch + t * p.o_token + head * p.o_head;
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    for (int i = 0; i < 2; i++)
        if (lane + 64 * i < p.width) o[lane + 64 * i] = (_Float16) (acc[i] * inv);
}

}  // namespace

size_t serving_attention_workspace(const ServingAttentionParams &) { return 0; }

int launch_serving_attention(const ServingAttentionParams &p, void *, ihipStream_t *stream) {
    const long long rows = (long long) p.batch * p.queries * p.heads;
    hipLaunchKernelGGL(masked_attention_kernel, dim3((unsigned) ((rows + WAVES - 1) / WAVES)), dim3(64 * WAVES), 0, stream, p);
    return (int) hipGetLastError();
}

}  // namespace kn
