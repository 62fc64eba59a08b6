// Attention over a paged cache and of whole prompts under caps, distance bias and masks (knhip_cached_attention,
// knhip_attention), f16 or quantised keys and values, on the CDNA4 matrix cores.
//
// Every mask of either operator is an interval [lo, hi) of keys per query: causal and prefix mask end it, window and document
// begin it. Blocks of keys that no query of a workgroup sees are not fetched, blocks that all of them see whole run
// without a comparison.
//
// The rows of a product are the queries that read the same head of keys: all heads of its group times all tokens, so
// that a block of keys is fetched once for them. Three kernels:
//   tile_attention_kernel   32 rows per wave, 128 or 256 per workgroup: prompts, prompts over a cache, and the shared prefix of a batch, whose
//                           rows are the queries of ALL sequences
//   row_attention_kernel    up to 16 or 32 rows per workgroup: the few queries of one sequence over its own keys, and over a
//                           prefix that is short
//   join_attention_kernel   the softmax of parts: keys are split between workgroups where rows are few, and a sequence with
//                           a prefix has its own part and the prefix's
// Scores are computed transposed, S^T = K Q^T, so that a lane owns a query and the accumulators of S^T are the operands of
// O^T += V^T P^T. The softmax runs in f32 in units of log2, with a running reference that follows the maximum lazily:
// it moves when a score exceeds it by more than SLACK. Weights enter the second product as f16 and are 2^LIFT at the reference, so that
// they use the type's range: at most 2^15, and normal numbers (rounded by half of 2^-10, the type's step) down to 2^-21 of the
// reference's. Their sum is that of the f32 numbers before the rounding, times 2^LIFT like them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../serving_kernels.h"

namespace kn {

namespace {

typedef _Float16 half_t;
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
// rows of prompts may start at any element: the hardware takes under-aligned 128 bit accesses
typedef _Float16 halfx8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 halfx4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float SLACK = 8.0f, LIFT = 7.0f;
constexpr int WAVES = 4;

// ---- which keys a query sees ---------------------------------------------------------------------------------------

enum Stretch { PROMPT, OWN, PREFIX };  // whose keys a workgroup reads

struct Row {
    int b, t, head;
    int at;      // place of the query, counted from the first key of the stretch
    int lo, hi;  // the keys of the stretch that it sees
};

__device__ __forceinline__ int own_length(const ServingAttentionParams &p, int b) { return min(max(p.lengths[b], 0), p.table_tokens); }

// Row `r` of kv head `kv_head`: (token, head of the group) of sequence `b`, of all sequences for the prefix
// (`length`: of the sequence, when the caller has it)
template <int STRETCH>
__device__ __forceinline__ Row row_of(const ServingAttentionParams &p, unsigned r, int b, int kv_head, int length = -1) {
    Row w;
    const unsigned token = p.group_div.div(r);
    w.head = kv_head * (int) p.group_div.d + (int) (r - token * p.group_div.d);
    w.b = b;
    w.t = (int) token;
    if (STRETCH == PREFIX) {
        w.b = (int) p.queries_div.div(token);
        w.t = (int) (token - (unsigned) w.b * p.queries_div.d);
    }
    w.lo = 0;
    if (STRETCH == PROMPT) {
        w.at = w.t + p.keys - p.queries;
        w.hi = p.keys;
        if (p.causal) w.hi = min(w.hi, max(w.at + 1, p.prefix ? p.prefix[w.b] : 0));
    } else {
        const int own = (length >= 0 ? length : own_length(p, w.b)) - p.queries + w.t;  // below 0: a query of padding
        w.at = STRETCH == OWN ? own : p.prefix_tokens + own;
        w.hi = own < 0 ? 0 : STRETCH == OWN ? own + 1 : p.prefix_tokens;
    }
    if (p.window) w.lo = max(w.lo, w.at - p.window + 1);
    if (STRETCH == PROMPT && p.spans) {
        const int2 span = *(const int2 *) (p.spans + 2 * ((long long) w.b * p.queries + w.t));
        w.lo = max(w.lo, span.x);
        w.hi = min(w.hi, span.y);
    }
    if (w.lo >= w.hi) w.lo = w.hi = 0;
    return w;
}

// tanh(x) = 1 - 2 / (1 + e^(2 x)): absolute error below 2^-22, and exact at both ends (e^(2 x) = 0 or infinity)
__device__ __forceinline__ float tanh_fast(float x) {
    return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * (2.0f * LOG2E))), 1.0f);
}

// a number that is the same in all lanes, into a scalar register
__device__ __forceinline__ float uniform(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); }

// The capped score c tanh(f s) in units of log2, off by a few units of its last place, or by 2^-16 where caps are small. Three forms:
//   series   |f s| <= 0.35 for a whole wave, the usual case: an odd series in s up to the 9th power; the next term is 1382 / 155925 x^10
//            of the result, below 2.5e-7. Half the time of the exponential and the reciprocal.
//   small    c <= SMALL: tanh_fast, whose 2^-22 of the cap are at most 2^-16, which moves a weight by a twentieth of its rounding to f16
//   any      the series where |f s| <= 0.35, tanh_fast beyond, where its error is small against its result too
// (8192 tokens whose scores lie around their cap: 1120 us if small caps went the last way, 830 so. All three in one tile kernel
// cost it registers: a capped prefix of 16384 tokens 96 us instead of 86; so its larger caps are an instantiation of their own.)
// `factor` is that of a score without a cap, c f: it is not formed from them, so that no cap near the end of f32 loses bits.
struct Cap {
    static constexpr float SMALL = 64.0f;
    static __host__ __device__ __forceinline__ bool large(float cap) { return cap * LOG2E > SMALL; }
    float c, f, near;  // near: up to which |s|; with caps so small that the coefficients would leave f32 nothing is
    float k[5];
    __device__ __forceinline__ Cap(float cap, float per_score, float factor) {
        c = uniform(cap);
        f = uniform(per_score);
        near = uniform(fabsf(f) < 4096.0f ? 0.35f / fabsf(f) : -1.0f);
        const float g = f * f;
        k[0] = uniform(factor);
        k[1] = uniform(factor * g * (-1.0f / 3));
        k[2] = uniform(factor * g * g * (2.0f / 15));
        k[3] = uniform(factor * g * g * g * (-17.0f / 315));
        k[4] = uniform(factor * g * g * g * g * (62.0f / 2835));
    }
    __device__ __forceinline__ float series(float s) const {
        const float q = s * s;
        return s * __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, k[4], k[3]), k[2]), k[1]), k[0]);
    }
    __device__ __forceinline__ float small(float s) const { return c * tanh_fast(s * f); }
    __device__ __forceinline__ float any(float s) const { return fabsf(s) <= near ? series(s) : small(s); }
};

// four keys (consecutive rows of the staged V) of one dim: 16 lanes hand in the addresses of 4 dims of 4 rows each
__device__ __forceinline__ halfx4 lds_read_transposed(const half_t *p) {
    return __builtin_bit_cast(halfx4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *) p));
}

__device__ __forceinline__ bool not_finite(halfx8 x) {
    const uint4 u = __builtin_bit_cast(uint4, x);
    unsigned any = 0;
    for (unsigned w : {u.x, u.y, u.z, u.w}) {
        any |= (w & 0x7c00u) == 0x7c00u;
        any |= (w & 0x7c000000u) == 0x7c000000u;
    }
    return any;
}

__device__ __forceinline__ halfx8 finite_or_zero(halfx8 x) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = x[e] - x[e] == (half_t) 0.0f ? x[e] : (half_t) 0.0f;
    return x;
}

// four words of two whole numbers plus 1152 each -> f16
__device__ __forceinline__ unsigned pk_sub_1152(unsigned x) {
    const halfx2 bias = {(half_t) -1152.0f, (half_t) -1152.0f};
    return __builtin_bit_cast(unsigned, __builtin_bit_cast(halfx2, x) + bias);
}

// 8 whole numbers of 8 bits as f16, in the order 0 2 1 3 4 6 5 7, without a conversion instruction: q + 128 in the low byte
// of 0x6400 is 1152 + q, the subtraction is exact
__device__ __forceinline__ halfx8 widen(unsigned a, unsigned b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    return __builtin_bit_cast(halfx8, uint4{pk_sub_1152((a & 0x00ff00ffu) | 0x64006400u), pk_sub_1152(((a >> 8) & 0x00ff00ffu) | 0x64006400u),
                                            pk_sub_1152((b & 0x00ff00ffu) | 0x64006400u), pk_sub_1152(((b >> 8) & 0x00ff00ffu) | 0x64006400u)});
}

// What the scale of an 8 bit value adds to its score (in units of log2), so that the weight is the softmax's times the scale, and what
// such a weight is multiplied by in the softmax's own sum. A key that a query does not see has the score -infinity, and with it
// the weight zero whatever its scale holds: not finite (or absurdly large) scales are NaN to the score and zero to the sum. Scales
// below 2^-40 count as that: values below 2^-33 are zeros of an f16 result.
struct ValueScale {
    float log, inv;
    __device__ __forceinline__ explicit ValueScale(float scale) {
        const float held = scale < 0x1p-40f ? 0x1p-40f : scale;
        const bool good = held <= 0x1p100f;
        log = good ? __builtin_amdgcn_logf(held) : __builtin_nanf("");
        inv = good ? __builtin_amdgcn_rcpf(held) : 0.0f;
    }
};

// ---- 32 rows per wave, 4 or 8 waves per workgroup ------------------------------------------------------------------

// The waves walk all blocks of 64 keys, which they stage together in one of two LDS buffers, one barrier per block: the
// block after the current one is in flight in registers meanwhile. KG = 2: twice the waves for the same rows, in two groups that take
// every other block each and are joined at the end through LDS. WP: the width, padded to 64 or 128 with zeros. SHAPE:
// whether there is a cap or a distance bias. I8: keys and values are staged as the whole numbers they are, exact in f16; the scale of a key is
// applied to its scores, that of a value to its weights, both in f32 and ahead of the exponential (ValueScale). The reference of a
// query's softmax follows score + log2(value scale), so that what the second product holds in f16 goes by what a key contributes:
// a large value of little weight takes no bits from the others.
enum Shape { PLAIN, SHAPED_SCORES, LARGE_CAP };
template <int WP, int STRETCH, bool I8, int SHAPE, int TW, int KG>
__global__ __launch_bounds__(64 * TW) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile_attention_kernel(ServingAttentionParams p) {
    constexpr int BKEYS = 64, RW = TW / KG, THREADS = 64 * RW;  // waves for the rows, threads that stage a block
    constexpr int PIECE = I8 ? 16 : 8;        // elements per 128 bit load
    constexpr int C = WP / PIECE;             // loads per row
    constexpr int VECS = BKEYS * C / THREADS;  // of K and of V, per lane and block
    constexpr int KS = WP + 8, VS = WP == 128 ? 160 : 96;  // halves per staged row: bank-conflict free reads
    constexpr int STAGE = BKEYS * (KS + VS);
    constexpr int OS = WP + 8, WAVE_ROWS = 32 * OS;
    constexpr int DT = WP / 32, QC = WP / 8;
    constexpr bool PAGED = STRETCH != PROMPT, SHAPED = SHAPE != PLAIN;
    constexpr int JOIN = KG > 1 ? RW * 64 * (DT * 16 + 2) * 2 : 0;  // the other group's accumulators, in halves
    constexpr int LDS_HALVES = std::max({2 * KG * STAGE, TW * WAVE_ROWS, JOIN + RW * WAVE_ROWS});
    static_assert(WP != 128 || VECS >= 1, "unsupported shape");
    __shared__ __attribute__((aligned(16))) half_t lds[LDS_HALVES];
    __shared__ __attribute__((aligned(16))) float kscale_s[2][BKEYS], vlog_s[2][BKEYS], vinv_s[2][BKEYS];
    __shared__ unsigned long long gone_s[2][TW], bad_s[2][TW];
    __shared__ int range_s[TW][4];
    static_assert(!I8 || KG == 1, "one group of waves stages the scales");

    const int lane = threadIdx.x & 63, all_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = all_wave % RW, group = all_wave / RW;  // rows of the tile, blocks of keys
    const int thread = (int) threadIdx.x % THREADS;
    const int c = lane & 31, h = lane >> 5;
    // workgroups of one head of keys are a multiple of the (sequence, head) pairs apart: with 8 pairs or a multiple of them
    // they run on one XCD and share its L2; the last tiles, with the most keys under a causal mask, come first
    const unsigned pairs = (unsigned) (STRETCH == PREFIX ? 1 : p.batch) * p.kv_heads;
    const unsigned pair = blockIdx.x % pairs, slab = blockIdx.x / pairs;
    const int tile = (int) (gridDim.x / pairs) - 1 - (int) slab, kv_head = (int) (pair % p.kv_heads), b = (int) (pair / p.kv_heads);
    const unsigned rows = (unsigned) (STRETCH == PREFIX ? p.batch : 1) * p.queries * p.group_div.d;
    const int split = blockIdx.y, splits = gridDim.y;

    const unsigned first_row = (unsigned) tile * (32 * RW) + wave * 32;
    const unsigned row = first_row + c, row_c = min(row, rows - 1);
    const Row w = row_of<STRETCH>(p, row_c, b, kv_head);

    // ---- the blocks that any of the rows needs, and those that all of them see whole
    int from, end, whole_from, whole_end;
    {
        const bool sees = w.hi > w.lo;
        int a[4] = {sees ? w.lo : INT_MAX, -(sees ? w.hi : 0), -w.lo, w.hi};
#pragma unroll
        for (int m = 1; m < 32; m <<= 1)
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = min(a[i], __shfl_xor(a[i], m));
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < 4; i++) range_s[all_wave][i] = a[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int m = range_s[0][i];
#pragma unroll
            for (int j = 1; j < TW; j++) m = min(m, range_s[j][i]);
            a[i] = __builtin_amdgcn_readfirstlane(m);
        }
        from = a[0];
        end = -a[1];
        whole_from = -a[2];
        whole_end = a[3];
    }
    const int count = __builtin_amdgcn_readfirstlane(STRETCH == PROMPT ? p.keys : STRETCH == OWN ? own_length(p, b) : p.prefix_tokens);
    int first_block = from < end ? from / BKEYS : 0, end_block = from < end ? (end + BKEYS - 1) / BKEYS : 0;
    if (splits > 1) {  // this workgroup's share of the blocks
        const int each = (end_block - first_block + splits - 1) / splits;
        first_block = min(first_block + split * each, end_block);
        end_block = min(first_block + each, end_block);
    }

    // ---- global -> registers -> LDS
    const int *table = STRETCH == OWN ? p.tables + b * p.table_stride : p.prefix_table;
    const char *kb = (const char *) p.k, *vb = (const char *) p.v;
    constexpr int ELEM = I8 ? 1 : 2;
    if (STRETCH == PROMPT) {
        kb += (b * p.k_batch + kv_head * p.k_head) * ELEM;
        vb += (b * p.v_batch + kv_head * p.v_head) * ELEM;
    } else {
        kb += kv_head * p.k_head * ELEM;
        vb += kv_head * p.v_head * ELEM;
    }
    const int stage_row = thread / C, part = thread % C;
    constexpr int ROW_STEP = THREADS / C;  // rows between a lane's loads
    const bool part_live = part * PIECE < p.width;
    const long long k_lane = stage_row * p.k_token * ELEM + 16 * part, v_lane = stage_row * p.v_token * ELEM + 16 * part;  // prompts
    uint4 kreg[VECS], vreg[VECS];
    float kscale[VECS], vscale[VECS];
    int pages[VECS];
    unsigned gone = 0;  // of the block in the registers: the lane's rows that are not there
#pragma unroll
    for (int i = 0; i < VECS; i++) kreg[i] = vreg[i] = uint4{0, 0, 0, 0};  // (what a row has behind the width stays zero)
    auto look_up = [&](int block) {  // the page numbers of a block, ahead of its loads
        if (!PAGED) return;
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const int j = block * BKEYS + stage_row + ROW_STEP * i;
            pages[i] = j < count ? table[p.page_tokens.div((unsigned) j)] : -1;
        }
    };
    auto fetch = [&](int block) {
        gone = 0;
        if (!PAGED && (block + 1) * BKEYS <= count) {
            if (part_live)
#pragma unroll
                for (int i = 0; i < VECS; i++) {
                    const long long r = block * BKEYS + ROW_STEP * i;
                    kreg[i] = __builtin_bit_cast(uint4, *(const halfx8_any *) (kb + r * p.k_token * ELEM + k_lane));
                    vreg[i] = __builtin_bit_cast(uint4, *(const halfx8_any *) (vb + r * p.v_token * ELEM + v_lane));
                }
            return;
        }
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const int j = block * BKEYS + stage_row + ROW_STEP * i;
            bool there = j < count;
            long long k_at, v_at, s_at = 0;
            if (PAGED) {
                there = (unsigned) pages[i] < (unsigned) p.pages;
                const unsigned in = (unsigned) j - p.page_tokens.div((unsigned) j) * p.page_tokens.d;
                k_at = v_at = pages[i] * p.k_page + in * p.k_token;  // (one layout for both)
                if (I8) s_at = ((long long) pages[i] * p.kv_heads + kv_head) * p.page_tokens.d + in;
            } else {
                k_at = j * p.k_token;
                v_at = j * p.v_token;
            }
            if (!there) {
                gone |= 1u << i;
                kreg[i] = vreg[i] = uint4{0, 0, 0, 0};
                kscale[i] = vscale[i] = 0.0f;
            } else if (part_live) {
                if (I8) {
                    kreg[i] = *(const uint4 *) (kb + k_at + 16 * part);
                    vreg[i] = *(const uint4 *) (vb + v_at + 16 * part);
                    kscale[i] = p.k_scales[s_at];
                    vscale[i] = p.v_scales[s_at];
                } else {
                    kreg[i] = __builtin_bit_cast(uint4, *(const halfx8_any *) (kb + 2 * k_at + 16 * part));
                    vreg[i] = __builtin_bit_cast(uint4, *(const halfx8_any *) (vb + 2 * v_at + 16 * part));
                }
            }
        }
    };
    // A scale of zero or less goes into Q (times -1, 0 or 1), so that the scores are multiplied by a positive number
    const float sign = uniform(p.scale > 0.0f ? 1.0f : p.scale < 0.0f ? -1.0f : 0.0f);
    const float scale2 = uniform(p.scale == 0.0f ? 1.0f : fabsf(p.scale) * LOG2E);
    const bool capped = SHAPED && p.cap > 0.0f;
    // (the scores of whole numbers have their factor already)
    const float cap2 = uniform(capped ? p.cap * LOG2E : 1.0f);
    const Cap cap(cap2, (I8 ? 1.0f : scale2) / cap2, I8 ? 1.0f : scale2);
    auto stage = [&](int buffer, bool masked) {
        half_t *ks = lds + (KG * buffer + group) * STAGE, *vs = ks + BKEYS * KS;
#pragma unroll
        for (int i = 0; i < VECS; i++) {
            const int r = stage_row + ROW_STEP * i;
            if (I8) {
                *(halfx8 *) &ks[r * KS + 16 * part] = widen(kreg[i].x, kreg[i].y);
                *(halfx8 *) &ks[r * KS + 16 * part + 8] = widen(kreg[i].z, kreg[i].w);
                *(halfx8 *) &vs[r * VS + 16 * part] = widen(vreg[i].x, vreg[i].y);
                *(halfx8 *) &vs[r * VS + 16 * part + 8] = widen(vreg[i].z, vreg[i].w);
                if (part == 0) {
                    kscale_s[buffer][r] = kscale[i] * scale2;
                    const ValueScale v(vscale[i]);
                    vlog_s[buffer][r] = v.log;
                    vinv_s[buffer][r] = v.inv;
                }
            } else {
                *(uint4 *) &ks[r * KS + 8 * part] = kreg[i];
                *(uint4 *) &vs[r * VS + 8 * part] = vreg[i];
            }
        }
        // which of the block's rows are not there, and which hold values that a product with a zero weight does not remove
        if (KG > 1 || PAGED || masked) {
            unsigned long long gone_rows = 0, bad_rows = 0;
#pragma unroll
            for (int i = 0; i < VECS; i++) {
                unsigned long long bad = 0;
                if (masked && !I8) bad = __ballot(not_finite(__builtin_bit_cast(halfx8, vreg[i])));
                const unsigned long long missing = __ballot((gone >> i) & 1);
                if (bad | missing)
#pragma unroll
                    for (int g = 0; g < 64 / C; g++) {  // rows of this wave's i-th load
                        const int r = wave * (64 / C) + g + ROW_STEP * i;
                        const unsigned long long lanes = ((1ull << C) - 1) << (g * C);
                        if (bad & lanes) bad_rows |= 1ull << r;
                        if (missing & lanes) gone_rows |= 1ull << r;
                    }
            }
            if (lane == 0) {
                gone_s[buffer][all_wave] = gone_rows;
                bad_s[buffer][all_wave] = bad_rows;
            }
        }
    };

    const int start = first_block + group;
    if (start < end_block) {
        look_up(start);
        fetch(start);
        look_up(min(start + KG, end_block - 1));
    }

    // ---- Q: the wave's 32 rows, whole lines at a time, through the wave's part of LDS; lane (query c, half h) holds elements
    // 16 t + 8 h .. + 7 for step t, in the order of the staged keys
    halfx8 qf[WP / 16];
    {
        half_t *qs = lds + all_wave * WAVE_ROWS;
#pragma unroll
        for (int i = 0; i < 32 * QC / 64; i++) {
            const int e = lane + 64 * i, r = e / QC, d = 8 * (e % QC);
            const Row o = row_of<STRETCH>(p, min(first_row + r, rows - 1), b, kv_head);
            halfx8 x = {0, 0, 0, 0, 0, 0, 0, 0};
            if (first_row + r < rows && d < p.width)
                x = *(const halfx8_any *) ((const half_t *) p.q + (o.b * p.q_batch + o.t * p.q_token + o.head * p.q_head + d)) * (half_t) sign;
            *(halfx8 *) &qs[r * OS + d] = I8 ? halfx8{x[0], x[2], x[1], x[3], x[4], x[6], x[5], x[7]} : x;
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < WP / 16; t++) qf[t] = *(const halfx8 *) &qs[c * OS + 16 * t + 8 * h];
        __syncthreads();  // (the buffers of K and V lie over these rows)
    }

    floatx16 oacc[DT];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int v = 0; v < 16; v++) oacc[t][v] = 0.0f;
    float ref = -INFINITY, sum = 0.0f;  // sum: this half's share of the keys
    const float slope2 = SHAPED && p.slopes ? p.slopes[w.head] * LOG2E : 0.0f;
    const int v_corner = BKEYS * KS + (4 * h + (lane & 15) / 4) * VS + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    constexpr bool LOG2_UNITS = SHAPED || I8;  // the scores have their factor before the exponential

    for (int turn = 0; first_block + KG * turn < end_block; turn++) {
        const int block = start + KG * turn, buffer = turn & 1, key0 = block * BKEYS;
        const bool live = KG == 1 || block < end_block;  // (the last turn may have one block less)
        bool masked = key0 < whole_from || key0 + BKEYS > whole_end;
        if (live) {
            stage(buffer, masked);
            if (block + KG < end_block) {
                fetch(block + KG);
                look_up(min(block + 2 * KG, end_block - 1));
            }
        } else if (lane == 0) {
            bad_s[buffer][all_wave] = 0;
        }
        __syncthreads();
        half_t *ks = lds + (KG * buffer + group) * STAGE;
        unsigned long long gone_rows = 0;
        if (KG > 1 || PAGED || masked) {
            unsigned long long bad_rows = 0, bad_anywhere = 0;
#pragma unroll
            for (int i = 0; i < RW; i++) {
                gone_rows |= gone_s[buffer][group * RW + i];
                if (!I8) bad_rows |= bad_s[buffer][group * RW + i];
            }
            if (!I8)
#pragma unroll
                for (int i = 0; i < TW; i++) bad_anywhere |= bad_s[buffer][i];
            gone_rows = ((unsigned long long) __builtin_amdgcn_readfirstlane((unsigned) (gone_rows >> 32)) << 32) | (unsigned) __builtin_amdgcn_readfirstlane((unsigned) gone_rows);
            if (PAGED) masked |= gone_rows != 0;
            bad_rows = ((unsigned long long) __builtin_amdgcn_readfirstlane((unsigned) (bad_rows >> 32)) << 32) | (unsigned) __builtin_amdgcn_readfirstlane((unsigned) bad_rows);
            if (!I8 && (__builtin_amdgcn_readfirstlane((unsigned) (bad_anywhere >> 32)) | __builtin_amdgcn_readfirstlane((unsigned) bad_anywhere)) != 0) {
                // Infinities or NaN among the values of a block that not every row sees whole: a weight of zero does not remove
                // them from a product, so they are added here for the queries that see their key, and then taken out.
                for (unsigned long long left = bad_rows; left; left &= left - 1) {
                    const int key = __builtin_ctzll(left);
                    if ((unsigned) (key0 + key - w.lo) < (unsigned) (w.hi - w.lo))
#pragma unroll
                        for (int t = 0; t < DT; t++)
#pragma unroll
                            for (int a = 0; a < 4; a++) {
                                const halfx4 x = *(const halfx4 *) &ks[BKEYS * KS + key * VS + 32 * t + 8 * a + 4 * h];
#pragma unroll
                                for (int u = 0; u < 4; u++) oacc[t][4 * a + u] += (float) x[u] - (float) x[u] == 0.0f ? 0.0f : (float) x[u];
                            }
                }
                __syncthreads();
                for (int e = thread; e < BKEYS * QC; e += THREADS) {
                    const int r = e / QC;
                    halfx8 *x = (halfx8 *) &ks[BKEYS * KS + r * VS + 8 * (e % QC)];
                    if ((bad_rows >> r) & 1) *x = finite_or_zero(*x);
                }
                __syncthreads();
            }
        }

        if (!live) break;  // (nothing comes behind it)
        floatx16 st[2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int v = 0; v < 16; v++) st[u][v] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int t = 0; t < WP / 16; t++) {
                const halfx8 a = *(const halfx8 *) &ks[(32 * u + c) * KS + 16 * t + 8 * h];
                st[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[t], st[u], 0, 0, 0);
            }
        // register v of tile u: key 32 u + 8 (v / 4) + 4 h + v % 4
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if (I8)
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const floatx4 f = *(const floatx4 *) &kscale_s[buffer][32 * u + 8 * a + 4 * h];
                    floatx4 l = {0, 0, 0, 0};
                    if (!SHAPED) l = *(const floatx4 *) &vlog_s[buffer][32 * u + 8 * a + 4 * h];
#pragma unroll
                    for (int e = 0; e < 4; e++) st[u][4 * a + e] = SHAPED ? st[u][4 * a + e] * f[e] : __builtin_fmaf(st[u][4 * a + e], f[e], l[e]);
                }
            if (SHAPED && capped) {
                // (the same choice for the whole wave; most scores lie far below the cap)
                float far = fabsf(st[u][0]);
#pragma unroll
                for (int v = 1; v < 16; v++) far = fmaxf(far, fabsf(st[u][v]));
                if (__all(far <= cap.near)) {
#pragma unroll
                    for (int v = 0; v < 16; v++) st[u][v] = cap.series(st[u][v]);
                } else {
#pragma unroll
                    for (int v = 0; v < 16; v++) st[u][v] = SHAPE == LARGE_CAP ? cap.any(st[u][v]) : cap.small(st[u][v]);
                }
            } else if (SHAPED && !I8) {
#pragma unroll
                for (int v = 0; v < 16; v++) st[u][v] *= scale2;
            }
            if (SHAPED && p.slopes) {
                const float away = (float) (w.at - (key0 + 32 * u + 4 * h));
#pragma unroll
                for (int v = 0; v < 16; v++) st[u][v] = __builtin_fmaf(-slope2, fabsf(away - (float) (8 * (v / 4) + v % 4)), st[u][v]);
            }
            if (SHAPED && I8)
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const floatx4 l = *(const floatx4 *) &vlog_s[buffer][32 * u + 8 * a + 4 * h];
#pragma unroll
                    for (int e = 0; e < 4; e++) st[u][4 * a + e] += l[e];
                }
            if (masked) {
                const unsigned missing = (unsigned) (gone_rows >> (32 * u)) >> (4 * h);
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const int e = 8 * (v / 4) + v % 4, j = key0 + 32 * u + 4 * h + e;
                    if ((unsigned) (j - w.lo) >= (unsigned) (w.hi - w.lo) || (PAGED && ((missing >> e) & 1))) st[u][v] = -INFINITY;
                }
            }
#pragma unroll
            for (int v = 0; v < 16; v++) top = fmaxf(top, st[u][v]);
        }
        if (!LOG2_UNITS) top *= scale2;
        if (__any(top > ref + SLACK)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            const float new_ref = fmaxf(ref, top);
            const float alpha = ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - new_ref);  // (what is not finite may have been added)
            ref = new_ref;
            sum *= alpha;
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int v = 0; v < 16; v++) oacc[t][v] *= alpha;
        }
        const float minus = ref == -INFINITY ? 0.0f : ref - LIFT;
        halfx8 pv[4];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int a = 0; a < 4; a++) {
                floatx4 f = {1, 1, 1, 1};
                if (I8) f = *(const floatx4 *) &vinv_s[buffer][32 * u + 8 * a + 4 * h];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int v = 4 * a + i;
                    const float e = __builtin_amdgcn_exp2f(LOG2_UNITS ? st[u][v] - minus : __builtin_fmaf(st[u][v], scale2, -minus));
                    sum = I8 ? __builtin_fmaf(e, f[i], sum) : sum + e;
                    pv[2 * u + v / 8][v % 8] = (half_t) e;
                }
            }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            halfx8 a[DT];
#pragma unroll
            for (int t = 0; t < DT; t++) {
                const halfx4 lo = lds_read_transposed(ks + v_corner + (16 * s) * VS + 32 * t);
                const halfx4 hi = lds_read_transposed(ks + v_corner + (16 * s + 8) * VS + 32 * t);
                a[t] = halfx8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            }
#pragma unroll
            for (int t = 0; t < DT; t++) oacc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[t], pv[s], oacc[t], 0, 0, 0);
        }
    }

    if (KG > 1) {  // the other group's blocks
        float *other = (float *) lds + wave * 64 * (DT * 16 + 2);
        __syncthreads();  // (every wave is done with the buffers)
        if (group == 1) {
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    *(floatx4 *) &other[(4 * t + a) * 256 + 4 * lane] = floatx4{oacc[t][4 * a], oacc[t][4 * a + 1], oacc[t][4 * a + 2], oacc[t][4 * a + 3]};
            *(float2 *) &other[DT * 16 * 64 + 2 * lane] = float2{ref, sum};
        }
        __syncthreads();
        if (group == 1) return;
        const float2 stats = *(const float2 *) &other[DT * 16 * 64 + 2 * lane];
        const float new_ref = fmaxf(ref, stats.x), minus = new_ref == -INFINITY ? 0.0f : new_ref;
        // (a group that saw nothing adds nothing but what is not finite, see above)
        const float own = ref == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - minus), its = stats.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(stats.x - minus);
        ref = new_ref;
        sum = sum * own + stats.y * its;
#pragma unroll
        for (int t = 0; t < DT; t++)
#pragma unroll
            for (int a = 0; a < 4; a++) {
                const floatx4 x = *(const floatx4 *) &other[(4 * t + a) * 256 + 4 * lane];
#pragma unroll
                for (int v = 0; v < 4; v++) oacc[t][4 * a + v] = oacc[t][4 * a + v] * own + x[v] * its;
            }
    }
    sum += __shfl_xor(sum, 32);
    // (dims 32 t + 8 a + 4 h + (0 .. 3) are registers 4 a .. 4 a + 3, the middle two changed over where widen() does)
    auto dims = [&](int t, int a) {
        return I8 ? floatx4{oacc[t][4 * a], oacc[t][4 * a + 2], oacc[t][4 * a + 1], oacc[t][4 * a + 3]}
                  : floatx4{oacc[t][4 * a], oacc[t][4 * a + 1], oacc[t][4 * a + 2], oacc[t][4 * a + 3]};
    };
    if (p.part_values) {
        // a part of the softmax: reference, sum and the sums of values as they are
        if (row < rows) {
            const long long at = ((long long) pair * splits + split) * rows + row;
            float *o = p.part_values + at * WP;
#pragma unroll
            for (int t = 0; t < DT; t++)
#pragma unroll
                for (int a = 0; a < 4; a++) *(floatx4 *) (o + 32 * t + 8 * a + 4 * h) = dims(t, a);
            if (h == 0) *(float2 *) (p.part_stats + 2 * at) = float2{ref, sum};
        }
        return;
    }
    // ---- the result: normalised, rounded, through the wave's rows of LDS into whole rows
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    if (KG == 1) __syncthreads();  // (every wave is done with the buffers)
    half_t *os = lds + JOIN + wave * WAVE_ROWS;
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
            const floatx4 o = dims(t, a);
            halfx4 x;
#pragma unroll
            for (int u = 0; u < 4; u++) x[u] = (half_t) (o[u] * inv);
            *(halfx4 *) &os[c * OS + 32 * t + 8 * a + 4 * h] = x;
        }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 32 * QC / 64; i++) {
        const int e = lane + 64 * i, r = e / QC, d = 8 * (e % QC);
        if (first_row + r >= rows || d >= p.width) continue;
        const Row o = row_of<STRETCH>(p, first_row + r, b, kv_head);
        *(halfx8_any *) ((half_t *) p.out + (o.b * p.o_batch + o.t * p.o_token + o.head * p.o_head + d)) = *(const halfx8 *) &os[r * OS + d];
    }
}

// ---- up to 16 NT rows per workgroup --------------------------------------------------------------------------------

// Decoding: bound by the bytes of the cache, which pass through once. A workgroup takes a stretch of keys of one sequence
// and head, its eight waves every eighth step of 32 keys; nothing is staged in LDS. The registers of a step's keys are
// loaded again as soon as the scores are there, those of its values as soon as they are summed, so that a wave always has
// loads in flight. Both products take 16 keys or dims by 16 rows (v_mfma_f32_16x16x32_f16):
//   S^T = K Q^T      lane (key i = lane % 16, g = lane / 16) reads 16 byte pieces of key i, 64 bytes of a row per load of four
//                    lanes; the order of a row's elements in the product is free, Q is loaded in the same one
//   O^T += V^T P^T   the accumulators of two tiles of S^T are the operand, keys 4 g + e and 16 + 4 g + e; lane (i, g) reads
//                    elements i DPL .. + DPL - 1 of those 8 keys and turns them in registers: product dt has dim i DPL + dt
// The scale of a key is applied to its score, that of a value to its weight, in f32 and ahead of the exponential (ValueScale); the
// reference of the softmax follows score + log2(value scale), which keeps the scaled weights inside the range of f16.

// Which keys a workgroup takes, decided on the device, where the lengths are: stretches (the prefix when it is done here, then
// every sequence's own keys) are cut into items of about the same size, ROW_ITEMS of them over all heads, and workgroup x
// takes item x / kv_heads. The grid covers the largest number of items that any lengths can give. Parts of less than
// ROW_MIN_KEYS keys are not made: four steps per wave take less time than the launch that joins two parts.
// Every wave looks its item up in the lengths of all sequences, 64 at a time. That takes each round of workgroups the longer the more
// sequences there are, so that for many of them a launch of one workgroup makes a list of the items first (LIST_FROM: sequences
// times pairs of a sequence and a head of keys). Looked up / listed, us, sequences x heads of keys x keys: 256 x 1 x 16 8.9 / 10.2,
// 96 x 8 x 200 25.2 / 25.7, 128 x 8 x 200 32.7 / 31.7, 256 x 8 x 200 68 / 55, 384 x 1 x 16 16.8 / 15.0, 1024 x 8 x 200 466 / 235,
// 65536 x 1 x 16 120700 / 1500.
constexpr int ROW_ITEMS = 512, ROW_MIN_KEYS = 1024, ROW_WAVES = 8, ROW_THREADS = 64 * ROW_WAVES;
constexpr int LIST_FROM = 1 << 17, LIST_THREADS = 1024, NO_ITEM = -2;

struct Item {
    int seg, length, from, end, nth, items;
};

// (length, first key that any row may see: a multiple of 32) of a sequence's own keys
__device__ __forceinline__ int2 own_range(const ServingAttentionParams &p, int b) {
    const int n = own_length(p, b);
    return int2{n, p.window ? max(0, n - p.queries + 1 - p.window) & ~31 : 0};
}
__device__ __forceinline__ int steps_of(int2 range) { return (range.x - range.y + 31) / 32; }
// steps per item, out of those of all stretches; no stretch has more than 2^26
__device__ __forceinline__ int steps_per_item(const ServingAttentionParams &p, long long steps) {
    return max(ROW_MIN_KEYS / 32, (int) min((steps * p.kv_heads + ROW_ITEMS - 1) / ROW_ITEMS, 1ll << 26));
}
__device__ __forceinline__ int items_of(int steps, int each) { return max(1, (steps + each - 1) / each); }

// the n-th of a segment's items, all of which have the same number of steps, but for the last
__device__ __forceinline__ void cut_item(int2 range, int steps, int nth, int items, Item &out) {
    const int per = 32 * ((steps + items - 1) / items);
    out.length = range.x;
    out.items = items;
    out.nth = nth;
    out.from = min(range.y + nth * per, range.x);
    out.end = min(range.y + nth * per + per, range.x);
}

// segments -1 (the prefix, when `with_prefix`) and 0 .. batch - 1; false when there is no such item. Every wave works it out
// for itself, a lane per segment, or takes it from the list.
__device__ __forceinline__ bool find_item(const ServingAttentionParams &p, int with_prefix, int item, Item &out) {
    if (p.item_list) {
        const int seg = __builtin_amdgcn_readfirstlane(p.item_list[item]);
        if (seg == NO_ITEM) return false;
        const int2 items = ((const int2 *) p.part_items)[seg + 1], range = own_range(p, seg);
        out.seg = seg;
        cut_item(range, steps_of(range), item - items.x, items.y, out);
        return true;
    }
    const int lane = threadIdx.x & 63, segs = p.batch + with_prefix;
    auto range = [&](int s) { return s >= segs ? int2{0, 0} : s < with_prefix ? int2{p.prefix_tokens, 0} : own_range(p, s - with_prefix); };
    const int2 first = range(lane);
    long long steps = 0;  // of 32 keys, of all stretches (64 bits: many long tables may share pages)
    for (int s0 = 0; s0 < segs; s0 += 64) steps += steps_of(s0 ? range(s0 + lane) : first);
    if (segs <= 64) {
        unsigned few = (unsigned) steps;  // (at most 64 stretches of 2^25 steps)
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) few += __shfl_xor(few, m);
        steps = few;
    } else {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) steps += __shfl_xor(steps, m);
    }
    const int each = steps_per_item(p, steps);
    int base = 0;
    for (int s0 = 0; s0 < segs; s0 += 64) {
        const int2 r = s0 ? range(s0 + lane) : first;
        const int own_steps = steps_of(r), n = s0 + lane < segs ? items_of(own_steps, each) : 0;
        int sums = n;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int other = __shfl_up(sums, m);
            if (lane >= m) sums += other;
        }
        const int before = base + sums - n;
        const unsigned long long hit = __ballot(n > 0 && item >= before && item < before + n);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            out.seg = s0 + l - with_prefix;
            cut_item(int2{__builtin_amdgcn_readlane(r.x, l), __builtin_amdgcn_readlane(r.y, l)}, __builtin_amdgcn_readlane(own_steps, l),
                     item - __builtin_amdgcn_readlane(before, l), __builtin_amdgcn_readlane(n, l), out);
            if (out.nth == 0 && threadIdx.x == 0) ((int2 *) p.part_items)[out.seg + 1] = int2{item, out.items};
            return true;
        }
        base += __builtin_amdgcn_readlane(sums, 63);
    }
    return false;
}

// The items of all sequences' own keys: a thread per sequence, one workgroup. part_items as find_item() writes them, and the
// sequence of each of the `items` that there may be.
__global__ __launch_bounds__(LIST_THREADS) void list_items_kernel(ServingAttentionParams p, int items) {
    constexpr int NWAVES = LIST_THREADS / 64;
    __shared__ long long wave_steps[NWAVES];
    __shared__ int wave_items[2][NWAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long long steps = 0;
    for (int b = threadIdx.x; b < p.batch; b += LIST_THREADS) steps += steps_of(own_range(p, b));
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) steps += __shfl_xor(steps, m);
    if (lane == 0) wave_steps[wave] = steps;
    __syncthreads();
    steps = 0;
    for (int w = 0; w < NWAVES; w++) steps += wave_steps[w];
    const int each = steps_per_item(p, steps);
    int base = 0;
    for (int b0 = 0, turn = 0; b0 < p.batch; b0 += LIST_THREADS, turn ^= 1) {
        const int b = b0 + (int) threadIdx.x, n = b < p.batch ? items_of(steps_of(own_range(p, b)), each) : 0;
        int sums = n;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int other = __shfl_up(sums, m);
            if (lane >= m) sums += other;
        }
        if (lane == 63) wave_items[turn][wave] = sums;
        __syncthreads();  // (two buffers: one barrier per turn keeps writers away from readers)
        int at = base + sums - n;
        for (int w = 0; w < NWAVES; w++) {
            if (w < wave) at += wave_items[turn][w];
            base += wave_items[turn][w];
        }
        if (b < p.batch) ((int2 *) p.part_items)[b + 1] = int2{at, n};
        for (int i = at; i < at + n && i < items; i++) p.item_list[i] = b;
    }
    for (int i = base + (int) threadIdx.x; i < items; i += LIST_THREADS) p.item_list[i] = NO_ITEM;
}

template <int WORDS>
__device__ __forceinline__ void load_words(const char *from, unsigned (&to)[WORDS]) {
    if constexpr (WORDS == 1) to[0] = *(const unsigned *) from;
    if constexpr (WORDS == 2) {
        const uint2 x = *(const uint2 *) from;
        to[0] = x.x;
        to[1] = x.y;
    }
    if constexpr (WORDS == 4) {
        const uint4 x = *(const uint4 *) from;
        to[0] = x.x;
        to[1] = x.y;
        to[2] = x.z;
        to[3] = x.w;
    }
}

// PAGE16: pages are multiples of 16 tokens and a tile of 16 keys spans less than 2 GiB, so that a tile lies in one page, whose
// number and address the whole wave shares, and lanes differ by 32 bit offsets
template <int WP, int NT, bool I8, bool SHAPED, bool PAGE16, bool INSIDE>
// (at least two waves per SIMD: with more registers than that leaves, the results of matrix instructions would lie in AGPRs, and
// the compiler reads such a result too early behind a branch; the build refuses kernels of this file that have any)
__global__ __launch_bounds__(ROW_THREADS) __attribute__((amdgpu_waves_per_eu(2))) void row_attention_kernel(ServingAttentionParams p, int with_prefix) {
    constexpr int ELEM = I8 ? 1 : 2;
    constexpr int KP = WP * ELEM / 64;    // 16 byte pieces of a key per lane
    constexpr int DPL = WP / 16;          // dims of a value per lane
    constexpr int VW = DPL * ELEM / 4;    // 32 bit words of a value per lane
    constexpr int STEPS = WP / 32;
    constexpr int OS = WP + 4;
    __shared__ __attribute__((aligned(16))) float os[ROW_WAVES][16 * NT][OS];
    __shared__ float refs[ROW_WAVES][16 * NT], sums[ROW_WAVES][16 * NT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int global_item = (int) (blockIdx.x / (unsigned) p.kv_heads), kv_head = (int) (blockIdx.x % (unsigned) p.kv_heads);
    Item item;
    if (!find_item(p, with_prefix, global_item, item)) return;
    const bool is_prefix = item.seg < 0;
    const int b = is_prefix ? 0 : item.seg;
    const int rows = (is_prefix ? p.batch : 1) * p.queries * (int) p.group_div.d;
    constexpr int STRIDE = 32 * ROW_WAVES;

    // ---- the rows: lane i of a tile of 16 owns row 16 n + i
    halfx8 qf[NT][STEPS];
    float slope2[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = 16 * n + i;
        const Row w = is_prefix ? row_of<PREFIX>(p, min(r, rows - 1), 0, kv_head) : row_of<OWN>(p, min(r, rows - 1), b, kv_head, item.length);
        slope2[n] = SHAPED && p.slopes ? p.slopes[w.head] * LOG2E : 0.0f;
        const half_t *q = (const half_t *) p.q + (w.b * p.q_batch + w.t * p.q_token + w.head * p.q_head);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int d = I8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
            halfx8 x = {0, 0, 0, 0, 0, 0, 0, 0};
            if (r < rows && d < p.width) x = *(const halfx8_any *) (q + d);
            qf[n][s] = I8 ? halfx8{x[0], x[2], x[1], x[3], x[4], x[6], x[5], x[7]} : x;
        }
    }
    floatx4 oacc[NT][DPL];
    float ref[NT], sum[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        ref[n] = -INFINITY;
        sum[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < DPL; d++) oacc[n][d] = floatx4{0, 0, 0, 0};
    }
    const float scale2 = p.scale * LOG2E;
    const bool capped = SHAPED && p.cap > 0.0f;
    const float cap2 = capped ? p.cap * LOG2E : 1.0f;
    const Cap cap(cap2, scale2 / cap2, scale2);
    const char *kb = (const char *) p.k + kv_head * p.k_head * ELEM, *vb = (const char *) p.v + kv_head * p.v_head * ELEM;
    const bool v_live = i * DPL < p.width, k_whole = p.width == WP;

    // INSIDE: two stretches one after the other, the sequence's first item begins with the prefix. (An instantiation of its own: the
    // loop costs the others a tenth of their time.)
    int taken = 0;  // steps of the stretch before, so that the waves go on in turn
#pragma unroll 1
    for (int stretch = INSIDE && item.nth == 0 ? 0 : 1; stretch < 2; stretch++) {
        const bool shared = is_prefix || stretch == 0;
        const int count = stretch == 0 ? p.prefix_tokens : item.length, item_from = stretch == 0 ? 0 : item.from, item_end = stretch == 0 ? count : item.end;
        const int *table = shared ? p.prefix_table : p.tables + b * p.table_stride;
        int pages[2] = {0, 0};
        auto look_up = [&](int key0) {  // the pages of a step's tiles, ahead of their loads; behind the last key: none
            if (PAGE16)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int j = key0 + 16 * u;
                    pages[u] = j < item_end ? table[p.page_tokens.div((unsigned) j)] : -1;
                }
        };
        const int first_key = 32 * ((wave - taken) & (ROW_WAVES - 1));
        if (item_from < item_end) look_up(item_from + first_key);

        int at[NT], lo[NT], hi[NT];
        int whole_from = 0, whole_end = INT_MAX, any_from = INT_MAX, any_end = 0;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = min(16 * n + i, rows - 1);
            const Row w = !shared ? row_of<OWN>(p, r, b, kv_head, item.length) : row_of<PREFIX>(p, b * rows + r, 0, kv_head, is_prefix ? -1 : item.length);
            at[n] = w.at;
            lo[n] = w.lo;
            hi[n] = w.hi;
            whole_from = max(whole_from, w.lo);
            whole_end = min(whole_end, w.hi);
            if (w.hi > w.lo) {
                any_from = min(any_from, w.lo);
                any_end = max(any_end, w.hi);
            }
        }
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) {
            whole_from = max(whole_from, __shfl_xor(whole_from, m));
            whole_end = min(whole_end, __shfl_xor(whole_end, m));
            any_from = min(any_from, __shfl_xor(any_from, m));
            any_end = max(any_end, __shfl_xor(any_end, m));
        }
        whole_from = __builtin_amdgcn_readfirstlane(whole_from);
        whole_end = __builtin_amdgcn_readfirstlane(whole_end);
        any_from = __builtin_amdgcn_readfirstlane(any_from);
        any_end = __builtin_amdgcn_readfirstlane(any_end);
        int from = max(item_from, any_from & ~31), end = min(item_end, any_end);
        if (from >= end) from = end = 0;  // (nothing to see: any_from may be INT_MAX, nothing may be added to it)

        uint4 kreg[2][KP];
        unsigned vreg[8][VW];
        floatx4 kscale[2], vscale[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            kscale[u] = vscale[u] = floatx4{1, 1, 1, 1};
#pragma unroll
            for (int c = 0; c < KP; c++) kreg[u][c] = uint4{0, 0, 0, 0};
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int x = 0; x < VW; x++) vreg[e][x] = 0;
        unsigned gone = 0, gone_next = 0;  // keys of the lane's 8 (4 u + e: key 16 u + 4 g + e) that are not there
        const unsigned k_lane = PAGE16 ? (unsigned) (i * (int) p.k_token * ELEM + 16 * g) : 0;
        const unsigned v_lane = PAGE16 ? (unsigned) ((4 * g * (int) p.v_token + i * DPL) * ELEM) : 0;

        // the places of a step's tiles: page and token inside it (PAGE16)
        int page_next[2] = {-1, -1};
        unsigned in_next[2] = {0, 0};
        auto place = [&](int key0) {
            if (PAGE16) {
                gone_next = 0;
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const unsigned j = (unsigned) (key0 + 16 * u);
                    page_next[u] = __builtin_amdgcn_readfirstlane(pages[u]);
                    in_next[u] = j - p.page_tokens.div(j) * p.page_tokens.d;
                    if ((unsigned) page_next[u] >= (unsigned) p.pages) gone_next |= 15u << (4 * u);
                }
            }
        };
        auto load_k = [&](int key0) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (PAGE16) {
                    if ((gone_next >> (4 * u)) & 1) continue;
                    const char *base = kb + (page_next[u] * p.k_page + in_next[u] * p.k_token) * ELEM;
#pragma unroll
                    for (int c = 0; c < KP; c++)
                        if (k_whole || 64 * c + 16 * g < p.width * ELEM) kreg[u][c] = *(const uint4 *) (base + (k_lane + 64 * c));
                } else {
                    const int j = key0 + 16 * u + i, pg = j < count ? table[p.page_tokens.div((unsigned) j)] : -1;
                    const unsigned at_j = (unsigned) j - p.page_tokens.div((unsigned) j) * p.page_tokens.d;
                    const char *base = kb + (pg * p.k_page + at_j * p.k_token) * ELEM;
                    if ((unsigned) pg < (unsigned) p.pages)
#pragma unroll
                        for (int c = 0; c < KP; c++)
                            if (64 * c + 16 * g < p.width * ELEM) kreg[u][c] = *(const uint4 *) (base + 64 * c + 16 * g);
                }
            }
        };
        auto load_scales = [&](int key0) {
            if (!I8) return;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (PAGE16) {
                    if ((gone_next >> (4 * u)) & 1) continue;
                    const long long s = ((long long) page_next[u] * p.kv_heads + kv_head) * p.page_tokens.d + in_next[u];
                    kscale[u] = *(const floatx4_any *) ((const char *) (p.k_scales + s) + (unsigned) (16 * g));
                    vscale[u] = *(const floatx4_any *) ((const char *) (p.v_scales + s) + (unsigned) (16 * g));
                }
            }
        };
        auto load_v = [&](int key0) {
            if (!PAGE16) gone_next = 0;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (PAGE16) {
                    if ((gone_next >> (4 * u)) & 1) continue;
                    const char *base = vb + (page_next[u] * p.v_page + in_next[u] * p.v_token) * ELEM;
                    if (v_live)
#pragma unroll
                        for (int e = 0; e < 4; e++) load_words(base + (long long) e * p.v_token * ELEM + v_lane, vreg[4 * u + e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = key0 + 16 * u + 4 * g + e, pg = j < count ? table[p.page_tokens.div((unsigned) j)] : -1;
                        const unsigned at_j = (unsigned) j - p.page_tokens.div((unsigned) j) * p.page_tokens.d;
                        if ((unsigned) pg < (unsigned) p.pages) {
                            if (v_live) load_words(vb + (pg * p.v_page + at_j * p.v_token + i * DPL) * ELEM, vreg[4 * u + e]);
                            if (I8) {
                                const long long s = ((long long) pg * p.kv_heads + kv_head) * p.page_tokens.d + at_j;
                                kscale[u][e] = p.k_scales[s];
                                vscale[u][e] = p.v_scales[s];
                            }
                        } else {
                            gone_next |= 1u << (4 * u + e);
                        }
                    }
                }
            }
        };

        int key0 = from + first_key;
        if (key0 < end) {
            if (from != item_from) look_up(key0);
            place(key0);
            load_k(key0);
            load_scales(key0);
            load_v(key0);
            look_up(key0 + STRIDE);
        }
        while (key0 < end) {
            gone = gone_next;
            const int next = key0 + STRIDE;
            const bool more = next < end;
            if (more) place(next);
            const bool masked = key0 < whole_from || key0 + 32 > min(whole_end, end) || __any(gone != 0);
            floatx4 st[NT][2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                halfx8 a[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; s++) {
                    if (I8) {
                        const uint4 x = kreg[u][s / 2];
                        a[s] = s % 2 ? widen(x.z, x.w) : widen(x.x, x.y);
                    } else {
                        a[s] = __builtin_bit_cast(halfx8, kreg[u][I8 ? 0 : s]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    st[n][u] = floatx4{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < STEPS; s++) st[n][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s], qf[n][s], st[n][u], 0, 0, 0);
                }
            }
            if (more) load_k(next);
            float value_log[8], value_inv[8];
            if (I8)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const ValueScale v(vscale[e / 4][e % 4]);
                    value_log[e] = v.log;
                    value_inv[e] = v.inv;
                }
            halfx8 weights[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float top = -INFINITY, s2[8];
#pragma unroll
                for (int e = 0; e < 8; e++) s2[e] = st[n][e / 4][e % 4] * (I8 ? kscale[e / 4][e % 4] : 1.0f);
                if (SHAPED && capped) {
                    float far = fabsf(s2[0]);
#pragma unroll
                    for (int e = 1; e < 8; e++) far = fmaxf(far, fabsf(s2[e]));
                    if (__all(far <= cap.near)) {
#pragma unroll
                        for (int e = 0; e < 8; e++) s2[e] = cap.series(s2[e]);
                    } else if (!Cap::large(p.cap)) {
#pragma unroll
                        for (int e = 0; e < 8; e++) s2[e] = cap.small(s2[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) s2[e] = cap.any(s2[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = key0 + 16 * (e / 4) + 4 * g + e % 4;
                    float x = s2[e];
                    if (!(SHAPED && capped)) x *= scale2;
                    if (SHAPED) x = __builtin_fmaf(-slope2[n], fabsf((float) (at[n] - key)), x);
                    if (I8) x += value_log[e];
                    if (masked && ((unsigned) (key - lo[n]) >= (unsigned) (hi[n] - lo[n]) || key >= end || ((gone >> e) & 1))) x = -INFINITY;
                    s2[e] = x;
                    top = fmaxf(top, x);
                }
                if (__any(top > ref[n] + SLACK)) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float new_ref = fmaxf(ref[n], top);
                    const float alpha = __builtin_amdgcn_exp2f(ref[n] - (new_ref == -INFINITY ? 0.0f : new_ref));
                    ref[n] = new_ref;
                    sum[n] *= alpha;
#pragma unroll
                    for (int d = 0; d < DPL; d++) oacc[n][d] *= alpha;
                }
                const float minus = ref[n] == -INFINITY ? 0.0f : ref[n] - LIFT;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = __builtin_amdgcn_exp2f(s2[e] - minus);
                    sum[n] = I8 ? __builtin_fmaf(x, value_inv[e], sum[n]) : sum[n] + x;
                    weights[n][e] = (half_t) x;
                }
            }
            if (more && PAGE16) load_scales(next);
            unsigned bad = 0;  // keys of the lane's 8 whose values hold an infinity or NaN, where not every row sees every key
            if (!I8 && masked) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool there = key0 + 16 * (e / 4) + 4 * g + e % 4 < count && !((gone >> e) & 1);
                    bool any = false;
#pragma unroll
                    for (int x = 0; x < VW; x++) {
                        if (!there) vreg[e][x] = 0;
                        any |= (vreg[e][x] & 0x7c00u) == 0x7c00u || (vreg[e][x] & 0x7c000000u) == 0x7c000000u;
                    }
                    // (of the 16 lanes of a group)
                    if ((__ballot(any) >> (16 * g)) & 0xffffu) bad |= 1u << e;
                }
            }
            const bool any_bad = !I8 && __any(bad != 0);
#pragma unroll
            for (int d = 0; d < DPL; d++) {
                unsigned pair[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (I8) {
                        const unsigned sel = (unsigned) (d % 4) | 0x0c00u | (unsigned) (4 + d % 4) << 16 | 0x0c000000u;
                        pair[k] = pk_sub_1152(__builtin_amdgcn_perm(vreg[2 * k + 1][d / 4] ^ 0x80808080u, vreg[2 * k][d / 4] ^ 0x80808080u, sel) | 0x64006400u);
                    } else {
                        pair[k] = __builtin_amdgcn_perm(vreg[2 * k + 1][I8 ? 0 : d / 2], vreg[2 * k][I8 ? 0 : d / 2], d % 2 ? 0x07060302u : 0x05040100u);
                    }
                }
                const halfx8 a = __builtin_bit_cast(halfx8, uint4{pair[0], pair[1], pair[2], pair[3]});
                const halfx8 good = any_bad ? finite_or_zero(a) : a;
#pragma unroll
                for (int n = 0; n < NT; n++) oacc[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(good, weights[n], oacc[n][d], 0, 0, 0);
            }
            if (any_bad) {
                // (as in the kernel above: what is not finite is added for the queries that see its key)
#pragma unroll 1
                for (int key = 0; key < 32; key++) {
                    const int group = (key % 16) / 4, nth = 4 * (key / 16) + key % 4;
                    if (!__any(g == group && ((bad >> nth) & 1))) continue;
#pragma unroll
                    for (int d = 0; d < DPL; d++)
#pragma unroll
                        for (int v = 0; v < 4; v++) {
                            // register v of product d: dim (4 g + v) DPL + d, which lane (4 g + v, group) holds
                            unsigned word = 0;
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (e == nth) word = vreg[e][I8 ? 0 : d / 2];
                            const unsigned got = __shfl(word, 16 * group + 4 * g + v);
                            const float x = (float) __builtin_bit_cast(half_t, (unsigned short) (d % 2 ? got >> 16 : got));
#pragma unroll
                            for (int n = 0; n < NT; n++)
                                if ((unsigned) (key0 + key - lo[n]) < (unsigned) (hi[n] - lo[n])) oacc[n][d][v] += x - x == 0.0f ? 0.0f : x;
                        }
                }
            }
            if (more) {
                load_v(next);
                look_up(next + STRIDE);
            }
            key0 = next;
        }
        taken = (end - from + 31) / 32;
    }

    // ---- the waves' parts into one
#pragma unroll
    for (int n = 0; n < NT; n++) {
        sum[n] += __shfl_xor(sum[n], 16);
        sum[n] += __shfl_xor(sum[n], 32);
        if (g == 0) {
            refs[wave][16 * n + i] = ref[n];
            sums[wave][16 * n + i] = sum[n];
        }
        // register v of product d: dim (4 g + v) DPL + d of row i
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int d = 0; d < DPL; d += 4)
                *(floatx4 *) &os[wave][16 * n + i][(4 * g + v) * DPL + d] = floatx4{oacc[n][d][v], oacc[n][d + 1][v], oacc[n][d + 2][v], oacc[n][d + 3][v]};
    }
    __syncthreads();
    const bool direct = !is_prefix && (p.prefix_tokens == 0 || INSIDE) && item.items == 1;
    for (int e = threadIdx.x; e < rows * (WP / 4); e += ROW_THREADS) {
        const int r = e / (WP / 4), d = 4 * (e % (WP / 4));
        float top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int w = 0; w < ROW_WAVES; w++) top = fmaxf(top, refs[w][r]);
        floatx4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < ROW_WAVES; w++) {
            const float weight = __builtin_amdgcn_exp2f(refs[w][r] - (top == -INFINITY ? 0.0f : top));
            total += weight * sums[w][r];
            x += weight * *(const floatx4 *) &os[w][r][d];
        }
        if (direct) {
            const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
            const Row w = row_of<OWN>(p, r, b, kv_head, item.length);
            if (d < p.width)
                *(halfx4_any *) ((half_t *) p.out + (w.b * p.o_batch + w.t * p.o_token + w.head * p.o_head + d)) =
                    halfx4{(half_t) (x[0] * inv), (half_t) (x[1] * inv), (half_t) (x[2] * inv), (half_t) (x[3] * inv)};
        } else {
            const long long part = is_prefix ? p.row_prefix_part : p.row_own_part;
            const long long at_part = part + ((long long) global_item * p.kv_heads + kv_head) * rows + r;
            *(floatx4 *) (p.part_values + at_part * WP + d) = x;
            if (d == 0) *(float2 *) (p.part_stats + 2 * at_part) = float2{top, total};
        }
    }
}

// ---- parts -> results ----------------------------------------------------------------------------------------------

// A wave per row of the result. WP / 4 lanes take a part's row, 16 bytes each, so that a wave reads 2 (4) parts at a time; up
// to PARTS (8 or 32) are in flight together, requested before their weights are known. Bound by the parts: they come out of the
// caches of other XCDs. (32 in flight where there are two parts: 59 us instead of 43 for a prompt of 1024 tokens.)
template <int WP, int PARTS>
__global__ __launch_bounds__(64 * WAVES) void join_attention_kernel(ServingAttentionParams p) {
    constexpr int LANES = WP / 4, SIDE = 64 / LANES, AHEAD = PARTS / SIDE;
    const int lane = threadIdx.x & 63, side = lane / LANES, d = 4 * (lane % LANES);
    const unsigned row = __builtin_amdgcn_readfirstlane(blockIdx.x * WAVES + (threadIdx.x >> 6));
    if (row >= (unsigned) p.batch * p.queries * p.heads) return;
    const unsigned token = row / (unsigned) p.heads, head = row - token * p.heads;
    const unsigned b = p.queries_div.div(token), t = token - b * p.queries_div.d;
    const unsigned kv_head = p.group_div.div(head), in_group = head - kv_head * p.group_div.d;
    const long long own_rows = (long long) p.queries * p.group_div.d, prefix_rows = p.batch * own_rows;
    const long long own_row = t * p.group_div.d + in_group, prefix_row = b * own_rows + own_row;
    // where the parts of either stretch start, how far apart they are and how many there are
    long long at[2] = {0, 0}, apart[2] = {0, 0};
    int count[2] = {0, 0};
    if (p.prefix_splits > 0) {
        at[0] = (long long) kv_head * p.prefix_splits * prefix_rows + prefix_row;
        apart[0] = prefix_rows;
        count[0] = p.prefix_splits;
    } else if (p.prefix_tokens > 0 && !p.prefix_inside) {
        const int2 items = ((const int2 *) p.part_items)[0];
        at[0] = p.row_prefix_part + ((long long) items.x * p.kv_heads + kv_head) * prefix_rows + prefix_row;
        apart[0] = p.kv_heads * prefix_rows;
        count[0] = items.y;
    }
    if (p.own_splits > 0) {
        at[1] = p.row_own_part + ((long long) b * p.kv_heads + kv_head) * p.own_splits * own_rows + own_row;
        apart[1] = own_rows;
        count[1] = p.own_splits;
    } else {
        const int2 items = ((const int2 *) p.part_items)[b + 1];
        if ((p.prefix_tokens == 0 || p.prefix_inside) && items.y == 1) return;  // (written where it was computed)
        at[1] = p.row_own_part + ((long long) items.x * p.kv_heads + kv_head) * own_rows + own_row;
        apart[1] = p.kv_heads * own_rows;
        count[1] = items.y;
    }
    float top = -INFINITY, total = 0.0f;
    floatx4 x = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < 2; s++)
        for (int i0 = 0; i0 < count[s]; i0 += PARTS) {
            const int n = min(PARTS, count[s] - i0);
            floatx4 part[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                const int i = a * SIDE + side;
                part[a] = floatx4{0, 0, 0, 0};
                if (i < n) part[a] = *(const floatx4 *) (p.part_values + (at[s] + (i0 + i) * apart[s]) * WP + d);
            }
            float2 stats = {-INFINITY, 0.0f};
            if (lane < n) stats = *(const float2 *) (p.part_stats + 2 * (at[s] + (i0 + lane) * apart[s]));
            float new_top = fmaxf(top, stats.x);
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) new_top = fmaxf(new_top, __shfl_xor(new_top, m));
            const float ref = new_top == -INFINITY ? 0.0f : new_top, old = __builtin_amdgcn_exp2f(top - ref);
            const float weight = __builtin_amdgcn_exp2f(stats.x - ref);
            top = new_top;
            total = total * old + weight * stats.y;
            x *= old;
#pragma unroll
            for (int a = 0; a < AHEAD; a++) x += __shfl(weight, a * SIDE + side) * part[a];
        }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) total += __shfl_xor(total, m);
#pragma unroll
    for (int m = LANES; m < 64; m <<= 1)
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] += __shfl_xor(x[k], m);
    const float inv = total > 0.0f || total != total ? 1.0f / total : 0.0f;
    if (side == 0 && d < p.width)
        *(halfx4_any *) ((half_t *) p.out + (b * p.o_batch + t * p.o_token + head * p.o_head + d)) =
            halfx4{(half_t) (x[0] * inv), (half_t) (x[1] * inv), (half_t) (x[2] * inv), (half_t) (x[3] * inv)};
}

// ---- plans ---------------------------------------------------------------------------------------------------------

// Waves for the rows of a tile, 32 rows each. Whole numbers are widened as they are staged, work that eight waves share better
// than four (16384 shared keys of width 128 for 256 rows of 8 heads, and what goes with them: 76 us against 99). f16 only
// passes through; eight waves still stage once for twice the rows, which pays where that leaves tiles enough to even out
// their lengths. Four / eight waves, us, causal prompts of 32 heads: 1024 tokens 32 / 46, 2048 67 / 84, 2816 93 / 99, 3328 119 / 118,
// 3584 138 / 127, 4096 177 / 159, 5000 250 / 255, 8192 633 / 595; four prompts of 1024 tokens 59 / 54, of 2048 184 / 174; 4096
// tokens in 4 documents 97 / 93, in 9 78 / 76, in 20 65 / 70; 8192 with a window of 256 79 / 83, of 1024 182 / 178. With 8 heads
// the longer tiles win earlier (8192 tokens 241 / 213, but 12000 381 / 397). `rows`: of a sequence and head of keys,
// `pairs` of which there are.
int tile_waves(int wp, bool i8, long long rows, long long pairs) { return wp == 128 && (i8 || (rows >= 1024 && rows * pairs >= 7 << 14)) ? 8 : 4; }

struct Plan {
    int own_rows;             // per sequence and head of keys
    long long prefix_rows;
    bool own_in_rows, prefix_in_rows;  // which kernel
    bool list;                         // of the row kernel's items
    bool prefix_inside;                // of every sequence's own rows, see row_attention_kernel
    long long own_tiles, prefix_tiles;
    int own_splits, prefix_splits;     // of the tile kernel
    int own_waves, prefix_waves;       // for the rows of a tile
    long long items;                   // of the row kernel, at most
    bool join;
    long long prefix_parts, own_parts;  // rows of partial results
    int wp;
};

// How many workgroups share the keys of a tile, by what that costs in the time of one block of keys (1.5 us with four waves on
// a compute unit, 2.6 with eight). `longest` and `mean`: keys of a tile. The longest tile is a chain of blocks, all of
// them together are work for 256 compute units. A part is written and read again: 5900 rows of parts cost as much as a
// block of four waves, and the launch of the join two blocks. (One prompt of 1024 tokens and 32 heads: 33 us whole, 43
// in two parts; of 8 heads: 32 us whole, 24 in four.)
int splits_for(long long workgroups, long long rows, long long longest, long long mean, int waves, bool join_anyway) {
    const long long blocks = std::max(1ll, (longest + 63) / 64);
    int best = 1;
    double least = 0.0;
    for (long long s = 1; s <= blocks && (s == 1 || workgroups * s <= 512); s++) {
        const double chain = (double) ((blocks + s - 1) / s), share = (double) mean / (double) std::max(1ll, longest);
        const double reading = chain * std::max(1.0, share * (double) ((workgroups * s + 255) / 256));
        const double joining = s == 1 && !join_anyway ? 0.0 : 2.0 + (double) (rows * s) * WAVES / (5900.0 * waves);
        if (s == 1 || reading + joining < least) {
            least = reading + joining;
            best = (int) s;
        }
    }
    return best;
}

Plan plan_for(const ServingAttentionParams &p) {
    Plan l = {};
    l.wp = p.width <= 64 ? 64 : 128;
    l.own_rows = p.queries * (p.heads / p.kv_heads);
    l.prefix_rows = (long long) p.batch * l.own_rows;
    // a tile of 16 or 32 rows keeps the keys streaming; more rows are worth staging them for
    l.own_in_rows = p.paged && l.own_rows <= 32;
    const long long pairs = (long long) p.batch * p.kv_heads;
    // A short prefix is read again for every sequence, which takes a workgroup, one per compute unit at a time, about a
    // microsecond for 128 keys, and saves the launch of the tiles and the join, or only the join where all rows of the batch fit this
    // kernel. (64 sequences of up to 700 tokens, 8 heads of keys, two rounds of workgroups: 18 shared tokens 27 us against
    // 45, 512 37 against 46, 1024 48 against 49, 2048 70 against 51. One sequence: 18 14 against 19, 1024 23 against 21.)
    const bool few_rows = l.prefix_rows <= 32;
    l.prefix_inside = l.own_in_rows && l.own_rows <= 16 && p.prefix_tokens > 0 && p.prefix_tokens * ((pairs + 255) / 256) <= (few_rows ? 768 : 1792);
    l.prefix_in_rows = !l.prefix_inside && p.prefix_tokens > 0 && few_rows;
    const bool prefix_apart = !l.prefix_inside && p.prefix_tokens > 0;
    const bool i8 = p.k_scales != nullptr;
    if (!l.own_in_rows) {
        l.own_waves = tile_waves(l.wp, i8, l.own_rows, pairs);
        const int tile_rows = 32 * l.own_waves;
        l.own_tiles = (l.own_rows + tile_rows - 1) / tile_rows;
        const long long keys = p.paged ? p.table_tokens : p.keys, tile_tokens = tile_rows / (p.heads / p.kv_heads) + 2;
        const long long longest = p.window > 0 ? std::min(keys, p.window + tile_tokens) : keys;
        const long long mean = p.paged || p.causal ? std::min(longest, std::max(keys - p.queries / 2, 1ll)) : longest;
        l.own_splits = splits_for(l.own_tiles * pairs, pairs * l.own_rows, longest, mean, l.own_waves, prefix_apart);
        l.own_parts = l.own_splits * pairs * l.own_rows;
    }
    if (prefix_apart && !l.prefix_in_rows) {
        l.prefix_waves = tile_waves(l.wp, i8, l.prefix_rows, p.kv_heads);
        l.prefix_tiles = (l.prefix_rows + 32 * l.prefix_waves - 1) / (32 * l.prefix_waves);
        l.prefix_splits = splits_for(l.prefix_tiles * p.kv_heads, p.kv_heads * l.prefix_rows, p.prefix_tokens, p.prefix_tokens, l.prefix_waves, true);
        l.prefix_parts = (long long) l.prefix_splits * p.kv_heads * l.prefix_rows;
    }
    if (l.own_in_rows) {
        // the stretches and the items beyond one of each, see find_item
        const long long stretches = p.batch + (l.prefix_in_rows ? 1 : 0);
        long long by_keys = p.batch * std::max(1ll, ((long long) p.table_tokens + ROW_MIN_KEYS - 1) / ROW_MIN_KEYS);
        if (l.prefix_in_rows) by_keys += std::max(1, (p.prefix_tokens + ROW_MIN_KEYS - 1) / ROW_MIN_KEYS);
        l.items = std::min(stretches + ROW_ITEMS / p.kv_heads, by_keys);
        l.list = p.batch > 64 && p.batch * pairs >= LIST_FROM;  // (a prefix in this kernel has rows of 32 sequences at most)
        l.own_parts = l.items * p.kv_heads * l.own_rows;
        if (l.prefix_in_rows) l.prefix_parts = l.items * p.kv_heads * l.prefix_rows;
    }
    l.join = prefix_apart || (l.own_in_rows ? l.items > p.batch : l.own_splits > 1);
    if (!l.join) l.own_parts = 0;
    return l;
}

size_t round256(size_t bytes) { return (bytes + 255) / 256 * 256; }

template <int WP, int STRETCH, bool I8, int RW, int KG>
int launch_tiles(const ServingAttentionParams &p, unsigned workgroups, int splits, hipStream_t stream) {
    constexpr int TW = RW * KG;
    const dim3 grid(workgroups, (unsigned) splits), block(64 * TW);
    if (Cap::large(p.cap)) hipLaunchKernelGGL((tile_attention_kernel<WP, STRETCH, I8, LARGE_CAP, TW, KG>), grid, block, 0, stream, p);
    else if (p.cap > 0.0f || p.slopes) hipLaunchKernelGGL((tile_attention_kernel<WP, STRETCH, I8, SHAPED_SCORES, TW, KG>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((tile_attention_kernel<WP, STRETCH, I8, PLAIN, TW, KG>), grid, block, 0, stream, p);
    return (int) hipGetLastError();
}

// Where compute units would have one workgroup of four waves each, a second group of waves takes every other block of keys. (Two
// workgroups overlap better than two groups, which wait at the same barriers: with 32 heads 1024 tokens, 256 workgroups, take 30
// us in two groups and 33 without, 1536 tokens, 384 workgroups, 44 and 52, but 3000 tokens, 752 workgroups, 128 and 104.)
template <int WP, int STRETCH>
int launch_tiles_of(const ServingAttentionParams &p, int waves, unsigned workgroups, int splits, hipStream_t stream) {
    if constexpr (STRETCH != PROMPT)
        if (p.k_scales) return launch_tiles<WP, STRETCH, true, WP == 128 ? 8 : 4, 1>(p, workgroups, splits, stream);
    if constexpr (WP == 128)
        if (waves == 8) return launch_tiles<WP, STRETCH, false, 8, 1>(p, workgroups, splits, stream);
    const int keys = STRETCH == PROMPT ? p.keys : STRETCH == OWN ? p.table_tokens : p.prefix_tokens;  // (one block cannot be shared)
    return (long long) workgroups * splits <= 384 && keys > 64 ? launch_tiles<WP, STRETCH, false, 4, 2>(p, workgroups, splits, stream)
                                                               : launch_tiles<WP, STRETCH, false, 4, 1>(p, workgroups, splits, stream);
}

template <int WP>
int launch_tiles_for(const ServingAttentionParams &p, int stretch, int waves, unsigned workgroups, int splits, hipStream_t stream) {
    return stretch == PROMPT ? launch_tiles_of<WP, PROMPT>(p, waves, workgroups, splits, stream)
         : stretch == OWN    ? launch_tiles_of<WP, OWN>(p, waves, workgroups, splits, stream)
                             : launch_tiles_of<WP, PREFIX>(p, waves, workgroups, splits, stream);
}

template <int WP, int NT, bool I8, bool INSIDE>
int launch_rows(const ServingAttentionParams &p, unsigned workgroups, int with_prefix, hipStream_t stream) {
    const bool shaped = p.cap > 0.0f || p.slopes, page16 = p.page_tokens.d % 16 == 0 && p.k_token <= 1 << 25;
    const dim3 grid(workgroups), block(ROW_THREADS);
    if (shaped && page16) hipLaunchKernelGGL((row_attention_kernel<WP, NT, I8, true, true, INSIDE>), grid, block, 0, stream, p, with_prefix);
    else if (shaped) hipLaunchKernelGGL((row_attention_kernel<WP, NT, I8, true, false, INSIDE>), grid, block, 0, stream, p, with_prefix);
    else if (page16) hipLaunchKernelGGL((row_attention_kernel<WP, NT, I8, false, true, INSIDE>), grid, block, 0, stream, p, with_prefix);
    else hipLaunchKernelGGL((row_attention_kernel<WP, NT, I8, false, false, INSIDE>), grid, block, 0, stream, p, with_prefix);
    return (int) hipGetLastError();
}

template <int WP, bool I8>
int launch_rows_of(const ServingAttentionParams &p, unsigned workgroups, bool two_tiles, int with_prefix, hipStream_t stream) {
    if (p.prefix_inside) return launch_rows<WP, 1, I8, true>(p, workgroups, with_prefix, stream);
    return two_tiles ? launch_rows<WP, 2, I8, false>(p, workgroups, with_prefix, stream) : launch_rows<WP, 1, I8, false>(p, workgroups, with_prefix, stream);
}

template <int WP>
int launch_rows_for(const ServingAttentionParams &p, unsigned workgroups, bool two_tiles, int with_prefix, hipStream_t stream) {
    return p.k_scales ? launch_rows_of<WP, true>(p, workgroups, two_tiles, with_prefix, stream)
                      : launch_rows_of<WP, false>(p, workgroups, two_tiles, with_prefix, stream);
}

template <int WP, int PARTS>
int launch_join(const ServingAttentionParams &p, hipStream_t stream) {
    const unsigned workgroups = (unsigned) (((long long) p.batch * p.queries * p.heads + WAVES - 1) / WAVES);
    hipLaunchKernelGGL((join_attention_kernel<WP, PARTS>), dim3(workgroups), dim3(64 * WAVES), 0, stream, p);
    return (int) hipGetLastError();
}

}  // namespace

// partial values, then their references and sums, then the items of the row kernel and their list
size_t serving_attention_workspace(const ServingAttentionParams &p) {
    const Plan l = plan_for(p);
    const size_t parts = (size_t) (l.prefix_parts + l.own_parts);
    size_t bytes = round256(parts * l.wp * 4) + round256(parts * 8);
    if (l.own_in_rows) bytes += round256(((size_t) p.batch + 1) * 8);
    if (l.list) bytes += round256((size_t) l.items * 4);
    return bytes;
}

int launch_serving_attention(const ServingAttentionParams &given, void *workspace, ihipStream_t *stream) {
    ServingAttentionParams p = given;
    const Plan l = plan_for(p);
    const size_t parts = (size_t) (l.prefix_parts + l.own_parts);
    p.group_div = FastDiv((uint32_t) (p.heads / p.kv_heads));
    p.queries_div = FastDiv((uint32_t) p.queries);
    float *values = (float *) workspace, *stats = (float *) ((char *) workspace + round256(parts * l.wp * 4));
    p.part_items = l.own_in_rows ? (int32_t *) ((char *) stats + round256(parts * 8)) : nullptr;
    p.item_list = l.list ? (int32_t *) ((char *) p.part_items + round256(((size_t) p.batch + 1) * 8)) : nullptr;
    p.row_prefix_part = 0;
    p.row_own_part = l.prefix_parts;
    p.prefix_inside = l.prefix_inside;
    p.prefix_splits = l.prefix_splits;
    p.own_splits = l.own_splits;
    const long long pairs = (long long) p.batch * p.kv_heads;
    if (l.prefix_tiles > 0) {
        p.part_values = values;
        p.part_stats = stats;
        const unsigned workgroups = (unsigned) (l.prefix_tiles * p.kv_heads);
        const int e = l.wp == 64 ? launch_tiles_for<64>(p, PREFIX, l.prefix_waves, workgroups, l.prefix_splits, stream) : launch_tiles_for<128>(p, PREFIX, l.prefix_waves, workgroups, l.prefix_splits, stream);
        if (e != 0) return e;
    }
    if (!l.own_in_rows) {
        p.part_values = l.join ? values + l.prefix_parts * l.wp : nullptr;
        p.part_stats = l.join ? stats + 2 * l.prefix_parts : nullptr;
        const unsigned workgroups = (unsigned) (l.own_tiles * pairs);
        const int stretch = p.paged ? OWN : PROMPT;
        const int e = l.wp == 64 ? launch_tiles_for<64>(p, stretch, l.own_waves, workgroups, l.own_splits, stream) : launch_tiles_for<128>(p, stretch, l.own_waves, workgroups, l.own_splits, stream);
        if (e != 0) return e;
    } else {
        p.part_values = values;
        p.part_stats = stats;
        const unsigned workgroups = (unsigned) (l.items * p.kv_heads);
        if (l.list) {
            hipLaunchKernelGGL(list_items_kernel, dim3(1), dim3(LIST_THREADS), 0, stream, p, (int) l.items);
            const int e = (int) hipGetLastError();
            if (e != 0) return e;
        }
        const bool two_tiles = (l.prefix_in_rows ? l.prefix_rows : l.own_rows) > 16;
        const int e = l.wp == 64 ? launch_rows_for<64>(p, workgroups, two_tiles, l.prefix_in_rows, stream) : launch_rows_for<128>(p, workgroups, two_tiles, l.prefix_in_rows, stream);
        if (e != 0) return e;
    }
    if (l.join) {
        p.part_values = values;
        p.part_stats = stats;
        // (which count decides only how many loads are in flight at a time: any number of parts comes out right)
        const bool few = !l.own_in_rows && l.own_splits <= 8 && l.prefix_splits <= 8;
        return l.wp == 64 ? few ? launch_join<64, 8>(p, stream) : launch_join<64, 32>(p, stream)
                          : few ? launch_join<128, 8>(p, stream) : launch_join<128, 32>(p, stream);
    }
    return 0;
}

}  // namespace kn
