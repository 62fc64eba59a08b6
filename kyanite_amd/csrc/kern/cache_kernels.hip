// Keys and values into a paged cache and back (knhip_cache_write, knhip_cache_read). A quantised row is whole numbers q and
// one scale: scale = max |x| / 127, q = rint(x / scale), standing for q * scale.
//
// Bound by HBM: a row is read once and written once (128 elements f16 -> i8: 256 + 132 bytes), which leaves a few
// instructions per element. A row belongs to a group of lanes of 8 elements each, so that its maximum is a handful of lane
// exchanges and no element is loaded twice; the group takes the row of the key and the row of the value of one (token,
// head) together, two loads in flight per lane. Quotients are products with the reciprocal of the scale, whose error is
// below 2^-15 of a step: only where one lies within 2^-13 of the middle between two whole numbers is the row's lane divided
// properly. With the division for every element 262144 rows of 128 took 57 us to write, bound by its instructions.
#include <hip/hip_runtime.h>

#include "../serving_kernels.h"

namespace kn {

namespace {

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
// rows outside the cache may start at any element: the hardware takes under-aligned 128 bit accesses
typedef _Float16 halfx8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));

constexpr int THREADS = 256;
constexpr float HALF_MAX = 65504.0f;

template <bool F32>
__device__ __forceinline__ void load_row(const void *base, long long offset, float (&x)[8]) {
    if (F32) {
        const floatx4_any *p = (const floatx4_any *) ((const float *) base + offset);
        const floatx4 a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    } else {
        const halfx8 a = *(const halfx8_any *) ((const _Float16 *) base + offset);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float) a[i];
    }
}

template <int CTRL>
__device__ __forceinline__ float from_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

// the largest of LANES neighbouring lanes: exchanges inside quads, halves of rows and rows of 16
template <int LANES>
__device__ __forceinline__ float group_max(float x) {
    x = fmaxf(x, from_lane<0xb1>(x));   // quad_perm 1 0 3 2
    x = fmaxf(x, from_lane<0x4e>(x));   // quad_perm 2 3 0 1
    x = fmaxf(x, from_lane<0x141>(x));  // row_half_mirror
    if (LANES > 8) x = fmaxf(x, from_lane<0x140>(x));  // row_mirror
    if (LANES > 16) x = fmaxf(x, __shfl_xor(x, 16));
    return x;
}

// (comparisons and not fmin / fmax: a NaN stays one)
__device__ __forceinline__ float clamped(float x) { return x > HALF_MAX ? HALF_MAX : x < -HALF_MAX ? -HALF_MAX : x; }

// LANES lanes of 8 elements per row
template <int LANES, bool QUANTISED, bool F32>
__global__ __launch_bounds__(THREADS) void cache_write_kernel(CacheParams p) {
    const unsigned row = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    const int e = 8 * (threadIdx.x % LANES);
    if (row >= (unsigned) (p.tokens * p.heads)) return;  // (whole groups leave together)
    const unsigned token = p.heads_div.div(row), head = row - token * (unsigned) p.heads;
    const bool live = e < p.width;
    const int slot = p.row_slots[token];
    float x[2][8] = {};
    if (live) {
        load_row<F32>(p.rows_k, (long long) token * p.k_token_stride + (long long) head * p.k_head_stride + e, x[0]);
        load_row<F32>(p.rows_v, (long long) token * p.v_token_stride + (long long) head * p.v_head_stride + e, x[1]);
    }
    if ((unsigned) slot >= (unsigned) p.slots) return;
    const unsigned page = p.page_tokens.div((unsigned) slot), at = (unsigned) slot - page * p.page_tokens.d;
    const long long to = (long long) page * p.page_stride + (long long) head * p.head_stride + (long long) at * p.token_stride + e;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (QUANTISED) {
            if (F32)
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = x[i][j] == x[i][j] ? x[i][j] : 0.0f;  // (an f16 NaN has zeros where the whole number is taken from)
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[i][j]));  // (fmax passes over a NaN)
            top = group_max<LANES>(top);
            if (top > HALF_MAX) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = clamped(x[i][j]);
                top = HALF_MAX;
            }
            const float scale = top / 127.0f, inv = __builtin_amdgcn_rcpf(scale);
            // adding 1.5 2^23 rounds to a whole number, ties to even, and leaves it in the low byte
            constexpr float MAGIC = 12582912.0f;
            unsigned whole[8];
            float off = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float m = __builtin_fmaf(x[i][j], inv, MAGIC);
                off = fmaxf(off, fabsf(__builtin_fmaf(x[i][j], inv, MAGIC - m)));
                whole[j] = __builtin_bit_cast(unsigned, m);
            }
            if (off > 0.5f - 0x1p-13f || scale < 0x1p-120f) {  // (below that the reciprocal and the scale itself are coarse; zero rows too)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float q = scale > 0.0f ? fminf(fmaxf(__builtin_rintf(x[i][j] / scale), -127.0f), 127.0f) : 0.0f;
                    whole[j] = x[i][j] == x[i][j] ? (unsigned) (int) q : 0u;
                }
            }
            // the low bytes of four numbers
            auto pack = [&](int j) {
                return __builtin_amdgcn_perm(__builtin_amdgcn_perm(whole[j + 3], whole[j + 2], 0x0c0c0400u), __builtin_amdgcn_perm(whole[j + 1], whole[j], 0x0c0c0400u), 0x05040100u);
            };
            if (live) *(uint2 *) ((signed char *) (i ? p.v : p.k) + to) = uint2{pack(0), pack(4)};
            if (e == 0) (i ? p.v_scales : p.k_scales)[((long long) page * p.heads + head) * p.page_tokens.d + at] = scale;
        } else {
            halfx8 h;
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = (_Float16) clamped(x[i][j]);
            if (live) *(halfx8 *) ((_Float16 *) (i ? p.v : p.k) + to) = h;
        }
    }
}

template <int LANES, bool QUANTISED, bool F32>
__global__ __launch_bounds__(THREADS) void cache_read_kernel(CacheParams p) {
    const unsigned row = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    const int e = 8 * (threadIdx.x % LANES);
    if (row >= (unsigned) (p.tokens * p.heads) || e >= p.width) return;
    const unsigned token = p.heads_div.div(row), head = row - token * (unsigned) p.heads;
    const int slot = p.row_slots[token];
    float x[2][8] = {};
    if ((unsigned) slot < (unsigned) p.slots) {
        const unsigned page = p.page_tokens.div((unsigned) slot), at = (unsigned) slot - page * p.page_tokens.d;
        const long long from = (long long) page * p.page_stride + (long long) head * p.head_stride + (long long) at * p.token_stride + e;
        if (QUANTISED) {
            const long long s = ((long long) page * p.heads + head) * p.page_tokens.d + at;
            const uint2 packed[2] = {*(const uint2 *) ((const signed char *) p.k + from), *(const uint2 *) ((const signed char *) p.v + from)};
            const float scale[2] = {p.k_scales[s], p.v_scales[s]};
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = (float) (signed char) ((j < 4 ? packed[i].x : packed[i].y) >> (8 * (j % 4))) * scale[i];
        } else {
            load_row<false>(p.k, from, x[0]);
            load_row<false>(p.v, from, x[1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        void *base = i ? p.rows_v : p.rows_k;
        const long long to = (long long) token * (i ? p.v_token_stride : p.k_token_stride) + (long long) head * (i ? p.v_head_stride : p.k_head_stride) + e;
        if (F32) {
            floatx4_any *o = (floatx4_any *) ((float *) base + to);
            o[0] = floatx4{x[i][0], x[i][1], x[i][2], x[i][3]};
            o[1] = floatx4{x[i][4], x[i][5], x[i][6], x[i][7]};
        } else {
            halfx8 h;
#pragma unroll
            for (int j = 0; j < 8; j++) h[j] = (_Float16) x[i][j];
            *(halfx8_any *) ((_Float16 *) base + to) = h;
        }
    }
}

template <int LANES, bool QUANTISED, bool F32>
int launch(const CacheParams &p, bool write, hipStream_t stream) {
    const unsigned rows = (unsigned) (p.tokens * p.heads), per = THREADS / LANES;
    if (write) hipLaunchKernelGGL((cache_write_kernel<LANES, QUANTISED, F32>), dim3((rows + per - 1) / per), dim3(THREADS), 0, stream, p);
    else hipLaunchKernelGGL((cache_read_kernel<LANES, QUANTISED, F32>), dim3((rows + per - 1) / per), dim3(THREADS), 0, stream, p);
    return (int) hipGetLastError();
}

template <int LANES>
int launch_lanes(const CacheParams &p, bool write, hipStream_t stream) {
    if (p.quantised) return p.rows_f32 ? launch<LANES, true, true>(p, write, stream) : launch<LANES, true, false>(p, write, stream);
    return p.rows_f32 ? launch<LANES, false, true>(p, write, stream) : launch<LANES, false, false>(p, write, stream);
}

// the lanes of a row: the power of two that covers its width (80 and 96 leave lanes of 16 idle)
int launch_any(const CacheParams &p, bool write, hipStream_t stream) {
    return p.width <= 64 ? launch_lanes<8>(p, write, stream) : p.width <= 128 ? launch_lanes<16>(p, write, stream) : launch_lanes<32>(p, write, stream);
}

}  // namespace

int launch_cache_write(const CacheParams &p, ihipStream_t *stream) { return launch_any(p, true, stream); }
int launch_cache_read(const CacheParams &p, ihipStream_t *stream) { return launch_any(p, false, stream); }

}  // namespace kn
