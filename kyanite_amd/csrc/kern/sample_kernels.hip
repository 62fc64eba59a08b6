// The draw of a token from a row of logits (knhip_sample).
//
// Weights are 64 bit fixed point, w = round(exp((x - max) / T) 2^bits), with `bits` chosen so that a whole row cannot overflow:
// sums of them are exact and the same in any order, so counting and adding may run in any order and with atomics. exp and its
// argument are f64: the nearest of 10^5 borders between tokens is then missed once in 10^10 rows or so.
//
// A row belongs to one workgroup of 16 waves, each of which owns a contiguous part of it. Rows that fit are held in LDS
// (f16: 60000 logits), so that they are read once. The filters end in one threshold, the last token that stays in the order of
// falling logits (ties: rising index). It is found without sorting:
//   1. a histogram over the distance to the maximum, 2048 buckets over the distances at which w is not zero, counts for
//      top_k, masses for top_p. (Buckets on the bits of x would put most of a row into two dozen of them: the atomics of a
//      wave would queue. Over the distance a normal distribution fills hundreds.)
//   2. the bucket where the count or the mass is reached; its tokens, usually a hundred, are ranked against each other.
// A bucket with more than 1024 tokens (flat rows) is searched by the bits of x instead, 8 at a time.
// The token is then found in two steps: the wave whose part holds the target, and the place inside that part.
#include <hip/hip_runtime.h>

#include "../serving_kernels.h"

namespace kn {

namespace {

constexpr int THREADS = 1024, NWAVES = THREADS / 64;
constexpr int BUCKETS = 2 * THREADS, CANDIDATES = THREADS;
constexpr int CACHE_BYTES = 120 * 1024;

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long mass_t;

// NaN counts as -inf, -0 as +0
__device__ __forceinline__ float plain(float x) { return x != x ? -INFINITY : x + 0.0f; }

// the bits of x as an unsigned number that grows with x
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    return u ^ ((unsigned) ((int) u >> 31) | 0x80000000u);
}

// 16 bytes of a row
template <bool F16>
struct Vec {
    static constexpr int N = F16 ? 8 : 4;
    float x[N];
};

template <bool F16>
__device__ __forceinline__ Vec<F16> unpack(uint4 raw) {
    Vec<F16> v;
    if constexpr (F16) {
        const halfx8 h = __builtin_bit_cast(halfx8, raw);
#pragma unroll
        for (int e = 0; e < 8; e++) v.x[e] = plain((float) h[e]);
    } else {
        const floatx4 f = __builtin_bit_cast(floatx4, raw);
#pragma unroll
        for (int e = 0; e < 4; e++) v.x[e] = plain(f[e]);
    }
    return v;
}

template <bool F16>
__device__ __forceinline__ float load_one(const void *row, int i) {
    return plain(F16 ? (float) ((const _Float16 *) row)[i] : ((const float *) row)[i]);
}

// vector n of a row of `vocab` logits; what lies behind its end reads as -inf
template <bool F16>
__device__ __forceinline__ uint4 load_raw(const void *row, int n, int vocab) {
    constexpr int N = Vec<F16>::N;
    if (n * N + N <= vocab) {
        if constexpr (F16) return __builtin_bit_cast(uint4, *(const halfx8_any *) ((const _Float16 *) row + n * N));
        else return __builtin_bit_cast(uint4, *(const floatx4_any *) ((const float *) row + n * N));
    }
    if constexpr (F16) {
        halfx8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = n * N + e < vocab ? ((const _Float16 *) row)[n * N + e] : (_Float16) -INFINITY;
        return __builtin_bit_cast(uint4, h);
    } else {
        floatx4 f;
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = n * N + e < vocab ? ((const float *) row)[n * N + e] : -INFINITY;
        return __builtin_bit_cast(uint4, f);
    }
}

// exp((x - top) / T) 2^bits for x <= top. 2^(n / 64 + r / 64) with |r| <= 1/2: a table of 64 roots of two, and the series of
// exp(r ln2 / 64) up to the 5th power, whose rest is below 4e-17.
struct Weigher {
    float top;
    double per;  // 64 log2(e) / T
    int bits;
    const double *roots;
    __device__ __forceinline__ double real(float x) const {
        constexpr double L = 0.010830424696249145;  // ln(2) / 64
        const double t = fmax(((double) x - (double) top) * per, -64.0 * 1000);
        const double n = __builtin_rint(t), z = (t - n) * L;
        const int i = (int) n;
        const double s = __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, __builtin_fma(z, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0);
        const double w = __builtin_ldexp(roots[i & 63] * s, (i >> 6) + bits);
        return x == top ? __builtin_ldexp(1.0, bits) : top == INFINITY || x == -INFINITY ? 0.0 : w;
    }
    // (bits <= 51: adding 2^52 rounds to a whole number and leaves it in the low bits)
    static __device__ __forceinline__ mass_t whole(double w) { return __builtin_bit_cast(mass_t, w + 0x1p52) & ((1ull << 52) - 1); }
    __device__ __forceinline__ mass_t operator()(float x) const { return whole(real(x)); }
};

struct Shared {
    mass_t hist[BUCKETS];
    unsigned cand_key[CANDIDATES], cand_index[CANDIDATES];
    mass_t cand_mass[CANDIDATES];
    double roots[64];
    mass_t wave_mass[NWAVES];
    float wave_top[NWAVES];
    int cand_count, bucket;
    mass_t above;
    unsigned last_key;  // the threshold: the last token that stays
    int last_index;
    mass_t search_mass;
    unsigned search_prefix, search_count;
};

__device__ __forceinline__ mass_t wave_scan(mass_t v, int lane) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const mass_t other = __shfl_up(v, m);
        if (lane >= m) v += other;
    }
    return v;
}

__device__ __forceinline__ mass_t wave_sum(mass_t v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

template <bool F16, bool CACHED>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p) {
    constexpr int N = Vec<F16>::N;
    __shared__ Shared sh;
    __shared__ uint4 cache[CACHED ? CACHE_BYTES / 16 : 1];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const void *row = (const char *) p.logits + r * p.row_stride * (F16 ? 2 : 4);
    const int vectors = (p.vocab + N - 1) / N, part = (vectors + NWAVES - 1) / NWAVES;
    const int begin = min(wave * part, vectors), end = min(begin + part, vectors);  // of this wave, in vectors

    // f(first index, values) for the vectors of this wave
    auto each = [&](auto f) {
        int n = begin + lane;
        constexpr int AHEAD = 4;
        for (; n + 64 * (AHEAD - 1) < end; n += 64 * AHEAD) {
            uint4 raw[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) raw[a] = CACHED ? cache[n + 64 * a] : load_raw<F16>(row, n + 64 * a, p.vocab);
#pragma unroll
            for (int a = 0; a < AHEAD; a++) f((n + 64 * a) * N, unpack<F16>(raw[a]));
        }
        for (; n < end; n += 64) f(n * N, unpack<F16>(CACHED ? cache[n] : load_raw<F16>(row, n, p.vocab)));
    };

    // ---- the maximum (and the row into LDS)
    float top = -INFINITY;
    {
        int n = begin + lane;
        constexpr int AHEAD = 8;
        auto take = [&](int at, uint4 raw) {
            if (CACHED) cache[at] = raw;
            const Vec<F16> v = unpack<F16>(raw);
#pragma unroll
            for (int e = 0; e < N; e++) top = fmaxf(top, v.x[e]);
        };
        for (; n + 64 * (AHEAD - 1) < end; n += 64 * AHEAD) {
            uint4 raw[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) raw[a] = load_raw<F16>(row, n + 64 * a, p.vocab);
#pragma unroll
            for (int a = 0; a < AHEAD; a++) take(n + 64 * a, raw[a]);
        }
        for (; n < end; n += 64) take(n, load_raw<F16>(row, n, p.vocab));
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
        if (lane == 0) sh.wave_top[wave] = top;
        if (threadIdx.x < 64) sh.roots[threadIdx.x] = exp2(threadIdx.x * (1.0 / 64));
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NWAVES; w++) top = fmaxf(top, sh.wave_top[w]);
    }
    if (top == -INFINITY) {
        if (threadIdx.x == 0) {
            p.tokens[r] = -1;
            if (p.probabilities) p.probabilities[r] = 0.0f;
        }
        return;
    }
    const float t = p.temperature ? p.temperature[r] : 1.0f;
    if (!(t > 0.0f)) {  // the first of the largest
        if (threadIdx.x == 0) sh.last_index = p.vocab;
        __syncthreads();
        int first = p.vocab;
        each([&](int i, const Vec<F16> &v) {
#pragma unroll
            for (int e = N - 1; e >= 0; e--)
                if (v.x[e] == top) first = min(first, i + e);
        });
        if (first < p.vocab) atomicMin(&sh.last_index, first);
        __syncthreads();
        if (threadIdx.x == 0) {
            p.tokens[r] = sh.last_index;
            if (p.probabilities) p.probabilities[r] = 1.0f;
        }
        return;
    }
    const Weigher weigh{top, 92.332482616893656877 / (double) t, p.bits, sh.roots};
    const int k = p.top_k ? p.top_k[r] : 0;
    const float top_p = p.top_p ? p.top_p[r] : 1.0f;
    const double min_w = p.min_p ? __builtin_ldexp((double) p.min_p[r], p.bits) : 0.0;
    // distances at which w may be more than zero: exp(-range / T) 2^bits = 1 / 4
    const float range = t * (0.6931472f * (p.bits + 2)), per_bucket = fminf(BUCKETS / range, 3e38f);
    const bool spread = range < 1e37f;
    auto bucket_of = [&](float x) {
        const float away = x == top ? 0.0f : top - x;
        return away < range ? min((int) (away * per_bucket), BUCKETS - 1) : BUCKETS;
    };
    unsigned last_key = 0;  // what stays: larger keys, and this key up to last_index
    int last_index = p.vocab;
    auto stays = [&](unsigned key, int i) { return key > last_key || (key == last_key && i <= last_index); };

    // The threshold at which `enough(tokens, mass)`, called with what lies at and above a token, first holds, among what stays
    // so far; tokens without weight have no part in it. `by_mass`: whether masses are needed.
    auto tighten = [&](bool by_mass, auto enough) {
        bool found = false;
        if (spread) {
            __syncthreads();
            for (int b = threadIdx.x; b < BUCKETS; b += THREADS) sh.hist[b] = 0;
            if (threadIdx.x == 0) {
                sh.cand_count = 0;
                sh.bucket = BUCKETS;
            }
            __syncthreads();
            each([&](int i, const Vec<F16> &v) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int b = bucket_of(v.x[e]);
                    if (b < BUCKETS && stays(key_of(v.x[e]), i + e)) {
                        if (by_mass) atomicAdd(&sh.hist[b], weigh(v.x[e]));
                        else atomicAdd((unsigned *) &sh.hist[b], 1u);
                    }
                }
            });
            __syncthreads();
            // a thread takes two neighbouring buckets
            const mass_t a = sh.hist[2 * threadIdx.x], both = a + sh.hist[2 * threadIdx.x + 1];
            mass_t sums = wave_scan(both, lane);
            if (lane == 63) sh.wave_mass[wave] = sums;
            __syncthreads();
            mass_t before = sums - both;
            for (int w = 0; w < wave; w++) before += sh.wave_mass[w];
            auto reached = [&](mass_t m) { return by_mass ? enough(0u, m) : enough((unsigned) m, (mass_t) 0); };
            if (both && !reached(before) && reached(before + both)) {
                const bool second = a == 0 || !reached(before + a);
                sh.bucket = 2 * threadIdx.x + second;
                sh.above = before + (second ? a : 0);
            }
            if (threadIdx.x == 0 && reached(0)) {  // (a top_p of zero: the largest stays)
                sh.bucket = 0;
                sh.above = 0;
            }
            __syncthreads();
            const int bucket = sh.bucket;
            if (bucket == BUCKETS) return;  // everything that weighs anything stays
            const mass_t above = sh.above;
            each([&](int i, const Vec<F16> &v) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const unsigned key = key_of(v.x[e]);
                    if (bucket_of(v.x[e]) != bucket || !stays(key, i + e)) continue;
                    const int c = atomicAdd(&sh.cand_count, 1);
                    if (c >= CANDIDATES) continue;
                    sh.cand_key[c] = key;
                    sh.cand_index[c] = i + e;
                    sh.cand_mass[c] = by_mass ? weigh(v.x[e]) : 1;
                }
            });
            __syncthreads();
            const int count = sh.cand_count;
            found = count <= CANDIDATES;
            if (found && (int) threadIdx.x < count) {
                const unsigned key = sh.cand_key[threadIdx.x], index = sh.cand_index[threadIdx.x];
                mass_t first = above;
                for (int c = 0; c < count; c++)
                    if (sh.cand_key[c] > key || (sh.cand_key[c] == key && sh.cand_index[c] < index)) first += sh.cand_mass[c];
                const mass_t with = first + sh.cand_mass[threadIdx.x];
                // (the largest token stays even if nothing is wanted)
                if ((!reached(first) || (bucket == 0 && first == 0)) && reached(with) && (with > first || first == 0)) {
                    sh.last_key = key;
                    sh.last_index = (int) index;
                }
            }
            __syncthreads();
        }
        if (!found) {
            // by the bits of x, from the top: the digit at which it is enough, four times
            mass_t *masses = sh.hist;
            unsigned *counts = (unsigned *) (sh.hist + 256);
            unsigned prefix = 0, above_count = 0;
            mass_t above_mass = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                if (threadIdx.x < 256) {
                    masses[threadIdx.x] = 0;
                    counts[threadIdx.x] = 0;
                }
                __syncthreads();
                each([&](int i, const Vec<F16> &v) {
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const unsigned key = key_of(v.x[e]);
                        if (v.x[e] == -INFINITY || !stays(key, i + e) || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
                        atomicAdd(&counts[(key >> shift) & 255], 1u);
                        if (by_mass) atomicAdd(&masses[(key >> shift) & 255], weigh(v.x[e]));
                    }
                });
                __syncthreads();
                if (threadIdx.x == 0) {
                    int last = -1, digit = 255;
                    for (; digit >= 0; digit--) {
                        if (counts[digit] == 0) continue;
                        last = digit;
                        if (enough(above_count + counts[digit], above_mass + masses[digit])) break;
                        above_count += counts[digit];
                        above_mass += masses[digit];
                    }
                    if (digit < 0) {  // all of them: end at the lowest
                        above_count -= counts[last];
                        above_mass -= masses[last];
                        digit = last;
                    }
                    sh.search_prefix = (prefix << 8) | (unsigned) digit;
                    sh.search_count = above_count;
                    sh.search_mass = above_mass;
                }
                __syncthreads();
                prefix = sh.search_prefix;
                above_count = sh.search_count;
                above_mass = sh.search_mass;
            }
            // how many of the tokens with this key stay, then the index of the last of them
            const unsigned equal = counts[prefix & 255];
            const mass_t one = by_mass ? masses[prefix & 255] / equal : 0;
            unsigned few = 1, most = equal;
            while (few < most) {
                const unsigned middle = (few + most) / 2;
                if (enough(above_count + middle, above_mass + middle * one)) most = middle;
                else few = middle + 1;
            }
            int mine = 0;
            each([&](int i, const Vec<F16> &v) {
#pragma unroll
                for (int e = 0; e < N; e++) mine += key_of(v.x[e]) == prefix && stays(prefix, i + e);
            });
            __syncthreads();
            mine = (int) wave_sum((mass_t) mine);
            if (lane == 0) sh.wave_mass[wave] = (mass_t) mine;
            if (threadIdx.x == 0) sh.last_key = prefix;
            __syncthreads();
            int before = 0;
            for (int w = 0; w < wave; w++) before += (int) sh.wave_mass[w];
            if (before < (int) most && (int) most <= before + mine) {  // in this wave's part
                for (int i0 = begin * N; i0 < end * N; i0 += 64) {
                    const int i = i0 + lane;
                    const bool hit = i < min(end * N, p.vocab) && key_of(load_one<F16>(row, i)) == prefix && stays(prefix, i);
                    const unsigned long long hits = __ballot(hit);
                    if (before + __popcll(hits) >= (int) most) {
                        if (hit && before + __popcll(hits & ((2ull << lane) - 1)) == (int) most) sh.last_index = i;
                        break;
                    }
                    before += __popcll(hits);
                }
            }
            __syncthreads();
        }
        last_key = sh.last_key;
        last_index = sh.last_index;
        __syncthreads();
    };
    if (k > 0 && k < p.vocab) tighten(false, [&](unsigned tokens, mass_t) { return tokens >= (unsigned) k; });
    auto weight_of = [&](float x, int i) -> mass_t {
        if (x == -INFINITY || !stays(key_of(x), i)) return 0;
        const double w = weigh.real(x);
        return w >= min_w || x == top ? Weigher::whole(w) : 0;
    };
    auto part_mass = [&](auto weight) {  // of this wave; all waves' in sh.wave_mass
        mass_t mass = 0;
        each([&](int i, const Vec<F16> &v) {
#pragma unroll
            for (int e = 0; e < N; e++) mass += weight(v.x[e], i + e);
        });
        mass = wave_sum(mass);
        __syncthreads();
        if (lane == 0) sh.wave_mass[wave] = mass;
        __syncthreads();
    };
    if (top_p < 1.0f) {
        part_mass([&](float x, int i) -> mass_t { return x == -INFINITY || !stays(key_of(x), i) ? 0 : weigh(x); });
        mass_t all = 0;
        for (int w = 0; w < NWAVES; w++) all += sh.wave_mass[w];
        const mass_t need = (mass_t) __builtin_ceil(fmax((double) top_p, 0.0) * (double) all);
        tighten(true, [&](unsigned, mass_t mass) { return mass >= need; });
    }

    // ---- the draw
    part_mass(weight_of);
    mass_t total = 0;
    for (int w = 0; w < NWAVES; w++) total += sh.wave_mass[w];
    const float u = p.uniform[r];
    const mass_t target = (mass_t) ((double) (u >= 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f) * (double) total);
    int chosen = 0;
    mass_t before = 0;
    while (chosen < NWAVES - 1 && before + sh.wave_mass[chosen] <= target) before += sh.wave_mass[chosen++];
    __syncthreads();
    // the part that holds the target, shared by all threads
    const int from = chosen * part * N, to = min(from + part * N, p.vocab), per = (to - from + THREADS - 1) / THREADS;
    const int mine = min(from + (int) threadIdx.x * per, to), mine_end = min(mine + per, to);
    mass_t mass = 0;
    for (int i = mine; i < mine_end; i++) mass += weight_of(load_one<F16>(row, i), i);
    const mass_t sums = wave_scan(mass, lane);
    if (lane == 63) sh.wave_mass[wave] = sums;
    __syncthreads();
    before += sums - mass;
    for (int w = 0; w < wave; w++) before += sh.wave_mass[w];
    if (!(before <= target && target < before + mass)) return;
    for (int i = mine; i < mine_end; i++) {
        const mass_t w = weight_of(load_one<F16>(row, i), i);
        before += w;
        if (before > target) {
            p.tokens[r] = i;
            if (p.probabilities) p.probabilities[r] = (float) ((double) w / (double) total);
            break;
        }
    }
}

}  // namespace

size_t sample_workspace(const SampleParams &) { return 0; }

int launch_sample(const SampleParams &given, void *, ihipStream_t *stream) {
    SampleParams p = given;
    int l = 0;
    while ((1 << l) < p.vocab) l++;
    p.bits = l < 11 ? 51 : 62 - l;
    const bool cached = (long long) p.vocab * (p.f16 ? 2 : 4) <= CACHE_BYTES;
    if (p.f16 && cached) hipLaunchKernelGGL((sample_kernel<true, true>), dim3((unsigned) p.rows), dim3(THREADS), 0, stream, p);
    else if (p.f16) hipLaunchKernelGGL((sample_kernel<true, false>), dim3((unsigned) p.rows), dim3(THREADS), 0, stream, p);
    else if (cached) hipLaunchKernelGGL((sample_kernel<false, true>), dim3((unsigned) p.rows), dim3(THREADS), 0, stream, p);
    else hipLaunchKernelGGL((sample_kernel<false, false>), dim3((unsigned) p.rows), dim3(THREADS), 0, stream, p);
    return (int) hipGetLastError();
}

}  // namespace kn
