// The draw of a token from a row of logits (knhip_sample).
//
// Weights are 64 bit fixed point, w = round(exp((x - max) / T) 2^bits), with `bits` chosen so that a whole row cannot overflow:
// sums of them are exact and the same in any order, so counting and adding may run in any order and with atomics. exp and its
// argument are f64: the nearest of 10^5 borders between tokens is then missed once in 10^10 rows or so.
//
// A row belongs to one workgroup of 16 waves, each of which owns a contiguous part of it. What bounds a row is the arithmetic
// per logit of one compute unit, and the fetch rate of one (60 GB/s where 64 of them read) for rows that do not fit LDS. So a row is read
// once where it fits (f16: 53000 logits), and the maxima of its groups of 8 logits are kept beside it, so that later passes
// touch only groups that can matter. The filters end in one threshold, the last token that stays in the order of falling
// logits (ties: rising index):
//   top_k   the group maxima go into a histogram over the distance to the largest. The bucket that holds the k-th largest of
//           them bounds the k-th largest logit from below: the logits of the groups that reach it, little more than k, are
//           listed, and the filters and the draw work on that list alone.
//   top_p   (and top_k beyond what the list holds) all logits go into the histogram, masses (counts) instead of ones; the
//           tokens of the bucket where the mass is reached, usually a few hundred, are sorted.
// The 2048 buckets span the distances at which w is not zero. (Buckets on the bits of x would put most of a row into two dozen
// of them: the atomics of a wave would queue. Over the distance a normal distribution fills hundreds.) A bucket with more
// than 2048 tokens (flat rows) is searched by the bits of x, 8 at a time. Without a list the token is found in two steps: the
// wave whose part holds the target, and the place inside that part.
// Measured: 8.4 us for one f16 row of 32000 (the best 40), of which reading is a third and the rest a chain of steps between
// barriers; 29 us for 64 f32 rows of 128001 (the best 1000), reading 8 us at 3.9 TB/s; 41 us for 256 f16 rows of 50001 by mass
// alone, half of it the f64 arithmetic of 50001 weights on one compute unit.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../serving_kernels.h"

namespace kn {

namespace {

constexpr int THREADS = 1024, NWAVES = THREADS / 64;
static_assert(NWAVES == 16, "a row of lanes adds up the waves");
constexpr int BUCKETS = 2 * THREADS, LISTED = 2 * THREADS;
constexpr int CACHE_BYTES = 104 * 1024, CACHED_MAXIMA_BYTES = CACHE_BYTES / 8, MAXIMA_BYTES = 112 * 1024;

typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long mass_t;

// NaN counts as -inf
__device__ __forceinline__ float plain(float x) { return fmaxf(x, -INFINITY); }

// the bits of x as an unsigned number that grows with x (-0 as +0, the two are equal)
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);
    return u ^ ((unsigned) ((int) u >> 31) | 0x80000000u);
}

constexpr int GROUP = 8;
template <bool F16>
struct Raw {  // a group as it lies in memory
    uint4 v[F16 ? 1 : 2];
};
struct Group {
    float x[GROUP];
};

template <bool F16>
__device__ __forceinline__ Group unpack(const Raw<F16> &raw) {
    Group g;
    if constexpr (F16) {
        const halfx8 h = __builtin_bit_cast(halfx8, raw.v[0]);
#pragma unroll
        for (int e = 0; e < 8; e++) g.x[e] = plain((float) h[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) g.x[e] = plain(__builtin_bit_cast(floatx4, raw.v[e / 4])[e % 4]);
    }
    return g;
}

template <bool F16>
__device__ __forceinline__ float load_one(const void *row, int i) {
    return plain(F16 ? (float) ((const _Float16 *) row)[i] : ((const float *) row)[i]);
}

// group n of a row of `vocab` logits; what lies behind its end reads as -inf
template <bool F16>
__device__ __forceinline__ Raw<F16> load_group(const void *row, int n, int vocab) {
    Raw<F16> raw;
    if (n * GROUP + GROUP <= vocab) {
        if constexpr (F16) {
            raw.v[0] = __builtin_bit_cast(uint4, *(const halfx8_any *) ((const _Float16 *) row + n * GROUP));
        } else {
            raw.v[0] = __builtin_bit_cast(uint4, *(const floatx4_any *) ((const float *) row + n * GROUP));
            raw.v[1] = __builtin_bit_cast(uint4, *(const floatx4_any *) ((const float *) row + n * GROUP + 4));
        }
        return raw;
    }
    if constexpr (F16) {
        halfx8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = n * GROUP + e < vocab ? ((const _Float16 *) row)[n * GROUP + e] : (_Float16) -INFINITY;
        raw.v[0] = __builtin_bit_cast(uint4, h);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            floatx4 f;
#pragma unroll
            for (int k = 0; k < 4; k++) f[k] = n * GROUP + e + k < vocab ? ((const float *) row)[n * GROUP + e + k] : -INFINITY;
            raw.v[e / 4] = __builtin_bit_cast(uint4, f);
        }
    }
    return raw;
}

// exp((x - top) / T) 2^bits for x <= top. 2^(n / 256 + y / 256) with |y| <= 1/2: a table of 256 roots of two, and the series of
// exp(y ln2 / 256) up to the 4th power, whose rest is below 4e-17.
constexpr int ROOTS = 256;
struct Weigher {
    float top;
    double per;  // 256 log2(e) / T
    int bits;
    const double *roots;
    // (exact at x = top: the argument is zero; far below, the result is 0 or a positive number below 1 / 4)
    __device__ __forceinline__ double core(double t) const {
        constexpr double L = 0.6931471805599453 / ROOTS, MAGIC = 0x1.8p52;
        // adding 1.5 2^52 rounds to a whole number and leaves it in the low bits
        const double m = t + MAGIC, y = t - (m - MAGIC);
        const int i = (int) __builtin_bit_cast(mass_t, m);
        const double s = __builtin_fma(y, __builtin_fma(y, __builtin_fma(y, __builtin_fma(y, L * L * L * L / 24, L * L * L / 6), L * L / 2), L), 1.0);
        const mass_t w = __builtin_bit_cast(mass_t, roots[i & (ROOTS - 1)] * s);
        return __builtin_bit_cast(double, w + ((mass_t) (unsigned) ((i >> 8) + bits) << 52));  // (times a power of two: normal numbers)
    }
    __device__ __forceinline__ double real(float x) const {
        if (top == INFINITY || x == -INFINITY) return x == top ? __builtin_ldexp(1.0, bits) : 0.0;
        return core(fmax(((double) x - (double) top) * per, -ROOTS * 200.0));
    }
    // (bits <= 51: adding 2^52 rounds to a whole number and leaves it in the low bits)
    static __device__ __forceinline__ mass_t whole(double w) { return __builtin_bit_cast(mass_t, w + 0x1p52) & ((1ull << 52) - 1); }
    __device__ __forceinline__ mass_t operator()(float x) const { return whole(real(x)); }
    // the same for finite logits within the distance of the histogram
    __device__ __forceinline__ double near_real(float x) const { return core(((double) x - (double) top) * per); }
    __device__ __forceinline__ mass_t near(float x) const { return whole(near_real(x)); }
};

__device__ __forceinline__ float logit_of(unsigned key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

struct Shared {
    mass_t hist[BUCKETS];
    mass_t list[LISTED];  // key and, below it, the complement of the index: falling order is the order of the filters
    double roots[ROOTS];
    mass_t wave_mass[NWAVES], part_mass[NWAVES];
    float wave_top[NWAVES];
    int list_count, bucket, place;
    unsigned short places[LISTED];
    mass_t above;
    unsigned last_key;  // the threshold: the last token that stays
    int last_index;
    mass_t search_mass;
    unsigned search_prefix, search_count;
};

// v of another lane by the pattern CTRL, 0 where it has none and in rows of 16 lanes outside the mask
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ mass_t from_lane(mass_t v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int) v, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int) (v >> 32), CTRL, ROWS, 0xf, false);
    return (mass_t) hi << 32 | lo;
}

__device__ __forceinline__ mass_t lane_of(mass_t v, int lane) {
    return (mass_t) (unsigned) __builtin_amdgcn_readlane((int) (v >> 32), lane) << 32 | (unsigned) __builtin_amdgcn_readlane((int) v, lane);
}

// sums over the lanes up to and with this one, in a row of 16 lanes and in the wave, without LDS
__device__ __forceinline__ mass_t row_scan(mass_t v) {
    v += from_lane<0x111>(v);  // one lane down
    v += from_lane<0x112>(v);
    v += from_lane<0x114>(v);
    return v + from_lane<0x118>(v);
}

__device__ __forceinline__ mass_t wave_scan(mass_t v) {
    v = row_scan(v);
    v += from_lane<0x142, 0xa>(v);         // the last lane of rows 0 and 2 to rows 1 and 3
    return v + from_lane<0x143, 0xc>(v);  // the last lane of row 1 to rows 2 and 3
}

__device__ __forceinline__ mass_t wave_sum(mass_t v) { return lane_of(wave_scan(v), 63); }

// sums over the first places, one per wave, of an array in LDS
__device__ __forceinline__ mass_t scan_of_waves(const mass_t *shared) {
    const int lane = threadIdx.x & 63;
    return row_scan(lane < NWAVES ? shared[lane] : 0);
}

// sums over the threads of the workgroup up to and with this one, and over all; `shared`: a place per wave
__device__ __forceinline__ mass_t block_scan(mass_t v, mass_t *shared, mass_t *all = nullptr) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) shared[wave] = v;
    __syncthreads();
    const mass_t waves = scan_of_waves(shared);
    if (all) *all = lane_of(waves, NWAVES - 1);
    return wave ? v + lane_of(waves, wave - 1) : v;
}

// places in a list for all that a lane asks for: one addition per wave
template <int N>
__device__ __forceinline__ void take_places(const bool (&live)[N], int (&place)[N], int *count) {
    const int lane = threadIdx.x & 63;
    int all = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
        const unsigned long long lanes = __ballot(live[e]);
        place[e] = all + __popcll(lanes & ((1ull << lane) - 1));
        all += __popcll(lanes);
    }
    if (all == 0) return;
    int base = 0;
    if (lane == 0) base = atomicAdd(count, all);
    base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
    for (int e = 0; e < N; e++) place[e] += base;
}

// The first `count` entries of the list into falling order: a bitonic network, a thread per pair. Steps of 64 and
// less stay inside the 128 entries of a wave and need no barrier.
__device__ __forceinline__ void sort_list(mass_t *list, int count) {
    int size = 2;
    while (size < count) size *= 2;
    __syncthreads();
    for (int i = count + (int) threadIdx.x; i < size; i += THREADS) list[i] = 0;
    __syncthreads();
    bool shared = false;  // whether other waves have written since the last barrier
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step > 0; step /= 2) {
            if (step > 64 || shared) __syncthreads();
            else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            shared = step > 64;
            if ((int) threadIdx.x < size / 2) {
                const int i = 2 * (int) threadIdx.x - ((int) threadIdx.x & (step - 1)), j = i + step;
                const mass_t a = list[i], b = list[j];
                const bool up = (i & run) != 0;
                if (up ? a > b : a < b) {
                    list[i] = b;
                    list[j] = a;
                }
            }
        }
    __syncthreads();
}

__device__ __forceinline__ mass_t target_of(float u, mass_t total) {
    return (mass_t) ((double) (u >= 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f) * (double) total);
}

template <bool F16, bool CACHED>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p) {
    __shared__ Shared sh;
    __shared__ Raw<F16> cache[CACHED ? CACHE_BYTES / sizeof(Raw<F16>) : 1];
    // the maxima of the groups; rows of more than that hold none
    using maximum_t = std::conditional_t<F16, _Float16, float>;
    constexpr int MAXIMA = (CACHED ? CACHED_MAXIMA_BYTES : MAXIMA_BYTES) / sizeof(maximum_t);
    __shared__ maximum_t maxima[MAXIMA];
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const void *row = (const char *) p.logits + r * p.row_stride * (F16 ? 2 : 4);
    const int groups = (p.vocab + GROUP - 1) / GROUP, part = (groups + NWAVES - 1) / NWAVES;
    const int begin = min(wave * part, groups), end = min(begin + part, groups);  // of this wave, in groups
    const bool has_maxima = CACHED || groups <= MAXIMA;
    auto logit_at = [&](int i) { return CACHED ? load_one<F16>(cache, i) : load_one<F16>(row, i); };
    auto group_at = [&](int n) { return CACHED ? cache[n] : load_group<F16>(row, n, p.vocab); };

    // f(first index, logits) for the groups of this wave
    auto each = [&](auto f) {
        int n = begin + lane;
        constexpr int AHEAD = 2;
        for (; n + 64 * (AHEAD - 1) < end; n += 64 * AHEAD) {
            Raw<F16> raw[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) raw[a] = group_at(n + 64 * a);
#pragma unroll
            for (int a = 0; a < AHEAD; a++) f((n + 64 * a) * GROUP, unpack<F16>(raw[a]));
        }
        for (; n < end; n += 64) f(n * GROUP, unpack<F16>(group_at(n)));
    };

    // ---- the maximum, of the row and of its groups (and the row into LDS)
    float top = -INFINITY;
    {
        int n = begin + lane;
        constexpr int AHEAD = F16 ? 8 : 4;
        auto take = [&](int at, const Raw<F16> &raw) {
            if (CACHED) cache[at] = raw;
            const Group g = unpack<F16>(raw);
            float m = g.x[0];
#pragma unroll
            for (int e = 1; e < GROUP; e++) m = fmaxf(m, g.x[e]);
            if (has_maxima) maxima[at] = (maximum_t) m;
            top = fmaxf(top, m);
        };
        for (; n + 64 * (AHEAD - 1) < end; n += 64 * AHEAD) {
            Raw<F16> raw[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) raw[a] = load_group<F16>(row, n + 64 * a, p.vocab);
#pragma unroll
            for (int a = 0; a < AHEAD; a++) take(n + 64 * a, raw[a]);
        }
        for (; n < end; n += 64) take(n, load_group<F16>(row, n, p.vocab));
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
        if (lane == 0) sh.wave_top[wave] = top;
        if (threadIdx.x < ROOTS) sh.roots[threadIdx.x] = exp2(threadIdx.x * (1.0 / ROOTS));
        for (int b = threadIdx.x; b < BUCKETS; b += THREADS) sh.hist[b] = 0;
        if (threadIdx.x == 0) {
            sh.list_count = 0;
            sh.bucket = BUCKETS;
            sh.last_index = p.vocab;
        }
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
    const float min_p = p.min_p ? p.min_p[r] : 0.0f;
    if (!(t > 0.0f) || min_p > 1.0f) {  // the first of the largest (no weight but the most probable token's stays above 1)
        int first = p.vocab;
        auto look = [&](int i, const Group &g) {
#pragma unroll
            for (int e = GROUP - 1; e >= 0; e--)
                if (g.x[e] == top) first = min(first, i + e);
        };
        if (has_maxima) {
            for (int n = threadIdx.x; n < groups; n += THREADS)
                if ((float) maxima[n] == top && n * GROUP < first) look(n * GROUP, unpack<F16>(group_at(n)));
        } else {
            each(look);
        }
        if (first < p.vocab) atomicMin(&sh.last_index, first);
        __syncthreads();
        if (threadIdx.x == 0) {
            p.tokens[r] = sh.last_index;
            if (p.probabilities) p.probabilities[r] = 1.0f;
        }
        return;
    }
    const Weigher weigh{top, 369.32993046757462751 / (double) t, p.bits, sh.roots};
    const int k = p.top_k ? p.top_k[r] : 0;
    const float top_p = p.top_p ? p.top_p[r] : 1.0f;
    const double min_w = min_p > 0.0f ? __builtin_ldexp((double) min_p, p.bits) : 0.0;  // (at most the weight of the maximum, which is exact)
    // distances at which w may be more than zero: exp(-range / T) 2^bits = 1 / 4
    const float range = t * (0.6931472f * (p.bits + 2)), per_bucket = BUCKETS / range;
    // (not for temperatures so low or high that f32 cannot hold buckets which end at the range, on which near() relies)
    const bool spread = range < 1e37f && per_bucket < 3e38f && top < INFINITY;
    auto bucket_of = [&](float x) { return (unsigned) ((top - x) * per_bucket); };  // (saturates: -inf falls behind the last)
    unsigned last_key = 0;  // what stays: larger keys, and this key up to last_index
    int last_index = p.vocab;
    bool restricted = false;
    auto stays = [&](unsigned key, int i) { return key > last_key || (key == last_key && i <= last_index); };
    const double mass_wanted = top_p < 1.0f ? fmax((double) top_p, 0.0) : 1.0;
    auto wanted_of = [&](mass_t all) { return max((mass_t) __builtin_ceil(mass_wanted * (double) all), 1ull); };  // (the most probable token stays)

    // ---- the bucket of the histogram where enough is reached
    auto clear_hist = [&] {
        __syncthreads();
        for (int b = threadIdx.x; b < BUCKETS; b += THREADS) sh.hist[b] = 0;
        if (threadIdx.x == 0) {
            sh.list_count = 0;
            sh.bucket = BUCKETS;
        }
        __syncthreads();
    };
    // sh.bucket, sh.above: the first bucket at whose end `need` is reached, and what lies before it; BUCKETS when it never is.
    // With `share`, `need` is mass_wanted of all. Returns `need`.
    auto find_bucket = [&](bool share, mass_t need) {
        __syncthreads();
        // a thread takes two neighbouring buckets
        const mass_t a = sh.hist[2 * threadIdx.x], both = a + sh.hist[2 * threadIdx.x + 1];
        mass_t all;
        const mass_t sums = block_scan(both, sh.wave_mass, &all), before = sums - both;
        if (share) {
            need = wanted_of(all);
        }
        if (before < need && need <= before + both) {
            const bool second = before + a < need;
            sh.bucket = 2 * threadIdx.x + second;
            sh.above = before + (second ? a : 0);
        }
        __syncthreads();
        return need;
    };
    auto append = [&](unsigned key, int i) {
        const int c = atomicAdd(&sh.list_count, 1);
        if (c < LISTED) sh.list[c] = (mass_t) key << 32 | ~(unsigned) i;
    };
    auto mass_of_entry = [&](mass_t entry) { return weigh(logit_of((unsigned) (entry >> 32))); };

    // the threshold by the bits of x, 8 from the top at a time: slow, for any row
    auto search = [&](bool by_mass, mass_t need) {
        mass_t *masses = sh.hist;
        unsigned *counts = (unsigned *) (sh.hist + 256);
        unsigned prefix = 0, above_count = 0;
        mass_t above_mass = 0;
        auto enough = [&](unsigned count, mass_t mass) { return (by_mass ? mass : (mass_t) count) >= need; };
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (threadIdx.x < 256) {
                masses[threadIdx.x] = 0;
                counts[threadIdx.x] = 0;
            }
            __syncthreads();
            each([&](int i, const Group &g) {
#pragma unroll
                for (int e = 0; e < GROUP; e++) {
                    const unsigned key = key_of(g.x[e]);
                    if (g.x[e] == -INFINITY || !stays(key, i + e) || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
                    atomicAdd(&counts[(key >> shift) & 255], 1u);
                    if (by_mass) atomicAdd(&masses[(key >> shift) & 255], weigh(g.x[e]));
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
        each([&](int i, const Group &g) {
#pragma unroll
            for (int e = 0; e < GROUP; e++) mine += key_of(g.x[e]) == prefix && stays(prefix, i + e);
        });
        __syncthreads();
        mine = (int) wave_sum((mass_t) mine);
        if (lane == 0) sh.wave_mass[wave] = (mass_t) mine;
        if (threadIdx.x == 0) sh.last_key = prefix;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < wave; w++) before += (int) sh.wave_mass[w];
        if (before < (int) most && (int) most <= before + mine) {  // in this wave's part
            for (int i0 = begin * GROUP; i0 < end * GROUP; i0 += 64) {
                const int i = i0 + lane;
                const bool hit = i < min(end * GROUP, p.vocab) && key_of(load_one<F16>(row, i)) == prefix && stays(prefix, i);
                const unsigned long long hits = __ballot(hit);
                if (before + __popcll(hits) >= (int) most) {
                    if (hit && before + __popcll(hits & ((2ull << lane) - 1)) == (int) most) sh.last_index = i;
                    break;
                }
                before += __popcll(hits);
            }
        }
        __syncthreads();
    };

    // ---- top_k from the group maxima: a list, in falling order for the filters, in the order of the indices for the draw
    const bool few = k > 0 && k < p.vocab && k <= LISTED / 2;
    if (few && spread && has_maxima) {
        constexpr int AHEAD = 4;  // reads before the first result is used
        for (int n0 = threadIdx.x; n0 < groups; n0 += AHEAD * THREADS) {
            unsigned b[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; e++) b[e] = n0 + THREADS * e < groups ? bucket_of((float) maxima[n0 + THREADS * e]) : BUCKETS;
#pragma unroll
            for (int e = 0; e < AHEAD; e++)
                if (b[e] < BUCKETS) atomicAdd((unsigned *) &sh.hist[b[e]], 1u);
        }
        find_bucket(false, (mass_t) k);
        // (fewer groups than k: the bucket behind the last, what lies there has no weight)
        const unsigned bucket = min(sh.bucket, BUCKETS - 1);
        // the groups that reach it, then, a thread per logit, their logits; places in the lists are taken by whole waves
        for (int n0 = 0; n0 < groups; n0 += AHEAD * THREADS) {
            bool live[AHEAD];
            int place[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; e++) {
                const int n = n0 + THREADS * e + (int) threadIdx.x;
                live[e] = n < groups && bucket_of((float) maxima[n]) <= bucket;
            }
            take_places(live, place, &sh.list_count);
#pragma unroll
            for (int e = 0; e < AHEAD; e++)
                if (live[e] && place[e] < LISTED) sh.places[place[e]] = (unsigned short) (n0 + THREADS * e + (int) threadIdx.x);
        }
        if (threadIdx.x == 0) sh.place = 0;
        __syncthreads();
        const int reaching = sh.list_count;
        if (reaching <= LISTED) {
            for (int n0 = 0; n0 < reaching * GROUP; n0 += AHEAD * THREADS) {
                bool live[AHEAD];
                int place[AHEAD], i[AHEAD];
                float x[AHEAD];
#pragma unroll
                for (int e = 0; e < AHEAD; e++) {
                    const int n = n0 + THREADS * e + (int) threadIdx.x;
                    i[e] = n < reaching * GROUP ? sh.places[n / GROUP] * GROUP + n % GROUP : p.vocab;
                }
#pragma unroll
                for (int e = 0; e < AHEAD; e++) x[e] = i[e] < p.vocab ? logit_at(i[e]) : -INFINITY;
#pragma unroll
                for (int e = 0; e < AHEAD; e++) live[e] = bucket_of(x[e]) <= bucket;
                take_places(live, place, &sh.place);
#pragma unroll
                for (int e = 0; e < AHEAD; e++)
                    if (live[e] && place[e] < LISTED) sh.list[place[e]] = (mass_t) key_of(x[e]) << 32 | ~(unsigned) i[e];
            }
        }
        __syncthreads();
        const int count = __builtin_amdgcn_readfirstlane(reaching <= LISTED ? sh.place : LISTED + 1);
        if (count <= 64) {
            // One wave does the rest, an entry per lane, without a barrier (12.6 -> 8.4 us for the best 40 of 32000 logits): all
            // entries are compared with all others, then put into the order of the logits and that of the indices.
            if (wave != 0) return;
            const mass_t entry = lane < count ? sh.list[lane] : 0;
            int rank = 0, place = 0;
            for (int o0 = 0; o0 < count; o0 += 8)  // (what lies behind the list comes last in both)
#pragma unroll
                for (int o = o0; o < o0 + 8; o++) {
                    const mass_t other = lane_of(entry, o);
                    rank += other > entry;
                    place += ~(unsigned) other < ~(unsigned) entry;
                }
            const bool listed = lane < count;
            auto sums_in_order = [&](mass_t v, int at) {  // lane n: the sum of the first n + 1 in an order
                sh.hist[lane] = 0;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                if (listed) sh.hist[at] = v;
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                return wave_scan(sh.hist[lane]);
            };
            const mass_t w = listed ? mass_of_entry(entry) : 0;
            const float x = logit_of((unsigned) (entry >> 32));
            bool kept = listed && rank < k;
            const mass_t sums = sums_in_order(kept ? w : 0, rank), wanted = wanted_of(lane_of(sums, 63));
            // (in the order of the logits: those before which less than `wanted` lies)
            const int stay = top_p < 1.0f ? 1 + (int) __popcll(__ballot(sums < wanted)) : 64;
            kept = kept && rank < stay && weigh.real(x) >= min_w;
            const mass_t parts = sums_in_order(kept ? w : 0, place), total = lane_of(parts, 63);
            const int chosen = (int) __popcll(__ballot(parts <= target_of(p.uniform[r], total)));
            if (listed && place == chosen) {
                p.tokens[r] = (int) ~(unsigned) entry;
                if (p.probabilities) p.probabilities[r] = (float) ((double) w / (double) total);
            }
            return;
        }
        if (count <= LISTED) {
            // A thread keeps two entries. Three times a histogram of what stays of the list finds the entry at which something is
            // reached: top_k tokens and top_p of the mass in the order of the logits, the target of the draw in the order of
            // the indices. The entries of the bucket where that is are compared with each other.
            mass_t entry[2], w[2], total = 0;
            bool kept[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int i = (int) threadIdx.x + THREADS * e;
                kept[e] = i < count;
                entry[e] = kept[e] ? sh.list[i] : 0;
                w[e] = kept[e] ? mass_of_entry(entry[e]) : 0;
            }
            int shift = 0;
            while ((p.vocab >> shift) >= BUCKETS) shift++;
#pragma unroll 1
            for (int what = 0; what < 3; what++) {
                if (what == 0 ? count <= k : what == 1 ? !(top_p < 1.0f) : false) continue;
                mass_t need = (mass_t) k;
                if (what == 2) {
                    mass_t mine = 0;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float x = logit_of((unsigned) (entry[e] >> 32));
                        kept[e] = kept[e] && weigh.real(x) >= min_w;
                        if (kept[e]) mine += w[e];
                    }
                    (void) block_scan(mine, sh.wave_mass, &total);
                    need = target_of(p.uniform[r], total) + 1;
                }
                clear_hist();
                unsigned b[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    b[e] = what == 2 ? ~(unsigned) entry[e] >> shift : min(bucket_of(logit_of((unsigned) (entry[e] >> 32))), BUCKETS - 1u);
                    if (kept[e]) atomicAdd(&sh.hist[b[e]], what == 0 ? 1ull : w[e]);
                }
                need = find_bucket(what == 1, need);
                const unsigned bucket = sh.bucket;
                const mass_t above = sh.above;
                // (the histogram has been read and the list is in registers: their rooms hold the bucket's entries and what they count)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (kept[e] && b[e] == bucket) {
                        const int c = atomicAdd(&sh.list_count, 1);
                        sh.list[c] = entry[e];
                        sh.hist[c] = what == 0 ? 1ull : w[e];
                    }
                __syncthreads();
                const int inside = sh.list_count;
                for (int c = threadIdx.x; c < inside; c += THREADS) {
                    const mass_t own = sh.list[c];
                    mass_t before = above;
#pragma unroll 4
                    for (int o = 0; o < inside; o++) {
                        const mass_t other = sh.list[o], counts = sh.hist[o];
                        if (what == 2 ? ~(unsigned) other < ~(unsigned) own : other > own) before += counts;
                    }
                    if (before < need && need <= before + sh.hist[c]) sh.place = c;
                }
                __syncthreads();
                const mass_t last = sh.list[sh.place];
                if (what == 2) {
                    if (threadIdx.x == 0) {
                        p.tokens[r] = (int) ~(unsigned) last;
                        if (p.probabilities) p.probabilities[r] = (float) ((double) mass_of_entry(last) / (double) total);
                    }
                    return;
                }
#pragma unroll
                for (int e = 0; e < 2; e++) kept[e] = kept[e] && entry[e] >= last;
            }
        }
    }

    // ---- otherwise: counts and then masses (one loop, so that each piece of code is there once), each a threshold
    if (threadIdx.x < NWAVES) sh.part_mass[threadIdx.x] = 0;
    bool masses_known = false;  // whether sh.part_mass holds the masses of the waves' parts
#pragma unroll 1
    for (int filter = 0; filter < 2; filter++) {
        const bool by_mass = filter == 1;
        if (by_mass ? !(top_p < 1.0f) : !(k > 0 && k < p.vocab)) continue;
        mass_t need = (mass_t) k;
        bool found = false;
        if (spread) {
            clear_hist();
            // (all weights first, then the atomics: branches in between would leave the reads of the table waiting one by one)
            each([&](int i, const Group &g) {
                unsigned b[GROUP];
#pragma unroll
                for (int e = 0; e < GROUP; e++) {
                    b[e] = bucket_of(g.x[e]);
                    if (restricted && !stays(key_of(g.x[e]), i + e)) b[e] = BUCKETS;
                }
                if (by_mass) {
#pragma unroll
                    for (int half = 0; half < GROUP; half += 4) {
                        mass_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = weigh.near(g.x[half + e]);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (b[half + e] < BUCKETS) atomicAdd(&sh.hist[b[half + e]], w[e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < GROUP; e++)
                        if (b[e] < BUCKETS) atomicAdd((unsigned *) &sh.hist[b[e]], 1u);
                }
            });
            need = find_bucket(by_mass, need);
            const unsigned bucket = sh.bucket;
            const mass_t above = sh.above;
            if (bucket == BUCKETS) continue;  // everything that weighs anything stays
            // The tokens of the bucket go into the list; with masses, the masses of what lies above it into the parts'. Where few
            // tokens lie so high, a wave would weigh 64 for the sake of some: they are queued until there are 64 of them, in
            // the room of the histogram, which has been read.
            mass_t mass = 0;
            int queued = 0;
            mass_t *queue = sh.hist + 128 * wave;
            auto kept = [&](float x) -> mass_t {
                const double w = weigh.near_real(x);
                return w >= min_w ? Weigher::whole(w) : 0;
            };
            auto settle = [&](mass_t item) {
                const float x = __builtin_bit_cast(float, (unsigned) (item >> 32));
                const int i = (int) (unsigned) item;
                const unsigned b = bucket_of(x);
                if (b > bucket || (restricted && !stays(key_of(x), i))) return;
                if (b < bucket) {
                    if (by_mass) mass += kept(x);
                } else {
                    append(key_of(x), i);
                }
            };
            // (one comparison per logit: buckets are a little wider here)
            const float lowest = top - ((float) bucket + 2.0f) / per_bucket;
            for (int n0 = begin; n0 < end; n0 += 64) {
                const int n = n0 + lane;
                const bool live = n < end && (!has_maxima || (float) maxima[n] >= lowest);
                if (!__any(live)) continue;
                Group g;
#pragma unroll
                for (int e = 0; e < GROUP; e++) g.x[e] = -INFINITY;
                if (live) g = unpack<F16>(group_at(n));
#pragma unroll
                for (int e = 0; e < GROUP; e++) {
                    const bool hit = live && g.x[e] >= lowest;
                    const unsigned long long hits = __ballot(hit);
                    if (hit) queue[queued + __popcll(hits & ((1ull << lane) - 1))] = (mass_t) __builtin_bit_cast(unsigned, g.x[e]) << 32 | (unsigned) (n * GROUP + e);
                    queued += __popcll(hits);
                    if (queued >= 64) {
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        settle(queue[lane]);
                        const mass_t rest = queue[64 + lane];
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        queue[lane] = rest;
                        queued -= 64;
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (lane < queued) settle(queue[lane]);
            if (by_mass) {
                mass = wave_sum(mass);
                if (lane == 0) atomicAdd(&sh.part_mass[wave], mass);
            }
            __syncthreads();
            const int count = sh.list_count;
            if (count <= LISTED) {
                found = true;
                sort_list(sh.list, count);
                mass_t entry[2], w[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = 2 * (int) threadIdx.x + e;
                    entry[e] = i < count ? sh.list[i] : 0;
                    w[e] = i >= count ? 0 : by_mass ? mass_of_entry(entry[e]) : 1;
                }
                // what of the bucket stays: the threshold is the last token before which less than `need` lies
                mass_t before = above + block_scan(w[0] + w[1], sh.wave_mass) - w[0] - w[1];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int i = (int) ~(unsigned) entry[e];
                    if (before < need && 2 * (int) threadIdx.x + e < count) {
                        if (by_mass) {
                            const mass_t own = kept(logit_of((unsigned) (entry[e] >> 32)));
                            if (own) atomicAdd(&sh.part_mass[i / (part * GROUP)], own);
                        }
                        if (need <= before + w[e]) {
                            sh.last_key = (unsigned) (entry[e] >> 32);
                            sh.last_index = i;
                        }
                    }
                    before += w[e];
                }
                masses_known = by_mass;
                __syncthreads();
            }
        } else if (by_mass) {
            mass_t mass = 0;
            each([&](int i, const Group &g) {
#pragma unroll
                for (int e = 0; e < GROUP; e++)
                    if (stays(key_of(g.x[e]), i + e)) mass += weigh(g.x[e]);
            });
            mass = wave_sum(mass);
            __syncthreads();
            if (lane == 0) sh.wave_mass[wave] = mass;
            __syncthreads();
            const mass_t all = lane_of(scan_of_waves(sh.wave_mass), NWAVES - 1);
            need = wanted_of(all);
        }
        if (!found) search(by_mass, need);
        last_key = sh.last_key;
        last_index = sh.last_index;
        restricted = true;
    }

    // ---- the draw: the wave whose part holds the target, then the place in that part
    auto weight_of = [&](float x, int i) -> mass_t {
        if (x == -INFINITY || !stays(key_of(x), i)) return 0;
        const double w = weigh.real(x);
        return w >= min_w ? Weigher::whole(w) : 0;
    };
    if (!masses_known) {
        mass_t mass = 0;
        each([&](int i, const Group &g) {
#pragma unroll
            for (int e = 0; e < GROUP; e++) mass += weight_of(g.x[e], i + e);
        });
        mass = wave_sum(mass);
        __syncthreads();
        if (lane == 0) sh.part_mass[wave] = mass;
    }
    __syncthreads();
    const mass_t parts = scan_of_waves(sh.part_mass), total = lane_of(parts, NWAVES - 1), target = target_of(p.uniform[r], total);
    const int chosen = min((int) __popcll(__ballot(lane < NWAVES && parts <= target)), NWAVES - 1);
    mass_t before = chosen ? lane_of(parts, chosen - 1) : 0;
    const int from = chosen * part * GROUP, to = min(from + part * GROUP, p.vocab), per = (to - from + THREADS - 1) / THREADS;
    const int mine = min(from + (int) threadIdx.x * per, to), mine_end = min(mine + per, to);
    mass_t mass = 0;
    for (int i = mine; i < mine_end; i++) mass += weight_of(load_one<F16>(row, i), i);
    before += block_scan(mass, sh.wave_mass) - mass;
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
