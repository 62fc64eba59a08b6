// The draw of a token from a row of logits (knhip_sample).
//
// Weights are 64 bit fixed point, w = round(exp((x - max) / T) 2^S) with S chosen so that a whole row cannot overflow: sums
// of them are exact and the same in any order, so counting and adding may run in any order and with atomics. exp and its
// argument are f64: the nearest of 10^5 borders between tokens is then missed once in 10^10 rows or so.
// Thresholds are found on ordered keys: the bits of x as an unsigned number that grows with x.
#include <hip/hip_runtime.h>

#include "../serving_kernels.h"

namespace kn {

namespace {

constexpr int THREADS = 1024, NWAVES = THREADS / 64;

template <bool F16>
__device__ __forceinline__ float load_logit(const void *row, int i) {
    const float x = F16 ? (float) ((const _Float16 *) row)[i] : ((const float *) row)[i];
    return x != x ? -INFINITY : x + 0.0f;  // (-0 becomes +0, the two compare equal)
}

__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    return u ^ ((unsigned) ((int) u >> 31) | 0x80000000u);
}

struct Weigher {
    float top;
    double inv_t, one;
    // exp((x - top) / T) as a real number
    __device__ __forceinline__ double real(float x) const {
        if (x == top) return 1.0;
        if (top == INFINITY || x == -INFINITY) return 0.0;
        return exp(((double) x - (double) top) * inv_t);
    }
    __device__ __forceinline__ unsigned long long operator()(float x) const { return (unsigned long long) __builtin_rint(real(x) * one); }
};

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T *shared, F f) {
    for (int m = 32; m; m >>= 1) v = f(v, __shfl_xor(v, m));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
    for (int w = 1; w < NWAVES; w++) v = f(v, shared[w]);
    return v;
}

struct Threshold {
    unsigned key;              // keys above stay
    int ties;                  // and this many of the keys equal to it, the lowest indices first
};

// One workgroup per row.
template <bool F16>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleParams p, int bits) {
    __shared__ unsigned long long masses[256], wave_mass[NWAVES];
    __shared__ unsigned counts[256];
    __shared__ float tops[NWAVES];
    __shared__ int wave_ties[NWAVES], found;
    __shared__ unsigned long long above_mass_s;
    __shared__ unsigned prefix_s, above_count_s;
    const int r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const void *row = (const char *) p.logits + r * p.row_stride * (F16 ? 2 : 4);
    float top = -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += THREADS) top = fmaxf(top, load_logit<F16>(row, i));
    top = block_reduce(top, tops, [](float a, float b) { return fmaxf(a, b); });
    if (top == -INFINITY) {
        if (threadIdx.x == 0) {
            p.tokens[r] = -1;
            if (p.probabilities) p.probabilities[r] = 0.0f;
        }
        return;
    }
    const float t = p.temperature ? p.temperature[r] : 1.0f;
    const bool greedy = !(t > 0.0f);
    const Weigher weigh{top, greedy ? 0.0 : 1.0 / (double) t, (double) (1ull << bits)};
    const int k = p.top_k ? p.top_k[r] : 0;
    const float top_p = p.top_p ? p.top_p[r] : 1.0f, min_p = p.min_p ? p.min_p[r] : 0.0f;

    // keeps everything finite, or +inf
    Threshold keep{key_of(-INFINITY), 0};
    unsigned long long kept_mass = 0;
    // the key at which `enough(count, mass)`, called with what lies above and at a key, first holds
    auto search = [&](auto enough) {
        unsigned prefix = 0, above_count = 0;
        unsigned long long above_mass = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (threadIdx.x < 256) {
                masses[threadIdx.x] = 0;
                counts[threadIdx.x] = 0;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < p.vocab; i += THREADS) {
                const float x = load_logit<F16>(row, i);
                const unsigned key = key_of(x);
                if (x == -INFINITY || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
                atomicAdd(&counts[(key >> shift) & 255], 1u);
                atomicAdd(&masses[(key >> shift) & 255], weigh(x));
            }
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
                prefix_s = (prefix << 8) | (unsigned) digit;
                above_count_s = above_count;
                above_mass_s = above_mass;
            }
            __syncthreads();
            prefix = prefix_s;
            above_count = above_count_s;
            above_mass = above_mass_s;
        }
        __syncthreads();
        struct {
            unsigned key, above, equal;
            unsigned long long above_mass, each;
        } got{prefix, above_count, counts[prefix & 255], above_mass, 0};
        got.each = masses[prefix & 255] / got.equal;
        __syncthreads();
        return got;
    };
    if (!greedy) {
        if (k > 0 && k < p.vocab) {
            const auto got = search([&](unsigned count, unsigned long long) { return count >= (unsigned) k; });
            keep.key = got.key;
            keep.ties = (int) min(got.equal, (unsigned) k - got.above);
            kept_mass = got.above_mass + keep.ties * got.each;
        } else {
            unsigned long long mass = 0;
            for (int i = threadIdx.x; i < p.vocab; i += THREADS) mass += weigh(load_logit<F16>(row, i));
            kept_mass = block_reduce(mass, wave_mass, [](unsigned long long a, unsigned long long b) { return a + b; });
        }
        if (top_p < 1.0f) {
            const double want = fmax((double) top_p, 0.0) * (double) kept_mass;
            const unsigned long long need = (unsigned long long) __builtin_ceil(want);
            const auto got = search([&](unsigned, unsigned long long mass) { return mass >= need; });
            const unsigned long long rest = need > got.above_mass ? need - got.above_mass : 0;
            const unsigned long long ties = got.each ? (rest + got.each - 1) / got.each : got.equal;
            const int most = (int) max(1ull, min(ties, (unsigned long long) got.equal));
            if (got.key > keep.key || (got.key == keep.key && most < keep.ties)) keep = Threshold{got.key, most};
        }
    }
    // ---- the draw: a wave takes a contiguous part of the row
    const int part = (p.vocab + NWAVES * 64 - 1) / (NWAVES * 64) * 64, begin = min(wave * part, p.vocab), end = min(begin + part, p.vocab);
    auto weight_at = [&](int i, float x, int tie_rank) -> unsigned long long {
        const unsigned key = key_of(x);
        if (greedy) return x == top ? 1ull << bits : 0;
        if (x == -INFINITY || key < keep.key || (key == keep.key && tie_rank >= keep.ties)) return 0;
        if (x != top && weigh.real(x) < (double) min_p) return 0;
        return weigh(x);
    };
    int ties = 0;
    for (int i = begin + lane; i < end; i += 64) ties += key_of(load_logit<F16>(row, i)) == keep.key;
    for (int m = 32; m; m >>= 1) ties += __shfl_xor(ties, m);
    if (lane == 0) wave_ties[wave] = ties;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    int tie_base = 0;
    for (int w = 0; w < wave; w++) tie_base += wave_ties[w];
    auto tile = [&](int i0, int &rank_base) {
        const int i = i0 + lane;
        const float x = i < end ? load_logit<F16>(row, i) : -INFINITY;
        const unsigned long long equal = __ballot(i < end && key_of(x) == keep.key);
        const int rank = rank_base + __popcll(equal & ((1ull << lane) - 1));
        rank_base += __popcll(equal);
        return weight_at(i, x, rank);
    };
    unsigned long long mass = 0;
    for (int i0 = begin, base = tie_base; i0 < end; i0 += 64) mass += tile(i0, base);
    for (int m = 32; m; m >>= 1) mass += __shfl_xor(mass, m);
    if (lane == 0) wave_mass[wave] = mass;
    __syncthreads();
    unsigned long long total = 0, before = 0;
    for (int w = 0; w < NWAVES; w++) {
        if (w == wave) before = total;
        total += wave_mass[w];
    }
    const float u = greedy ? 0.0f : p.uniform[r];
    const unsigned long long target = (unsigned long long) ((double) (u >= 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f) * (double) total);
    if (!(before <= target && target < before + wave_mass[wave])) return;
    for (int i0 = begin, base = tie_base; i0 < end; i0 += 64) {
        const unsigned long long w = tile(i0, base);
        unsigned long long sums = w;
        for (int m = 1; m < 64; m <<= 1) {
            const unsigned long long other = __shfl_up(sums, m);
            if (lane >= m) sums += other;
        }
        const unsigned long long hit = __ballot(before + sums > target);
        if (hit) {
            if (lane == __ffsll((long long) hit) - 1) {
                p.tokens[r] = i0 + lane;
                if (p.probabilities) p.probabilities[r] = greedy ? 1.0f : (float) ((double) w / (double) total);
            }
            return;
        }
        before += __shfl(sums, 63);
    }
}

int bits_for(int vocab) {
    int l = 0;
    while ((1 << l) < vocab) l++;
    return 62 - l;
}

}  // namespace

size_t sample_workspace(const SampleParams &) { return 0; }

int launch_sample(const SampleParams &p, void *, ihipStream_t *stream) {
    if (p.f16) hipLaunchKernelGGL(sample_kernel<true>, dim3((unsigned) p.rows), dim3(THREADS), 0, stream, p, bits_for(p.vocab));
    else hipLaunchKernelGGL(sample_kernel<false>, dim3((unsigned) p.rows), dim3(THREADS), 0, stream, p, bits_for(p.vocab));
    return (int) hipGetLastError();
}

}  // namespace kn
