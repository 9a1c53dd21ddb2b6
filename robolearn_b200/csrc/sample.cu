// Drawing tokens: temperature, top-k, top-p and min-p from given uniforms.
//
// Order the row's tokens by logit, descending, equal logits by index. With
//   e_i = exp((l_i - max) / T),   w_i = round(2^30 e_i)   (an integer)
// the token is drawn among those that
//   K  are the first k of the order,
//   P  have less than p W_K of K's mass before them in the order (the first always),
//   M  have e_i >= min_p,
// as the first index whose cumulative w over the kept ones exceeds floor(u W).
//
// The weights are integers so that every sum is exact, whatever the order it is added in: the
// result does not depend on how the row is split over threads. 2^30 resolves e to 24 bits down
// to 2^-6 and gives weight 0 below 2^-31 of the best token's probability (such a token is never
// drawn); a row of 2^20 tokens sums to at most 2^50.
//
// One CTA per row. The two cuts are found as thresholds on an order-preserving integer key of the
// logit, by fixing its bits from the highest down.

#include "common.cuh"
#include "../../include/rl2.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>

namespace rl2 {
namespace sample {

constexpr int kMaxVocab = 1 << 20;
constexpr float kUnit = 1073741824.0f;  // 2^30

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// NaN counts as -inf (never drawn), +inf as the largest finite value, -0 as 0
__device__ __forceinline__ float clean(float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX) + 0.0f; }

__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }

typedef unsigned long long u64;

// What a row is drawn with.
struct Row {
    float inverse, top_p, min_p, uniform;
    int top_k;
    bool greedy, valid;
};

__device__ __forceinline__ Row row_of(const rl2_sample_args& a, long long row) {
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    Row r;
    r.greedy = t < FLT_MIN;  // 0, or so little that its reciprocal is not finite
    r.inverse = 1.0f / t;
    r.top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    r.top_p = a.top_ps ? a.top_ps[row] : a.top_p;
    r.min_p = a.min_ps ? a.min_ps[row] : a.min_p;
    r.uniform = a.uniforms[row];
    r.valid = t >= 0.0f && r.top_p == r.top_p && r.min_p <= 1.0f;
    return r;
}

__device__ __forceinline__ float exp_of(float v, float best, float inverse) { return expf((v - best) * inverse); }
__device__ __forceinline__ u64 weight_of(float e) { return __float2uint_rn(e * kUnit); }

// tokens of the last value that P keeps: those before which less than `limit` of mass stands
__device__ __forceinline__ u64 kept_of_last(u64 before, u64 w, double limit, u64 count) {
    if (w == 0) return count;
    u64 n = static_cast<u64>((limit - static_cast<double>(before)) / static_cast<double>(w));
    while (n > 0 && static_cast<double>(before + (n - 1) * w) >= limit) --n;
    while (n < count && static_cast<double>(before + n * w) < limit) ++n;
    return min(n, count);
}

__device__ __forceinline__ u64 target_of(float u, u64 total) {
    const double at = static_cast<double>(u > 0.0f ? u : 0.0f) * static_cast<double>(total);
    return at < static_cast<double>(total) ? min(static_cast<u64>(at), total - 1) : total - 1;
}

__device__ __forceinline__ float log_share(u64 w, u64 total) {
    const float share = static_cast<float>(w) / static_cast<float>(total);
    return share > 0.5f ? log1pf(-static_cast<float>(total - w) / static_cast<float>(total)) : logf(share);
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int THREADS>
__device__ __forceinline__ u64 block_sum64(u64 v, u64* red) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < THREADS / 32 ? red[threadIdx.x & 31] : 0;
    return warp_sum64(v);
}

template <typename L, int THREADS>
__global__ void __launch_bounds__(THREADS) row_kernel(const rl2_sample_args a) {
    constexpr int kWarps = THREADS / 32;
    __shared__ u64 red[32];
    __shared__ u64 seg_eq[kWarps], seg_mass[kWarps];
    __shared__ float redf[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int V = a.vocab;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits;
        const Row r = row_of(a, row);
        auto at = [&](int j) { return clean(to_float(s[j])); };
        float best = -INFINITY;
        for (int j = tid; j < V; j += THREADS) best = fmaxf(best, at(j));
        best = warp_max(best);
        __syncthreads();
        if (lane == 0) redf[warp] = best;
        __syncthreads();
        best = warp_max(lane < kWarps ? redf[lane] : -INFINITY);
        if (best == -INFINITY || !r.valid) {
            if (tid == 0) {
                a.tokens[row] = -1;
                if (a.log_probs) a.log_probs[row] = -INFINITY;
                if (!r.valid && a.health) atomicOr(a.health, kHealthIndex);
            }
            continue;
        }
        const uint32_t best_key = key_of(best);
        auto mass_above = [&](uint32_t key) {
            u64 m = 0;
            for (int j = tid; j < V; j += THREADS) {
                const float v = at(j);
                if (key_of(v) > key) m += weight_of(exp_of(v, best, r.inverse));
            }
            return block_sum64<THREADS>(m, red);
        };
        auto count_from = [&](uint32_t key) {
            u64 c = 0;
            for (int j = tid; j < V; j += THREADS) c += key_of(at(j)) >= key;
            return block_sum64<THREADS>(c, red);
        };
        // cut: tokens above `key` and the first `ties` tokens at it
        uint32_t key = 0;
        u64 ties = V;
        if (r.greedy || r.top_p <= 0.0f) {
            key = best_key;
            ties = 1;
        } else {
            if (r.top_k > 0 && r.top_k < V) {
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t trial = key | (1u << bit);
                    if (count_from(trial) >= static_cast<u64>(r.top_k)) key = trial;
                }
                ties = r.top_k - (key == 0xFFFFFFFFu ? 0 : count_from(key + 1));
            }
            if (r.top_p < 1.0f) {
                u64 total = mass_above(key);
                if (key) total += ties * weight_of(exp_of(value_of(key), best, r.inverse));
                const double limit = static_cast<double>(r.top_p) * static_cast<double>(total);
                // the lowest key above which less than `limit` of mass stands
                uint32_t low = key;
                if (static_cast<double>(mass_above(key)) >= limit) {
                    uint32_t under = 0;  // highest key above which there still is `limit`, bit by bit
                    for (int bit = 31; bit >= 0; --bit) {
                        const uint32_t trial = under | (1u << bit);
                        if (static_cast<double>(mass_above(trial)) >= limit) under = trial;
                    }
                    low = under + 1;
                    ties = V;
                }
                const u64 n = kept_of_last(mass_above(low), weight_of(exp_of(value_of(low), best, r.inverse)), limit, V);
                ties = min(ties, n);
                key = low;
            }
        }
        // segments of the row, one per warp: mass above the cut, tokens at it
        const int span = (V + kWarps - 1) / kWarps;
        const int from = min(V, warp * span), to = min(V, from + span);
        const bool greedy = r.greedy;
        auto weigh = [&](float v) {
            if (greedy) return static_cast<u64>(1);
            const float e = exp_of(v, best, r.inverse);
            return e >= r.min_p ? weight_of(e) : 0;
        };
        u64 mass = 0, eq = 0;
        for (int j = from + lane; j < to; j += 32) {
            const float v = at(j);
            const uint32_t k = key_of(v);
            if (k > key) mass += weigh(v);
            eq += k == key;
        }
        mass = warp_sum64(mass);
        eq = warp_sum64(eq);
        __syncthreads();
        if (lane == 0) {
            seg_eq[warp] = eq;
            seg_mass[warp] = mass;
        }
        __syncthreads();
        const u64 tie_weight = key ? weigh(value_of(key)) : 0;
        u64 total = 0, before_mass = 0, ties_left = 0, seen = 0;
        for (int w = 0; w < kWarps; ++w) {
            const u64 kept = seen < ties ? min(seg_eq[w], ties - seen) : 0;
            if (w == warp) {
                before_mass = total;
                ties_left = kept;
            }
            total += seg_mass[w] + kept * tie_weight;
            seen += seg_eq[w];
        }
        const u64 target = target_of(r.uniform, total);
        const u64 own = mass + ties_left * tie_weight;
        if (target >= before_mass && target < before_mass + own) {  // this warp's segment holds the token
            u64 cum = before_mass;
            for (int j0 = from; j0 < to; j0 += 32) {
                const int j = j0 + lane;
                const float v = j < to ? at(j) : -INFINITY;
                const uint32_t k = j < to ? key_of(v) : 0;
                const bool tie = j < to && k == key;
                const uint32_t tied = __ballot_sync(0xffffffffu, tie);
                const u64 rank = __popc(tied & ((1u << lane) - 1));
                u64 w = 0;
                if (k > key || (tie && rank < ties_left)) w = weigh(v);
                ties_left -= min(ties_left, static_cast<u64>(__popc(tied)));
                u64 sum = w;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += up;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, cum + sum > target);
                if (hit) {
                    if (lane == __ffs(hit) - 1) {
                        a.tokens[row] = j;
                        if (a.log_probs) a.log_probs[row] = log_share(w, total);
                    }
                    break;
                }
                cum += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        __syncthreads();
    }
}

template <typename L>
void launch(const rl2_sample_args& a, cudaStream_t stream) {
    if (a.vocab <= 4096)
        row_kernel<L, 128><<<std::min(a.rows, 148 * 16), 128, 0, stream>>>(a);
    else
        row_kernel<L, 1024><<<std::min(a.rows, 148 * 2), 1024, 0, stream>>>(a);
}

}  // namespace sample
}  // namespace rl2

extern "C" int rl2_sample_tokens(const rl2_sample_args* a, void* stream) {
    using namespace rl2;
    using namespace rl2::sample;
    clear_error();
    if (!a) {
        set_error("token sampling: null arguments");
        return -1;
    }
    if (a->rows < 0 || a->vocab < 1 || a->vocab > kMaxVocab) {
        set_error("token sampling: rows >= 0 and 1..%d tokens are needed", kMaxVocab);
        return -1;
    }
    if (a->logits_dtype < 0 || a->logits_dtype > 2) {
        set_error("token sampling: types are 0 (fp32), 1 (fp16) or 2 (bf16)");
        return -1;
    }
    if ((!a->temperatures && !(a->temperature >= 0.0f)) || (!a->top_ps && a->top_p != a->top_p) ||
        (!a->min_ps && !(a->min_p <= 1.0f))) {
        set_error("token sampling: temperature >= 0, a number for top_p and min_p <= 1 are needed");
        return -1;
    }
    if (a->rows == 0) return 0;
    if (!a->logits || !a->uniforms || !a->tokens) {
        set_error("token sampling: logits, uniforms and tokens must be non-null");
        return -1;
    }
    if (a->ld_logits < a->vocab || !aligned(a->logits, a->logits_dtype == 0 ? 4 : 2)) {
        set_error("token sampling: the row stride is shorter than a row, or the logits are not aligned to their element");
        return -1;
    }
    if (a->logits_dtype == 0)
        launch<float>(*a, as_stream(stream));
    else if (a->logits_dtype == 1)
        launch<__half>(*a, as_stream(stream));
    else
        launch<__nv_bfloat16>(*a, as_stream(stream));
    return launch_status("token sampling");
}
