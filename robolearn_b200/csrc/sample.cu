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
// A cut of the order (the k-th token; the token at which p is reached) is the lowest value v such that
// the tokens above v count, or weigh, less than a limit. Up to 1024 tokens: one warp per row, the row
// in registers, v from a histogram. More tokens: a CTA, or with few rows a cluster of CTAs that each
// read a part of the row, on a short list of candidates.
//
// Measured, a call among others: 8.5 us at 4096 x 256 fp32, top-p (16.4 with the cuts by halving the interval of
// values, two warp reductions a step); 69 us at 256 x 131072 bf16, top-k 2000 (67 MB; 118 with the list's cuts by
// halving); 22.5 us at 1 x 128257 fp32, top-k 50 and top-p.

#include "common.cuh"
#include "../../include/rl2.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <type_traits>

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
    r.inverse = r.greedy ? 1.0f : 1.0f / t;
    r.top_k = a.top_ks ? a.top_ks[row] : a.top_k;
    r.top_p = a.top_ps ? a.top_ps[row] : a.top_p;
    r.min_p = a.min_ps ? a.min_ps[row] : a.min_p;
    r.uniform = a.uniforms[row];
    r.valid = t >= 0.0f && r.top_p == r.top_p && r.min_p <= 1.0f;
    return r;
}

__device__ __forceinline__ float exp_of(float v, float best, float inverse) { return expf((v - best) * inverse); }
__device__ __forceinline__ u64 weight_of(float e) { return __float2uint_rn(e * kUnit); }

// The share p of a weight as an integer: a sum is below the product exactly if it is below this.
__device__ __forceinline__ u64 share_of(float p, u64 total) {
    return static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(total)));
}

// tokens of the last value that P keeps: those before which less than `limit` of mass stands
__device__ __forceinline__ u64 kept_of_last(u64 before, u64 w, u64 limit, u64 count) {
    return w == 0 ? count : min((limit - before + w - 1) / w, count);
}

__device__ __forceinline__ u64 target_of(float u, u64 total) {
    const double at = static_cast<double>(u > 0.0f ? u : 0.0f) * static_cast<double>(total);
    return at < static_cast<double>(total) ? min(static_cast<u64>(at), total - 1) : total - 1;
}

__device__ __forceinline__ float log_share(u64 w, u64 total) {
    const float share = static_cast<float>(w) / static_cast<float>(total);
    return share > 0.5f ? log1pf(-static_cast<float>(total - w) / static_cast<float>(total)) : logf(share);
}

// The drawn token (weight w of `total` kept) and its log-probability: that of the draw, log(w / W), or the logits' own,
// (l - max) / T - log sum e, where w's rounding to 2^-30 would show (a token at 2^-24 of the best: 0.002; the sum holds
// the best token's 2^30 and is hardly touched). One thread.
__device__ __forceinline__ void write_token(const rl2_sample_args& a, long long row, const Row& r, float best, int token, u64 w, u64 total) {
    a.tokens[row] = token;
    if (!a.log_probs) return;
    if (!a.log_probs_of_logits) {
        a.log_probs[row] = log_share(w, total);
        return;
    }
    const long long at = row * a.ld_logits + token;
    const float v = clean(a.logits_dtype == 0   ? static_cast<const float*>(a.logits)[at]
                          : a.logits_dtype == 1 ? __half2float(static_cast<const __half*>(a.logits)[at])
                                                : __bfloat162float(static_cast<const __nv_bfloat16*>(a.logits)[at]));
    const u64 unit = 1ull << 30;
    a.log_probs[row] = r.greedy ? 0.0f : (v - best) * r.inverse - log1pf(static_cast<float>(total - unit) * (1.0f / kUnit));
}

// ---- sums over a group of threads ------------------------------------------------

struct Sum {
    uint32_t count;
    u64 mass;
};

// 26 + 24 bits: a warp's lanes hold at most 2^45 each (2^15 tokens), so neither half overflows
__device__ __forceinline__ u64 warp_sum64(u64 v) {
    const uint32_t lo = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v) & 0x3FFFFFFu);
    const uint32_t hi = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 26));
    return (static_cast<u64>(hi) << 26) + lo;
}

struct WarpGroup {
    __device__ __forceinline__ u64 mass(u64 m) { return warp_sum64(m); }
    __device__ __forceinline__ uint32_t count(uint32_t c) { return __reduce_add_sync(0xffffffffu, c); }
    __device__ __forceinline__ Sum sum(Sum s) { return Sum{__reduce_add_sync(0xffffffffu, s.count), warp_sum64(s.mass)}; }
    __device__ __forceinline__ uint32_t max_key(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
};

// Where a cut falls: tokens above `value` are kept, and so many of those at it; what is above it.
struct Cut {
    float value;
    Sum above;
};

// The cut among N tokens a thread (w = 0: no token) of a range of values, `above` it the tokens that
// are not among them. The limit is not reached by `above` alone, and is by all of them. MASS: the
// limit is on the weight above, else on the count.
template <bool MASS, int N, typename Group>
__device__ __forceinline__ Cut find_cut(Group& group, const float (&v)[N], const uint32_t (&w)[N], u64 limit, Sum above) {
    auto over = [&](float x) {
        Sum s{0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (v[i] > x) {
                s.count += w[i] != 0;
                s.mass += w[i];
            }
        s = group.sum(s);
        return Sum{s.count + above.count, s.mass + above.mass};
    };
    auto less = [&](Sum s) { return (MASS ? s.mass : static_cast<u64>(s.count)) < limit; };
    // highest and lowest token, as keys (the lowest through the complement)
    auto extremes = [&](float lo, float hi, float& least, float& most) {
        uint32_t up = 0, down = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (w[i] && v[i] > lo && v[i] <= hi) {
                up = max(up, key_of(v[i]));
                down = max(down, ~key_of(v[i]));
            }
        most = value_of(group.max_key(up));
        least = value_of(~group.max_key(down));
    };
    float lo, hi;
    extremes(-INFINITY, FLT_MAX, lo, hi);
    Sum at_lo = over(lo), at_hi = above;
    if (less(at_lo)) return Cut{lo, at_lo};
    // now the limit stands above lo and not above hi: halve; now and then move the ends onto tokens
    for (int step = 1;; ++step) {
        if (step % 8 == 0 || at_lo.count - at_hi.count == 1) {
            float least, most;
            extremes(lo, hi, least, most);
            if (least == most) return Cut{most, at_hi};
            hi = most;
        }
        const float mid = 0.5f * lo + 0.5f * hi;
        if (!(mid > lo && mid < hi)) return Cut{hi, at_hi};  // neighbouring floats: what is between is at hi
        const Sum s = over(mid);
        if (less(s)) {
            hi = mid;
            at_hi = s;
        } else {
            lo = mid;
            at_lo = s;
        }
    }
}

// What is kept of a row: tokens above `cut`, the first `ties` at it, with e >= min_p.
struct Kept {
    float cut;
    u64 ties;
};

// Both cuts of a row whose tokens (at least those that the cuts can reach) are N a thread. `given`: the
// limit of the second where the tokens are not all that weigh, else 0. CUT(by_mass, limit) finds a cut.
template <typename CUT>
__device__ __forceinline__ Kept both_cuts(const Row& r, int vocab, float best, Sum all, u64 given, CUT&& cut) {
    if (r.greedy || r.top_p <= 0.0f) return Kept{best, 1};
    Kept kept{-INFINITY, 0};
    Sum above = all;  // above -inf
    u64 total = all.mass;
    if (r.top_k > 0 && r.top_k < vocab && all.count > static_cast<uint32_t>(r.top_k)) {
        const Cut c = cut(std::false_type{}, static_cast<u64>(r.top_k));
        kept = Kept{c.value, static_cast<u64>(r.top_k) - c.above.count};
        above = c.above;
        total = above.mass + kept.ties * weight_of(exp_of(kept.cut, best, r.inverse));
    }
    if (r.top_p < 1.0f) {
        const u64 limit = given ? given : share_of(r.top_p, total);
        u64 most = kept.ties;
        if (above.mass >= limit) {
            const Cut c = cut(std::true_type{}, limit);
            kept.cut = c.value;
            above = c.above;
            most = ~0ull;
        }
        if (kept.cut != -INFINITY)
            kept.ties = kept_of_last(above.mass, weight_of(exp_of(kept.cut, best, r.inverse)), limit, most);
    }
    return kept;
}

// ---- up to 1024 tokens: a warp per row, N tokens a lane (token lane * N + i) -----------------
//
// A cut comes from a histogram of the row over 128 bins of (max - l) / T in shared memory (two words a bin: the
// count above the weights' low 11 bits, and the weights' high 20), then from counting among the tokens of its bin.

constexpr int kRowWarps = 4;
constexpr int kRowBins = 128;
constexpr float kReach = 21.6f;  // exp(-21.6) 2^30 rounds to 0: what is further from the best has no weight

struct RowShared {
    alignas(16) uint32_t low[kRowBins], high[kRowBins];
    float few_value[32];
    uint32_t few_w[32];
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {  // exclusive
    const int lane = threadIdx.x & 31;
    uint32_t in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += up;
    }
    return in - v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v) {  // exclusive
    const int lane = threadIdx.x & 31;
    u64 in = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += up;
    }
    return in - v;
}

template <typename L, int N>
__global__ void __launch_bounds__(32 * kRowWarps) warp_kernel(const rl2_sample_args a) {
    __shared__ RowShared all_shared[kRowWarps];
    RowShared& sh = all_shared[threadIdx.x >> 5];
    const int lane = threadIdx.x & 31;
    const int V = a.vocab;
    WarpGroup group;
    ptx::grid_release();
    ptx::grid_wait();
    for (long long row = static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5); row < a.rows;
         row += static_cast<long long>(gridDim.x) * kRowWarps) {
        const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits + lane * N;
        const int here = V - lane * N;  // tokens of this lane (more than N: N)
        float v[N];
        constexpr int kVec = N * sizeof(L) >= 16 ? 16 / sizeof(L) : 1;
        if (kVec > 1 && here >= N && (reinterpret_cast<uintptr_t>(s) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < N; i += kVec) {
                L x[kVec];
                *reinterpret_cast<uint4*>(x) = ptx::load_vector(s + i);
#pragma unroll
                for (int k = 0; k < kVec; ++k) v[i + k] = clean(to_float(x[k]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i < here ? clean(to_float(s[i])) : -INFINITY;
        }
        const Row r = row_of(a, row);
        float best = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) best = fmaxf(best, v[i]);
        best = warp_max(best);
        if (best == -INFINITY || !r.valid) {
            if (lane == 0) {
                a.tokens[row] = -1;
                if (a.log_probs) a.log_probs[row] = -INFINITY;
                if (!r.valid && a.health) atomicOr(a.health, kHealthIndex);
            }
            continue;
        }
        uint32_t w[N];
        Sum all{0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = weight_of(exp_of(v[i], best, r.inverse));
            all.count += w[i] != 0;
            all.mass += w[i];
        }
        all = group.sum(all);
        const float per_value = fminf(r.inverse * (kRowBins / kReach), FLT_MAX);
        auto bin_of = [&](float x) {
            const float at = (best - x) * per_value;
            return at < kRowBins - 1 ? static_cast<int>(at) : kRowBins - 1;
        };
        bool counted = false;
        auto cut_of = [&](auto by_mass, u64 limit) {
            constexpr bool kMass = decltype(by_mass)::value;
            static_assert(kRowBins == 128, "four bins a lane");
            if (!counted) {
                counted = true;
                __syncwarp();
                reinterpret_cast<uint4*>(sh.low)[lane] = make_uint4(0, 0, 0, 0);
                reinterpret_cast<uint4*>(sh.high)[lane] = make_uint4(0, 0, 0, 0);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (w[i]) {
                        const int bin = bin_of(v[i]);
                        // at most 1024 tokens of at most 2^30: the low words sum to less than 2^21, the high to 2^29
                        atomicAdd(&sh.low[bin], (1u << 21) | (w[i] & 0x7FFu));
                        atomicAdd(&sh.high[bin], w[i] >> 11);
                    }
                __syncwarp();
            }
            Sum mine[4], sum{0, 0};
            const uint4 lo = reinterpret_cast<const uint4*>(sh.low)[lane], hi = reinterpret_cast<const uint4*>(sh.high)[lane];
            auto bin_sum = [](uint32_t low, uint32_t high) { return Sum{low >> 21, (static_cast<u64>(high) << 11) + (low & 0x1FFFFFu)}; };
            mine[0] = bin_sum(lo.x, hi.x);
            mine[1] = bin_sum(lo.y, hi.y);
            mine[2] = bin_sum(lo.z, hi.z);
            mine[3] = bin_sum(lo.w, hi.w);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum.count += mine[e].count;
                sum.mass += mine[e].mass;
            }
            Sum at{kMass ? 0u : warp_scan(sum.count), warp_scan64(sum.mass)};  // a cut by weight needs no counts
            // the bin at which the limit is reached: in one lane
            int bin = -1;
            uint32_t inside = 0;
            Sum before{0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const Sum next{at.count + mine[e].count, at.mass + mine[e].mass};
                if ((kMass ? at.mass : at.count) < limit && (kMass ? next.mass : next.count) >= limit) {
                    bin = lane * 4 + e;
                    inside = mine[e].count;
                    before = at;
                }
                at = next;
            }
            const int from = __ffs(__ballot_sync(0xffffffffu, bin >= 0)) - 1;
            bin = __shfl_sync(0xffffffffu, bin, from);
            inside = __shfl_sync(0xffffffffu, inside, from);
            before.count = __shfl_sync(0xffffffffu, before.count, from);
            before.mass = __shfl_sync(0xffffffffu, before.mass, from);
            if (inside > 32) {
                uint32_t y[N];
#pragma unroll
                for (int i = 0; i < N; ++i) y[i] = bin_of(v[i]) == bin ? w[i] : 0u;
                return find_cut<kMass>(group, v, y, limit, before);
            }
            // what is above each of the bin's tokens; the cut is the lowest that has less than the limit there
            uint32_t own = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) own |= (w[i] && bin_of(v[i]) == bin ? 1u : 0u) << i;
            uint32_t to = warp_scan(__popc(own));
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (own >> i & 1u) {
                    sh.few_value[to] = v[i];
                    sh.few_w[to++] = w[i];
                }
            __syncwarp();
            const float x = lane < inside ? sh.few_value[lane] : INFINITY;
            Sum above = before;
            for (uint32_t k = 0; k < inside; ++k)
                if (sh.few_value[k] > x) {
                    above.count += 1;
                    above.mass += sh.few_w[k];
                }
            const bool less = lane < inside && (kMass ? above.mass : static_cast<u64>(above.count)) < limit;
            const uint32_t lowest = ~__reduce_max_sync(0xffffffffu, less ? ~key_of(x) : 0u);
            const int owner = __ffs(__ballot_sync(0xffffffffu, less && key_of(x) == lowest)) - 1;
            __syncwarp();
            return Cut{value_of(lowest), Sum{__shfl_sync(0xffffffffu, above.count, owner), __shfl_sync(0xffffffffu, above.mass, owner)}};
        };
        const Kept kept = both_cuts(r, V, best, all, 0, cut_of);
        // the first ties by index, then the kept weights in order
        uint32_t ties = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) ties += v[i] == kept.cut && w[i] != 0;
        uint32_t rank = kept.cut != -INFINITY ? warp_scan(ties) : 0u;
        u64 sum = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool tie = v[i] == kept.cut && w[i] != 0;
            const bool in = v[i] > kept.cut || (tie && rank < kept.ties);
            rank += tie;
            if (!in || (!r.greedy && r.min_p > 0.0f && exp_of(v[i], best, r.inverse) < r.min_p)) w[i] = 0;
            sum += w[i];
        }
        const u64 total = warp_sum64(sum);
        const u64 target = target_of(r.uniform, total);
        u64 cum = warp_scan64(sum);
        if (cum <= target && target < cum + sum) {
            int chosen = 0;
            uint32_t its = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (cum <= target && target < cum + w[i]) {
                    chosen = lane * N + i;
                    its = w[i];
                }
                cum += w[i];
            }
            write_token(a, row, r, best, chosen, its, total);
        }
    }
}

// ---- more tokens: a CTA, or a cluster of CTAs, per row ---------------------------------
//
// The row is read once. A thread keeps the maxima of small groups of its tokens (16-byte vectors, or
// several); the k-th largest of all maxima bounds the k-th token from below, so only the groups whose
// maximum reaches the bound are read again and give a list of a little more than k candidates, on which
// cuts and draw are made. The bound comes from a histogram of the maxima over 2048 bins of (max - l) / T,
// whose 21.6 cover every token that has a weight. min-p bounds the candidates in the same way.
// Without a bound (no top-k, or the list does not fit) the cuts come from a histogram of all tokens
// (count and weight a bin) and the list of those in the bin of the cut, and the draw from the kept
// weight of each stretch of 2^shift tokens.
// Histograms leave a bin of a few tokens, which one warp finishes without barriers.

constexpr int kT = 512;
constexpr int kWarps = kT / 32;
constexpr int kBins = 2048;
constexpr int kEach = kBins / kT;
constexpr int kPer = 8;          // list entries per thread
constexpr int kList = kT * kPer;
constexpr int kFewPer = 8;
constexpr int kFew = 32 * kFewPer;  // tokens that one warp takes
constexpr int kStretches = 1024;
constexpr int kMaxStretch = 2048;  // tokens: 2^20 of them in fewer than 1024 stretches

// A bin of a histogram (or a stretch): what is in it, what is before it, the whole.
struct Found {
    Sum here, before, whole;
    int bin, pad;
};

struct Shared {
    alignas(16) u64 mass[kBins];  // histogram / stretches
    alignas(16) uint32_t count[kBins];
    uint8_t maxima[64 * kT];      // L [slot][thread]
    float value[kList];
    int index[kList];
    union {
        struct {
            uint32_t slot_w[kMaxStretch];  // the drawn stretch: weight, tie
            uint8_t slot_tie[kMaxStretch];
        };
        struct {
            float few_value[kFew];
            int few_index[kFew];
            uint32_t few_w[kFew];
        };
    };
    uint32_t red_count[2][kWarps];
    u64 red_mass[2][kWarps];
    uint2 red_pair[2][kWarps];
    uint32_t scan_count[kWarps];
    u64 scan_mass[kWarps];
    Found found;
    Cut cut;
    int listed, groups, few, answer;
};

__device__ __forceinline__ uint32_t peer(const void* p, uint32_t rank) { return ptx::cluster_addr(p, rank); }
__device__ __forceinline__ uint32_t load32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ u64 load64(uint32_t at) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void store32(uint32_t at, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void add32(uint32_t at, uint32_t v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void add64(uint32_t at, u64 v) {
    asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

// A warp's lanes append `mine` entries each to a list: the place of this lane's first.
__device__ __forceinline__ int append(int* length, int mine) {
    const int lane = threadIdx.x & 31;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    int base = 0;
    if (lane == 31 && sum) base = atomicAdd(length, sum);
    return __shfl_sync(0xffffffffu, base, 31) + sum - mine;
}

// The threads of one CTA. At most 2^12 tokens of weight up to 2^30 a sum: the count shares a word with
// the weight's high bits. One barrier a reduction: the slots alternate, and a slot is written again only
// after the barrier of the reduction between, which every reader has reached.
struct Block {
    Shared* sh;
    int parity;
    __device__ __forceinline__ Sum sum(Sum s) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const uint32_t lo = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(s.mass) & 0x3FFFFFFu);
        uint32_t hi = __reduce_add_sync(0xffffffffu, (s.count << 18) | static_cast<uint32_t>(s.mass >> 26));
        if (lane == 0) sh->red_pair[parity][warp] = make_uint2(lo, hi);
        __syncthreads();
        const uint2 x = lane < kWarps ? sh->red_pair[parity][lane] : make_uint2(0, 0);
        parity ^= 1;
        // the warps' low parts have 31 bits: added as two halves
        const uint32_t l0 = __reduce_add_sync(0xffffffffu, x.x & 0xFFFFu), l1 = __reduce_add_sync(0xffffffffu, x.x >> 16);
        hi = __reduce_add_sync(0xffffffffu, x.y);
        return Sum{hi >> 18, (static_cast<u64>(hi & 0x3FFFFu) << 26) + (static_cast<u64>(l1) << 16) + l0};
    }
    __device__ __forceinline__ u64 mass(u64 m) { return sum(Sum{0, m}).mass; }
    __device__ __forceinline__ uint32_t count(uint32_t c) { return sum(Sum{c, 0}).count; }
    __device__ __forceinline__ uint32_t max_key(uint32_t k) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        k = __reduce_max_sync(0xffffffffu, k);
        if (lane == 0) sh->red_count[parity][warp] = k;
        __syncthreads();
        k = lane < kWarps ? sh->red_count[parity][lane] : 0u;
        parity ^= 1;
        return __reduce_max_sync(0xffffffffu, k);
    }
};

// The threads of a cluster's CTAs (of the CTA alone where it has one), any number of tokens.
struct Cluster {
    Shared* sh;
    uint32_t size, rank;
    int parity;

    __device__ __forceinline__ void sync() {
        if (size > 1)
            ptx::cluster_sync();
        else
            __syncthreads();
    }
    __device__ __forceinline__ Sum sum(Sum s) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        s.count = __reduce_add_sync(0xffffffffu, s.count);
        s.mass = warp_sum64(s.mass);
        if (lane == 0) {
            sh->red_count[parity][warp] = s.count;
            sh->red_mass[parity][warp] = s.mass;
        }
        sync();
        Sum t{0, 0};
        for (uint32_t i = lane; i < size * kWarps; i += 32) {
            t.count += load32(peer(&sh->red_count[parity][i % kWarps], i / kWarps));
            t.mass += load64(peer(&sh->red_mass[parity][i % kWarps], i / kWarps));
        }
        parity ^= 1;
        t.count = __reduce_add_sync(0xffffffffu, t.count);
        t.mass = warp_sum64(t.mass);
        return t;
    }
    __device__ __forceinline__ uint32_t max_key(uint32_t k) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        k = __reduce_max_sync(0xffffffffu, k);
        if (lane == 0) sh->red_count[parity][warp] = k;
        sync();
        uint32_t t = 0;
        for (uint32_t i = lane; i < size * kWarps; i += 32)
            t = max(t, load32(peer(&sh->red_count[parity][i % kWarps], i / kWarps)));
        parity ^= 1;
        return __reduce_max_sync(0xffffffffu, t);
    }
};

// Exclusive scan over the CTA's threads; `all` receives the total.
__device__ __forceinline__ Sum block_scan(Shared* sh, Sum s, Sum& all) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Sum in = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t c = __shfl_up_sync(0xffffffffu, in.count, o);
        const u64 m = __shfl_up_sync(0xffffffffu, in.mass, o);
        if (lane >= o) {
            in.count += c;
            in.mass += m;
        }
    }
    __syncthreads();
    if (lane == 31) {
        sh->scan_count[warp] = in.count;
        sh->scan_mass[warp] = in.mass;
    }
    __syncthreads();
    Sum before{in.count - s.count, in.mass - s.mass};
    all = Sum{0, 0};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) {
            before.count += sh->scan_count[w];
            before.mass += sh->scan_mass[w];
        }
        all.count += sh->scan_count[w];
        all.mass += sh->scan_mass[w];
    }
    return before;
}

__device__ __forceinline__ uint32_t block_scan(Shared* sh, uint32_t s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t in = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += up;
    }
    if (lane == 31) sh->scan_count[warp] = in;
    __syncthreads();
    return in - s + __reduce_add_sync(0xffffffffu, lane < warp ? sh->scan_count[lane] : 0u);
}

__device__ __forceinline__ void clear_histogram(Shared* sh) {
    for (int i = threadIdx.x; i < kBins / 2; i += kT) reinterpret_cast<uint4*>(sh->mass)[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < kBins / 4; i += kT) reinterpret_cast<uint4*>(sh->count)[i] = make_uint4(0, 0, 0, 0);
}

// Adds a weight to a bin: its low word, and the carry where there is one. (A 64-bit add in shared memory is a
// loop of compare and swap.)
__device__ __forceinline__ void add_mass(Shared* sh, int bin, uint32_t w) {
    uint32_t* word = reinterpret_cast<uint32_t*>(&sh->mass[bin]);
    const uint32_t old = atomicAdd(word, w);
    if (old + w < old) atomicAdd(word + 1, 1u);
}

// Of a complete histogram: into sh->found the first bin up to which (itself included) the count, or the
// weight, reaches the limit (kBins where none does). All threads; a barrier before it is read.
__device__ __forceinline__ void find_bin(Shared* sh, bool by_mass, u64 limit, const Sum (&mine)[kEach], Sum at) {
    auto value = [&](Sum x) { return by_mass ? x.mass : static_cast<u64>(x.count); };
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const Sum next{at.count + mine[e].count, at.mass + mine[e].mass};
        if (value(at) < limit && value(next) >= limit) {
            sh->found.bin = threadIdx.x * kEach + e;
            sh->found.here = mine[e];
            sh->found.before = at;
        }
        at = next;
    }
}

// This thread's bins and what is before them.
__device__ __forceinline__ Sum scan_histogram(Shared* sh, Sum (&mine)[kEach], Sum& whole) {
    Sum s{0, 0};
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        mine[e] = Sum{sh->count[threadIdx.x * kEach + e], sh->mass[threadIdx.x * kEach + e]};
        s.count += mine[e].count;
        s.mass += mine[e].mass;
    }
    return block_scan(sh, s, whole);
}

// ---- a row from its list ------------------------------------------------------------

// One warp on a few tokens of the list: value, weight and index of entry i * 32 + lane in each lane.
template <int N>
struct Few {
    float v[N];
    uint32_t w[N];
    int token[N];
    WarpGroup group;

    __device__ __forceinline__ Cut cut(bool by_mass, u64 limit, Sum before) {
        return by_mass ? find_cut<true>(group, v, w, limit, before) : find_cut<false>(group, v, w, limit, before);
    }
    // the last of the first `ties` indexes (in lo .. hi] among the tokens marked, which are more than that
    __device__ __forceinline__ int last_of(const bool (&marked)[N], u64 ties, int lo, int hi) {
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) c += marked[i] && token[i] <= mid;
            (group.count(c) > ties ? hi : lo) = mid;
        }
        return lo;
    }
    // the first index (in lo .. hi] through which the tokens' weight and what is before them exceeds the target
    __device__ __forceinline__ int first_over(u64 before, u64 target, int lo, int hi) {
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            u64 m = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) m += token[i] <= mid ? w[i] : 0u;
            (before + group.mass(m) > target ? hi : lo) = mid;
        }
        return hi;
    }
    __device__ __forceinline__ void write(const rl2_sample_args& a, long long row, const Row& r, float best, int chosen, u64 total) const {
        uint32_t its = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (token[i] == chosen) its = w[i];
        if (its) write_token(a, row, r, best, chosen, its, total);
    }
};

// A list of up to 32 N candidates: one warp, no barriers.
template <int N>
__device__ __noinline__ void draw_few(Shared* sh, int n, const Row r, int vocab, float best, u64 given, const rl2_sample_args& a,
                                      long long row) {
    const int lane = threadIdx.x & 31;
    Few<N> few;
    Sum all{0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = i * 32 + lane;
        few.v[i] = at < n ? sh->value[at] : -INFINITY;
        few.token[i] = at < n ? sh->index[at] : vocab;
        few.w[i] = at < n ? static_cast<uint32_t>(weight_of(exp_of(few.v[i], best, r.inverse))) : 0u;
        all.count += few.w[i] != 0;
        all.mass += few.w[i];
    }
    all = few.group.sum(all);
    const Kept kept = both_cuts(r, vocab, best, all, given,
                                [&](auto by_mass, u64 limit) { return few.cut(decltype(by_mass)::value, limit, Sum{0, 0}); });
    bool tie[N];
    uint32_t ties = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) ties += tie[i] = few.v[i] == kept.cut && few.w[i] != 0;
    const int last = few.group.count(ties) > kept.ties ? few.last_of(tie, kept.ties, -1, vocab - 1) : vocab;
    u64 total = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool in = few.v[i] > kept.cut || (tie[i] && few.token[i] <= last);
        if (!in || (!r.greedy && exp_of(few.v[i], best, r.inverse) < r.min_p)) few.w[i] = 0;
        total += few.w[i];
    }
    total = few.group.mass(total);
    few.write(a, row, r, best, few.first_over(0, target_of(r.uniform, total), -1, vocab - 1), total);
}

// A longer list: histograms of it (by value for the cuts, by index for the draw), one warp on the bin found.
// `fine` bins a unit of value below the best spread the list over all bins. A bin with more tokens than one
// warp takes is halved by the block.
__device__ __noinline__ void draw_many(Shared* sh, int n, const Row r, int vocab, float best, float fine, u64 given,
                                       const rl2_sample_args& a, long long row) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Block group{sh, 0};
    float v[kPer];
    uint32_t w[kPer];
    auto bin_of = [&](float x) {
        const float at = (best - x) * fine;
        return at < kBins - 1 ? static_cast<int>(at) : kBins - 1;
    };
    auto token_of = [&](int i) { return i * kT + tid < n ? sh->index[i * kT + tid] : vocab; };
    clear_histogram(sh);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        v[i] = -INFINITY;
        w[i] = 0;
        if (i * kT + tid < n) {
            v[i] = sh->value[i * kT + tid];
            w[i] = static_cast<uint32_t>(weight_of(exp_of(v[i], best, r.inverse)));
            if (w[i]) {
                atomicAdd(&sh->count[bin_of(v[i])], 1u);
                add_mass(sh, bin_of(v[i]), w[i]);
            }
        }
    }
    __syncthreads();
    Sum mine[kEach], whole;
    const Sum at = scan_histogram(sh, mine, whole);
    // the cut whose limit the histogram reaches
    auto cut_of = [&](auto by_mass, u64 limit) {
        constexpr bool kMass = decltype(by_mass)::value;
        if (tid == 0) sh->few = 0;
        find_bin(sh, kMass, limit, mine, at);
        __syncthreads();
        const int bin = sh->found.bin;
        const Sum before = sh->found.before;
        if (sh->found.here.count <= 32) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (w[i] && bin_of(v[i]) == bin) {
                    const int to = atomicAdd(&sh->few, 1);
                    sh->few_value[to] = v[i];
                    sh->few_w[to] = w[i];
                }
            __syncthreads();
            if (warp == 0) {
                // what is above each of the few; the cut is the lowest that has less than the limit there
                const int few = sh->few;
                const float x = lane < few ? sh->few_value[lane] : INFINITY;
                Sum above = before;
                for (int k = 0; k < few; ++k)
                    if (sh->few_value[k] > x) {
                        above.count += 1;
                        above.mass += sh->few_w[k];
                    }
                const bool less = lane < few && (kMass ? above.mass : static_cast<u64>(above.count)) < limit;
                const uint32_t lowest = ~__reduce_max_sync(0xffffffffu, less ? ~key_of(x) : 0u);
                if (less && key_of(x) == lowest) sh->cut = Cut{x, above};  // equal values write the same
            }
            __syncthreads();
            const Cut c = sh->cut;
            __syncthreads();
            return c;
        }
        uint32_t y[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) y[i] = bin_of(v[i]) == bin ? w[i] : 0u;
        return find_cut<kMass>(group, v, y, limit, before);
    };
    const Kept kept = both_cuts(r, vocab, best, whole, given, cut_of);
    // ---- what is kept, by index ----
    uint32_t ties = 0;
    __syncthreads();  // sh->few and the histogram are read
    if (tid == 0) sh->few = 0;
    clear_histogram(sh);
    auto tie = [&](int i) { return v[i] == kept.cut && w[i] != 0; };
#pragma unroll
    for (int i = 0; i < kPer; ++i) ties += tie(i);
    ties = group.count(ties);
    int last = vocab;
    if (ties > kept.ties) {
        if (ties <= 32) {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (tie(i)) sh->few_index[atomicAdd(&sh->few, 1)] = token_of(i);
            __syncthreads();
            if (warp == 0) {
                // rank among the few by index; the one of rank ties - 1 is the last kept
                const int mine_index = lane < sh->few ? sh->few_index[lane] : vocab;
                int rank = 0;
                for (int k = 0; k < sh->few; ++k) rank += sh->few_index[k] < mine_index;
                if (lane < sh->few && rank + 1 == static_cast<int>(kept.ties)) sh->answer = mine_index;
            }
            __syncthreads();
            last = sh->answer;
        } else {
            int lo = -1, hi = vocab - 1;  // more than kept.ties through hi, not through lo
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                uint32_t c = 0;
#pragma unroll
                for (int i = 0; i < kPer; ++i) c += tie(i) && token_of(i) <= mid;
                (group.count(c) > kept.ties ? hi : lo) = mid;
            }
            last = lo;
        }
    }
    int shift = 0;
    while ((vocab - 1) >> shift >= kBins) ++shift;
    __syncthreads();  // the histogram is clear, sh->answer and sh->few are read
    if (tid == 0) sh->few = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (!w[i]) continue;
        const int token = token_of(i);
        const bool in = v[i] > kept.cut || (v[i] == kept.cut && token <= last);
        if (!in || (!r.greedy && r.min_p > 0.0f && exp_of(v[i], best, r.inverse) < r.min_p)) {
            w[i] = 0;
        } else {
            atomicAdd(&sh->count[token >> shift], 1u);
            add_mass(sh, token >> shift, w[i]);
        }
    }
    __syncthreads();
    Sum kept_all;
    const Sum kept_at = scan_histogram(sh, mine, kept_all);
    const u64 target = target_of(r.uniform, kept_all.mass);
    find_bin(sh, true, target + 1, mine, kept_at);
    __syncthreads();
    const int bin = sh->found.bin;
    const u64 before = sh->found.before.mass;
    const int lo = (bin << shift) - 1, hi = min(vocab, (bin + 1) << shift) - 1;
    if (sh->found.here.count <= 32) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (w[i] && token_of(i) >> shift == bin) {
                const int to = atomicAdd(&sh->few, 1);
                sh->few_index[to] = token_of(i);
                sh->few_w[to] = w[i];
            }
        __syncthreads();
        const int few = sh->few;
        if (warp != 0 || lane >= few) return;
        const int mine_index = sh->few_index[lane];
        u64 cum = before;
        for (int k = 0; k < few; ++k)
            if (sh->few_index[k] < mine_index) cum += sh->few_w[k];
        if (cum <= target && target < cum + sh->few_w[lane]) write_token(a, row, r, best, mine_index, sh->few_w[lane], kept_all.mass);
        return;
    }
    int from = lo, to = hi;
    while (to - from > 1) {
        const int mid = (from + to) >> 1;
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int token = token_of(i);
            m += token > lo && token <= mid ? w[i] : 0u;
        }
        (before + group.mass(m) > target ? to : from) = mid;
    }
    uint32_t its = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (token_of(i) == to) its = w[i];
    if (its) write_token(a, row, r, best, to, its, kept_all.mass);
}

// ---- reading a row ------------------------------------------------------------------

template <typename L>
struct Reader {
    static constexpr int kN = 16 / sizeof(L);
    const L* s;      // the row
    int vocab, mis;  // elements between the 16-byte boundary at or before the row and the row
    int vectors;

    __device__ __forceinline__ Reader(const L* row, int v) : s(row), vocab(v) {
        mis = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(L));
        vectors = (mis + vocab + kN - 1) / kN;
    }
    // token of the first element of vector b; whether the vector lies in the row, and the 32 from b on
    __device__ __forceinline__ int first(int b) const { return b * kN - mis; }
    __device__ __forceinline__ bool whole(int j) const { return j >= 0 && j + kN <= vocab; }
    __device__ __forceinline__ bool inside(int b) const { return b * kN >= mis && (b + 32) * kN - mis <= vocab; }
    __device__ __forceinline__ uint4 raw(int b) const { return ptx::load_vector(s + first(b)); }
    __device__ __forceinline__ float at(int j) const { return clean(to_float(s[j])); }
    // elements outside the row are -inf
    __device__ __forceinline__ void load(int b, float (&v)[kN]) const {
        const int j = first(b);
        if (whole(j)) {
            const uint4 x = raw(b);
            L y[kN];
            *reinterpret_cast<uint4*>(y) = x;
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = clean(to_float(y[e]));
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = j + e >= 0 && j + e < vocab ? at(j + e) : -INFINITY;
        }
    }
};

// Maximum of a 16-byte vector's elements, NaN left out (not cleaned otherwise).
template <typename L>
__device__ __forceinline__ L most(uint4 x);
template <>
__device__ __forceinline__ float most<float>(uint4 x) {
    return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)), fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
}
template <>
__device__ __forceinline__ __half most<__half>(uint4 x) {
    const __half2* h = reinterpret_cast<const __half2*>(&x);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return __hmax(__low2half(m), __high2half(m));
}
template <>
__device__ __forceinline__ __nv_bfloat16 most<__nv_bfloat16>(uint4 x) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return __hmax(__low2bfloat16(m), __high2bfloat16(m));
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ __half larger(__half a, __half b) { return __hmax(a, b); }
__device__ __forceinline__ __nv_bfloat16 larger(__nv_bfloat16 a, __nv_bfloat16 b) { return __hmax(a, b); }

// One row as a CTA of its cluster sees it: stretches [from, to) are this CTA's, a warp each in turn.
template <typename L>
struct Work {
    static constexpr int kN = Reader<L>::kN;
    static constexpr int kSlots = 64 / sizeof(L);  // group maxima per thread: 64 bytes of them
    Shared* sh;
    Cluster group;
    Reader<L> in;
    Row r;
    int shift, log_per;    // log2 of the tokens of a stretch, and of a lane's vectors in it
    int from, to;
    int steps, slot_steps; // vectors of this lane; of one of its groups
    float best, per_value; // bins a unit of value below the best
    bool cut_k, first_only;

    __device__ __forceinline__ int vectors_of(int warp) const { return max(0, (to - from - warp + kWarps - 1) / kWarps) << log_per; }
    __device__ __forceinline__ int vector_of(int warp, int lane, int step) const {
        return (((from + warp + kWarps * (step >> log_per)) << log_per) + (step & ((1 << log_per) - 1))) * 32 + lane;
    }
    // bin 0 holds the best token; -inf and what has no weight: the last
    __device__ __forceinline__ int bin_of(float v) const {
        const float at = (best - v) * per_value;
        return at < kBins - 1 ? static_cast<int>(at) : kBins - 1;
    }
    // f(step, token of the first element, elements) for every vector of this lane, whole warps in step;
    // elements outside the row are -inf
    template <typename F>
    __device__ __forceinline__ void every_vector(F&& f) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        constexpr int kAhead = 4;  // loads in flight
        int i = 0;
        for (; i + kAhead <= steps; i += kAhead) {
            if (in.inside(vector_of(warp, 0, i)) && in.inside(vector_of(warp, 0, i + kAhead - 1))) {
                uint4 raw[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) raw[k] = in.raw(vector_of(warp, lane, i + k));
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    L y[kN];
                    *reinterpret_cast<uint4*>(y) = raw[k];
                    float x[kN];
#pragma unroll
                    for (int e = 0; e < kN; ++e) x[e] = clean(to_float(y[e]));
                    f(i + k, in.first(vector_of(warp, lane, i + k)), x);
                }
            } else {
                for (int k = 0; k < kAhead; ++k) {
                    float x[kN];
                    in.load(vector_of(warp, lane, i + k), x);
                    f(i + k, in.first(vector_of(warp, lane, i + k)), x);
                }
            }
        }
        for (; i < steps; ++i) {
            float x[kN];
            in.load(vector_of(warp, lane, i), x);
            f(i, in.first(vector_of(warp, lane, i)), x);
        }
    }
    template <typename F>
    __device__ __forceinline__ void every(F&& f) const {
        every_vector([&](int, int, const float(&x)[kN]) {
#pragma unroll
            for (int e = 0; e < kN; ++e) f(x[e]);
        });
    }
    // hands the first CTA's sh->found to the others; a barrier
    __device__ __forceinline__ void share_found() {
        __syncthreads();
        if (group.size > 1) {
            constexpr int kWords = sizeof(Found) / 4;
            if (group.rank == 0)
                for (int i = threadIdx.x; i < kWords * static_cast<int>(group.size - 1); i += kT) {
                    const uint32_t* word = reinterpret_cast<const uint32_t*>(&sh->found) + i % kWords;
                    store32(peer(word, 1 + i / kWords), *word);
                }
            group.sync();
        }
    }
    // adds the cluster's histograms on its first CTA: bins [0, n); a barrier
    __device__ __forceinline__ void merge(int n) {
        group.sync();
        if (group.size > 1) {
            if (group.rank != 0)
                for (int i = threadIdx.x; i < n; i += kT) {
                    if (const uint32_t c = sh->count[i]) add32(peer(&sh->count[i], 0), c);
                    if (const u64 m = sh->mass[i]) add64(peer(&sh->mass[i], 0), m);
                }
            group.sync();
        }
    }
    // the counts alone
    __device__ __forceinline__ void merge_counts() {
        group.sync();
        if (group.size > 1) {
            if (group.rank != 0)
                for (int i = threadIdx.x; i < kBins; i += kT)
                    if (const uint32_t c = sh->count[i]) add32(peer(&sh->count[i], 0), c);
            group.sync();
        }
    }
    // The bin of the merged histogram at which the limit is reached; on every CTA.
    __device__ __forceinline__ Found search(bool by_mass, u64 limit) {
        if (group.rank == 0) {
            Sum mine[kEach], whole;
            const Sum at = scan_histogram(sh, mine, whole);
            if (threadIdx.x == 0) {
                sh->found.bin = kBins;
                sh->found.whole = whole;
            }
            __syncthreads();
            find_bin(sh, by_mass, limit, mine, at);
        }
        share_found();
        const Found f = sh->found;
        group.sync();  // read by all before it is written again
        return f;
    }
};

// Group maxima and the row's maximum: the one pass over the row.
template <typename L>
__device__ __forceinline__ float read_row(const Work<L>& work) {
    constexpr int kN = Work<L>::kN, kSlots = Work<L>::kSlots;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    L* maxima = reinterpret_cast<L*>(work.sh->maxima);
    const Reader<L>& in = work.in;
    const L none = L(-INFINITY);
    L m = none, all = none;
    int slot = 0, left = work.slot_steps;
    auto put = [&](L x) {
        m = larger(m, x);
        if (--left == 0) {
            all = larger(all, m);
            maxima[slot++ * kT + tid] = m;
            m = none;
            left = work.slot_steps;
        }
    };
    auto edge = [&](int i) {  // a vector that may lie across an end of the row
        const int j = in.first(work.vector_of(warp, lane, i));
        L x = none;
        for (int e = max(0, -j); e < kN && j + e < in.vocab; ++e) x = larger(x, in.s[j + e]);
        return x;
    };
    constexpr int kAhead = 8;  // loads in flight
    int i = 0;
    for (; i + kAhead <= work.steps; i += kAhead) {
        if (in.inside(work.vector_of(warp, 0, i)) && in.inside(work.vector_of(warp, 0, i + kAhead - 1))) {
            uint4 x[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) x[k] = in.raw(work.vector_of(warp, lane, i + k));
#pragma unroll
            for (int k = 0; k < kAhead; ++k) put(most<L>(x[k]));
        } else {
            for (int k = 0; k < kAhead; ++k) put(edge(i + k));
        }
    }
    for (; i < work.steps; ++i) put(in.inside(work.vector_of(warp, 0, i)) ? most<L>(in.raw(work.vector_of(warp, lane, i))) : edge(i));
    all = larger(all, m);
    for (; slot < kSlots; ++slot) {
        maxima[slot * kT + tid] = m;
        m = none;
    }
    return clean(to_float(all));
}

// The list of the tokens in bins [0, bound], on the cluster's first CTA: whether it fits.
template <typename L>
__device__ __forceinline__ bool build_list(Work<L>& work, int bound) {
    constexpr int kN = Work<L>::kN, kSlots = Work<L>::kSlots;
    const int tid = threadIdx.x;
    Shared* sh = work.sh;
    const Reader<L>& in = work.in;
    const L* maxima = reinterpret_cast<const L*>(sh->maxima);
    uint16_t* groups = reinterpret_cast<uint16_t*>(sh->mass);
    const float best = work.best, per_value = work.per_value, limit = static_cast<float>(bound + 1);
    // bin_of(v) <= bound, without cleaning: NaN fails, +inf passes
    auto passes = [&](float v) { return (best - v) * per_value < limit; };
    if (tid == 0) sh->listed = sh->groups = 0;
    __syncthreads();
    // groups with a candidate, then their tokens, both appended a warp at a time
    uint32_t passed = 0;
#pragma unroll
    for (int slot = 0; slot < kSlots; ++slot) passed |= (passes(to_float(maxima[slot * kT + tid])) ? 1u : 0u) << slot;
    int at = append(&sh->groups, __popc(passed));
    for (; passed; passed &= passed - 1, ++at)
        if (at < kList) groups[at] = static_cast<uint16_t>((__ffs(passed) - 1) * kT + tid);
    __syncthreads();
    if (sh->groups <= kList) {  // each group has a token
        const int n = sh->groups * work.slot_steps;  // vectors to read again
        constexpr int kAhead = 4;
        for (int i0 = 0; i0 < n; i0 += kAhead * kT) {
            uint4 x[kAhead];
            int first[kAhead];  // token of the vector's first element
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int i = i0 + k * kT + tid;
                first[k] = in.vocab;
                if (i < n) {
                    const int g = work.slot_steps == 1 ? groups[i] : groups[i / work.slot_steps];
                    const int step = (g / kT) * work.slot_steps + (work.slot_steps == 1 ? 0 : i % work.slot_steps);
                    const int its_warp = (g & (kT - 1)) >> 5;
                    if (step < work.vectors_of(its_warp)) {
                        const int b = work.vector_of(its_warp, g & 31, step);
                        first[k] = in.first(b);
                        if (in.whole(first[k])) x[k] = in.raw(b);
                    }
                }
            }
            uint32_t has = 0;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (in.whole(first[k])) {
                    L y[kN];
                    *reinterpret_cast<uint4*>(y) = x[k];
#pragma unroll
                    for (int e = 0; e < kN; ++e) has |= (passes(to_float(y[e])) ? 1u : 0u) << (k * kN + e);
                } else {
                    for (int e = max(0, -first[k]); e < kN && first[k] + e < in.vocab; ++e)
                        has |= (passes(to_float(in.s[first[k] + e])) ? 1u : 0u) << (k * kN + e);
                }
            }
            // indexes first, values once the list is whole: a lane has its tokens in any of the vectors
            int slot = append(&sh->listed, __popc(has));
            for (; has; has &= has - 1, ++slot) {
                const int bit = __ffs(has) - 1;
                int j = first[0];
#pragma unroll
                for (int k = 1; k < kAhead; ++k)
                    if (bit / kN == k) j = first[k];
                if (slot < kList) sh->index[slot] = j + bit % kN;
            }
        }
        __syncthreads();
        const int listed = min(sh->listed, kList);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (i * kT + tid < listed) sh->value[i * kT + tid] = in.at(sh->index[i * kT + tid]);
    } else if (tid == 0) {
        sh->listed = kList + 1;
    }
    work.group.sync();
    const int size = static_cast<int>(work.group.size);
    if (size == 1) return sh->listed <= kList;
    int before = 0, all = 0;
    for (int c = 0; c < size; ++c) {
        const int n_c = static_cast<int>(load32(peer(&sh->listed, c)));
        if (c < static_cast<int>(work.group.rank)) before += n_c;
        all = min(all + n_c, kList + 1);
    }
    const int own = sh->listed;
    if (all <= kList && work.group.rank != 0)
        for (int i = tid; i < own; i += kT) {
            store32(peer(&sh->value[before + i], 0), __float_as_uint(sh->value[i]));
            store32(peer(&sh->index[before + i], 0), static_cast<uint32_t>(sh->index[i]));
        }
    work.group.sync();
    if (tid == 0) sh->listed = all;
    __syncthreads();
    return all <= kList;
}

// The cut of all tokens: histogram, then the list of the cut's bin; a bin that does not fit is divided
// again between its own extremes, by keys.
template <typename L>
__device__ __noinline__ Cut wide_cut(Work<L>& work, bool by_mass, u64 limit, const Found* known) {
    Shared* sh = work.sh;
    const int tid = threadIdx.x;
    const float best = work.best, inverse = work.r.inverse;
    float high = best, low = -INFINITY;
    uint32_t width = 1;  // keys a bin, after the first division
    Sum above{0, 0};
    for (bool first = true;; first = false) {
        // bin of a token of weight in the range divided; -1 elsewhere
        auto bin_in = [&](float x, uint32_t& w) {
            if (!(x >= low && x <= high)) return -1;
            w = static_cast<uint32_t>(weight_of(exp_of(x, best, inverse)));
            if (!w) return -1;
            return first ? work.bin_of(x) : static_cast<int>((key_of(high) - key_of(x)) / width);
        };
        Found f;
        if (first && known) {
            f = *known;
        } else {
            clear_histogram(sh);
            work.group.sync();
            work.every([&](float x) {
                uint32_t w;
                const int bin = bin_in(x, w);
                if (bin < 0) return;
                atomicAdd(&sh->count[bin], 1u);
                add_mass(sh, bin, w);
            });
            work.merge(kBins);
            f = work.search(by_mass, limit - (by_mass ? above.mass : static_cast<u64>(above.count)));
        }
        if (f.bin == kBins) return Cut{-INFINITY, f.whole};  // fewer tokens of weight than top-k asks for
        above.count += f.before.count;
        above.mass += f.before.mass;
        if (tid == 0) sh->listed = 0;
        work.group.sync();
        work.every([&](float x) {
            uint32_t w;
            if (bin_in(x, w) != f.bin) return;
            const int at = atomicAdd(&sh->listed, 1);
            if (at < kList) sh->value[at] = x;
        });
        __syncthreads();
        if (work.group.max_key(static_cast<uint32_t>(sh->listed)) <= kList) {
            float v[kPer];
            uint32_t w[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int at = i * kT + tid;
                v[i] = at < sh->listed ? sh->value[at] : -INFINITY;
                w[i] = at < sh->listed ? static_cast<uint32_t>(weight_of(exp_of(v[i], best, inverse))) : 0u;
            }
            return by_mass ? find_cut<true>(work.group, v, w, limit, above) : find_cut<false>(work.group, v, w, limit, above);
        }
        uint32_t up = 0, down = 0;
        work.every([&](float x) {
            uint32_t w;
            if (bin_in(x, w) != f.bin) return;
            up = max(up, key_of(x));
            down = max(down, ~key_of(x));
        });
        high = value_of(work.group.max_key(up));
        low = value_of(~work.group.max_key(down));
        if (high == low) return Cut{high, above};
        width = (key_of(high) - key_of(low)) / kBins + 1;  // the ends never share a bin: each division gains
    }
}

// Weight of the whole row, and the bin of its tokens up to which a share p < 1 of it stands. Tokens that all
// together weigh less than the rest, 1 - p, cannot reach the share: they are left out of the histogram. The
// weight's lower bound is that of the group maxima.
template <typename L>
__device__ __noinline__ Found share_bin(Work<L>& work, u64& limit) {
    constexpr int kSlots = Work<L>::kSlots;
    Shared* sh = work.sh;
    const float best = work.best, inverse = work.r.inverse;
    const L* maxima = reinterpret_cast<const L*>(sh->maxima);
    clear_histogram(sh);
    u64 mass = 0;
#pragma unroll 4
    for (int slot = 0; slot < kSlots; ++slot)
        mass += weight_of(exp_of(clean(to_float(maxima[slot * kT + threadIdx.x])), best, inverse));
    const u64 least = work.group.sum(Sum{0, mass}).mass;
    // token weights below this sum to less than half of the rest (the other half is slack for roundings to weights)
    const float rest = (1.0f - work.r.top_p) * 0.5f * static_cast<float>(least) / static_cast<float>(work.in.vocab);
    const uint32_t floor_w = rest > 2.0f ? static_cast<uint32_t>(fminf(rest, kUnit)) : 1u;
    mass = 0;
    work.every([&](float x) {
        const uint32_t w = static_cast<uint32_t>(weight_of(exp_of(x, best, inverse)));
        mass += w;
        if (w >= floor_w) add_mass(sh, work.bin_of(x), w);
    });
    limit = share_of(work.r.top_p, work.group.sum(Sum{0, mass}).mass);
    work.merge(kBins);
    return work.search(true, limit);
}

// Cuts and draw from the whole row.
template <typename L>
__device__ __noinline__ void draw_wide(Work<L>& work, u64 given, const Found* known, const rl2_sample_args& a, long long row) {
    constexpr int kN = Work<L>::kN;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Shared* sh = work.sh;
    const Row r = work.r;
    const float best = work.best;
    const Reader<L>& in = work.in;
    const int shift = work.shift, per = 1 << work.log_per;
    Kept kept{-INFINITY, 0};
    if (work.first_only) {
        kept = Kept{best, 1};
    } else {
        Sum above{~0u, ~0ull};
        u64 total = 0;
        if (work.cut_k) {
            const Cut c = wide_cut(work, false, static_cast<u64>(r.top_k), nullptr);
            above = c.above;
            total = c.above.mass;
            if (c.value != -INFINITY) {
                kept = Kept{c.value, static_cast<u64>(r.top_k) - c.above.count};
                total += kept.ties * weight_of(exp_of(kept.cut, best, r.inverse));
            }
        }
        if (r.top_p < 1.0f) {
            u64 most = kept.ties;
            const u64 limit = given ? given : share_of(r.top_p, total);
            if (above.mass >= limit) {
                const Cut c = wide_cut(work, true, limit, known);
                kept.cut = c.value;
                above = c.above;
                most = ~0ull;
            }
            if (kept.cut != -INFINITY)
                kept.ties = kept_of_last(above.mass, weight_of(exp_of(kept.cut, best, r.inverse)), limit, most);
        }
    }
    // kept weight above the cut and tokens at it, by stretch
    auto weigh = [&](float x) {
        if (r.greedy) return static_cast<u64>(1);
        const float e = exp_of(x, best, r.inverse);
        return e >= r.min_p ? weight_of(e) : 0;
    };
    const u64 tie_weight = kept.ties ? weigh(kept.cut) : 0;
    work.group.sync();
    clear_histogram(sh);
    work.group.sync();
    u64 mass = 0;
    uint32_t ties = 0;
    auto end_of_step = [&](int step) {
        if (((step + 1) & (per - 1)) != 0) return;  // not the stretch's last
        mass = warp_sum64(mass);
        ties = __reduce_add_sync(0xffffffffu, ties);
        if (lane == 0) {
            const int st = work.from + warp + kWarps * (step >> work.log_per);
            sh->mass[st] = mass;
            sh->count[st] = ties;
        }
        mass = 0;
        ties = 0;
    };
    if (kept.cut == -INFINITY && !(r.min_p > 0.0f)) {  // all that weighs
        work.every_vector([&](int step, int, const float(&x)[kN]) {
#pragma unroll
            for (int e = 0; e < kN; ++e) mass += weight_of(exp_of(x[e], best, r.inverse));
            end_of_step(step);
        });
    } else {
        work.every_vector([&](int step, int, const float(&x)[kN]) {
#pragma unroll
            for (int e = 0; e < kN; ++e) {
                if (x[e] > kept.cut) mass += weigh(x[e]);
                ties += x[e] == kept.cut;
            }
            end_of_step(step);
        });
    }
    work.merge(kStretches);
    if (work.group.rank == 0) {
        constexpr int kEachStretch = kStretches / kT;
        Sum mine[kEachStretch], s{0, 0}, all;
#pragma unroll
        for (int e = 0; e < kEachStretch; ++e) {
            mine[e] = Sum{sh->count[tid * kEachStretch + e], sh->mass[tid * kEachStretch + e]};
            s.count += mine[e].count;
            s.mass += mine[e].mass;
        }
        Sum at = block_scan(sh, s, all);
        const u64 total = all.mass + min(static_cast<u64>(all.count), kept.ties) * tie_weight;
        const u64 target = target_of(r.uniform, total);
#pragma unroll
        for (int e = 0; e < kEachStretch; ++e) {
            // kept weight before this stretch, and through it
            const u64 cum = at.mass + min(static_cast<u64>(at.count), kept.ties) * tie_weight;
            const Sum next{at.count + mine[e].count, at.mass + mine[e].mass};
            if (cum <= target && target < next.mass + min(static_cast<u64>(next.count), kept.ties) * tie_weight)
                sh->found = Found{mine[e], Sum{at.count, cum}, Sum{0, total}, tid * kEachStretch + e, 0};
            at = next;
        }
    }
    work.share_found();
    const int chosen = sh->found.bin;
    const u64 start = sh->found.before.mass, ties_seen = sh->found.before.count, total = sh->found.whole.mass;
    const u64 target = target_of(r.uniform, total);
    if (chosen < work.from || chosen >= work.to) return;
    // the CTA that owns the stretch draws within it
    for (int i = tid; i < (1 << shift); i += kT) {
        sh->slot_w[i] = 0;
        sh->slot_tie[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < 32 * per; i += kT) {
        const int b = chosen * per * 32 + i;
        if (b >= in.vectors) break;
        float x[kN];
        in.load(b, x);
#pragma unroll
        for (int e = 0; e < kN; ++e) {
            sh->slot_w[i * kN + e] = x[e] > kept.cut || (x[e] == kept.cut && kept.ties) ? static_cast<uint32_t>(weigh(x[e])) : 0u;
            sh->slot_tie[i * kN + e] = x[e] == kept.cut;
        }
    }
    __syncthreads();
    if (warp != 0) return;
    u64 cum = start, left = kept.ties - min(kept.ties, ties_seen);
    for (int i = lane; i < (1 << shift); i += 32) {
        uint32_t mine = sh->slot_w[i];
        const bool tie = sh->slot_tie[i];
        const uint32_t tied = __ballot_sync(0xffffffffu, tie);
        if (tie && __popc(tied & ((1u << lane) - 1)) >= left) mine = 0;
        left -= min(left, static_cast<u64>(__popc(tied)));
        const u64 step = warp_sum64(mine);
        if (cum + step > target) {
            u64 sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, cum + sum > target);
            if (lane == __ffs(hit) - 1) write_token(a, row, r, best, (chosen << shift) + i - in.mis, mine, total);
            return;
        }
        cum += step;
    }
}

// The arguments are a grid constant: what is called here takes their address, which would put a copy on each thread's stack.
template <typename L>
__global__ void __launch_bounds__(kT, 2) row_kernel(const __grid_constant__ rl2_sample_args a, const int size, const int shift) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared* sh = reinterpret_cast<Shared*>(raw);
    constexpr int kN = Work<L>::kN, kSlots = Work<L>::kSlots;
    const int tid = threadIdx.x, warp = tid >> 5;
    const int V = a.vocab;
    const uint32_t rank = size > 1 ? ptx::cluster_rank() : 0u;
    ptx::grid_release();
    ptx::grid_wait();
    for (long long row = blockIdx.x / size; row < a.rows; row += gridDim.x / size) {
        const Reader<L> in(static_cast<const L*>(a.logits) + row * a.ld_logits, V);
        const int log_per = shift - 5 - (kN == 8 ? 3 : 2);
        const int stretches = (in.vectors + (32 << log_per) - 1) >> (5 + log_per);
        Work<L> work{sh, Cluster{sh, static_cast<uint32_t>(size), rank, 0}, in, row_of(a, row), shift, log_per,
                     static_cast<int>(static_cast<long long>(stretches) * rank / size),
                     static_cast<int>(static_cast<long long>(stretches) * (rank + 1) / size), 0, 0, 0.0f, 0.0f, false, false};
        work.steps = work.vectors_of(warp);
        work.slot_steps = max(1, (work.vectors_of(0) + kSlots - 1) / kSlots);
        work.best = value_of(work.group.max_key(key_of(read_row(work))));
        if (work.best == -INFINITY || !work.r.valid) {
            if (tid == 0 && rank == 0) {
                a.tokens[row] = -1;
                if (a.log_probs) a.log_probs[row] = -INFINITY;
                if (!work.r.valid && a.health) atomicOr(a.health, kHealthIndex);
            }
            work.group.sync();
            continue;
        }
        const Row& r = work.r;
        work.per_value = fminf(r.inverse * (kBins / kReach), FLT_MAX);
        work.cut_k = r.top_k > 0 && r.top_k < V;
        work.first_only = r.greedy || r.top_p <= 0.0f || (work.cut_k && r.top_k == 1);
        // ---- the bound on the candidates ----
        int bound = kBins - 1;
        if (work.first_only) {
            bound = 0;
        } else {
            if (work.cut_k) {
                clear_histogram(sh);
                __syncthreads();
                const L* maxima = reinterpret_cast<const L*>(sh->maxima);
#pragma unroll
                for (int slot = 0; slot < kSlots; ++slot) {
                    const int bin = work.bin_of(clean(to_float(maxima[slot * kT + tid])));
                    if (bin < kBins - 1) atomicAdd(&sh->count[bin], 1u);
                }
                static_assert(kEach == 4, "four bins a thread");
                work.merge_counts();
                if (rank == 0) {
                    if (tid == 0) sh->found.bin = kBins;
                    __syncthreads();
                    const uint4 mine = *reinterpret_cast<const uint4*>(&sh->count[tid * kEach]);
                    const uint32_t in_order[kEach] = {mine.x, mine.y, mine.z, mine.w};
                    uint32_t at = block_scan(sh, mine.x + mine.y + mine.z + mine.w);
                    const uint32_t k = static_cast<uint32_t>(r.top_k);
#pragma unroll
                    for (int e = 0; e < kEach; ++e) {
                        if (at < k && at + in_order[e] >= k) sh->found.bin = tid * kEach + e;
                        at += in_order[e];
                    }
                    __syncthreads();
                    if (tid > 0 && tid < size) store32(peer(&sh->found.bin, tid), static_cast<uint32_t>(sh->found.bin));
                }
                if (size > 1) work.group.sync();
                bound = min(bound, sh->found.bin);
            }
            if (r.top_p >= 1.0f && r.min_p > 0.0f)  // one bin of slack for the rounding of the logarithm
                bound = min(bound, static_cast<int>(min(-logf(r.min_p) * (kBins / kReach) + 1.0f, kBins - 1.0f)));
        }
        u64 given = 0;
        Found share;
        if (!work.cut_k && !work.first_only && r.top_p < 1.0f) {
            share = share_bin(work, given);
            bound = min(bound, share.bin);
        }
        if (bound < kBins - 1 && build_list(work, bound)) {
            if (rank == 0) {
                const int n = sh->listed;
                if (n <= 64) {
                    if (warp == 0) draw_few<2>(sh, n, r, V, work.best, given, a, row);
                } else if (n <= kFew) {
                    if (warp == 0) draw_few<kFewPer>(sh, n, r, V, work.best, given, a, row);
                } else {
                    draw_many(sh, n, r, V, work.best, fminf(work.per_value * (static_cast<float>(kBins) / (bound + 1)), FLT_MAX), given, a, row);
                }
            }
        } else {
            draw_wide(work, given, given ? &share : nullptr, a, row);
        }
        work.group.sync();
    }
    if (size > 1) ptx::cluster_sync();  // no CTA leaves while another may read its shared memory
}

int launched(cudaError_t e) {
    if (e == cudaSuccess) return launch_status("token sampling");
    set_error("token sampling: %s", cudaGetErrorString(e));
    return -1;
}

template <typename L, int N>
int launch_warps(const rl2_sample_args& a, cudaStream_t stream) {
    const int blocks = static_cast<int>(std::min<long long>((static_cast<long long>(a.rows) + kRowWarps - 1) / kRowWarps, 148 * 16));
    return launched(launch_early(warp_kernel<L, N>, blocks, 32 * kRowWarps, 0, stream, a));
}

template <typename L>
int launch(const rl2_sample_args& a, cudaStream_t stream) {
    if (a.vocab <= 32) return launch_warps<L, 1>(a, stream);
    if (a.vocab <= 64) return launch_warps<L, 2>(a, stream);
    if (a.vocab <= 128) return launch_warps<L, 4>(a, stream);
    if (a.vocab <= 256) return launch_warps<L, 8>(a, stream);
    if (a.vocab <= 512) return launch_warps<L, 16>(a, stream);
    if (a.vocab <= 1024) return launch_warps<L, 32>(a, stream);
    // stretches of 32 vectors, or more where that gives over kStretches of them
    constexpr int kN = Reader<L>::kN;
    int shift = 5 + (kN == 8 ? 3 : 2);
    while (((a.vocab + kN - 1 + kN - 1) >> shift) + 1 > kStretches) ++shift;
    // few rows: more CTAs a row, while each has 4096 tokens or more
    int size = 1;
    while (size < 8 && static_cast<long long>(a.rows) * size * 2 <= 148 && a.vocab / (2 * size) >= 4096) size *= 2;
    const long long clusters = std::min<long long>(a.rows, std::max(1, 148 * 2 / size));
    static std::atomic<unsigned long long> allowed{0};  // devices (up to 64) whose limit is raised
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && (device > 63 || !(allowed.load() >> device & 1))) {
        e = cudaFuncSetAttribute(reinterpret_cast<const void*>(row_kernel<L>), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 sizeof(Shared));
        if (e == cudaSuccess && device <= 63) allowed.fetch_or(1ull << device);
    }
    if (e == cudaSuccess)
        e = launch_early_clusters(row_kernel<L>, size, static_cast<unsigned>(clusters * size), kT, sizeof(Shared), stream, a, size, shift);
    return launched(e);
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
    if (a->logits_dtype == 0) return launch<float>(*a, as_stream(stream));
    if (a->logits_dtype == 1) return launch<__half>(*a, as_stream(stream));
    return launch<__nv_bfloat16>(*a, as_stream(stream));
}
