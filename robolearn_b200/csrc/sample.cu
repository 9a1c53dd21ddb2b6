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
// in registers, v found by halving the interval of values, two warp reductions a step. More tokens: a
// CTA, or with few rows a cluster of CTAs that each read a part of the row, see row_kernel.

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
__device__ __forceinline__ Cut find_cut(Group& group, const float (&v)[N], const uint32_t (&w)[N], double limit, Sum above) {
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
    auto less = [&](Sum s) { return (MASS ? static_cast<double>(s.mass) : static_cast<double>(s.count)) < limit; };
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

// Both cuts of a row whose tokens (at least those that the cuts can reach) are N a thread.
template <int N, typename Group>
__device__ __forceinline__ Kept both_cuts(Group& group, const Row& r, int vocab, float best, const float (&v)[N],
                                          const uint32_t (&w)[N], Sum all) {
    Kept kept{-INFINITY, 0};
    if (r.greedy || r.top_p <= 0.0f) return Kept{best, 1};
    Sum above = all;  // above -inf
    u64 total = all.mass;
    if (r.top_k > 0 && r.top_k < vocab && all.count > static_cast<uint32_t>(r.top_k)) {
        const Cut c = find_cut<false>(group, v, w, static_cast<double>(r.top_k), Sum{0, 0});
        kept = Kept{c.value, static_cast<u64>(r.top_k) - c.above.count};
        above = c.above;
        total = above.mass + kept.ties * weight_of(exp_of(kept.cut, best, r.inverse));
    }
    if (r.top_p < 1.0f) {
        const double limit = static_cast<double>(r.top_p) * static_cast<double>(total);
        u64 most = kept.ties;
        if (!(static_cast<double>(above.mass) < limit)) {
            const Cut c = find_cut<true>(group, v, w, limit, Sum{0, 0});
            kept.cut = c.value;
            above = c.above;
            most = ~0ull;
        }
        if (kept.cut != -INFINITY)
            kept.ties = kept_of_last(above.mass, weight_of(exp_of(kept.cut, best, r.inverse)), limit, most);
    }
    return kept;
}

// ---- up to 1024 tokens: a warp per row, N tokens a lane (token i * 32 + lane) --------------

constexpr int kRowWarps = 4;

template <typename L, int N>
__global__ void __launch_bounds__(32 * kRowWarps) warp_kernel(const rl2_sample_args a) {
    const int lane = threadIdx.x & 31;
    const int V = a.vocab;
    WarpGroup group;
    for (long long row = static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5); row < a.rows;
         row += static_cast<long long>(gridDim.x) * kRowWarps) {
        const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits;
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = i * 32 + lane;
            v[i] = j < V ? clean(to_float(s[j])) : -INFINITY;
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
        const Kept kept = both_cuts(group, r, V, best, v, w, all);
        u64 ties_left = kept.ties, total = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool tie = v[i] == kept.cut && w[i] != 0;
            const uint32_t tied = __ballot_sync(0xffffffffu, tie);
            const bool in = v[i] > kept.cut || (tie && __popc(tied & ((1u << lane) - 1)) < ties_left);
            ties_left -= min(ties_left, static_cast<u64>(__popc(tied)));
            if (!in || (!r.greedy && exp_of(v[i], best, r.inverse) < r.min_p)) w[i] = 0;
            total += w[i];
        }
        total = warp_sum64(total);
        const u64 target = target_of(r.uniform, total);
        u64 cum = 0;
        for (int i = 0; i < N; ++i) {
            uint32_t mine = 0;
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (k == i) mine = w[k];
            const u64 step = warp_sum64(mine);
            if (cum + step > target) {  // the token is one of these 32
                u64 sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += up;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, cum + sum > target);
                if (lane == __ffs(hit) - 1) {
                    a.tokens[row] = i * 32 + lane;
                    if (a.log_probs) a.log_probs[row] = log_share(mine, total);
                }
                break;
            }
            cum += step;
        }
    }
}

// ---- more tokens: a CTA, or a cluster of CTAs, per row ---------------------------------
//
// The row is read once. A thread keeps the maxima of small groups of its tokens (16-byte vectors, or
// several); the k-th largest of all maxima bounds the k-th token from below, so only the groups whose
// maximum reaches the bound are read again and give a list of a little more than k candidates, on which
// both cuts are found. The bound comes from a histogram of the maxima over 2048 bins of (l - max) / T,
// whose 21.6 cover every token that has a weight. min-p bounds the candidates in the same way.
// Without a bound (no top-k, or the list does not fit) the cuts come from a histogram of all tokens
// (count and weight a bin) and the list of those in the bin of the cut.
// The draw: the kept weight of each stretch of 2^shift tokens, a scan, and one warp on the stretch that
// holds the target.

constexpr int kT = 512;
constexpr int kWarps = kT / 32;
constexpr int kBins = 2048;
constexpr float kReach = 21.6f;  // exp(-21.6) 2^30 rounds to 0
constexpr int kSlots = 16;       // group maxima per thread
constexpr int kPer = 8;          // list entries per thread
constexpr int kList = kT * kPer;
constexpr int kStretches = 1024;
constexpr int kMaxStretch = 2048;  // tokens: 2^20 of them in fewer than 1024 stretches

struct Shared {
    u64 mass[kBins];       // histogram / stretches
    uint32_t count[kBins];
    float maxima[kSlots][kT];
    float value[kList];
    int index[kList];
    uint32_t slot_w[kMaxStretch];  // the drawn stretch: weight, tie
    uint8_t slot_tie[kMaxStretch];
    uint32_t red_count[2][kWarps];
    u64 red_mass[2][kWarps];
    uint32_t scan_count[kWarps];
    u64 scan_mass[kWarps];
    int found;
    u64 found_mass;
    uint32_t found_count;
    u64 found_total;
    int listed;
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

// All threads of the cluster's CTAs (of the CTA alone where it has one).
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
    // One barrier a reduction: the slots alternate, and a slot is written again only after the
    // barrier of the reduction between, which every reader has reached.
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

template <typename L>
struct Reader {
    static constexpr int kN = 16 / sizeof(L);
    const L* s;     // the row
    int vocab, mis; // elements between the 16-byte boundary at or before the row and the row
    int vectors;

    __device__ __forceinline__ Reader(const L* row, int v) : s(row), vocab(v) {
        mis = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(L));
        vectors = (mis + vocab + kN - 1) / kN;
    }
    // token of element e of vector b: b kN + e - mis; elements outside the row are -inf
    __device__ __forceinline__ void load(int b, float (&v)[kN]) const {
        const int j = b * kN - mis;
        if (j >= 0 && j + kN <= vocab) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(s + j));
            L x[kN];
            *reinterpret_cast<uint4*>(x) = raw;
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = clean(to_float(x[e]));
        } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = j + e >= 0 && j + e < vocab ? clean(to_float(s[j + e])) : -INFINITY;
        }
    }
};

template <typename L>
__global__ void __launch_bounds__(kT, 2) row_kernel(const rl2_sample_args a, const int size, const int shift) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared* sh = reinterpret_cast<Shared*>(raw);
    constexpr int kN = Reader<L>::kN;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int V = a.vocab;
    Cluster group{sh, static_cast<uint32_t>(size), size > 1 ? ptx::cluster_rank() : 0u, 0};
    const int per = (1 << shift) / (32 * kN);  // vectors a lane has in a stretch
    for (long long row = blockIdx.x / size; row < a.rows; row += gridDim.x / size) {
        const Reader<L> in(static_cast<const L*>(a.logits) + row * a.ld_logits, V);
        const Row r = row_of(a, row);
        const int stretches = (in.vectors + 32 * per - 1) / (32 * per);
        // this CTA's stretches, a warp each in turn
        const int from = static_cast<int>(static_cast<long long>(stretches) * group.rank / size);
        const int to = static_cast<int>(static_cast<long long>(stretches) * (group.rank + 1) / size);
        const int steps = max(0, (to - from - warp + kWarps - 1) / kWarps) * per;  // vectors of this lane
        const int slot_steps = (((to - from + kWarps - 1) / kWarps) * per + kSlots - 1) / kSlots;
        auto vector_of = [&](int step) {
            return ((from + warp + kWarps * (step / per)) * per + step % per) * 32 + lane;
        };
        // ---- the one pass over the row: group maxima and the maximum ----
        float best = -INFINITY;
        for (int slot = 0; slot < kSlots; ++slot) {
            float m = -INFINITY;
            const int end = min(steps, (slot + 1) * slot_steps);
#pragma unroll 4
            for (int i = slot * slot_steps; i < end; ++i) {
                const int b = vector_of(i);
                if (b < in.vectors) {
                    float v[kN];
                    in.load(b, v);
#pragma unroll
                    for (int e = 0; e < kN; ++e) m = fmaxf(m, v[e]);
                }
            }
            sh->maxima[slot][tid] = m;
            best = fmaxf(best, m);
        }
        best = value_of(group.max_key(key_of(best)));
        if (best == -INFINITY || !r.valid) {
            if (tid == 0 && group.rank == 0) {
                a.tokens[row] = -1;
                if (a.log_probs) a.log_probs[row] = -INFINITY;
                if (!r.valid && a.health) atomicOr(a.health, kHealthIndex);
            }
            continue;
        }
        const float per_bin = kBins / kReach;
        auto bin_of = [&](float v) {  // bin 0 holds the best token; -inf and what has no weight: the last
            const float at = (best - v) * r.inverse * per_bin;
            return at < kBins - 1 ? static_cast<int>(at) : kBins - 1;
        };
        auto clear = [&]() {
            for (int i = tid; i < kBins; i += kT) {
                sh->mass[i] = 0;
                sh->count[i] = 0;
            }
        };
        // totals of a bin over the cluster
        auto bin_total = [&](int i) {
            Sum t{sh->count[i], sh->mass[i]};
            if (size > 1) {
                t = Sum{0, 0};
                for (int c = 0; c < size; ++c) {
                    t.count += load32(peer(&sh->count[i], c));
                    t.mass += load64(peer(&sh->mass[i], c));
                }
            }
            return t;
        };
        // The first bin up to which (itself included) the count, or the weight, reaches the limit; what is before
        // it; the whole. kBins where none does. The histogram is complete and stays.
        auto find_bin = [&](bool by_mass, double limit, Sum& before, Sum& whole) {
            constexpr int kEach = kBins / kT;
            Sum mine[kEach], s{0, 0};
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                mine[e] = bin_total(tid * kEach + e);
                s.count += mine[e].count;
                s.mass += mine[e].mass;
            }
            if (tid == 0) sh->found = kBins;
            Sum at = block_scan(sh, s, whole);
            auto value = [&](Sum x) { return by_mass ? static_cast<double>(x.mass) : static_cast<double>(x.count); };
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const Sum next{at.count + mine[e].count, at.mass + mine[e].mass};
                if (value(at) < limit && value(next) >= limit) {
                    sh->found = tid * kEach + e;
                    sh->found_count = at.count;
                    sh->found_mass = at.mass;
                }
                at = next;
            }
            __syncthreads();
            before = Sum{sh->found_count, sh->found_mass};
            const int bin = sh->found;
            __syncthreads();
            return bin;
        };
        // List of the tokens of weight in a range of values; false where it does not fit on some CTA.
        auto push = [&](float v, int token) {
            const int at = atomicAdd(&sh->listed, 1);
            if (at < kList) {
                sh->value[at] = v;
                sh->index[at] = token;
            }
        };
        const bool cut_k = r.top_k > 0 && r.top_k < V;
        const bool first_only = r.greedy || r.top_p <= 0.0f || (cut_k && r.top_k == 1);

        // ---- the bound on the candidates ----
        int bound = kBins - 1;
        Sum before, whole;
        if (first_only) {
            bound = 0;
        } else {
            if (cut_k) {
                clear();
                group.sync();
                for (int slot = 0; slot < kSlots; ++slot) {
                    const float m = sh->maxima[slot][tid];
                    if (m != -INFINITY) atomicAdd(&sh->count[bin_of(m)], 1u);
                }
                group.sync();
                bound = min(bound, find_bin(false, r.top_k, before, whole));
                group.sync();
            }
            if (r.top_p >= 1.0f && r.min_p > 0.0f)  // one bin of slack for the rounding of the logarithm
                bound = min(bound, static_cast<int>(min(-logf(r.min_p) * per_bin + 1.0f, kBins - 1.0f)));
        }
        float v[kPer];
        uint32_t w[kPer];
        auto take_list = [&]() {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int at = i * kT + tid;
                v[i] = at < sh->listed ? sh->value[at] : -INFINITY;
                w[i] = at < sh->listed ? static_cast<uint32_t>(weight_of(exp_of(v[i], best, r.inverse))) : 0u;
            }
        };
        bool listed = false;
        if (bound < kBins - 1) {
            if (tid == 0) sh->listed = 0;
            __syncthreads();
            for (int slot = 0; slot < kSlots; ++slot) {
                if (bin_of(sh->maxima[slot][tid]) > bound) continue;
                const int end = min(steps, (slot + 1) * slot_steps);
                for (int i = slot * slot_steps; i < end; ++i) {
                    const int b = vector_of(i);
                    if (b >= in.vectors) break;
                    float x[kN];
                    in.load(b, x);
#pragma unroll
                    for (int e = 0; e < kN; ++e)
                        if (bin_of(x[e]) <= bound) push(x[e], b * kN + e - in.mis);
                }
            }
            __syncthreads();
            listed = group.max_key(sh->listed > kList ? 1u : 0u) == 0;
        }
        Kept kept{-INFINITY, 0};
        if (listed) {
            take_list();
            Sum all{0, 0};
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                all.count += w[i] != 0;
                all.mass += w[i];
            }
            all = group.sum(all);
            kept = both_cuts(group, r, V, best, v, w, all);
        } else if (first_only) {
            kept = Kept{best, 1};
        } else if (cut_k || r.top_p < 1.0f) {
            // ---- cuts from a histogram of every token ----
            auto every = [&](auto&& f) {
                for (int i = 0; i < steps; ++i) {
                    const int b = vector_of(i);
                    if (b >= in.vectors) break;
                    float x[kN];
                    in.load(b, x);
#pragma unroll
                    for (int e = 0; e < kN; ++e) f(x[e], b * kN + e - in.mis);
                }
            };
            // The cut of all tokens: histogram over [.., high], then the list of the cut's bin; a bin that does
            // not fit is divided again between its own extremes.
            auto wide_cut = [&](bool by_mass, double limit_or_share, bool is_share, double& limit) {
                float high = best, low = -INFINITY, scale = r.inverse * per_bin;
                Sum above{0, 0};
                for (bool first = true;; first = false) {
                    auto bin_in = [&](float x) {
                        const float at = (high - x) * scale;
                        return at < kBins - 1 ? static_cast<int>(at) : kBins - 1;
                    };
                    auto inside = [&](float x) { return x >= low && x <= high; };
                    clear();
                    group.sync();
                    every([&](float x, int) {
                        if (!inside(x)) return;
                        const u64 weight = weight_of(exp_of(x, best, r.inverse));
                        if (!weight) return;
                        const int bin = bin_in(x);
                        atomicAdd(&sh->count[bin], 1u);
                        atomicAdd(&sh->mass[bin], weight);
                    });
                    group.sync();
                    Sum part, all;
                    if (first && is_share) {
                        find_bin(by_mass, 0.0, part, all);
                        limit = limit_or_share * static_cast<double>(all.mass);
                    } else if (first) {
                        limit = limit_or_share;
                    }
                    const double rest = limit - (by_mass ? static_cast<double>(above.mass) : static_cast<double>(above.count));
                    const int bin = find_bin(by_mass, rest, part, all);
                    if (bin == kBins) {  // fewer tokens of weight than top-k asks for
                        group.sync();
                        return Cut{-INFINITY, all};
                    }
                    above.count += part.count;
                    above.mass += part.mass;
                    const Sum here = bin_total(bin);
                    if (tid == 0) sh->listed = 0;
                    group.sync();
                    if (here.count <= kList) {
                        every([&](float x, int token) {
                            if (inside(x) && bin_in(x) == bin && weight_of(exp_of(x, best, r.inverse))) push(x, token);
                        });
                        __syncthreads();
                        take_list();
                        return by_mass ? find_cut<true>(group, v, w, limit, above) : find_cut<false>(group, v, w, limit, above);
                    }
                    uint32_t up = 0, down = 0;
                    every([&](float x, int) {
                        if (inside(x) && bin_in(x) == bin && weight_of(exp_of(x, best, r.inverse))) {
                            up = max(up, key_of(x));
                            down = max(down, ~key_of(x));
                        }
                    });
                    high = value_of(group.max_key(up));
                    low = value_of(~group.max_key(down));
                    if (high == low) return Cut{high, above};
                    // at most kBins - 1 for the lowest, so the ends never share a bin
                    scale = fminf((kBins - 1) / (high - low), FLT_MAX);
                }
            };
            Sum above{0, 0};
            u64 total = 0;
            double limit = 0.0;
            bool have_k = false;
            if (cut_k) {
                const Cut c = wide_cut(false, r.top_k, false, limit);
                above = c.above;
                total = c.above.mass;
                if (c.value != -INFINITY) {
                    have_k = true;
                    kept = Kept{c.value, static_cast<u64>(r.top_k) - c.above.count};
                    total += kept.ties * weight_of(exp_of(kept.cut, best, r.inverse));
                }
            }
            if (r.top_p < 1.0f) {
                u64 most = kept.ties;
                limit = static_cast<double>(r.top_p) * static_cast<double>(total);
                if (!have_k || !(static_cast<double>(above.mass) < limit)) {
                    const Cut c = have_k || cut_k ? wide_cut(true, limit, false, limit) : wide_cut(true, r.top_p, true, limit);
                    kept.cut = c.value;
                    above = c.above;
                    most = ~0ull;
                }
                if (kept.cut != -INFINITY)
                    kept.ties = kept_of_last(above.mass, weight_of(exp_of(kept.cut, best, r.inverse)), limit, most);
            }
        }
        // ---- the draw: kept weight above the cut and tokens at it, by stretch ----
        auto weigh = [&](float x) {
            if (r.greedy) return static_cast<u64>(1);
            const float e = exp_of(x, best, r.inverse);
            return e >= r.min_p ? weight_of(e) : 0;
        };
        const u64 tie_weight = kept.ties ? weigh(kept.cut) : 0;
        group.sync();
        clear();
        group.sync();
        if (listed) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int at = i * kT + tid;
                if (at < sh->listed && v[i] >= kept.cut) {
                    const int b = (sh->index[at] + in.mis) >> shift;
                    if (v[i] == kept.cut)
                        atomicAdd(&sh->count[b], 1u);
                    else
                        atomicAdd(&sh->mass[b], weigh(v[i]));
                }
            }
        } else {
            for (int st = from + warp; st < to; st += kWarps) {
                u64 mass = 0;
                uint32_t ties = 0;
                for (int i = 0; i < per; ++i) {
                    const int b = (st * per + i) * 32 + lane;
                    if (b >= in.vectors) break;
                    float x[kN];
                    in.load(b, x);
#pragma unroll
                    for (int e = 0; e < kN; ++e) {
                        if (x[e] > kept.cut) mass += weigh(x[e]);
                        ties += x[e] == kept.cut;
                    }
                }
                mass = warp_sum64(mass);
                ties = __reduce_add_sync(0xffffffffu, ties);
                if (lane == 0) {
                    sh->mass[st] = mass;
                    sh->count[st] = ties;
                }
            }
        }
        group.sync();
        constexpr int kEach = kStretches / kT;
        Sum mine[kEach], s{0, 0}, all;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            mine[e] = bin_total(tid * kEach + e);
            s.count += mine[e].count;
            s.mass += mine[e].mass;
        }
        Sum at = block_scan(sh, s, all);
        const u64 total = all.mass + min(static_cast<u64>(all.count), kept.ties) * tie_weight;
        const u64 target = target_of(r.uniform, total);
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            // before this stretch, and through it
            const u64 cum = at.mass + min(static_cast<u64>(at.count), kept.ties) * tie_weight;
            at.count += mine[e].count;
            at.mass += mine[e].mass;
            const u64 next = at.mass + min(static_cast<u64>(at.count), kept.ties) * tie_weight;
            if (cum <= target && target < next) {
                sh->found = tid * kEach + e;
                sh->found_mass = cum;
                sh->found_count = at.count - mine[e].count;
            }
        }
        __syncthreads();
        const int chosen = sh->found;
        const u64 start = sh->found_mass;
        const u64 ties_seen = sh->found_count;
        // the CTA that owns the stretch draws within it
        if (chosen >= from && chosen < to) {
            for (int i = tid; i < (1 << shift); i += kT) {
                sh->slot_w[i] = 0;
                sh->slot_tie[i] = 0;
            }
            __syncthreads();
            if (listed) {
                for (int i = tid; i < sh->listed; i += kT) {
                    const float x = sh->value[i];
                    const int j = sh->index[i] + in.mis;
                    if ((j >> shift) == chosen && x >= kept.cut) {
                        sh->slot_w[j & ((1 << shift) - 1)] = static_cast<uint32_t>(weigh(x));
                        sh->slot_tie[j & ((1 << shift) - 1)] = x == kept.cut;
                    }
                }
            } else {
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
            }
            __syncthreads();
            if (warp == 0) {
                u64 cum = start, left = kept.ties - min(kept.ties, ties_seen);
                for (int i = lane; i < (1 << shift); i += 32) {
                    uint32_t mine_w = sh->slot_w[i];
                    const bool tie = sh->slot_tie[i];
                    const uint32_t tied = __ballot_sync(0xffffffffu, tie);
                    if (tie && __popc(tied & ((1u << lane) - 1)) >= left) mine_w = 0;
                    left -= min(left, static_cast<u64>(__popc(tied)));
                    const u64 step = warp_sum64(mine_w);
                    if (cum + step > target) {
                        u64 sum = mine_w;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const u64 up = __shfl_up_sync(0xffffffffu, sum, o);
                            if (lane >= o) sum += up;
                        }
                        const uint32_t hit = __ballot_sync(0xffffffffu, cum + sum > target);
                        if (lane == __ffs(hit) - 1) {
                            a.tokens[row] = (chosen << shift) + i - in.mis;
                            if (a.log_probs) a.log_probs[row] = log_share(mine_w, total);
                        }
                        break;
                    }
                    cum += step;
                }
            }
        }
        group.sync();
    }
    if (size > 1) ptx::cluster_sync();  // no CTA leaves while another may read its shared memory
}

template <typename L, int N>
void launch_warps(const rl2_sample_args& a, cudaStream_t stream) {
    const int blocks = static_cast<int>(std::min<long long>((static_cast<long long>(a.rows) + kRowWarps - 1) / kRowWarps, 148 * 16));
    warp_kernel<L, N><<<blocks, 32 * kRowWarps, 0, stream>>>(a);
}

template <typename L>
int launch(const rl2_sample_args& a, cudaStream_t stream) {
    if (a.vocab <= 1024) {
        if (a.vocab <= 32)
            launch_warps<L, 1>(a, stream);
        else if (a.vocab <= 64)
            launch_warps<L, 2>(a, stream);
        else if (a.vocab <= 128)
            launch_warps<L, 4>(a, stream);
        else if (a.vocab <= 256)
            launch_warps<L, 8>(a, stream);
        else if (a.vocab <= 512)
            launch_warps<L, 16>(a, stream);
        else
            launch_warps<L, 32>(a, stream);
        return launch_status("token sampling");
    }
    // stretches of 32 vectors, or more where that gives over kStretches of them
    constexpr int kN = Reader<L>::kN;
    int shift = 5 + (kN == 8 ? 3 : 2);
    while (((a.vocab + kN - 1 + kN - 1) >> shift) + 1 > kStretches) ++shift;
    // few rows: more CTAs a row, while each has 4096 tokens or more
    int size = 1;
    while (size < 8 && static_cast<long long>(a.rows) * size * 2 <= 148 && a.vocab / (2 * size) >= 4096) size *= 2;
    const long long clusters = std::min<long long>(a.rows, std::max(1, 148 * 2 / size));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * size));
    cfg.blockDim = dim3(kT);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(row_kernel<L>),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, row_kernel<L>, a, size, shift);
    if (e != cudaSuccess) {
        set_error("token sampling: %s", cudaGetErrorString(e));
        return -1;
    }
    return launch_status("token sampling");
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
