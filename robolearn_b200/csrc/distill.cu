// Distillation of a head from a teacher's top logits: loss and gradient in one kernel.
//
//   q = softmax(t / T) over the k teacher entries that are there (index >= 0)
//   p = softmax(s / T) over all V logits of the student
//   row_loss = T^2 sum_k q_k (log q_k - log p[i_k])
//   loss     = c sum_n w_n row_loss_n
//   ds_j     = c w_n T (p_j - sum_{k: i_k = j} q_k) (* *grad_scale)
//
// A row is read from memory once and stays on the chip between its two passes (running maximum and
// sum of the softmax; gradient): in a warp's registers (up to 256 tokens, 1024 of fp32), in L1 behind a
// warp (up to 1024) or a CTA (up to 2048), and above that in shared memory and L2 (long_kernel). All sums
// are fp32; exponentials are the hardware's exp2 of s log2(e) / T less the same of the maximum, so every
// value is within a few units in the last place of fp32 times 1 + its argument.

#include "common.cuh"
#include "../../include/rl2.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <type_traits>

namespace rl2 {
namespace distill {

constexpr int kMaxTop = 1024;
constexpr int kMaxVocab = 1 << 30;  // a column plus a grid's stride stays below 2^31
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 2^x on the special-function unit (2 units in the last place; 2^-inf = 0)
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two fp32 operations in one instruction, each rounded as by itself
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
    return static_cast<unsigned long long>(__float_as_uint(hi)) << 32 | __float_as_uint(lo);
}
__device__ __forceinline__ float2 halves_of(unsigned long long x) {
    return make_float2(__uint_as_float(static_cast<uint32_t>(x)), __uint_as_float(static_cast<uint32_t>(x >> 32)));
}
__device__ __forceinline__ float2 fma_pair(float2 a, float b, float c) {
    unsigned long long y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(pair_of(a.x, a.y)), "l"(pair_of(b, b)), "l"(pair_of(c, c)));
    return halves_of(y);
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
    unsigned long long y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(pair_of(a.x, a.y)), "l"(pair_of(b.x, b.y)));
    return halves_of(y);
}
__device__ __forceinline__ float2 mul_pair(float2 a, float b) {
    unsigned long long y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(pair_of(a.x, a.y)), "l"(pair_of(b, b)));
    return halves_of(y);
}

// two values as one word of 16-bit elements, rounded to nearest
template <typename T>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t narrow2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t narrow2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
struct alignas(16) Pack {
    static constexpr int kN = 16 / sizeof(T);
    T v[kN];
};
template <typename G, int N>
struct alignas(N * sizeof(G)) Out {
    G v[N];
};

// running maximum (of the logits) and sum of 2^((s - max) scale)
struct Running {
    float max, sum;
};

__device__ __forceinline__ Running merge(Running a, Running b, float scale) {
    const float m = fmaxf(a.max, b.max);
    const float base = m == -INFINITY ? 0.0f : m;
    Running r;
    r.max = m;
    // a side without a finite maximum has sum 0, or NaN if it saw one
    r.sum = a.sum * (a.max == -INFINITY ? 1.0f : exp2_fast((a.max - base) * scale)) +
            b.sum * (b.max == -INFINITY ? 1.0f : exp2_fast((b.max - base) * scale));
    return r;
}

template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    if (THREADS == 32) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < THREADS / 32 ? red[lane] : 0.0f;
    return warp_sum(v);
}

template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* red) {
    v = warp_max(v);
    if (THREADS == 32) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    v = lane < THREADS / 32 ? red[lane] : -INFINITY;
    return warp_max(v);
}

__device__ __forceinline__ long long teacher_index(const rl2_distill_args& a, long long row, int k) {
    const long long at = row * a.ld_indices + k;
    return a.index_bits == 64 ? static_cast<const long long*>(a.teacher_indices)[at]
                              : static_cast<const int*>(a.teacher_indices)[at];
}

__device__ __forceinline__ float teacher_value(const rl2_distill_args& a, long long row, int k) {
    const long long at = row * a.ld_values + k;
    if (a.values_dtype == 0) return static_cast<const float*>(a.teacher_values)[at];
    if (a.values_dtype == 1) return __half2float(static_cast<const __half*>(a.teacher_values)[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher_values)[at]);
}

// Row's loss and gradient by a group of THREADS threads (a warp or a CTA) that reads the row where it lies.
// The arrays q_s and i_s hold the teacher's entries.
template <typename L, typename G, int THREADS>
__device__ __forceinline__ void row_by_group(const rl2_distill_args& a, long long row, int tid, float* red, float* red2, float* q_s,
                                             int* i_s) {
    constexpr int kN = Pack<L>::kN;
    auto sync = [] {
        if (THREADS == 32)
            __syncwarp();
        else
            __syncthreads();
    };
    const int V = a.vocab, K = a.top;
    const float scale = kLog2e / a.temperature;
    const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits;
    G* ds = a.dlogits ? static_cast<G*>(a.dlogits) + row * a.ld_dlogits : nullptr;
    const float weight = a.row_weight ? a.row_weight[row] : 1.0f;
    if (weight == 0.0f) {
        if (ds)
            for (int j = tid; j < V; j += THREADS) ds[j] = narrow<G>(0.0f);
        if (tid == 0) a.row_loss[row] = 0.0f;
        return;
    }
    // teacher
    float top = -INFINITY;
    bool bad = false;
    for (int k = tid; k < K; k += THREADS) {
        const long long i = teacher_index(a, row, k);
        const bool out = i >= V;
        bad |= out;
        const float v = i >= 0 && !out ? teacher_value(a, row, k) : -INFINITY;
        i_s[k] = i >= 0 && !out ? static_cast<int>(i) : -1;
        q_s[k] = v;
        top = fmaxf(top, v);
    }
    if (bad && a.health) atomicOr(a.health, kHealthIndex);
    top = block_max<THREADS>(top, red);
    float total = 0.0f;
    for (int k = tid; k < K; k += THREADS) {
        const float v = q_s[k];
        if (v != -INFINITY) total += exp2_fast((v - top) * scale);
    }
    total = block_sum<THREADS>(total, red);

    // student: running maximum and sum
    const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(s) % 16 / sizeof(L));
    const int head = min(V, mis ? kN - mis : 0);
    const int packs = (V - head) / kN;
    const int tail = head + packs * kN;
    Running r{-INFINITY, 0.0f};
    auto take = [&](float v) { r = merge(r, Running{v, v == -INFINITY ? 0.0f : (v == v ? 1.0f : v)}, scale); };
    for (int j = tid; j < head; j += THREADS) take(to_float(s[j]));
    for (int j = tail + tid; j < V; j += THREADS) take(to_float(s[j]));
    const Pack<L>* body = reinterpret_cast<const Pack<L>*>(s + head);
    for (int b = tid; b < packs; b += THREADS) {
        const Pack<L> x = body[b];
        float v[kN], m = r.max;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
            v[e] = to_float(x.v[e]);
            m = fmaxf(m, v[e]);
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float sum = r.max == -INFINITY ? r.sum : r.sum * exp2_fast((r.max - base) * scale);
#pragma unroll
        for (int e = 0; e < kN; ++e) sum += exp2_fast((v[e] - base) * scale);
        r.max = m;
        r.sum = sum;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1)
        r = merge(r, Running{__shfl_xor_sync(0xffffffffu, r.max, o), __shfl_xor_sync(0xffffffffu, r.sum, o)}, scale);
    if (THREADS > 32) {
        __syncthreads();
        if ((tid & 31) == 0) {
            red[tid >> 5] = r.max;
            red2[tid >> 5] = r.sum;
        }
        __syncthreads();
        r = Running{-INFINITY, 0.0f};
        for (int w = 0; w < THREADS / 32; ++w) r = merge(r, Running{red[w], red2[w]}, scale);
    }
    const float base = r.max == -INFINITY ? 0.0f : r.max;
    const bool some = total != 0.0f && r.sum != 0.0f;  // a teacher entry and a logit that are not -inf (NaN passes)

    // loss
    const float log_total = logf(total), log_sum = logf(r.sum);
    float loss = 0.0f;
    const float inv_total = 1.0f / total;
    for (int k = tid; k < K; k += THREADS) {
        const float v = q_s[k];
        const float z = (v - top) * scale;
        const float q = v == -INFINITY ? 0.0f : exp2_fast(z) * inv_total;
        if (some && q != 0.0f) loss += q * ((z * kLn2 - log_total) - ((to_float(s[i_s[k]]) - base) * scale * kLn2 - log_sum));
        q_s[k] = q;
    }
    loss = block_sum<THREADS>(loss, red);
    if (tid == 0) a.row_loss[row] = some ? a.temperature * (a.temperature * loss) : 0.0f;
    if (ds) {
        // gradient
        const float factor = weight * a.loss_weight * a.temperature * (a.grad_scale ? *a.grad_scale : 1.0f);
        const float p_factor = factor / r.sum;
        auto grad = [&](float v, float q) { return some ? exp2_fast((v - base) * scale) * p_factor - factor * q : 0.0f; };
        for (int j = tid; j < head; j += THREADS) ds[j] = narrow<G>(grad(to_float(s[j]), 0.0f));
        for (int j = tail + tid; j < V; j += THREADS) ds[j] = narrow<G>(grad(to_float(s[j]), 0.0f));
        using O = Out<G, sizeof(G) * kN <= 16 ? kN : 16 / sizeof(G)>;
        constexpr int kO = sizeof(O) / sizeof(G);
        const bool vec = reinterpret_cast<uintptr_t>(ds + head) % sizeof(O) == 0;
        for (int b = tid; b < packs; b += THREADS) {
            const Pack<L> x = body[b];
#pragma unroll
            for (int o = 0; o < kN / kO; ++o) {
                O out;
#pragma unroll
                for (int e = 0; e < kO; ++e) out.v[e] = narrow<G>(grad(to_float(x.v[o * kO + e]), 0.0f));
                G* at = ds + head + b * kN + o * kO;
                if (vec) {
                    *reinterpret_cast<O*>(at) = out;
                } else {
#pragma unroll
                    for (int e = 0; e < kO; ++e) at[e] = out.v[e];
                }
            }
        }
        sync();
        // the teacher's entries: the first entry of each token writes the token's gradient
        for (int k = tid; k < K; k += THREADS) {
            const int i = i_s[k];
            if (i < 0) continue;
            float q = 0.0f;
            bool first = true;
            for (int j = 0; j < K; ++j)
                if (i_s[j] == i) {
                    first &= j >= k;
                    q += q_s[j];
                }
            if (first) ds[i] = narrow<G>(grad(to_float(s[i]), q));
        }
    }
    sync();
}

// The total with a row added (one of weight 0 whatever its loss). The loss weight goes in first: a mean of large losses
// does not overflow on the way. A select and no branch, so that the loop's loads stay together (32768 rows: 8 us for 12).
__device__ __forceinline__ float with_row(float sum, const rl2_distill_args& a, float w, float loss) {
    return fmaf(a.loss_weight * w, w != 0.0f ? loss : 0.0f, sum);
}

// The last CTA to finish adds the rows' losses in a fixed order (all threads of the CTA).
__device__ __forceinline__ void finish(const rl2_distill_args& a) {
    __shared__ bool last;
    __shared__ float part[32];
    if (!a.loss_out) return;
    const int tid = threadIdx.x, threads = blockDim.x;
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(a.counter, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    float sum = 0.0f;
#pragma unroll 8
    for (int n = tid; n < a.rows; n += threads) {
        const float w = a.row_weight ? a.row_weight[n] : 1.0f, loss = __ldcg(a.row_loss + n);
        sum = with_row(sum, a, w, loss);
    }
    sum = warp_sum(sum);
    if ((tid & 31) == 0) part[tid >> 5] = sum;
    __syncthreads();
    if (tid < 32) {
        sum = warp_sum(tid < threads / 32 ? part[tid] : 0.0f);
        if (tid == 0) {
            *a.loss_out = sum;
            *a.counter = 0;
        }
    }
}

// Up to kFewTop teacher entries and 1024 tokens: a warp per row, N tokens a lane in registers (pairs 64 tokens apart),
// read once; the exponentials of the sum are the gradient's. The row's loads and the teacher's are on their way
// together. 25 us at 32768 x 101 fp32 (48 with the row read twice through L1), 9 us a call at 512 x 101.
constexpr int kRowWarps = 4;
constexpr int kFewTop = 256;

__device__ __forceinline__ float2 load_pair(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load_pair(const __half* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 load_pair(const __nv_bfloat16* p) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

template <typename L, typename G, int N>
__device__ __forceinline__ void row_by_warp(const rl2_distill_args& a, long long row, int lane, float* q_s, int* i_s) {
    const int V = a.vocab, K = a.top;
    const float scale = kLog2e / a.temperature;
    const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits;
    G* ds = a.dlogits ? static_cast<G*>(a.dlogits) + row * a.ld_dlogits : nullptr;
    const float weight = a.row_weight ? a.row_weight[row] : 1.0f;
    if (weight == 0.0f) {
        if (ds)
            for (int j = lane; j < V; j += 32) ds[j] = narrow<G>(0.0f);
        if (lane == 0) a.row_loss[row] = 0.0f;
        return;
    }
    float v[N];
    const bool pairs = reinterpret_cast<uintptr_t>(s) % (2 * sizeof(L)) == 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const int j = i * 32 + lane * 2;
        if (pairs && j + 1 < V) {
            const float2 x = load_pair(s + j);
            v[i] = x.x, v[i + 1] = x.y;
        } else {
            v[i] = j < V ? to_float(s[j]) : -INFINITY;
            v[i + 1] = j + 1 < V ? to_float(s[j + 1]) : -INFINITY;
        }
    }
    // teacher
    float top = -INFINITY;
    bool bad = false;
    for (int k = lane; k < K; k += 32) {
        const long long i = teacher_index(a, row, k);
        const bool out = i >= V;
        bad |= out;
        const float given = teacher_value(a, row, k);
        const float t = i >= 0 && !out ? given : -INFINITY;
        i_s[k] = i >= 0 && !out ? static_cast<int>(i) : -1;
        q_s[k] = t;
        top = fmaxf(top, t);
    }
    if (bad && a.health) atomicOr(a.health, kHealthIndex);
    top = warp_max(top);
    float total = 0.0f;
    for (int k = lane; k < K; k += 32) {
        const float t = q_s[k];
        if (t != -INFINITY) total += exp2_fast((t - top) * scale);
    }
    // student
    float base = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) base = fmaxf(base, v[i]);
    base = warp_max(base);
    if (!(base > -INFINITY)) base = 0.0f;  // none, or NaN alone
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = exp2_fast((v[i] - base) * scale);
        sum += v[i];
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const bool some = total != 0.0f && sum != 0.0f;  // a teacher entry and a logit that are not -inf (NaN passes)
    const float factor = weight * a.loss_weight * a.temperature * (a.grad_scale ? *a.grad_scale : 1.0f);
    const float p_factor = factor / sum;
    if (ds) {
        const bool whole = reinterpret_cast<uintptr_t>(ds) % (2 * sizeof(G)) == 0;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const int j = i * 32 + lane * 2;
            const float x = some ? v[i] * p_factor : 0.0f, y = some ? v[i + 1] * p_factor : 0.0f;
            if (whole && j + 1 < V) {
                if constexpr (sizeof(G) == 4)
                    *reinterpret_cast<float2*>(ds + j) = make_float2(x, y);
                else
                    *reinterpret_cast<uint32_t*>(ds + j) = narrow2<G>(x, y);
            } else {
                if (j < V) ds[j] = narrow<G>(x);
                if (j + 1 < V) ds[j + 1] = narrow<G>(y);
            }
        }
    }
    // the teacher's entries: loss, and the gradient of each token by its first entry
    const float log_total = logf(total), log_sum = logf(sum), inv_total = 1.0f / total;
    auto share = [&](float t) { return t == -INFINITY ? 0.0f : exp2_fast((t - top) * scale) * inv_total; };
    float loss = 0.0f;
    __syncwarp();  // q_s and i_s are whole, the gradients are written
    for (int k0 = 0; k0 < K; k0 += 32) {
        const int k = k0 + lane, i = k < K ? i_s[k] : -1;
        // other entries of this token: among 32 by a match, among more by a count
        int same = __popc(__match_any_sync(0xffffffffu, i));
        if (K > 32) {
            same = 0;
#pragma unroll 4
            for (int j = 0; j < K; ++j) same += i_s[j] == i;
        }
        if (i < 0) continue;
        const float t = q_s[k], z = (to_float(s[i]) - base) * scale, q = share(t);
        if (some && q != 0.0f) loss += q * (((t - top) * scale * kLn2 - log_total) - (z * kLn2 - log_sum));
        if (!ds) continue;
        float all = q;
        bool first = true;
        if (same > 1) {
            all = 0.0f;
            for (int j = 0; j < K; ++j)
                if (i_s[j] == i) {
                    first &= j >= k;
                    all += share(q_s[j]);
                }
        }
        if (first) ds[i] = narrow<G>(some ? exp2_fast(z) * p_factor - factor * all : 0.0f);
    }
    loss = warp_sum(loss);
    if (lane == 0) a.row_loss[row] = some ? a.temperature * (a.temperature * loss) : 0.0f;
    __syncwarp();  // q_s and i_s are the next row's
}

// N = 0: the row stays in L1 instead
template <typename L, typename G, int N>
__global__ void __launch_bounds__(32 * kRowWarps) warp_kernel(const rl2_distill_args a) {
    __shared__ float q_s[kRowWarps][kFewTop];
    __shared__ int i_s[kRowWarps][kFewTop];
    const int warp = threadIdx.x >> 5;
    ptx::grid_release();
    ptx::grid_wait();
    for (long long row = static_cast<long long>(blockIdx.x) * kRowWarps + warp; row < a.rows;
         row += static_cast<long long>(gridDim.x) * kRowWarps)
        if constexpr (N > 0)
            row_by_warp<L, G, N>(a, row, threadIdx.x & 31, q_s[warp], i_s[warp]);
        else
            row_by_group<L, G, 32>(a, row, threadIdx.x & 31, nullptr, nullptr, q_s[warp], i_s[warp]);
    finish(a);
}

// A CTA per row.
template <typename L, typename G, int THREADS>
__global__ void __launch_bounds__(THREADS) row_kernel(const rl2_distill_args a) {
    __shared__ float red[32], red2[32];
    __shared__ float q_s[kMaxTop];
    __shared__ int i_s[kMaxTop];
    ptx::grid_release();
    ptx::grid_wait();
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x)
        row_by_group<L, G, THREADS>(a, row, threadIdx.x, red, red2, q_s, i_s);
    finish(a);
}

// ---- long rows: a CTA each, or with few rows a cluster of CTAs ---------------------------
//
// T threads read the row (of a cluster: each CTA its part) four vectors each at a time, the next four on their way,
// and keep the first eight in shared memory; the second pass takes those from there and the rest from L2, the last read
// first. 1024 threads an SM, so that one row's reading goes along with another's writing: 512 a CTA for the longest rows
// and for few of them, fewer for shorter ones, whose barriers and first loads weigh more (4096 x 4096 bf16: 77 us with
// 512, 40 with 256, 26 with 128; 2048 x 50257 bf16: 104, 87, 98; 2047 x 128257 bf16: 214, 241). What bounds it is DRAM:
// 1.05 GB in 214 us at 2047 x 128257 bf16 (4.9 TB/s; 224 in a row of calls on other inputs each); the second pass misses
// L2 for 0.12 of the row. 246 us when it read forward and kept nothing.
// Slower there: rows held in registers by clusters of four CTAs (389 us), rows streamed through a ring in
// shared memory by bulk copies (308 us), both waiting for one another at each row.
//
// The CTAs of a cluster exchange their maxima and sums through shared memory. The teacher's entries are a
// thread's each: their loads and their softmax go along with the row's. The first entry of each token writes the
// token's gradient over what the second pass wrote. The few elements of a row outside its 16-byte vectors are
// one thread's each.
//
// The passes use the offset o = max log2(e) / T: p = 2^(s c - o) / sum needs one multiply-add and one exp2 an
// element. o is rounded, the product in the multiply-add is not, so every exponent carries the same error of up to
// half a unit in o's last place, which the division by the sum takes out as long as 2 to that error is an ordinary
// number: while |o| < 2^24 it is at most a factor of sqrt 2. Rows whose maximum lies outside (a mask's large finite fill; no
// logit that is not -inf), or with NaN, are done again from (s - max) c.

constexpr int kLongThreads = 1024;  // of an SM, in CTAs of T
constexpr int kMaxCluster = 8;
constexpr int kHeld = 4;                      // vectors a thread has in registers
constexpr int kSteps = 2;                     // times that, a thread, are kept in shared memory
constexpr float kTame = 16777216.0f;  // 2^24

template <int WARPS>
struct Meeting {
    uint64_t met[2];
    float2 meet[2][kMaxCluster];
    float top[2][WARPS], sum[2][WARPS];
    Running teacher[WARPS];
    float loss[WARPS];
};

// mbarrier that other CTAs of the cluster arrive on; bounded to 4 s (then the timeout bit of *health)
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t phase, int* health) {
    auto done = [&] {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(ptx::smem_u32(bar)), "r"(phase) : "memory");
        return ok != 0;
    };
    if (done()) return true;
    uint64_t start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    for (uint32_t i = 1;; ++i) {
        if (done()) return true;
        if ((i & 1023u) == 0) {
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (now - start > 4000000000ull) {
                if (health) atomicOr(health, kHealthTimeout);
                return false;
            }
        }
    }
}

// A row's 16-byte vectors and the slice of them that this CTA holds.
template <typename L>
struct Slice {
    static constexpr int kN = 16 / sizeof(L);
    const L* s;
    int head, vectors, tail;  // elements before the first vector, vectors, first element after them
    int from, count;

    __device__ __forceinline__ Slice(const rl2_distill_args& a, long long row, uint32_t rank, uint32_t size) {
        s = static_cast<const L*>(a.logits) + row * a.ld_logits;
        const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(s) % 16 / sizeof(L));
        head = min(a.vocab, mis ? kN - mis : 0);
        vectors = (a.vocab - head) / kN;
        tail = head + vectors * kN;
        const int shift = 31 - __clz(size);  // a power of two
        from = static_cast<int>(static_cast<unsigned long long>(vectors) * rank >> shift);
        count = static_cast<int>(static_cast<unsigned long long>(vectors) * (rank + 1) >> shift) - from;
    }
};

__device__ __forceinline__ void unpack_as(uint4 x, float (&v)[4], float) {
    v[0] = __uint_as_float(x.x), v[1] = __uint_as_float(x.y), v[2] = __uint_as_float(x.z), v[3] = __uint_as_float(x.w);
}
__device__ __forceinline__ void unpack_as(uint4 x, float (&v)[8], __half) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack_as(uint4 x, float (&v)[8], __nv_bfloat16) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) v[2 * k] = __uint_as_float(w[k] << 16), v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
}
// a vector of -inf
__device__ __forceinline__ uint4 nothing(float) { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }
__device__ __forceinline__ uint4 nothing(__half) { return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
__device__ __forceinline__ uint4 nothing(__nv_bfloat16) { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }

template <typename L>
__device__ __forceinline__ void unpack(uint4 x, float (&v)[16 / sizeof(L)]) {
    unpack_as(x, v, L(0.0f));
}
// maximum of a vector's elements, NaN left out
__device__ __forceinline__ float most_as(uint4, const float (&v)[4], float) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); }
__device__ __forceinline__ float most_as(uint4 x, const float (&)[8], __half) {
    const __half2* h = reinterpret_cast<const __half2*>(&x);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float most_as(uint4 x, const float (&)[8], __nv_bfloat16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&x);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}

// N values to an address aligned to N elements (16 bytes where they are more)
template <typename G, int N>
__device__ __forceinline__ void store_vector(G* to, const float (&y)[N]) {
    if constexpr (sizeof(G) == 4) {
#pragma unroll
        for (int e = 0; e < N; e += 4) __stcs(reinterpret_cast<float4*>(to + e), make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]));
    } else if constexpr (N == 8) {
        __stcs(reinterpret_cast<uint4*>(to), make_uint4(narrow2<G>(y[0], y[1]), narrow2<G>(y[2], y[3]), narrow2<G>(y[4], y[5]), narrow2<G>(y[6], y[7])));
    } else {
        __stcs(reinterpret_cast<uint2*>(to), make_uint2(narrow2<G>(y[0], y[1]), narrow2<G>(y[2], y[3])));
    }
}

template <typename L, typename G, int T>
__global__ void __launch_bounds__(T, kLongThreads / T) long_kernel(const rl2_distill_args a, const int size) {
    extern __shared__ __align__(16) uint8_t raw[];  // the row's first vectors; the teacher's entries
    constexpr int kWarps = T / 32, kKept = kSteps * kHeld * T;
    __shared__ Meeting<kWarps> sh;
    constexpr int kN = Slice<L>::kN;
    uint4* kept = reinterpret_cast<uint4*>(raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = size > 1 ? ptx::cluster_rank() : 0u;
    const long long row = blockIdx.x / size;
    const Slice<L> in(a, row, rank, size);
    const int K = a.top, padded = (K + 3) / 4 * 4;
    int* token = reinterpret_cast<int*>(kept + kKept);         // -1: absent
    float* given = reinterpret_cast<float*>(token + padded);   // the teacher's value
    const float scale = kLog2e / a.temperature;
    ptx::grid_release();
    ptx::grid_wait();
    const float weight = a.row_weight ? a.row_weight[row] : 1.0f;
    G* ds = a.dlogits ? static_cast<G*>(a.dlogits) + row * a.ld_dlogits : nullptr;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) ptx::mbar_init(&sh.met[i], size);
        ptx::fence_barrier_init();
    }
    // this thread's vectors, and its element outside them
    uint4 x[kHeld];
    const uint4* data = reinterpret_cast<const uint4*>(in.s + in.head) + in.from + tid;
    auto load = [&](uint4 (&to)[kHeld], int first) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            to[k] = first + k * T + tid < in.count ? ptx::load_vector(data + first + k * T) : nothing(L(0.0f));
    };
    // the second pass's: from shared memory where the first kept them
    auto load_again = [&](uint4 (&to)[kHeld], int first) {
        if (first < 0) return;
        if (first < kKept) {
#pragma unroll
            for (int k = 0; k < kHeld; ++k) to[k] = kept[first + k * T + tid];
        } else {
            load(to, first);
        }
    };
    load(x, 0);
    const bool has_edge = rank == 0 && tid < in.head + (a.vocab - in.tail);
    const int edge_at = tid < in.head ? tid : in.tail + tid - in.head;
    const float edge = has_edge ? to_float(in.s[edge_at]) : -INFINITY;
    // the teacher: its softmax as a running one
    Running teacher{-INFINITY, 0.0f};
    for (int k = tid; k < padded; k += T) {
        const long long i = k < K ? teacher_index(a, row, k) : -1;
        if (i >= a.vocab && weight != 0.0f && a.health) atomicOr(a.health, kHealthIndex);
        const bool here = i >= 0 && i < a.vocab;
        const float v = here ? teacher_value(a, row, k) : -INFINITY;
        token[k] = here ? static_cast<int>(i) : -1;
        given[k] = v;
        teacher = merge(teacher, Running{v, v == -INFINITY ? 0.0f : (v == v ? 1.0f : v)}, scale);
    }
    if (warp * 32 < K) {
#pragma unroll
        for (int o = 16; o; o >>= 1)
            teacher = merge(teacher, Running{__shfl_xor_sync(0xffffffffu, teacher.max, o), __shfl_xor_sync(0xffffffffu, teacher.sum, o)}, scale);
    }
    if (lane == 0) sh.teacher[warp] = teacher;
    if (weight == 0.0f) {
        const int lo = rank == 0 ? 0 : in.head + in.from * kN, hi = static_cast<int>(rank) == size - 1 ? a.vocab : in.head + (in.from + in.count) * kN;
        if (ds)
            for (int j = lo + tid; j < hi; j += T) ds[j] = narrow<G>(0.0f);
        if (tid == 0 && rank == 0) a.row_loss[row] = 0.0f;
        return;
    }
    if (size > 1) ptx::cluster_sync();  // the peers' barriers exist
    const float factor = weight * a.loss_weight * a.temperature * (a.grad_scale ? *a.grad_scale : 1.0f);
    int meeting = 0;
    // over the CTA, then the cluster: a maximum and the sum (unless `plain`, relative to it as powers of two)
    auto meet = [&](float top, float sum, bool plain) {
        auto relative = [&](float t, float all) { return plain ? 1.0f : exp2_fast(t - all); };
        float all = warp_max(top);
        sum = warp_sum(sum * relative(top, all));
        const int buf = meeting & 1;
        if (lane == 0) {
            sh.top[buf][warp] = all;
            sh.sum[buf][warp] = sum;
        }
        __syncthreads();
        top = sh.top[buf][lane % kWarps];
        all = warp_max(top);
        sum = warp_sum(lane < kWarps ? sh.sum[buf][lane % kWarps] * relative(top, all) : 0.0f);
        if (size > 1) {
            if (warp == 0 && lane < size) {
                const uint32_t to = ptx::cluster_addr(&sh.meet[buf][rank], lane);
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(all), "f"(sum) : "memory");
                ptx::mbar_arrive_cluster(ptx::cluster_addr(&sh.met[buf], lane));
            }
            wait_bar(&sh.met[buf], (meeting >> 1) & 1, a.health);
            const float2 y = sh.meet[buf][lane & (size - 1)];
            all = warp_max(y.x);
            sum = warp_sum(lane < size ? y.y * relative(y.x, all) : 0.0f);
        }
        ++meeting;
        return make_float2(all, sum);
    };
    // ---- first pass ----
    float o = fmaxf(edge * scale, -kTame);
    float sum = exp2_fast(fmaf(edge, scale, -o));  // 0 without one (-inf)
    for (int first = 0;;) {
        const int after = first + kHeld * T;
        uint4 next[kHeld];
        load(next, after);  // on its way while this is worked on
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            float v[kN];
            unpack<L>(x[k], v);
            m = fmaxf(m, most_as(x[k], v, L(0.0f)));
        }
        const float up = fmaxf(o, m * scale);
        sum *= exp2_fast(o - up);
        o = up;
        float2 part = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            float v[kN];
            unpack<L>(x[k], v);
#pragma unroll
            for (int e = 0; e < kN; e += 2) {
                const float2 z = fma_pair(make_float2(v[e], v[e + 1]), scale, -o);
                part = add_pair(part, make_float2(exp2_fast(z.x), exp2_fast(z.y)));
            }
        }
        sum += part.x + part.y;
        if (first < kKept) {
#pragma unroll
            for (int k = 0; k < kHeld; ++k) kept[first + k * T + tid] = x[k];
        }
        first = after;
        if (first >= in.count) break;
#pragma unroll
        for (int k = 0; k < kHeld; ++k) x[k] = next[k];
    }
    // the student's logit of this thread's teacher entry
    const int own_token = tid < K ? token[tid] : -1;
    const float own = own_token >= 0 ? to_float(in.s[own_token]) : 0.0f;
    const float2 whole = meet(o, sum, false);
    o = whole.x;
    sum = whole.y;
    teacher = sh.teacher[lane % kWarps];
#pragma unroll
    for (int w = kWarps / 2; w; w >>= 1)
        teacher = merge(teacher, Running{__shfl_xor_sync(0xffffffffu, teacher.max, w), __shfl_xor_sync(0xffffffffu, teacher.sum, w)}, scale);
    float base = 0.0f;
    const bool tame = fabsf(o) < kTame && sum > 0.0f;  // at -kTame nothing is above it
    if (!tame) {  // from (s - max) c
        auto each = [&](auto&& f) {
            if (has_edge) f(edge);
            for (int first = 0; first < in.count; first += kHeld * T) {
                load_again(x, first);
#pragma unroll
                for (int k = 0; k < kHeld; ++k) {
                    if (first + k * T + tid >= in.count) continue;
                    float v[kN];
                    unpack<L>(x[k], v);
#pragma unroll
                    for (int e = 0; e < kN; ++e) f(v[e]);
                }
            }
        };
        float m = -INFINITY;
        each([&](float v) { m = fmaxf(m, v); });
        base = meet(m, 0.0f, true).x;
        if (base == -INFINITY) base = 0.0f;
        sum = 0.0f;
        each([&](float v) { sum += exp2_fast((v - base) * scale); });
        sum = meet(0.0f, sum, true).y;
    }
    const bool some = teacher.sum != 0.0f && sum != 0.0f;  // a teacher entry and a logit that are not -inf (NaN passes)
    const float f = factor / sum;
    auto grad = [&](float v) {
        if (tame) return exp2_fast(fmaf(v, scale, -o)) * f;
        return exp2_fast((v - base) * scale) * f;
    };
    // ---- second pass ----
    if (ds) {
        if (has_edge) ds[edge_at] = narrow<G>(some ? grad(edge) : 0.0f);
        G* out = ds + in.head + (static_cast<long long>(in.from) + tid) * kN;
        const bool vec = reinterpret_cast<uintptr_t>(out) % (sizeof(G) * kN <= 16 ? sizeof(G) * kN : 16) == 0;
        auto write = [&](auto is_plain) {
            // the last read first: they are the likeliest still in L2
            const int last = in.count > 0 ? (in.count - 1) / (kHeld * T) * (kHeld * T) : -1;
            load_again(x, last);
            for (int first = last; first >= 0; first -= kHeld * T) {
                uint4 next[kHeld];
                load_again(next, first - kHeld * T);
#pragma unroll
                for (int k = 0; k < kHeld; ++k) {
                    float v[kN];
                    unpack<L>(x[k], v);
#pragma unroll
                    for (int e = 0; e < kN; e += 2) {
                        if (decltype(is_plain)::value) {
                            const float2 z = fma_pair(make_float2(v[e], v[e + 1]), scale, -o);
                            const float2 y = mul_pair(make_float2(exp2_fast(z.x), exp2_fast(z.y)), f);
                            v[e] = y.x, v[e + 1] = y.y;
                        } else {
                            v[e] = some ? grad(v[e]) : 0.0f;
                            v[e + 1] = some ? grad(v[e + 1]) : 0.0f;
                        }
                    }
                    if (first + k * T + tid >= in.count) break;
                    G* to = out + (first + k * T) * static_cast<long long>(kN);
                    if (vec) {
                        store_vector<G, kN>(to, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < kN; ++e) to[e] = narrow<G>(v[e]);
                    }
                }
#pragma unroll
                for (int k = 0; k < kHeld; ++k) x[k] = next[k];
            }
        };
        if (tame && some)
            write(std::true_type{});
        else
            write(std::false_type{});
    }
    __syncthreads();
    // ---- the teacher's entries: loss, and the gradient of the tokens of this CTA's part of the row ----
    const float inverse = 1.0f / teacher.sum, log_total = logf(teacher.sum), log_sum = logf(sum);
    auto share = [&](int k) { return given[k] == -INFINITY ? 0.0f : exp2_fast((given[k] - teacher.max) * scale) * inverse; };
    const int lo = rank == 0 ? 0 : in.head + in.from * kN, hi = in.head + (in.from + in.count) * kN;
    float loss = 0.0f;
    if (some) {
        for (int k = tid; k < K; k += T) {
            const int i = token[k];
            const float s = k == tid || i < 0 ? own : to_float(in.s[i]);
            float q = share(k);
            if (rank == 0 && q != 0.0f)
                loss += q * (((given[k] - teacher.max) * scale * kLn2 - log_total) -
                             ((tame ? fmaf(s, scale, -o) : (s - base) * scale) * kLn2 - log_sum));
            if (!ds || i < 0 || !((i >= lo && i < hi) || (rank == 0 && i >= in.tail))) continue;
            int same = 0;
#pragma unroll 4
            for (int j = 0; j < padded; j += 4) {
                const int4 t = *reinterpret_cast<const int4*>(token + j);
                same += (t.x == i) + (t.y == i) + (t.z == i) + (t.w == i);
            }
            bool first = true;
            if (same > 1) {
                q = 0.0f;
                for (int j = 0; j < K; ++j)
                    if (token[j] == i) {
                        first &= j >= k;
                        q += share(j);
                    }
            }
            if (first) ds[i] = narrow<G>(grad(s) - factor * q);
        }
    }
    if (rank == 0) {
        loss = warp_sum(loss);
        if (lane == 0) sh.loss[warp] = loss;
        __syncthreads();
        if (warp == 0) {
            loss = warp_sum(lane < kWarps ? sh.loss[lane] : 0.0f);
            if (lane == 0) a.row_loss[row] = some ? a.temperature * (a.temperature * loss) : 0.0f;
        }
    }
}

// The total of long rows, in a fixed order, by one CTA of a launch of its own: a ticket and a fence at the end of
// every CTA of long_kernel cost 14 us at 2047 rows of 128257, this 3 us.
__global__ void __launch_bounds__(1024) total_kernel(const rl2_distill_args a) {
    __shared__ float part[32];
    const int tid = threadIdx.x;
    float sum = 0.0f;
    ptx::grid_release();
    ptx::grid_wait();
#pragma unroll 4
    for (int n = tid; n < a.rows; n += 1024) {
        const float w = a.row_weight ? a.row_weight[n] : 1.0f, loss = a.row_loss[n];
        sum = with_row(sum, a, w, loss);
    }
    sum = warp_sum(sum);
    if ((tid & 31) == 0) part[tid >> 5] = sum;
    __syncthreads();
    if (tid < 32) {
        sum = warp_sum(part[tid]);
        if (tid == 0) *a.loss_out = sum;
    }
}

int launched(cudaError_t e) {
    if (e == cudaSuccess) return launch_status("distillation");
    set_error("distillation: %s", cudaGetErrorString(e));
    return -1;
}

template <typename L, typename G, int T>
int launch_long(const rl2_distill_args& a, cudaStream_t stream) {
    // few rows: more CTAs a row, while each has four vectors a thread
    constexpr int kResident = 148 * (kLongThreads / T);
    int size = 1;
    while (size < kMaxCluster && static_cast<long long>(a.rows) * size * 2 <= kResident && a.vocab / Slice<L>::kN / (size * 2) >= kHeld * T)
        size *= 2;
    constexpr int kMost = kSteps * kHeld * T * 16 + kMaxTop * 8;
    const size_t smem = kMost - (kMaxTop - (a.top + 3) / 4 * 4) * 8;
    static std::atomic<unsigned long long> allowed{0};  // devices (up to 64) whose limit is raised
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && (device > 63 || !(allowed.load() >> device & 1))) {
        e = cudaFuncSetAttribute(reinterpret_cast<const void*>(long_kernel<L, G, T>), cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (e == cudaSuccess && device <= 63) allowed.fetch_or(1ull << device);
    }
    if (e == cudaSuccess)
        e = launch_early_clusters(long_kernel<L, G, T>, size, static_cast<unsigned>(static_cast<long long>(a.rows) * size), T, smem, stream, a, size);
    if (e == cudaSuccess && a.loss_out) e = launch_early(total_kernel, 1, 1024, 0, stream, a);
    return launched(e);
}

template <typename L, typename G>
int launch(const rl2_distill_args& a, cudaStream_t stream) {
    if (a.vocab > 2048) {
        // more and smaller CTAs while the rows under way stay in L2 (148 x 4 of 140 KB, read and written), a row gives
        // every thread work in each step, and the teacher has at most an entry a thread
        const long long bytes = a.vocab * static_cast<long long>(sizeof(L));
        const bool many = a.rows > 148 * 2;
        if (many && bytes <= 48 << 10 && a.top <= 128) return launch_long<L, G, 128>(a, stream);
        if (many && bytes <= 140000 && a.top <= 256) return launch_long<L, G, 256>(a, stream);
        return launch_long<L, G, 512>(a, stream);
    }
    // short rows: the total by the last CTA, or with many rows (whose losses one small CTA takes long to add: 22 us
    // for 6 + 3 at 4096 x 101) by a launch of its own
    rl2_distill_args each = a;
    cudaError_t e;
    if (a.rows > 1024) each.loss_out = nullptr;
    if (a.vocab <= 1024 && a.top <= kFewTop) {
        // registers up to 256 tokens, and up to 1024 of fp32 (8192 x 1024: 23 us for 28 with the row in L1; of 16 bits,
        // whose rows L1 takes in 16-byte vectors, 50 for 23, and 32768 x 256 35 for 46)
        constexpr int kMid = sizeof(L) == 4 ? 16 : 0, kWide = sizeof(L) == 4 ? 32 : 0;
        const auto kernel = a.vocab <= 128 ? warp_kernel<L, G, 4> : a.vocab <= 256 ? warp_kernel<L, G, 8>
                          : a.vocab <= 512 ? warp_kernel<L, G, kMid> : warp_kernel<L, G, kWide>;
        const long long blocks = (static_cast<long long>(a.rows) + kRowWarps - 1) / kRowWarps;
        e = launch_early(kernel, static_cast<unsigned>(blocks), 32 * kRowWarps, 0, stream, each);
    } else {
        e = launch_early(row_kernel<L, G, 128>, std::min(a.rows, 148 * 16), 128, 0, stream, each);
    }
    if (e == cudaSuccess && a.loss_out && !each.loss_out) e = launch_early(total_kernel, 1, 1024, 0, stream, a);
    return launched(e);
}

template <typename L>
int launch_for(const rl2_distill_args& a, cudaStream_t stream) {
    if (a.dlogits_dtype == 0) return launch<L, float>(a, stream);
    if (a.dlogits_dtype == 1) return launch<L, __half>(a, stream);
    return launch<L, __nv_bfloat16>(a, stream);
}

}  // namespace distill
}  // namespace rl2

extern "C" int rl2_distill_topk(const rl2_distill_args* a, void* stream) {
    using namespace rl2;
    using namespace rl2::distill;
    clear_error();
    if (!a) {
        set_error("distillation: null arguments");
        return -1;
    }
    if (a->rows < 0 || a->vocab < 1 || a->vocab > kMaxVocab || a->top < 1 || a->top > kMaxTop) {
        set_error("distillation: rows >= 0, vocab >= 1 (up to 2^30) and 1..%d teacher entries are needed", kMaxTop);
        return -1;
    }
    const int esize[3] = {4, 2, 2};
    for (int d : {a->logits_dtype, a->values_dtype, a->dlogits_dtype})
        if (d < 0 || d > 2) {
            set_error("distillation: types are 0 (fp32), 1 (fp16) or 2 (bf16)");
            return -1;
        }
    if (a->index_bits != 32 && a->index_bits != 64) {
        set_error("distillation: teacher indices have 32 or 64 bits");
        return -1;
    }
    if (!(a->temperature > 0.0f) || a->temperature > 1e30f || kLog2e / a->temperature > FLT_MAX) {
        set_error("distillation: the temperature must be positive and finite, and so must its reciprocal");
        return -1;
    }
    if (a->loss_out && !a->counter) {
        set_error("distillation: the total loss needs the counter");
        return -1;
    }
    if (a->rows == 0) {
        if (a->loss_out && cudaMemsetAsync(a->loss_out, 0, sizeof(float), as_stream(stream)) != cudaSuccess) {
            set_error("distillation: clearing the loss failed");
            return -1;
        }
        return 0;
    }
    if (!a->logits || !a->teacher_values || !a->teacher_indices || !a->row_loss) {
        set_error("distillation: logits, teacher values and indices and row_loss must be non-null");
        return -1;
    }
    if (a->ld_logits < a->vocab || (a->dlogits && a->ld_dlogits < a->vocab)) {
        set_error("distillation: a row stride is shorter than its row");
        return -1;
    }
    auto extent = [&](const void* base, long long ld, int size) {
        return Extent{base, a->rows, static_cast<long long>(a->vocab) * size, ld * size};
    };
    if (overlap(extent(a->logits, a->ld_logits, esize[a->logits_dtype]), extent(a->dlogits, a->ld_dlogits, esize[a->dlogits_dtype]))) {
        set_error("distillation: the gradient may not overwrite the logits");
        return -1;
    }
    if (a->ld_values < a->top || a->ld_indices < a->top) {
        set_error("distillation: a row stride is shorter than its row");
        return -1;
    }
    if (!aligned(a->logits, esize[a->logits_dtype]) || !aligned(a->teacher_values, esize[a->values_dtype]) ||
        !aligned(a->teacher_indices, a->index_bits / 8) || !aligned(a->dlogits, esize[a->dlogits_dtype])) {
        set_error("distillation: a matrix is not aligned to its element");
        return -1;
    }
    if (a->logits_dtype == 0) return launch_for<float>(*a, as_stream(stream));
    if (a->logits_dtype == 1) return launch_for<__half>(*a, as_stream(stream));
    return launch_for<__nv_bfloat16>(*a, as_stream(stream));
}
