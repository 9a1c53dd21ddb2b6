// Distillation of a head from a teacher's top logits: loss and gradient in one kernel.
//
//   q = softmax(t / T) over the k teacher entries that are there (index >= 0)
//   p = softmax(s / T) over all V logits of the student
//   row_loss = T^2 sum_k q_k (log q_k - log p[i_k])
//   loss     = c sum_n w_n row_loss_n
//   ds_j     = c w_n T (p_j - sum_{k: i_k = j} q_k) (* *grad_scale)
//
// A row is read from memory once and stays on the chip between its two passes (running maximum and
// sum of the softmax; gradient): in a warp's registers up to 1024 tokens, in L1 / L2 behind a CTA up to
// 8192, and above that in the shared memory of a CTA or of a cluster of CTAs (stream_kernel). All sums
// are fp32; exponentials are the hardware's exp2 of s log2(e) / T less the same of the maximum, so every
// value is within a few units in the last place of fp32 times 1 + its argument.

#include "common.cuh"
#include "../../include/rl2.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace rl2 {
namespace distill {

constexpr int kMaxTop = 1024;
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
    if (tid == 0) a.row_loss[row] = some ? a.temperature * a.temperature * loss : 0.0f;
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
    for (int n = tid; n < a.rows; n += threads) {
        const float w = a.row_weight ? a.row_weight[n] : 1.0f;
        if (w != 0.0f) sum += w * __ldcg(a.row_loss + n);
    }
    sum = warp_sum(sum);
    if ((tid & 31) == 0) part[tid >> 5] = sum;
    __syncthreads();
    if (tid < 32) {
        sum = warp_sum(tid < threads / 32 ? part[tid] : 0.0f);
        if (tid == 0) {
            *a.loss_out = a.loss_weight * sum;
            *a.counter = 0;
        }
    }
}

// Up to kFewTop teacher entries and 1024 tokens: a warp per row.
constexpr int kRowWarps = 4;
constexpr int kFewTop = 256;

template <typename L, typename G>
__global__ void __launch_bounds__(32 * kRowWarps) warp_kernel(const rl2_distill_args a) {
    __shared__ float q_s[kRowWarps][kFewTop];
    __shared__ int i_s[kRowWarps][kFewTop];
    const int warp = threadIdx.x >> 5;
    for (long long row = static_cast<long long>(blockIdx.x) * kRowWarps + warp; row < a.rows;
         row += static_cast<long long>(gridDim.x) * kRowWarps)
        row_by_group<L, G, 32>(a, row, threadIdx.x & 31, nullptr, nullptr, q_s[warp], i_s[warp]);
    finish(a);
}

// A CTA per row.
template <typename L, typename G, int THREADS>
__global__ void __launch_bounds__(THREADS) row_kernel(const rl2_distill_args a) {
    __shared__ float red[32], red2[32];
    __shared__ float q_s[kMaxTop];
    __shared__ int i_s[kMaxTop];
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x)
        row_by_group<L, G, THREADS>(a, row, threadIdx.x, red, red2, q_s, i_s);
    finish(a);
}

// ---- long rows: streamed through shared memory -------------------------------------------
//
// A cluster of CTAs holds a row, each CTA a slice of its 16-byte vectors, in a ring of 16 KB chunks that a
// producer warp fills with bulk copies: while the second pass over a row frees chunks, the next row's are on
// their way. Another warp prepares the next row's teacher (softmax, first entry of each token). 512 consumer
// threads make the two passes; the CTAs of a cluster exchange their maxima and sums through shared
// memory with one barrier a row. The few elements of a row outside its 16-byte vectors are read where they lie.
//
// The passes keep the offset o = max log2(e) / T instead of the maximum: p = 2^(s c - o) / sum needs one
// multiply-add and one exp2 an element, and the rounding of o cancels. Rows where that does not hold (no logit
// above -1e30, or one above 1e30 after scaling, or NaN) are done again from (s - max) c.

constexpr int kChunk = 16384;
constexpr int kConsumers = 512;
constexpr int kMaxSlots = 13;
constexpr int kMaxCluster = 8;
constexpr float kTame = 1e30f;

// A row's teacher entries, in arrays of kMaxTop or fewer (a multiple of 4).
struct Entries {
    int* token;    // -1: absent
    float* q;      // this entry's
    float* all_q;  // of all entries of the token, at its first entry; -1 elsewhere
    float* value;  // the student's logit

    __host__ __device__ static constexpr int padded(int top) { return (top + 3) / 4 * 4; }
    __host__ __device__ static constexpr int bytes(int top) { return padded(top) * 16; }
    __device__ __forceinline__ Entries(uint8_t* at, int top) {
        token = reinterpret_cast<int*>(at);
        q = reinterpret_cast<float*>(token + padded(top));
        all_q = q + padded(top);
        value = all_q + padded(top);
    }
};

// A row's softmax after the first pass: p = 2^(s c - o) / sum where tame, else 2^((s - base) c) / sum.
struct Softmax {
    float o, base, sum;
    bool tame;
};

struct Stream {
    uint64_t full[kMaxSlots], empty[kMaxSlots];
    uint64_t teacher_full[2], passed[2], written[2];
    uint64_t met[2];
    float2 meet[2][kMaxCluster];
    float red[2][kConsumers / 32], red2[2][kConsumers / 32];
    float some[2];  // sum of the teacher's weights: 0 without an entry
    Softmax softmax[2];
    int abort;
};

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t phase, int* health, volatile int* abort_flag, bool cluster = false) {
    auto done = [&] {
        uint32_t ok;
        if (cluster)
            asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                         : "=r"(ok) : "r"(ptx::smem_u32(bar)), "r"(phase) : "memory");
        else
            ok = ptx::mbar_try_wait(bar, phase);
        return ok != 0;
    };
    if (done()) return true;
    uint64_t start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    for (uint32_t i = 1;; ++i) {
        if (done()) return true;
        if ((i & 1023u) == 0) {
            if (*abort_flag) return false;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (now - start > 4000000000ull) {
                if (health) atomicOr(health, kHealthTimeout);
                *abort_flag = 1;
                return false;
            }
        }
    }
}

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); }

// A row's 16-byte vectors and the slice of them that this CTA holds.
template <typename L>
struct Slice {
    static constexpr int kN = 16 / sizeof(L);
    const L* s;
    int head, vectors, tail;  // elements before the first vector, vectors, first element after them
    int from, count, chunks;

    __device__ __forceinline__ Slice(const rl2_distill_args& a, long long row, uint32_t rank, uint32_t size) {
        s = static_cast<const L*>(a.logits) + row * a.ld_logits;
        const int mis = static_cast<int>(reinterpret_cast<uintptr_t>(s) % 16 / sizeof(L));
        head = min(a.vocab, mis ? kN - mis : 0);
        vectors = (a.vocab - head) / kN;
        tail = head + vectors * kN;
        const int shift = 31 - __clz(size);  // a power of two
        from = static_cast<int>(static_cast<unsigned long long>(vectors) * rank >> shift);
        count = static_cast<int>(static_cast<unsigned long long>(vectors) * (rank + 1) >> shift) - from;
        chunks = (count * 16 + kChunk - 1) / kChunk;
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
        for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(to + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
    } else if constexpr (N == 8) {
        *reinterpret_cast<uint4*>(to) = make_uint4(narrow2<G>(y[0], y[1]), narrow2<G>(y[2], y[3]), narrow2<G>(y[4], y[5]), narrow2<G>(y[6], y[7]));
    } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(narrow2<G>(y[0], y[1]), narrow2<G>(y[2], y[3]));
    }
}

// One warp: the row's teacher; returns the sum of its weights. Entries go four to a lane, so that the loads of
// 128 are in flight together.
template <typename L>
__device__ __forceinline__ float prepare_teacher(const rl2_distill_args& a, long long row, const Entries entry, float scale) {
    constexpr int kEach = 4;
    const int lane = threadIdx.x & 31;
    const int K = a.top, padded = Entries::padded(K);
    const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits;
    float top = -INFINITY;
    bool bad = false;
    for (int k0 = 0; k0 < padded; k0 += 32 * kEach) {
        long long i[kEach];
        float v[kEach], z[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int k = k0 + e * 32 + lane;
            i[e] = k < K ? teacher_index(a, row, k) : -1;
            v[e] = k < K ? teacher_value(a, row, k) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) z[e] = i[e] >= 0 && i[e] < a.vocab ? to_float(s[i[e]]) : 0.0f;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int k = k0 + e * 32 + lane;
            const bool here = i[e] >= 0 && i[e] < a.vocab;
            bad |= i[e] >= a.vocab;
            if (!here) v[e] = -INFINITY;
            top = fmaxf(top, v[e]);
            if (k < padded) {
                entry.token[k] = here ? static_cast<int>(i[e]) : -1;
                entry.q[k] = v[e];
                entry.value[k] = z[e];
            }
        }
    }
    if (bad && a.health) atomicOr(a.health, kHealthIndex);
    top = warp_max(top);
    float total = 0.0f;
    for (int k = lane; k < K; k += 32)
        if (entry.q[k] != -INFINITY) total += exp2_fast((entry.q[k] - top) * scale);
    total = warp_sum(total);
    const float inverse = 1.0f / total;
    bool repeated = false;
    __syncwarp();
    for (int k0 = 0; k0 < K; k0 += 32 * kEach) {
        int token[kEach], same[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int k = k0 + e * 32 + lane;
            token[e] = k < K ? entry.token[k] : -1;
            same[e] = 0;
            if (k < K) {
                const float q = entry.q[k] == -INFINITY ? 0.0f : exp2_fast((entry.q[k] - top) * scale) * inverse;
                entry.q[k] = q;
                entry.all_q[k] = token[e] >= 0 ? q : -1.0f;
            }
        }
#pragma unroll 4
        for (int j = 0; j < padded; j += 4) {
            const int4 t = *reinterpret_cast<const int4*>(entry.token + j);
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                same[e] += (t.x == token[e]) + (t.y == token[e]) + (t.z == token[e]) + (t.w == token[e]);
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) repeated |= token[e] >= 0 && same[e] > 1;
    }
    if (__any_sync(0xffffffffu, repeated)) {
        for (int k = lane; k < K; k += 32) {
            float q = 0.0f;
            bool first = entry.token[k] >= 0;
            for (int j = 0; j < K; ++j)
                if (entry.token[j] == entry.token[k]) {
                    first &= j >= k;
                    q += entry.q[j];
                }
            entry.all_q[k] = first ? q : -1.0f;
        }
    }
    __syncwarp();
    return total;
}

template <typename L, typename G>
__global__ void __launch_bounds__(kConsumers + 64, 2) stream_kernel(const rl2_distill_args a, const int size, const int slots) {
    extern __shared__ __align__(128) uint8_t ring[];  // chunks, then two rows' teacher entries
    __shared__ Stream sh;
    constexpr int kN = Slice<L>::kN;
    const int tid = threadIdx.x;
    const uint32_t rank = size > 1 ? ptx::cluster_rank() : 0u;
    volatile int* abort_flag = &sh.abort;
    const float scale = kLog2e / a.temperature;
    const Entries entries[2] = {Entries(ring + slots * kChunk, a.top), Entries(ring + slots * kChunk + Entries::bytes(a.top), a.top)};
    if (tid == 0) {
        for (int i = 0; i < slots; ++i) {
            ptx::mbar_init(&sh.full[i], 1);
            ptx::mbar_init(&sh.empty[i], kConsumers / 32);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&sh.teacher_full[i], 1);
            ptx::mbar_init(&sh.passed[i], 1);
            ptx::mbar_init(&sh.written[i], kConsumers / 32);
            ptx::mbar_init(&sh.met[i], size);
        }
        sh.abort = 0;
        ptx::fence_barrier_init();
    }
    __syncthreads();
    if (size > 1) ptx::cluster_sync();
    const long long first_row = blockIdx.x / size, step = gridDim.x / size;

    const float grad_factor = a.loss_weight * a.temperature * (a.grad_scale ? *a.grad_scale : 1.0f);
    if (tid >= kConsumers + 32) {
        // ---- teacher warp: the next row's teacher, then the row's loss and its teacher's tokens ----
        const int lane = tid & 31;
        auto next_row = [&](long long row) {
            while (row < a.rows && a.row_weight && a.row_weight[row] == 0.0f) row += step;
            return row;
        };
        int n = 0;
        auto prepare = [&](long long row, int buf) {
            const float total = prepare_teacher<L>(a, row, entries[buf], scale);
            if (lane == 0) {
                sh.some[buf] = total;
                ptx::mbar_arrive(&sh.teacher_full[buf]);
            }
        };
        long long row = next_row(first_row);
        if (row < a.rows) prepare(row, 0);
        while (row < a.rows) {
            const long long after = next_row(row + step);
            const int buf = n & 1;
            const Entries& entry = entries[buf];
            if (after < a.rows) prepare(after, buf ^ 1);  // its last user was this warp
            wait_bar(&sh.passed[buf], (n >> 1) & 1, a.health, abort_flag);
            __syncwarp();
            const Softmax soft = sh.softmax[buf];
            const bool some = sh.some[buf] != 0.0f && soft.sum != 0.0f;
            if (rank == 0) {
                const float log_sum = logf(soft.sum);
                float loss = 0.0f;
                for (int k = lane; k < a.top; k += 32) {
                    const float q = entry.q[k], v = entry.value[k];
                    const float log_p = (soft.tame ? fmaf(v, scale, -soft.o) : (v - soft.base) * scale) * kLn2 - log_sum;
                    if (some && q != 0.0f) loss += q * (logf(q) - log_p);
                }
                loss = warp_sum(loss);
                if (lane == 0) a.row_loss[row] = some ? a.temperature * a.temperature * loss : 0.0f;
            }
            wait_bar(&sh.written[buf], (n >> 1) & 1, a.health, abort_flag);
            __syncwarp();
            if (a.dlogits && some) {
                // over what the pass wrote: each CTA the tokens of its own slice
                const Slice<L> in(a, row, rank, size);
                const int lo = rank == 0 ? 0 : in.head + in.from * kN, hi = static_cast<int>(rank) == size - 1 ? in.tail : in.head + (in.from + in.count) * kN;
                const float factor = (a.row_weight ? a.row_weight[row] : 1.0f) * grad_factor;
                const float f = factor / soft.sum;
                G* ds = static_cast<G*>(a.dlogits) + row * a.ld_dlogits;
                for (int k = lane; k < a.top; k += 32) {
                    const int token = entry.token[k];
                    const float q = entry.all_q[k], v = entry.value[k];
                    const bool own = (token >= lo && token < hi) || (rank == 0 && token >= in.tail);
                    const float p = exp2_fast(soft.tame ? fmaf(v, scale, -soft.o) : (v - soft.base) * scale) * f;
                    if (q != -1.0f && own) ds[token] = narrow<G>(p - factor * q);
                }
            }
            __syncwarp();
            row = after;
            ++n;
        }
    } else if (tid >= kConsumers) {  // ---- producer warp: one lane ----
        if (tid == kConsumers) {
            long long issued = 0;
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (long long row = first_row; row < a.rows && ok; row += step) {
                if (a.row_weight && a.row_weight[row] == 0.0f) continue;
                const Slice<L> in(a, row, rank, size);
                const uint8_t* from = reinterpret_cast<const uint8_t*>(in.s + in.head) + in.from * 16ll;
                for (int c = 0; c < in.chunks; ++c) {
                    ok = wait_bar(&sh.empty[slot], phase ^ 1, a.health, abort_flag);
                    if (!ok) break;
                    const uint32_t bytes = static_cast<uint32_t>(min(kChunk, in.count * 16 - c * kChunk));
                    ptx::mbar_arrive_expect_tx(&sh.full[slot], bytes);
                    ptx::bulk_load(ring + slot * kChunk, from + c * static_cast<long long>(kChunk), bytes, &sh.full[slot]);
                    ++issued;
                    if (++slot == slots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
            // every chunk asked for has landed before the CTA may end, also after an abort
            for (int i = 0; i < slots; ++i) {
                const long long armed = issued > i ? (issued - 1 - i) / slots + 1 : 0;
                volatile int none = 0;
                if (armed > 0) wait_bar(&sh.full[i], static_cast<uint32_t>((armed - 1) & 1), a.health, &none);
            }
        }
    } else {  // ---- consumers ----
        const int lane = tid & 31, warp = tid >> 5;
        int slot = 0, n = 0, meeting = 0;
        uint32_t phase = 0;
        // A wait that fails (bounded, then the abort word) does not change the path: every barrier keeps its threads.
        // over the CTA, then the cluster: a maximum and the sum (unless `plain`, relative to it as powers of two)
        auto meet = [&](float top, float sum, bool plain) {
            auto relative = [&](float t, float all) { return plain ? 1.0f : exp2_fast(t - all); };
            float all = warp_max(top);
            sum = warp_sum(sum * relative(top, all));
            const int buf = meeting & 1;
            if (lane == 0) {
                sh.red[buf][warp] = all;
                sh.red2[buf][warp] = sum;
            }
            consumer_sync();
            top = sh.red[buf][lane & 15];
            all = warp_max(top);
            sum = warp_sum(lane < kConsumers / 32 ? sh.red2[buf][lane & 15] * relative(top, all) : 0.0f);
            if (size > 1) {
                if (warp == 0 && lane < size) {
                    const uint32_t to = ptx::cluster_addr(&sh.meet[buf][rank], lane);
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(all), "f"(sum) : "memory");
                    ptx::mbar_arrive_cluster(ptx::cluster_addr(&sh.met[buf], lane));
                }
                wait_bar(&sh.met[buf], (meeting >> 1) & 1, a.health, abort_flag, true);
                const float2 x = sh.meet[buf][lane & (size - 1)];
                all = warp_max(x.x);
                sum = warp_sum(lane < size ? x.y * relative(x.x, all) : 0.0f);
            }
            ++meeting;
            return make_float2(all, sum);
        };
        // the next row's weight and edge, loaded while this row is worked on
        struct Ahead {
            float weight, edge;
        };
        auto load_ahead = [&](long long row) {
            Ahead x{0.0f, -INFINITY};
            if (row < a.rows) {
                const Slice<L> in(a, row, rank, size);
                x.weight = a.row_weight ? a.row_weight[row] : 1.0f;
                if (rank == 0 && tid < in.head + (a.vocab - in.tail)) x.edge = to_float(in.s[tid < in.head ? tid : in.tail + tid - in.head]);
            }
            return x;
        };
        Ahead ahead = load_ahead(first_row);
        for (long long row = first_row; row < a.rows; row += step) {
            const Slice<L> in(a, row, rank, size);
            G* ds = a.dlogits ? static_cast<G*>(a.dlogits) + row * a.ld_dlogits : nullptr;
            const float weight = ahead.weight, edge_now = ahead.edge;
            ahead = load_ahead(row + step);
            if (weight == 0.0f) {
                if (ds) {
                    const int lo = rank == 0 ? 0 : in.head + in.from * kN, hi = static_cast<int>(rank) == size - 1 ? a.vocab : in.head + (in.from + in.count) * kN;
                    for (int j = lo + tid; j < hi; j += kConsumers) ds[j] = narrow<G>(0.0f);
                }
                if (tid == 0 && rank == 0) a.row_loss[row] = 0.0f;
                continue;
            }
            // elements outside the vectors: one a thread, on the first CTA
            const int outside = in.head + (a.vocab - in.tail);
            const bool has_edge = rank == 0 && tid < outside;
            const int edge_at = tid < in.head ? tid : in.tail + tid - in.head;
            const float edge = has_edge ? edge_now : -INFINITY;
            // f(vector of the slice, its elements) for this thread's vectors of chunk c in ring slot `at`
            auto chunk = [&](int c, int at, auto&& f) {
                const uint4* data = reinterpret_cast<const uint4*>(ring + at * kChunk);
                const int left = in.count - c * (kChunk / 16);
#pragma unroll
                for (int k = 0; k < kChunk / 16 / kConsumers; ++k) {
                    const int i = k * kConsumers + tid;
                    if (i < left) f(c * (kChunk / 16) + i, data[i]);
                }
            };
            auto next = [&](int& at, uint32_t& ph) {
                if (++at == slots) {
                    at = 0;
                    ph ^= 1;
                }
            };
            // ---- first pass ----
            float o = -kTame, sum = 0.0f;
            int at = slot;
            uint32_t ph = phase;
            if (has_edge && edge * scale > o) {
                o = edge * scale;
                sum = exp2_fast(fmaf(edge, scale, -o));
            } else if (edge != edge) {
                sum = edge;
            }
            for (int c = 0; c < in.chunks; ++c) {
                wait_bar(&sh.full[at], ph, a.health, abort_flag);
                chunk(c, at, [&](int, uint4 x) {
                    float v[kN];
                    unpack<L>(x, v);
                    const float up = fmaxf(o, most_as(x, v, L(0.0f)) * scale);
                    sum *= exp2_fast(o - up);
                    float part = 0.0f;
#pragma unroll
                    for (int e = 0; e < kN; e += 2) {
                        sum += exp2_fast(fmaf(v[e], scale, -up));
                        part += exp2_fast(fmaf(v[e + 1], scale, -up));
                    }
                    sum += part;
                    o = up;
                });
                next(at, ph);
            }
            const float2 whole = meet(o, sum, false);
            o = whole.x;
            sum = whole.y;
            float base = 0.0f;
            const bool tame = o < kTame && sum > 0.0f;
            if (!tame) {  // from (s - max) c
                float m = edge;
                auto again = [&](auto&& f) {
                    int s2 = slot;
                    uint32_t p2 = phase;
                    for (int c = 0; c < in.chunks; ++c) {
                        chunk(c, s2, [&](int, uint4 x) {
                            float v[kN];
                            unpack<L>(x, v);
#pragma unroll
                            for (int e = 0; e < kN; ++e) f(v[e]);
                        });
                        next(s2, p2);
                    }
                };
                again([&](float v) { m = fmaxf(m, v); });
                base = meet(m, 0.0f, true).x;
                if (base == -INFINITY) base = 0.0f;
                sum = has_edge ? exp2_fast((edge - base) * scale) : 0.0f;
                again([&](float v) { sum += exp2_fast((v - base) * scale); });
                sum = meet(0.0f, sum, true).y;
            }
            const int buf = n & 1;
            // the teacher warp arrives here for a row once it is done with the row before the last, so the
            // slots of that one are free
            wait_bar(&sh.teacher_full[buf], (n >> 1) & 1, a.health, abort_flag);
            if (tid == 0) {
                sh.softmax[buf] = Softmax{o, base, sum, tame};
                ptx::mbar_arrive(&sh.passed[buf]);
            }
            // ---- gradient ----
            const bool some = sh.some[buf] != 0.0f && sum != 0.0f;
            const float f = weight * grad_factor / sum;
            auto grad = [&](float v) {
                if (tame) return exp2_fast(fmaf(v, scale, -o)) * f;
                return exp2_fast((v - base) * scale) * f;
            };
            if (has_edge && ds) ds[edge_at] = narrow<G>(some ? grad(edge) : 0.0f);
            G* out = ds ? ds + in.head + static_cast<long long>(in.from) * kN : nullptr;
            const bool vec = reinterpret_cast<uintptr_t>(out) % (sizeof(G) * kN <= 16 ? sizeof(G) * kN : 16) == 0;
            auto write = [&](auto is_tame) {
                for (int c = 0; c < in.chunks; ++c) {
                    if (out)
                        chunk(c, slot, [&](int i, uint4 x) {
                            float v[kN];
                            unpack<L>(x, v);
#pragma unroll
                            for (int e = 0; e < kN; ++e)
                                v[e] = decltype(is_tame)::value ? exp2_fast(fmaf(v[e], scale, -o)) * f : (some ? grad(v[e]) : 0.0f);
                            G* to = out + static_cast<long long>(i) * kN;
                            if (vec) {
                                store_vector<G, kN>(to, v);
                            } else {
#pragma unroll
                                for (int e = 0; e < kN; ++e) to[e] = narrow<G>(v[e]);
                            }
                        });
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&sh.empty[slot]);
                    next(slot, phase);
                }
            };
            if (tame && some)
                write(std::true_type{});
            else
                write(std::false_type{});
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&sh.written[buf]);
            ++n;
        }
    }
    __syncthreads();
    if (size > 1) ptx::cluster_sync();  // no CTA leaves while another may write into its shared memory
    finish(a);
}

template <typename L, typename G>
int launch(const rl2_distill_args& a, cudaStream_t stream) {
    if (a.vocab <= 1024 && a.top <= kFewTop) {
        const long long blocks = std::min<long long>((static_cast<long long>(a.rows) + kRowWarps - 1) / kRowWarps, 148 * 8);
        warp_kernel<L, G><<<static_cast<int>(blocks), 32 * kRowWarps, 0, stream>>>(a);
        return launch_status("distillation");
    }
    if (a.vocab <= 2048) {
        row_kernel<L, G, 128><<<std::min(a.rows, 148 * 16), 128, 0, stream>>>(a);
        return launch_status("distillation");
    }
    // two CTAs an SM; the smallest cluster whose slices leave two chunks of the ring to the next row
    constexpr int kBudget = 113 * 1024 - static_cast<int>(sizeof(Stream)) - 1024;
    const int slots = std::min(kMaxSlots, (kBudget - 2 * Entries::bytes(a.top)) / kChunk);
    auto chunks = [&](int size) {
        return static_cast<int>(((a.vocab / Slice<L>::kN + size - 1) / size * 16ll + kChunk - 1) / kChunk);
    };
    int size = 1;
    while (size < kMaxCluster && chunks(size) > slots - 2) size *= 2;
    if (a.vocab <= 8192 || chunks(size) > slots) {
        // short rows (a CTA each, several an SM), or a row that no cluster holds
        if (a.vocab <= 8192)
            row_kernel<L, G, 256><<<std::min(a.rows, 148 * 8), 256, 0, stream>>>(a);
        else
            row_kernel<L, G, 512><<<std::min(a.rows, 148 * 4), 512, 0, stream>>>(a);
        return launch_status("distillation");
    }
    const int smem = slots * kChunk + 2 * Entries::bytes(a.top);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kConsumers + 64);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    // clusters resident at once (each walks over its rows, so one that started later would end as much later):
    // asked once a device, cluster size and type, at the largest shared memory
    static std::atomic<int> resident[64][4];
    int device = 0, log_size = 0;
    while ((1 << log_size) < size) ++log_size;
    cudaError_t e = cudaGetDevice(&device);
    int most = device < 64 ? resident[device][log_size].load() : 0;
    if (e == cudaSuccess && most == 0) {
        e = cudaFuncSetAttribute(reinterpret_cast<const void*>(stream_kernel<L, G>), cudaFuncAttributeMaxDynamicSharedMemorySize, kBudget);
        cudaLaunchConfig_t full = cfg;
        full.dynamicSmemBytes = kBudget;
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&most, stream_kernel<L, G>, &full);
        most = std::max(most, 1);
        if (e == cudaSuccess && device < 64) resident[device][log_size].store(most);
    }
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(a.rows, most)) * size);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, stream_kernel<L, G>, a, size, slots);
    if (e != cudaSuccess) {
        set_error("distillation: %s", cudaGetErrorString(e));
        return -1;
    }
    return launch_status("distillation");
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
    if (a->rows < 0 || a->vocab < 1 || a->top < 1 || a->top > kMaxTop) {
        set_error("distillation: rows >= 0, vocab >= 1 and 1..%d teacher entries are needed", kMaxTop);
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
    if (!(a->temperature > 0.0f) || a->temperature > 1e30f) {
        set_error("distillation: the temperature must be positive and finite");
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
    if (a->ld_logits < a->vocab || a->ld_values < a->top || a->ld_indices < a->top || (a->dlogits && a->ld_dlogits < a->vocab)) {
        set_error("distillation: a row stride is shorter than its row");
        return -1;
    }
    if (!aligned(a->logits, esize[a->logits_dtype]) || !aligned(a->teacher_values, esize[a->values_dtype]) ||
        !aligned(a->teacher_indices, a->index_bits / 8) || !aligned(a->dlogits, esize[a->dlogits_dtype])) {
        set_error("distillation: a matrix is not aligned to its element");
        return -1;
    }
    if (a->dlogits == a->logits) {
        set_error("distillation: the gradient may not overwrite the logits");
        return -1;
    }
    if (a->logits_dtype == 0) return launch_for<float>(*a, as_stream(stream));
    if (a->logits_dtype == 1) return launch_for<__half>(*a, as_stream(stream));
    return launch_for<__nv_bfloat16>(*a, as_stream(stream));
}
