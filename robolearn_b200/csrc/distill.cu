// Distillation of a head from a teacher's top logits: loss and gradient in one kernel.
//
//   q = softmax(t / T) over the k teacher entries that are there (index >= 0)
//   p = softmax(s / T) over all V logits of the student
//   row_loss = T^2 sum_k q_k (log q_k - log p[i_k])
//   loss     = c sum_n w_n row_loss_n
//   ds_j     = c w_n T (p_j - sum_{k: i_k = j} q_k) (* *grad_scale)
//
// A row is read from memory once: the running maximum and the running sum of a softmax make the
// first pass, the gradient is written by a second one that finds the row in L2. All sums are
// fp32; exponentials are the hardware's exp2 of (s - max) log2(e) / T, whose argument is at most
// 0, so every value is within a few units in the last place of fp32.

#include "common.cuh"
#include "../../include/rl2.h"

#include <cuda_bf16.h>

#include <algorithm>

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

// One CTA per row.
template <typename L, typename G, int THREADS>
__global__ void __launch_bounds__(THREADS) row_kernel(const rl2_distill_args a) {
    __shared__ float red[32];
    __shared__ float red2[32];
    __shared__ float q_s[kMaxTop];
    __shared__ int i_s[kMaxTop];
    __shared__ bool last;
    constexpr int kN = Pack<L>::kN;
    const int tid = threadIdx.x;
    const int V = a.vocab, K = a.top;
    const float scale = kLog2e / a.temperature;
    const float grad_scale = a.loss_weight * a.temperature * (a.grad_scale ? *a.grad_scale : 1.0f);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const L* s = static_cast<const L*>(a.logits) + row * a.ld_logits;
        G* ds = a.dlogits ? static_cast<G*>(a.dlogits) + row * a.ld_dlogits : nullptr;
        const float weight = a.row_weight ? a.row_weight[row] : 1.0f;
        if (weight == 0.0f) {
            if (ds)
                for (int j = tid; j < V; j += THREADS) ds[j] = narrow<G>(0.0f);
            if (tid == 0) a.row_loss[row] = 0.0f;
            continue;
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
            top = v != v ? v : fmaxf(top, v);
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
        __syncthreads();
        if ((tid & 31) == 0) {
            red[tid >> 5] = r.max;
            red2[tid >> 5] = r.sum;
        }
        __syncthreads();
        r = Running{-INFINITY, 0.0f};
        for (int w = 0; w < THREADS / 32; ++w) r = merge(r, Running{red[w], red2[w]}, scale);
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
            const float factor = some ? weight * grad_scale : 0.0f;
            const float inv_sum = some ? 1.0f / r.sum : 0.0f;
            auto grad = [&](float v, float q) { return some ? factor * (exp2_fast((v - base) * scale) * inv_sum - q) : 0.0f; };
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
            __syncthreads();
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
        __syncthreads();
    }
    if (!a.loss_out) return;
    // the last block adds the rows' losses in a fixed order
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(a.counter, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    float sum = 0.0f;
    for (int n = tid; n < a.rows; n += THREADS) {
        const float w = a.row_weight ? a.row_weight[n] : 1.0f;
        if (w != 0.0f) sum += w * __ldcg(a.row_loss + n);
    }
    sum = block_sum<THREADS>(sum, red);
    if (tid == 0) {
        *a.loss_out = a.loss_weight * sum;
        *a.counter = 0;
    }
}

template <typename L, typename G>
void launch(const rl2_distill_args& a, cudaStream_t stream) {
    if (a.vocab <= 2048)
        row_kernel<L, G, 128><<<std::min(a.rows, 148 * 16), 128, 0, stream>>>(a);
    else
        row_kernel<L, G, 512><<<std::min(a.rows, 148 * 4), 512, 0, stream>>>(a);
}

template <typename L>
void launch_for(const rl2_distill_args& a, cudaStream_t stream) {
    if (a.dlogits_dtype == 0)
        launch<L, float>(a, stream);
    else if (a.dlogits_dtype == 1)
        launch<L, __half>(a, stream);
    else
        launch<L, __nv_bfloat16>(a, stream);
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
    if (a->logits_dtype == 0)
        launch_for<float>(*a, as_stream(stream));
    else if (a->logits_dtype == 1)
        launch_for<__half>(*a, as_stream(stream));
    else
        launch_for<__nv_bfloat16>(*a, as_stream(stream));
    return launch_status("distillation");
}
