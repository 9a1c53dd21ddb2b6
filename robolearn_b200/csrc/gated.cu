// Gated feed-forward block on tcgen05: h = act(x Wg^T) * (x Wu^T), and its backward pass.
//
//   forward     g = x Wg^T, u = x Wu^T, h = act(g) * u                      [M][F]
//   backward    dg = dh * u * act'(g), du = dh * act(g)                     [M][F] each
//               dx = dg Wg + du Wu                                          [M][K]
//               dWg = dg^T x, dWu = du^T x                                  [F][K]
//
// x [M][K], Wg and Wu [F][K] (the layout of a linear layer's weight), fp16 or bf16 operands,
// fp32 accumulation. g and u are never stored: the forward's epilogue consumes them from
// TMEM, and the backward computes them again (2 of its 6 products; storing them in fp32 would
// write and read 16 bytes per element of [M][F], which costs more than the two products up to
// K = 1024 or so, and storing them rounded would add their rounding to every gradient). dg and
// du are rounded once to the operand type: they are the operands of the last two products.
//
// One kernel, four modes. All run 256 x (2 BNC) tiles on CTA pairs (tcgen05 cta_group::2, M =
// 256): each CTA stages its 128 rows of A and BNC rows of B per 64-deep k-block.
//   kForward, kGate   the pair's B rows are BNC rows of Wg (even CTA) and the same BNC rows of
//                     Wu (odd CTA), so one MMA makes both projections of BNC hidden units and
//                     a TMEM lane holds g in columns [0, BNC) and u in [BNC, 2 BNC). kGate also
//                     brings the tile's dh by TMA and stores dg and du.
//   kInput            contraction over the 2F concatenated hidden units: A = [dg | du]
//                     (K-major), B = [Wg ; Wu] read N-contiguous, no transposed copies.
//   kWeight           contraction over the M rows: A = dg or du read M-contiguous, B = x read
//                     N-contiguous; split over rows when the tiles do not fill the GPU.
// dg and du live in the workspace in blocks of 128 rows by 64 hidden units, 16 KB each in one piece, because the
// last two products read them so: as rows of the matrix, a block is 128 pieces of 128 bytes in as many DRAM pages,
// and dx at 8192 x 512 x 2048 took 0.53 us a k-block for the 0.38 that the tensor cores take. Rows and hidden units
// past the matrix are zeros there (the projections of zero-filled operands).
// Warp roles as in the dense products: TMA producer, MMA issuer, eight or sixteen epilogue warps on a
// double-buffered accumulator. Outputs leave through shared-memory boxes and TMA stores, which
// clip at the output's extents. Every wait is bounded by wall-clock time.
//
// Two forms without these tiles, forward only: few_rows_kernel (up to 16 rows) and strip_kernel (up to 128).
//
// Measured: forward 65536 x 1024 x 4096 bf16 794 us (1385 TFLOP/s, the rate that the card sustains under its power
// limit); backward 32768 x 1024 x 4096 bf16 1382 to 1429 us (1154 to 1193 TFLOP/s). At 8192 x 512 x 2048 fp16 the forward takes 29
// us (a library product of its shape 35) and the backward 101: the projections again 40, dx 27, dW 34 (split over rows, then
// summed). What bounds these is the way between L2 and the SMs: 313 MB in the forward, 449 MB where dh comes in and dg and du go
// out, 10 to 11 TB/s (27 us without the stores). Stores of dg and du in whole 4 KB pieces instead of
// tensor boxes change that by less than 1%.

#include "common.cuh"
#include "../../include/rl2.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <initializer_list>
#include <new>

namespace rl2 {
namespace gated {

constexpr int kBM = 128;  // rows of A per CTA (256 per pair)
constexpr int kBK = 64;   // 128 bytes of 16-bit operands
constexpr int kMaxEpiWarps = 16;
constexpr int kMaxSmem = 232448;
constexpr int kMaxStages = 8;

enum Mode { kForward = 0, kGate = 1, kInput = 2, kWeight = 3 };
enum Act { kSilu = 0, kGelu = 1, kRelu = 2 };

// Epilogue warps: four per TMEM lane quarter where the epilogue computes (the activation's two special-function
// steps an element need the warps to hide them), two where it only rounds and stores.
__host__ __device__ constexpr int epi_warps(int mode) { return mode == kForward || mode == kGate ? 16 : 8; }
__host__ __device__ constexpr int threads_of(int mode) { return 64 + 32 * epi_warps(mode); }
// Boxes: 32 rows of 32 (or 16) hidden units, one a warp (kForward) or three (kGate: dg, du, and dh, which is on its way
// while the tile before is stored); or of 128 bytes, one a warp.
__host__ __device__ constexpr int box_bytes(int mode) { return mode == kForward || mode == kGate ? 2048 : 4096; }
__host__ __device__ constexpr int boxes_of(int mode) { return mode == kGate ? 3 : 1; }

struct Params {
    int b_merged;       // N-contiguous operand: one copy brings all its 64-wide chunks
    int row_blocks;     // 128-row blocks of dg (of du) in the workspace
    int kblocks;        // k-blocks of the whole contraction
    int kb_segment;     // kInput: k-blocks of one half (F / 64, rounded up)
    int splits, kb_per_split;
    int bnc;            // B rows staged per CTA
    int tile_cols;      // output columns per tile: bnc (kForward, kGate) or 2 bnc
    int tiles_n, tiles_m, tiles_z, tiles_total;
    int stages;
    int box_cols;       // columns per store box
    int out_rows, out_cols;
    int store_cols;     // columns that the store engine writes; the rest of a row (less than 16 bytes) by plain stores
    void* out[2];       // kForward, kInput: out[0]; kWeight: by gate / up
    long long ld_out[2];
    const float* scale; // kWeight, not split: multiplies the output
    int* health;
    int* found_inf;     // the backward's: a rounded value is not finite (see Rounded)
};

struct Maps {
    CUtensorMap a, b0, b1, d0, d1, in;
};

// ---- small device helpers ---------------------------------------------------

__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);  // descriptor version, 128-byte swizzle
}

// mbarrier wait bounded to 4 s; gives up early once another role raised the CTA's abort word
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t phase, int* health, volatile int* abort_flag) {
    if (ptx::mbar_try_wait(bar, phase)) return true;
    uint64_t start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    for (uint32_t i = 1;; ++i) {
        if (ptx::mbar_try_wait(bar, phase)) return true;
        if ((i & 1023u) == 0) {
            if (abort_flag && *abort_flag) return false;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
            if (now - start > 4000000000ull) {
                if (health) atomicOr(health, kHealthTimeout);
                if (abort_flag) *abort_flag = 1;
                return false;
            }
        }
    }
}

// The same for all lanes of a warp: they go on together, and all or none of them. (After a wait that ran out, one lane may
// see another role's abort word and the next the barrier's phase; what follows is for whole warps.)
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t phase, int* health, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, wait_bar(bar, phase, health, abort_flag));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Whether all 16-bit words that a thread has rounded are finite: their largest magnitude, in which a NaN stays (two
// instructions a word).
template <bool BF16>
struct Rounded {
    uint32_t most = 0;
    __device__ __forceinline__ void add(uint32_t w) {
        if (BF16) {
            const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&most), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
            most = *reinterpret_cast<const uint32_t*>(&m);
        } else {
            const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&most), __habs2(*reinterpret_cast<const __half2*>(&w)));
            most = *reinterpret_cast<const uint32_t*>(&m);
        }
    }
    __device__ __forceinline__ bool finite() const {
        constexpr uint32_t kInf = BF16 ? 0x7F80u : 0x7C00u;
        return (most & 0xFFFFu) < kInf && (most >> 16) < kInf;
    }
};

// A step whose gradients are not finite: *found_inf, or without one the overflow bit of *health.
__device__ __forceinline__ void report_overflow(int* found_inf, int* health) {
    if (found_inf)
        atomicOr(found_inf, 1);
    else if (health)
        atomicOr(health, kHealthOverflow);
}

// The normal distribution function Phi(g), and exp(-g^2 / 2), which its density shares. Phi(-|g|) is taken itself, not as
// what 1 leaves: exp(-g^2 / 2) t P(t) with t = 1 / (1 + 0.3 |g|), the form of Hastings (Abramowitz and Stegun 7.1.26), P
// fitted here to erfcx(|g| / sqrt 2) / 2 over 0 .. 13.4 in the relative error: 1.3e-7, 4e-7 with the roundings. The
// exponent's rounding adds g^2 2^-24. So the lower tail keeps its digits down to g = -13 (1e-38), where a form with 1 + erf has
// lost 4% at -5 and all at -6. 8192 x 512 x 2048 forward: 33 us with that form, 50 with the library's erfcf, which has too many steps for
// an epilogue.
__device__ __forceinline__ float normal_cdf(float g, float& bell) {
    const float z = fabsf(g), t = __fdividef(1.0f, fmaf(0.3f, z, 1.0f));
    float s = 0.0359838195f;
    s = fmaf(s, t, -0.158493891f);
    s = fmaf(s, t, 0.208583847f);
    s = fmaf(s, t, -0.0557430983f);
    s = fmaf(s, t, 0.129655257f);
    s = fmaf(s, t, 0.0995806456f);
    s = fmaf(s, t, 0.120807566f);
    s = fmaf(s, t, 0.119625784f);
    bell = __expf(-0.5f * g * g);
    const float tail = bell * (s * t);
    return g < 0.0f ? tail : 1.0f - tail;
}

// act(g) and act'(g). The exponential and the division are the fast fp32 forms (a few units in
// the last place of fp32): the result is rounded to 16 bits, 2^13 to 2^16 times coarser. SiLU and its slope are 0 below -87
// (1e-36), where the exponential leaves fp32.
template <int ACT>
__device__ __forceinline__ float act_value(float g) {
    if (ACT == kSilu) return __fdividef(g, 1.0f + __expf(-g));
    if (ACT == kGelu) {
        float bell;
        return g * normal_cdf(g, bell);
    }
    return g > 0.0f ? g : (g == g ? 0.0f : g);
}

template <int ACT>
__device__ __forceinline__ void act_both(float g, float& value, float& slope) {
    if (ACT == kSilu) {
        const float s = __fdividef(1.0f, 1.0f + __expf(-g));
        value = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if (ACT == kGelu) {
        float bell;
        const float cdf = normal_cdf(g, bell);
        value = g * cdf;
        slope = fmaf(g * 0.39894228f, bell, cdf);
    } else {
        value = g > 0.0f ? g : (g == g ? 0.0f : g);
        slope = g > 0.0f ? 1.0f : 0.0f;
    }
}

struct Tile {
    int n, m, z, split, kb0, kb1;
};

__device__ __forceinline__ Tile decode(const Params& p, int t) {
    Tile w;
    w.n = t % p.tiles_n;
    t /= p.tiles_n;
    w.m = t % p.tiles_m;
    t /= p.tiles_m;
    w.z = t % p.tiles_z;
    w.split = t / p.tiles_z;
    w.kb0 = w.split * p.kb_per_split;
    w.kb1 = min(p.kblocks, w.kb0 + p.kb_per_split);
    return w;
}

// ---- roles --------------------------------------------------------------------

// `chunks` 64-wide pieces (from column n0 on) of 64 k-rows of an N-contiguous operand: one behind the other in
// shared memory. Merged maps see the matrix as {64, rows, columns / 64}.
__device__ __forceinline__ void load_chunks(uint8_t* to, const CUtensorMap* map, uint32_t bar, int n0, int k0, int chunks,
                                            int merged) {
    if (merged) {
        ptx::tma_load_3d_pair(to, map, bar, 0, k0, n0 / 64);
    } else {
        for (int c = 0; c < chunks; ++c) ptx::tma_load_3d_pair(to + c * (kBK * 128), map, bar, n0 + c * 64, k0, 0);
    }
}

template <int MODE>
__device__ __forceinline__ void produce(const Maps& maps, const Params& p, uint8_t* smem, uint32_t stage_bytes,
                                        uint64_t* full, uint64_t* empty, volatile int* abort_flag) {
    const int rank = static_cast<int>(blockIdx.x & 1u);
    ptx::prefetch_tensormap(&maps.a);
    ptx::prefetch_tensormap(&maps.b0);
    int s = 0;
    uint32_t phase = 0;
    long long issued = 0;
    bool ok = true;
    for (int t = blockIdx.x >> 1; t < p.tiles_total && ok; t += gridDim.x >> 1) {
        const Tile w = decode(p, t);
        const int row0 = w.m * 2 * kBM + rank * kBM;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
            if (!wait_bar(&empty[s], phase ^ 1, p.health, abort_flag)) {
                ok = false;
                break;
            }
            if (rank == 0) ptx::mbar_arrive_expect_tx(&full[s], 2 * stage_bytes);
            ++issued;
            const uint32_t bar = ptx::cluster_addr(&full[s], 0);
            uint8_t* sa = smem + s * stage_bytes;
            uint8_t* sb = sa + kBM * 128;
            if (MODE == kForward || MODE == kGate) {
                ptx::tma_load_3d_pair(sa, &maps.a, bar, kb * kBK, row0, 0);
                ptx::tma_load_3d_pair(sb, rank == 0 ? &maps.b0 : &maps.b1, bar, kb * kBK, w.n * p.bnc, 0);
            } else if (MODE == kInput) {
                const int seg = kb >= p.kb_segment ? 1 : 0;
                const int f0 = (kb - seg * p.kb_segment) * kBK;
                const int n0 = w.n * p.tile_cols + rank * p.bnc;
                ptx::tma_load_4d_pair(sa, &maps.a, bar, 0, 0, f0 / 64, row0 / kBM + seg * p.row_blocks);
                load_chunks(sb, seg ? &maps.b1 : &maps.b0, bar, n0, f0, p.bnc / 64, p.b_merged);
            } else {
                const int n0 = w.n * p.tile_cols + rank * p.bnc;
                ptx::tma_load_4d_pair(sa, &maps.a, bar, 0, kb % 2 * kBK, row0 / 64, kb / 2 + w.z * p.row_blocks);
                load_chunks(sb, &maps.b0, bar, n0, kb * kBK, p.bnc / 64, p.b_merged);
            }
            if (++s == p.stages) {
                s = 0;
                phase ^= 1;
            }
        }
    }
    // Every armed stage has landed before the pair may exit, also after an abort (the even
    // CTA's barriers count both CTAs' loads; the odd CTA leaves after the even one).
    if (rank != 0) return;
    for (int st = 0; st < p.stages; ++st) {
        const long long armed = issued > st ? (issued - 1 - st) / p.stages + 1 : 0;
        if (armed > 0) wait_bar(&full[st], static_cast<uint32_t>((armed - 1) & 1), p.health, nullptr);
    }
}

// One thread of the even CTA issues every MMA of the pair.
template <int MODE, bool BF16>
__device__ __forceinline__ void issue(const Params& p, uint8_t* smem, uint32_t stage_bytes, uint64_t* full,
                                      uint64_t* empty, uint64_t* acc_full, uint64_t* acc_empty, uint32_t tmem,
                                      volatile int* abort_flag) {
    constexpr uint32_t a_mn = MODE == kWeight ? 1u : 0u;
    constexpr uint32_t b_mn = MODE == kWeight || MODE == kInput ? 1u : 0u;
    constexpr uint32_t fmt = BF16 ? 1u : 0u;
    const uint32_t n = 2u * p.bnc;
    const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) |
                           ((2u * kBM >> 4) << 24);
    auto commit = [&](uint64_t* bar) {
        ptx::mma_commit_pair(ptx::cluster_addr(bar, 0));
        ptx::mma_commit_pair(ptx::cluster_addr(bar, 1));
    };
    int s = 0, i = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x >> 1; t < p.tiles_total; t += gridDim.x >> 1, ++i) {
        const Tile w = decode(p, t);
        const int buf = i & 1;
        if (!wait_bar(&acc_empty[buf], ((i >> 1) & 1) ^ 1, p.health, abort_flag)) return;
        ptx::tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(buf) * n;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
            if (!wait_bar(&full[s], phase, p.health, abort_flag)) return;
            ptx::tc_fence_after();
            const uint32_t sa = ptx::smem_u32(smem + s * stage_bytes);
            const uint32_t sb = sa + kBM * 128;
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j) {
                // K-major: 32 bytes further inside the swizzle atom; MN-major: 16 k-rows further
                const uint64_t da = a_mn ? desc(sa + j * 2048, kBK * 128, 1024) : desc(sa + j * 32, 16, 1024);
                const uint64_t db = b_mn ? desc(sb + j * 2048, kBK * 128, 1024) : desc(sb + j * 32, 16, 1024);
                ptx::mma_f16_pair(d, da, db, idesc, kb > w.kb0 || j > 0 ? 1u : 0u);
            }
            commit(&empty[s]);
            if (++s == p.stages) {
                s = 0;
                phase ^= 1;
            }
        }
        commit(&acc_full[buf]);
    }
}

// Byte offset of 16-byte chunk j of row r in a store box whose rows are 128, 64 or 32 bytes (the swizzle of that
// width): lane = row writes without bank conflicts.
__device__ __forceinline__ uint32_t box_at(int r, int j, int row_bytes) {
    const int swizzled = row_bytes == 128 ? j ^ (r & 7) : row_bytes == 64 ? j ^ ((r >> 1) & 3) : j ^ ((r >> 2) & 1);
    return static_cast<uint32_t>(r * row_bytes + (swizzled << 4));
}

// Columns [store_cols, out_cols) of this lane's row, if its box (columns col0 .. col0 + box_cols - 1)
// holds them: the store engine clips a row at 16-byte granules, so it would also write the columns
// beside a row that ends inside one.
template <int ELEM>
__device__ __forceinline__ void store_tail(const Params& p, const uint8_t* box, int row_bytes, void* base, long long ld,
                                           int col0, int row0, int lane) {
    constexpr int kPer = 16 / ELEM;
    if (p.store_cols >= p.out_cols || p.store_cols < col0 || p.store_cols >= col0 + p.box_cols || row0 + lane >= p.out_rows)
        return;
    const uint4 v = *reinterpret_cast<const uint4*>(box + box_at(lane, (p.store_cols - col0) / kPer, row_bytes));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < kPer - 1; ++e) {
        if (p.store_cols + e >= p.out_cols) break;
        const long long at = (row0 + lane) * ld + p.store_cols + e;
        if (ELEM == 4)
            static_cast<uint32_t*>(base)[at] = w[e];
        else
            static_cast<uint16_t*>(base)[at] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
    }
}

// Epilogue warps: warp w reads TMEM lanes 32 (w % 4) .. + 31 (rows of the tile), the warps of a lane quarter
// share the tile's output columns.
template <int MODE, bool BF16, int ACT, bool OUT32>
__device__ __forceinline__ void drain(const Maps& maps, const Params& p, uint8_t* boxes, uint64_t* in_full,
                                      uint64_t* acc_full, uint64_t* acc_empty, uint32_t tmem,
                                      volatile int* abort_flag) {
    constexpr bool kGated = MODE == kForward || MODE == kGate;
    constexpr int kSlots = epi_warps(MODE) / 4;  // warps of a lane quarter
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = warp & 3, slot = (warp - 2) >> 2;
    const int rank = static_cast<int>(blockIdx.x & 1u);
    uint8_t* box = boxes + (warp - 2) * boxes_of(MODE) * box_bytes(MODE);
    uint8_t* box1 = box + box_bytes(MODE);
    uint8_t* in_box = box1 + box_bytes(MODE);
    uint64_t* in_bar = in_full + (warp - 2);
    const uint32_t n = 2u * p.bnc;
    const int row_bytes = OUT32 ? 128 : p.box_cols * 2;
    const float scale = MODE == kWeight && p.scale ? *p.scale : 1.0f;
    const int mine = kGated ? p.bnc / kSlots : 2 * p.bnc / kSlots;  // this warp's output columns
    auto load_in = [&](int t) {  // a tile's dh, by one lane
        const Tile w = decode(p, t);
        ptx::mbar_arrive_expect_tx(in_bar, 32u * p.box_cols * 2u);
        ptx::tma_load_3d(in_box, &maps.in, in_bar, w.n * p.tile_cols + slot * mine, w.m * 2 * kBM + rank * kBM + q * 32, 0);
    };
    if (MODE == kGate && lane == 0 && (blockIdx.x >> 1) < p.tiles_total) load_in(blockIdx.x >> 1);
    // Rounded values past the matrices are zeros (so are the operands there), or NaN where an operand within is not finite.
    Rounded<BF16> rounded;
    bool over = false;
    int i = 0;
    for (int t = blockIdx.x >> 1; t < p.tiles_total; t += gridDim.x >> 1, ++i) {
        const Tile w = decode(p, t);
        const int buf = i & 1;
        const int row0 = w.m * 2 * kBM + rank * kBM + q * 32;
        const int col0 = w.n * p.tile_cols + slot * mine;
        const bool ready = wait_bar_warp(&acc_full[buf], (i >> 1) & 1, p.health, abort_flag);
        if (MODE == kGate) {  // the copy has landed before the CTA goes on (the next is not under way yet)
            const bool in = wait_bar_warp(in_bar, i & 1, p.health, nullptr);
            if (!in || !ready) break;
        } else if (!ready) {
            break;
        }
        ptx::tc_fence_after();
        const uint32_t base = tmem + static_cast<uint32_t>(buf) * n + (static_cast<uint32_t>(q * 32) << 16);
        if (kGated) {
            // the accumulators, then their buffer is the next tile's
            uint32_t gs[2][16], us[2][16];
            ptx::tmem_ld16_issue(base + slot * mine, gs[0]);
            ptx::tmem_ld16_issue(base + p.bnc + slot * mine, us[0]);
            if (mine == 32) {
                ptx::tmem_ld16_issue(base + slot * mine + 16, gs[1]);
                ptx::tmem_ld16_issue(base + p.bnc + slot * mine + 16, us[1]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ptx::tmem_ld_wait(gs[h]);
                ptx::tmem_ld_wait(us[h]);
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                ptx::mbar_arrive_cluster_relaxed(ptx::cluster_addr(&acc_empty[buf], 0));
                ptx::bulk_wait_read0();
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && mine != 32) break;
                const int c = 16 * h;
                const uint32_t(&gr)[16] = gs[h];
                const uint32_t(&ur)[16] = us[h];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t at = box_at(lane, c / 8 + e, row_bytes);
                    uint32_t o0[4], o1[4];
                    uint4 in4 = make_uint4(0, 0, 0, 0);
                    if (MODE == kGate) in4 = *reinterpret_cast<const uint4*>(in_box + at);
                    const uint32_t in[4] = {in4.x, in4.y, in4.z, in4.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float g0 = __uint_as_float(gr[8 * e + 2 * k]), g1 = __uint_as_float(gr[8 * e + 2 * k + 1]);
                        const float u0 = __uint_as_float(ur[8 * e + 2 * k]), u1 = __uint_as_float(ur[8 * e + 2 * k + 1]);
                        if (MODE == kForward) {
                            o0[k] = pack2<BF16>(act_value<ACT>(g0) * u0, act_value<ACT>(g1) * u1);
                        } else {
                            const float2 dh = unpack2<BF16>(in[k]);
                            float a0, s0, a1, s1;
                            act_both<ACT>(g0, a0, s0);
                            act_both<ACT>(g1, a1, s1);
                            o0[k] = pack2<BF16>(dh.x * u0 * s0, dh.y * u1 * s1);
                            o1[k] = pack2<BF16>(dh.x * a0, dh.y * a1);
                            rounded.add(o0[k]);
                            rounded.add(o1[k]);
                        }
                    }
                    *reinterpret_cast<uint4*>(box + at) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
                    if (MODE == kGate) *reinterpret_cast<uint4*>(box1 + at) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
                }
            }
            if (MODE == kForward) store_tail<2>(p, box, row_bytes, p.out[0], p.ld_out[0], col0, row0, lane);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (MODE == kGate) {
                    ptx::tma_store_4d(&maps.d0, box, col0 % 64, row0 % kBM, col0 / 64, row0 / kBM);
                    ptx::tma_store_4d(&maps.d0, box1, col0 % 64, row0 % kBM, col0 / 64, row0 / kBM + p.row_blocks);
                } else if (col0 < p.store_cols && row0 < p.out_rows) {  // the store engine clips a box, it needs one to start inside
                    ptx::tma_store_3d(&maps.d0, box, col0, row0, 0);
                }
                ptx::bulk_commit();
                if (MODE == kGate && t + (gridDim.x >> 1) < p.tiles_total) load_in(t + (gridDim.x >> 1));
            }
        } else {
            const int z = p.splits > 1 ? (MODE == kWeight ? w.split * 2 + w.z : w.split) : 0;
            const CUtensorMap* dst = MODE == kWeight && p.splits == 1 && w.z ? &maps.d1 : &maps.d0;
            for (int c = 0; c < mine; c += p.box_cols) {
                if (lane == 0) ptx::bulk_wait_read0();
                __syncwarp();
                for (int e = 0; e < p.box_cols; e += 32) {
                    float r[32];
                    ptx::tmem_ld32(base + slot * mine + c + e, r);
                    if (c + e + 32 >= mine) {  // the accumulators are read: their buffer is the next tile's
                        ptx::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive_cluster_relaxed(ptx::cluster_addr(&acc_empty[buf], 0));
                    }
                    if (MODE == kWeight) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) r[k] *= scale;
                    }
                    if (OUT32) {
                        if (p.splits == 1) {  // else partial sums: the reduction reports
#pragma unroll
                            for (int k = 0; k < 32; ++k) over |= !(fabsf(r[k]) <= FLT_MAX);
                        }
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            *reinterpret_cast<float4*>(box + box_at(lane, e / 4 + k, 128)) =
                                make_float4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 o = make_uint4(pack2<BF16>(r[8 * k], r[8 * k + 1]), pack2<BF16>(r[8 * k + 2], r[8 * k + 3]),
                                                       pack2<BF16>(r[8 * k + 4], r[8 * k + 5]), pack2<BF16>(r[8 * k + 6], r[8 * k + 7]));
                            for (uint32_t w : {o.x, o.y, o.z, o.w}) rounded.add(w);
                            *reinterpret_cast<uint4*>(box + box_at(lane, e / 8 + k, row_bytes)) = o;
                        }
                    }
                }
                store_tail<OUT32 ? 4 : 2>(p, box, row_bytes, w.z ? p.out[1] : p.out[0], w.z ? p.ld_out[1] : p.ld_out[0], col0 + c, row0, lane);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (col0 + c < p.store_cols && row0 < p.out_rows) ptx::tma_store_3d(dst, box, col0 + c, row0, z);
                    ptx::bulk_commit();
                }
            }
        }
    }
    if (MODE != kForward && (over || !rounded.finite())) report_overflow(p.found_inf, p.health);
    if (lane == 0) ptx::bulk_wait0();
}

template <int MODE, bool BF16, int ACT, bool OUT32>
__global__ void __launch_bounds__(threads_of(MODE), 1) __cluster_dims__(2, 1, 1)
    product_kernel(const __grid_constant__ Maps maps, const Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], mma_done, in_full[kMaxEpiWarps];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t stage_bytes = static_cast<uint32_t>(kBM + p.bnc) * 128;
    uint8_t* boxes = smem + p.stages * stage_bytes;
    const int warp = threadIdx.x >> 5;
    const bool leader = (blockIdx.x & 1u) == 0;
    const uint32_t tmem_cols = 4u * p.bnc;  // two buffers of 2 bnc columns

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(&acc_full[b], 1);
            ptx::mbar_init(&acc_empty[b], 2 * epi_warps(MODE));
        }
        for (int e = 0; e < kMaxEpiWarps; ++e) ptx::mbar_init(&in_full[e], 1);
        ptx::mbar_init(&mma_done, 1);
        abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(&tmem_slot, tmem_cols);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();  // both CTAs' barriers exist before any remote use
    ptx::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    ptx::grid_release();
    ptx::grid_wait();

    if (warp == 0) {
        if (ptx::elect_one()) produce<MODE>(maps, p, smem, stage_bytes, full, empty, &abort_flag);
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            if (leader) {
                issue<MODE, BF16>(p, smem, stage_bytes, full, empty, acc_full, acc_empty, tmem, &abort_flag);
                // all MMAs have completed before TMEM is released, also after an abort
                ptx::mma_commit_pair(ptx::cluster_addr(&mma_done, 0));
                ptx::mma_commit_pair(ptx::cluster_addr(&mma_done, 1));
            }
            wait_bar(&mma_done, 0, p.health, nullptr);
        }
    } else {
        drain<MODE, BF16, ACT, OUT32>(maps, p, boxes, in_full, acc_full, acc_empty, tmem, &abort_flag);
    }
    ptx::tc_fence_before();
    __syncthreads();
    __syncwarp();
    ptx::cluster_sync();  // neither CTA leaves while the other may still address its memory
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem, tmem_cols);
    }
}

// ---- few rows: forward without tiles ------------------------------------------------
//
// Up to 16 rows the weights are nearly all there is to read, and a 256-row tile would be mostly padding. A CTA
// takes 16 hidden units of both weights; its eight warps share the contraction in steps of 32, each lane loading
// 16 bytes of two rows of each weight straight into the operand registers of m16n8k16 products (hidden units by
// rows of x). A lane's 8 consecutive features stand for the k positions of two products; x is loaded the same
// way, so both see the same order. The warps' sums meet in shared memory. Measured against the tiles: 14 us for 20
// at 2048 x 8192 (4.7 TB/s of weights), 2.4 us for 7.3 at 512 x 2048, 1 to 16 rows; with more rows the loads of x
// per CTA take over (32 rows: 29 us for 20).

constexpr int kFewRows = 16;
constexpr int kFewWarps = 8;
constexpr int kFewUnits = 16;

template <bool BF16>
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct FewArgs {
    const uint16_t* x;
    const uint16_t* gate;
    const uint16_t* up;
    uint16_t* out;
    long long ldx, ld_gate, ld_up, ld_out;
    int rows, features, hidden, act;
};

// 8 elements of a row from column k on where it may end before: 0 past `cols` (the rows' padding is neither data nor
// read: the last row's need not exist)
__device__ __forceinline__ uint4 load_end(const uint16_t* row, int k, int cols) {
    if (k + 8 <= cols) return ptx::load_vector(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (k + e < cols) w[e / 2] |= static_cast<uint32_t>(row[k + e]) << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// NT: 8-row groups of x
template <bool BF16, int NT>
__global__ void __launch_bounds__(32 * kFewWarps) few_rows_kernel(const FewArgs a) {
    extern __shared__ float sums[];  // [warp][gate, up][unit][row]
    constexpr int kRows = 8 * NT;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int f0 = blockIdx.x * kFewUnits;
    ptx::grid_release();
    ptx::grid_wait();
    // Rows past the end repeat the last one: what they give is not stored.
    const uint16_t* w[4];  // gate rows g and g + 8, up rows g and g + 8
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int f = min(f0 + g + (i & 1) * 8, a.hidden - 1);
        w[i] = (i < 2 ? a.gate + f * a.ld_gate : a.up + f * a.ld_up) + t * 8;
    }
    const uint16_t* xr[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xr[n] = a.x + min(n * 8 + g, a.rows - 1) * a.ldx + t * 8;
    float acc[2][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][n][e] = acc[1][n][e] = 0.0f;
    auto multiply = [&](const uint4 (&m)[4], const uint4 (&b)[NT]) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                mma_16x8x16<BF16>(acc[z][n], m[2 * z].x, m[2 * z + 1].x, m[2 * z].y, m[2 * z + 1].y, b[n].x, b[n].y);
                mma_16x8x16<BF16>(acc[z][n], m[2 * z].z, m[2 * z + 1].z, m[2 * z].w, m[2 * z + 1].w, b[n].z, b[n].w);
            }
    };
    // whole steps of 32 features, a warp every kFewWarps-th group of kAhead; the step at the end by the last warp
    const int steps = a.features / 32;
    constexpr int kAhead = 4;
    for (int step0 = warp * kAhead; step0 < steps; step0 += kFewWarps * kAhead) {
        uint4 m[kAhead][4], b[kAhead][NT];
        const int n_here = min(kAhead, steps - step0);
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            const int k = (step0 + min(s, n_here - 1)) * 32;
#pragma unroll
            for (int i = 0; i < 4; ++i) m[s][i] = ptx::load_vector(w[i] + k);
#pragma unroll
            for (int n = 0; n < NT; ++n) b[s][n] = ptx::load_vector(xr[n] + k);
        }
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
            if (s < n_here) multiply(m[s], b[s]);
    }
    if (a.features % 32 && warp == kFewWarps - 1) {
        uint4 m[4], b[NT];
        const int k = steps * 32, left = a.features - t * 8;  // the pointers stand at column t * 8
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = load_end(w[i], k, left);
#pragma unroll
        for (int n = 0; n < NT; ++n) b[n] = load_end(xr[n], k, left);
        multiply(m, b);
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int unit = g + (e >> 1) * 8, row = n * 8 + 2 * t + (e & 1);
                sums[((warp * 2 + z) * kRows + row) * kFewUnits + unit] = acc[z][n][e];
            }
    __syncthreads();
    for (int i = tid; i < kRows * kFewUnits; i += 32 * kFewWarps) {
        const int unit = i % kFewUnits, row = i / kFewUnits;
        if (row >= a.rows || f0 + unit >= a.hidden) continue;
        float gate = 0.0f, up = 0.0f;
#pragma unroll
        for (int s = 0; s < kFewWarps; ++s) {
            gate += sums[(s * 2) * kRows * kFewUnits + i];
            up += sums[(s * 2 + 1) * kRows * kFewUnits + i];
        }
        const float value = a.act == kSilu ? act_value<kSilu>(gate) : a.act == kGelu ? act_value<kGelu>(gate) : act_value<kRelu>(gate);
        a.out[row * a.ld_out + f0 + unit] = static_cast<uint16_t>(pack2<BF16>(value * up, 0.0f));
    }
}

// ---- up to 128 rows: forward with the weights as the MMA's rows -------------------------
//
// The weights are still most of what is read, so they are the MMA's rows: a CTA multiplies `units` (up to 64, so
// many that the CTAs fill the SMs) rows of Wg and the same of Wu by all rows of x (N = rows, rounded up to 16), with
// a ring in shared memory that holds most of the SM's weights on their way. MMA rows past 2 units are whatever
// lies there and go nowhere. Gate and up of a unit (TMEM lanes u and units + u) meet through shared memory, from
// where whole row segments are stored. Measured against 256-row tiles: see launch_strip.

constexpr int kStripRows = 128;
constexpr int kStripStages = 16;
constexpr int kStripThreads = 192;  // producer, MMA issuer, four epilogue warps
constexpr int kStripPitch = kBM + 1;

struct StripParams {
    int kblocks, stages, n;  // n: columns of the MMA
    int units;
    int rows, hidden;
    uint16_t* out;
    long long ld_out;
    int* health;
};

template <bool BF16, int ACT>
__global__ void __launch_bounds__(kStripThreads, 1) strip_kernel(const __grid_constant__ Maps maps, const StripParams p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t full[kStripStages], empty[kStripStages], acc_full;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t stage_bytes = static_cast<uint32_t>(2 * p.units + p.n) * 128;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int f0 = blockIdx.x * p.units;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        ptx::mbar_init(&acc_full, 1);
        abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == 1) {
        ptx::tmem_alloc(&tmem_slot, 128);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    ptx::grid_release();
    ptx::grid_wait();
    if (warp == 0) {
        if (ptx::elect_one()) {
            int issued = 0;
            for (int kb = 0; kb < p.kblocks; ++kb) {
                const int s = kb % p.stages;
                if (!wait_bar(&empty[s], ((kb / p.stages) & 1) ^ 1, p.health, &abort_flag)) break;
                uint8_t* at = smem + s * stage_bytes;
                ptx::mbar_arrive_expect_tx(&full[s], stage_bytes);
                ptx::tma_load_3d(at, &maps.b0, &full[s], kb * kBK, f0, 0);
                ptx::tma_load_3d(at + p.units * 128, &maps.b1, &full[s], kb * kBK, f0, 0);
                ptx::tma_load_3d(at + 2 * p.units * 128, &maps.a, &full[s], kb * kBK, 0, 0);
                ++issued;
            }
            // every armed stage has landed before the CTA may end
            for (int s = 0; s < p.stages; ++s) {
                const int armed = issued > s ? (issued - 1 - s) / p.stages + 1 : 0;
                if (armed > 0) wait_bar(&full[s], (armed - 1) & 1, p.health, nullptr);
            }
        }
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            constexpr uint32_t fmt = BF16 ? 1u : 0u;
            const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((static_cast<uint32_t>(p.n) >> 3) << 17) | ((kBM >> 4) << 24);
            for (int kb = 0; kb < p.kblocks; ++kb) {
                const int s = kb % p.stages;
                if (!wait_bar(&full[s], (kb / p.stages) & 1, p.health, &abort_flag)) break;
                ptx::tc_fence_after();
                const uint32_t sa = ptx::smem_u32(smem + s * stage_bytes), sb = sa + 2 * p.units * 128;
#pragma unroll
                for (int j = 0; j < kBK / 16; ++j)
                    ptx::mma_f16(tmem, desc(sa + j * 32, 16, 1024), desc(sb + j * 32, 16, 1024), idesc, kb > 0 || j > 0 ? 1u : 0u);
                ptx::mma_commit(&empty[s]);
            }
            ptx::mma_commit(&acc_full);
            wait_bar(&acc_full, 0, p.health, nullptr);  // all MMAs have completed before TMEM is released
        }
    } else {
        const int q = warp & 3;  // TMEM lanes 32 q .. + 31
        const bool ready = wait_bar_warp(&acc_full, 0, p.health, &abort_flag);
        ptx::tc_fence_after();
        float* sums = reinterpret_cast<float*>(smem);  // [row][lane]: the ring is done with
        for (int c = 0; c < p.n; c += 16) {
            uint32_t r[16];
            ptx::tmem_ld16_issue(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, r);
            ptx::tmem_ld_wait(r);
            if (ready) {
#pragma unroll
                for (int e = 0; e < 16; ++e) sums[(c + e) * kStripPitch + q * 32 + lane] = __uint_as_float(r[e]);
            }
        }
        ptx::tc_fence_before();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int tid = threadIdx.x - 64, groups = p.units / 8;
        const bool vec = f0 + p.units <= p.hidden;  // the rows of h are 16-byte aligned
        for (int i = tid; i < p.rows * groups && ready; i += 128) {
            const int row = i / groups, u = i % groups * 8;
            const float* g = sums + row * kStripPitch + u;
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                h[e] = pack2<BF16>(act_value<ACT>(g[2 * e]) * g[p.units + 2 * e], act_value<ACT>(g[2 * e + 1]) * g[p.units + 2 * e + 1]);
            uint16_t* to = p.out + row * p.ld_out + f0 + u;
            if (vec) {
                *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (f0 + u + e < p.hidden) to[e] = static_cast<uint16_t>(h[e / 2] >> (16 * (e & 1)));
            }
        }
    }
    __syncthreads();
    __syncwarp();
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 128);
    }
}

// out_z[f][k] = sum over splits, in split order, of part[split][z][f][k]; z = gate, up (or one matrix alone)
template <typename OUT>
__device__ __forceinline__ OUT narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename OUT>
__global__ void reduce_kernel(const float* part, const float* scale, int splits, int matrices, int rows, int cols, int ld_part,
                              OUT* gate, long long ld_gate, OUT* up, long long ld_up, int* found_inf, int* health) {
    ptx::grid_release();
    ptx::grid_wait();
    const int quads = (cols + 3) / 4;
    const long long per = static_cast<long long>(rows) * quads;
    const long long plane = static_cast<long long>(rows) * ld_part;
    const float factor = scale ? *scale : 1.0f;
    bool over = false;
    auto rounded = [&](float v) {
        const OUT y = narrow<OUT>(v);
        over |= !(fabsf(static_cast<float>(y)) <= FLT_MAX);
        return y;
    };
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < matrices * per;
         i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int z = i >= per;
        const long long j = i - z * per;
        const long long row = j / quads;
        const int col = static_cast<int>(j - row * quads) * 4;
        const float* src = part + z * plane + row * ld_part + col;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
            const float4 v = *reinterpret_cast<const float4*>(src + static_cast<long long>(matrices) * s * plane);
            sum.x += v.x;
            sum.y += v.y;
            sum.z += v.z;
            sum.w += v.w;
        }
        OUT* dst = (z ? up + row * ld_up : gate + row * ld_gate) + col;
        dst[0] = rounded(sum.x * factor);
        if (col + 1 < cols) dst[1] = rounded(sum.y * factor);
        if (col + 2 < cols) dst[2] = rounded(sum.z * factor);
        if (col + 3 < cols) dst[3] = rounded(sum.w * factor);
    }
    if (over) report_overflow(found_inf, health);
}

// ---- host ---------------------------------------------------------------------

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static const EncodeTiled fn = [] {
        void* q = nullptr;
        cudaDriverEntryPointQueryResult r;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess &&
                       r == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<EncodeTiled>(q)
                   : nullptr;
    }();
    return fn;
}

struct Plan {
    int rows, features, hidden, bf16, act;
    int device, pairs;  // CTA pairs resident at once
};

// Tensor map of `rank` dimensions (extents and box in elements, strides in bytes from the second dimension on), the
// box's rows swizzled over their width.
bool encode(CUtensorMap* map, const char* what, CUtensorMapDataType type, const void* base, int rank,
            std::initializer_list<long long> extents, std::initializer_list<long long> strides, std::initializer_list<int> box) {
    cuuint64_t dims[4], steps[3];
    cuuint32_t boxes[4];
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    std::copy(extents.begin(), extents.end(), dims);
    std::copy(strides.begin(), strides.end(), steps);
    std::copy(box.begin(), box.end(), boxes);
    const int row_bytes = *box.begin() * (type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2);
    const CUtensorMapSwizzle swizzle = row_bytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                       : row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                         : CU_TENSOR_MAP_SWIZZLE_32B;
    const CUresult r = encoder()(map, type, rank, const_cast<void*>(base), dims, steps, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return true;
    set_error("gated MLP: tensor map of %s failed (%d) for %lld x %lld", what, static_cast<int>(r), *extents.begin(),
              *(extents.begin() + 1));
    return false;
}

// {inner, outer, depth} elements at base; boxes of box_inner x box_outer
bool make_map(CUtensorMap* map, const char* what, CUtensorMapDataType type, const void* base, long long inner,
              long long outer, long long depth, long long ld, long long depth_stride, int box_inner, int box_outer) {
    const int elem = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
    return encode(map, what, type, base, 3, {inner, outer, depth}, {ld * elem, depth_stride * elem}, {box_inner, box_outer, 1});
}

// An N-contiguous 16-bit operand (`cols` contiguous, contraction over `rows`) for load_chunks: with whole 64-wide
// chunks the matrix is seen as {64, rows, cols / 64} and one box takes `chunks` of them; otherwise (the last chunk
// would read past the last row) as it is, a box a chunk.
bool make_chunk_map(CUtensorMap* map, int* merged, const char* what, CUtensorMapDataType type, const void* base, long long cols,
                    long long rows, long long ld, int chunks) {
    *merged = cols % 64 == 0;
    return encode(map, what, type, base, 3, {*merged ? 64 : cols, rows, *merged ? cols / 64 : 1},
                  {ld * 2, *merged ? 128 : ld * rows * 2}, {64, kBK, *merged ? chunks : 1});
}

// The workspace's blocks of dg and du: {64 hidden units, 128 rows, blocks of hidden units, blocks of rows of both}.
bool make_block_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long hidden_blocks, long long row_blocks,
                    int box_units, int box_rows, int box_blocks) {
    return encode(map, "hidden gradients", type, base, 4, {64, kBM, hidden_blocks, 2 * row_blocks},
                  {128, kBM * 128, hidden_blocks * kBM * 128}, {box_units, box_rows, box_blocks, 1});
}

bool matrix_ok(const char* what, const void* base, long long ld, long long cols, int elem) {
    if (base && aligned(base, 16) && ld >= cols && (ld * elem) % 16 == 0) return true;
    set_error("gated MLP: %s must be non-null, 16-byte aligned, with a row stride >= %lld that is a multiple of 16 bytes "
              "(got stride %lld)", what, cols, ld);
    return false;
}

// What of a call may not share memory: an output and what is still read, or written, when it is written.
bool apart(const char* what, const Extent& out, std::initializer_list<Extent> others) {
    for (const Extent& other : others)
        if (overlap(out, other)) {
            set_error("gated MLP: %s may not overlap the operands or another output", what);
            return false;
        }
    return true;
}

typedef void (*KernelFn)(const Maps, const Params);

int launched(cudaError_t e) {
    if (e == cudaSuccess) return launch_status("gated MLP");
    set_error("gated MLP launch: %s", cudaGetErrorString(e));
    return -1;
}

template <bool BF16>
int launch_few(const FewArgs& a, cudaStream_t stream) {
    const int blocks = (a.hidden + kFewUnits - 1) / kFewUnits;
    constexpr int kSums = kFewWarps * 2 * 8 * kFewUnits * 4;  // bytes per 8 rows
    const bool eight = a.rows <= 8;
    return launched(launch_early(eight ? few_rows_kernel<BF16, 1> : few_rows_kernel<BF16, 2>, blocks, 32 * kFewWarps,
                                 eight ? kSums : 2 * kSums, stream, a));
}

template <bool BF16>
KernelFn gated_kernel(int mode, int act) {
    if (mode == kForward)
        return act == kSilu ? product_kernel<kForward, BF16, kSilu, false>
                            : act == kGelu ? product_kernel<kForward, BF16, kGelu, false>
                                           : product_kernel<kForward, BF16, kRelu, false>;
    return act == kSilu ? product_kernel<kGate, BF16, kSilu, false>
                        : act == kGelu ? product_kernel<kGate, BF16, kGelu, false>
                                       : product_kernel<kGate, BF16, kRelu, false>;
}

KernelFn kernel_of(const Plan* plan, int mode, bool out32) {
    if (mode == kForward || mode == kGate)
        return plan->bf16 ? gated_kernel<true>(mode, plan->act) : gated_kernel<false>(mode, plan->act);
    if (mode == kInput && out32) return plan->bf16 ? product_kernel<kInput, true, 0, true> : product_kernel<kInput, false, 0, true>;
    if (mode == kInput) return plan->bf16 ? product_kernel<kInput, true, 0, false> : product_kernel<kInput, false, 0, false>;
    if (out32) return plan->bf16 ? product_kernel<kWeight, true, 0, true> : product_kernel<kWeight, false, 0, true>;
    return plan->bf16 ? product_kernel<kWeight, true, 0, false> : product_kernel<kWeight, false, 0, false>;
}

constexpr int kStaticSmem = 1024;  // room left for the barriers, the TMEM slot and the abort word

int launch(const Plan* plan, int mode, bool out32, Params& p, const Maps& maps, cudaStream_t stream) {
    const int stage = (kBM + p.bnc) * 128;
    const int fixed = 1024 + epi_warps(mode) * boxes_of(mode) * box_bytes(mode);
    p.stages = std::min(kMaxStages, (kMaxSmem - kStaticSmem - fixed) / stage);
    const long long total = static_cast<long long>(p.tiles_n) * p.tiles_m * p.tiles_z * p.splits;
    if (total > 0x3FFFFFFF) {
        set_error("gated MLP: too many output tiles");
        return -1;
    }
    p.tiles_total = static_cast<int>(total);
    const int pairs = static_cast<int>(std::min<long long>(total, plan->pairs));
    return launched(launch_early(kernel_of(plan, mode, out32), 2 * pairs, threads_of(mode), p.stages * stage + fixed, stream, maps, p));
}

// Tile width: 128 B rows per CTA, or 64 where that ends sooner, by waves of tiles times a tile's cost (its width,
// and its share of the A rows as much as 16 columns). The backward at 8192 x 512 x 2048 took 118 us with 128
// throughout and takes 104 so.
int width_for(const Plan* plan, long long row_tiles, long long cols, int per_row) {
    auto cost = [&](int width) {
        const long long tiles = row_tiles * ((cols + width * per_row - 1) / (width * per_row));
        return (tiles + plan->pairs - 1) / plan->pairs * (width + 16);
    };
    return cost(64) < cost(128) ? 64 : 128;
}

// Splits of the weight gradients' contraction over `rows`: one tile per pair where the splits stay at least 16
// k-blocks long; and chains that keep the tensor cores' fp32 accumulation error (about 7e-9 a product, measured)
// below a quarter of the operands' rounding: 16384 rows for fp16, 65536 for bf16.
int splits_for(const Plan* plan, int rows) {
    const long long row_tiles = 2LL * ((plan->hidden + 255) / 256);
    const int width = 2 * width_for(plan, row_tiles, plan->features, 2);
    const long long tiles = row_tiles * ((plan->features + width - 1) / width);
    const int kblocks = (rows + kBK - 1) / kBK;
    const long long fill = std::max<long long>(1, std::min<long long>(plan->pairs / tiles, kblocks / 16));
    const int chain = plan->bf16 ? 1024 : 256;
    return static_cast<int>(std::max<long long>(fill, (kblocks + chain - 1) / chain));
}

long long pad(long long cols, long long to) { return (cols + to - 1) / to * to; }

// inner extent of an output's tensor map: whole granules (rows shorter than one are not stored by it)
long long stored(long long cols, long long granule) { return std::max(granule, cols / granule * granule); }

// blocks of dg (of du) for so many rows: of 128 rows (whole pair tiles), and of 64 hidden units (whole tiles)
int row_blocks(int rows) { return (rows + 2 * kBM - 1) / (2 * kBM) * 2; }
int hidden_blocks(const Plan* plan, int rows) {
    const int width = width_for(plan, row_blocks(rows) / 2, plan->hidden, 1);
    return (plan->hidden + width - 1) / width * (width / 64);
}

// workspace: dg and du, then (when split) the fp32 partial weight gradients
long long gate_bytes(const Plan* plan) {
    return 2LL * row_blocks(plan->rows) * ((plan->hidden + 127) / 128 * 2) * kBM * 128;
}
long long part_bytes(const Plan* plan) {  // the weight gradients' splits grow with the rows
    const long long s = splits_for(plan, plan->rows);
    const long long weights = s > 1 ? s * 2 * plan->hidden * pad(plan->features, 4) * 4 : 0;
    // the input gradient's partial sums: at most a 256 x 128 tile (its last columns padded to 4) per pair
    return std::max(weights, plan->pairs * 256LL * 132 * 4);
}

bool ready(const Plan* plan, int rows) {
    if (!plan) {
        set_error("null gated MLP plan");
        return false;
    }
    if (rows < 0 || rows > plan->rows) {
        set_error("gated MLP: rows must be 0..%d (got %d)", plan->rows, rows);
        return false;
    }
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess || device != plan->device) {
        set_error("gated MLP: the plan belongs to device %d, the current device is %d", plan->device, device);
        return false;
    }
    return true;
}

// The two projections: forward (out = h) or backward (grad_out in, dg and du out).
int project(const Plan* plan, int rows, const void* x, long long ldx, const void* wg, long long ldg, const void* wu,
            long long ldu, const void* grad_out, long long ld_grad, void* out, long long ld_out, int* found_inf, int* health,
            cudaStream_t stream) {
    const int K = plan->features, F = plan->hidden;
    const CUtensorMapDataType type = plan->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const int mode = grad_out ? kGate : kForward;
    Params p{};
    p.tiles_m = (rows + 2 * kBM - 1) / (2 * kBM);
    p.bnc = width_for(plan, p.tiles_m, F, 1);
    p.tile_cols = p.bnc;
    p.tiles_n = (F + p.bnc - 1) / p.bnc;
    p.tiles_z = p.splits = 1;
    p.kblocks = p.kb_per_split = (K + kBK - 1) / kBK;
    p.box_cols = p.bnc / (epi_warps(mode) / 4);
    p.out_rows = rows;
    p.out_cols = F;
    p.store_cols = F / 8 * 8;
    p.row_blocks = row_blocks(rows);
    p.out[0] = out;
    p.ld_out[0] = ld_out;
    p.found_inf = found_inf;
    p.health = health;
    Maps maps;
    if (!make_map(&maps.a, "x", type, x, K, rows, 1, ldx, ldx * rows, kBK, kBM) ||
        !make_map(&maps.b0, "gate weight", type, wg, K, F, 1, ldg, ldg * F, kBK, p.bnc) ||
        !make_map(&maps.b1, "up weight", type, wu, K, F, 1, ldu, ldu * F, kBK, p.bnc) ||
        !(grad_out ? make_block_map(&maps.d0, type, out, hidden_blocks(plan, rows), p.row_blocks, p.box_cols, 32, 1)
                   : make_map(&maps.d0, "output", type, out, stored(F, 8), rows, 1, ld_out, ld_out * rows, p.box_cols, 32)))
        return -1;
    maps.d1 = maps.in = maps.d0;
    if (grad_out && !make_map(&maps.in, "output gradient", type, grad_out, F, rows, 1, ld_grad, ld_grad * rows, p.box_cols, 32))
        return -1;
    return launch(plan, mode, false, p, maps, stream);
}

template <typename OUT>
cudaError_t reduce_as(const float* part, const float* scale, int splits, int matrices, int rows, int cols, int ld, void* first, long long ld_first,
               void* second, long long ld_second, int* found_inf, int* health, cudaStream_t stream) {
    const long long quads = static_cast<long long>(matrices) * rows * ((cols + 3) / 4);
    const int blocks = static_cast<int>(std::min<long long>((quads + 255) / 256, 148 * 8));
    return launch_early(reduce_kernel<OUT>, blocks, 256, 0, stream, part, scale, splits, matrices, rows, cols, ld, static_cast<OUT*>(first),
                        ld_first, static_cast<OUT*>(second), ld_second, found_inf, health);
}

int reduce(const Plan* plan, bool fp32, const float* part, const float* scale, int splits, int matrices, int rows, int cols, int ld, void* first,
           long long ld_first, void* second, long long ld_second, int* found_inf, int* health, cudaStream_t stream) {
    const auto run = fp32 ? reduce_as<float> : plan->bf16 ? reduce_as<__nv_bfloat16> : reduce_as<__half>;
    return launched(run(part, scale, splits, matrices, rows, cols, ld, first, ld_first, second, ld_second, found_inf, health, stream));
}

// 17 to 128 rows, forward. Device time for that of the 256-row tiles: 15.0 us for 20.3 (32 rows) and 17.5 for 22.2
// (128 rows) at 2048 x 8192 fp16, 6.5 for 7.4 (64 rows) at 512 x 2048 bf16; 4.5 TB/s of weights.
int launch_strip(const Plan* plan, const rl2_gated_forward_args* g, cudaStream_t stream) {
    const int K = plan->features, F = plan->hidden;
    const CUtensorMapDataType type = plan->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    StripParams p{};
    p.kblocks = (K + kBK - 1) / kBK;
    p.n = (g->rows + 15) / 16 * 16;
    p.rows = g->rows;
    p.hidden = F;
    p.out = static_cast<uint16_t*>(g->out);
    p.ld_out = g->ld_out;
    p.health = g->health;
    // units a CTA: the least (waves of CTAs) x (units + a CTA's own cost, about that of 8 units)
    p.units = 64;
    auto cost = [&](int units) { return ((F + units - 1) / units + 2 * plan->pairs - 1) / (2 * plan->pairs) * (units + 8); };
    for (int units = 56; units >= 16; units -= 8)
        if (cost(units) < cost(p.units)) p.units = units;
    // the MMA reads kBM rows from a stage's start on, past the last stage's end where 2 units are fewer
    const int stage = (2 * p.units + p.n) * 128, tail = std::max(0, kBM * 128 - stage);
    p.stages = std::min({kStripStages, p.kblocks, (kMaxSmem - kStaticSmem - 1024 - tail) / stage});
    const int smem = std::max(p.stages * stage + tail, p.n * kStripPitch * 4) + 1024;
    Maps maps;
    if (!make_map(&maps.a, "x", type, g->x, K, g->rows, 1, g->ldx, g->ldx * g->rows, kBK, p.n) ||
        !make_map(&maps.b0, "gate weight", type, g->gate_weight, K, F, 1, g->ld_gate, g->ld_gate * F, kBK, p.units) ||
        !make_map(&maps.b1, "up weight", type, g->up_weight, K, F, 1, g->ld_up, g->ld_up * F, kBK, p.units))
        return -1;
    maps.d0 = maps.d1 = maps.in = maps.a;
    void (*const kernels[2][3])(const Maps, const StripParams) = {
        {strip_kernel<false, kSilu>, strip_kernel<false, kGelu>, strip_kernel<false, kRelu>},
        {strip_kernel<true, kSilu>, strip_kernel<true, kGelu>, strip_kernel<true, kRelu>}};
    const auto kernel = kernels[plan->bf16][plan->act];
    static std::atomic<unsigned long long> allowed[2][3];  // devices (up to 64) whose limit is raised
    std::atomic<unsigned long long>& seen = allowed[plan->bf16][plan->act];
    if (plan->device > 63 || !(seen.load() >> plan->device & 1)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem - kStaticSmem);
        if (e != cudaSuccess) {
            set_error("gated MLP: %s", cudaGetErrorString(e));
            return -1;
        }
        if (plan->device <= 63) seen.fetch_or(1ull << plan->device);
    }
    return launched(launch_early(kernel, (F + p.units - 1) / p.units, kStripThreads, smem, stream, maps, p));
}

int input_gradient(const Plan* plan, const rl2_gated_backward_args* g, cudaStream_t stream) {
    const int K = plan->features, F = plan->hidden, rows = g->rows;
    const CUtensorMapDataType type = plan->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    Params p{};
    p.row_blocks = row_blocks(rows);
    p.tiles_m = (rows + 2 * kBM - 1) / (2 * kBM);
    p.bnc = width_for(plan, p.tiles_m, K, 2);
    p.tile_cols = 2 * p.bnc;
    p.tiles_n = (K + p.tile_cols - 1) / p.tile_cols;
    p.tiles_z = 1;
    p.kb_segment = (F + kBK - 1) / kBK;
    p.kblocks = 2 * p.kb_segment;
    // few tiles: the contraction in pieces of at least 16 k-blocks, while each adds pairs at work
    p.splits = static_cast<int>(std::max<long long>(1, std::min<long long>(plan->pairs / (static_cast<long long>(p.tiles_m) * p.tiles_n), p.kblocks / 16)));
    p.kb_per_split = (p.kblocks + p.splits - 1) / p.splits;
    p.splits = (p.kblocks + p.kb_per_split - 1) / p.kb_per_split;  // every split non-empty
    const bool split = p.splits > 1;
    const long long ldp = pad(K, 4);
    float* part = reinterpret_cast<float*>(static_cast<char*>(g->workspace) + gate_bytes(plan));
    p.box_cols = split ? 32 : 64;
    p.out_rows = rows;
    p.out_cols = K;
    p.store_cols = split ? K : K / 8 * 8;
    p.out[0] = g->grad_x;
    p.ld_out[0] = g->ld_grad_x;
    p.found_inf = g->found_inf;
    p.health = g->health;
    Maps maps;
    if (!make_block_map(&maps.a, type, g->workspace, hidden_blocks(plan, rows), p.row_blocks, 64, kBM, 1) ||
        !make_chunk_map(&maps.b0, &p.b_merged, "gate weight", type, g->gate_weight, K, F, g->ld_gate, p.bnc / 64) ||
        !make_chunk_map(&maps.b1, &p.b_merged, "up weight", type, g->up_weight, K, F, g->ld_up, p.bnc / 64) ||
        !(split ? make_map(&maps.d0, "partial input gradients", CU_TENSOR_MAP_DATA_TYPE_FLOAT32, part, K, rows, p.splits, ldp, ldp * rows, 32, 32)
                : make_map(&maps.d0, "input gradient", type, g->grad_x, stored(K, 8), rows, 1, g->ld_grad_x, g->ld_grad_x * rows, 64, 32)))
        return -1;
    maps.d1 = maps.in = maps.d0;
    if (launch(plan, kInput, split, p, maps, stream)) return -1;
    return split ? reduce(plan, false, part, nullptr, p.splits, 1, rows, K, static_cast<int>(ldp), g->grad_x, g->ld_grad_x, nullptr, 0, g->found_inf, g->health, stream) : 0;
}


int weight_gradients(const Plan* plan, const rl2_gated_backward_args* g, cudaStream_t stream) {
    const int K = plan->features, F = plan->hidden, rows = g->rows;
    const CUtensorMapDataType type = plan->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const long long ldp = pad(K, 4);
    Params p{};
    p.row_blocks = row_blocks(rows);
    p.tiles_m = (F + 2 * kBM - 1) / (2 * kBM);
    p.tiles_z = 2;
    p.kblocks = (rows + kBK - 1) / kBK;
    p.splits = splits_for(plan, rows);
    p.kb_per_split = (p.kblocks + p.splits - 1) / p.splits;
    p.splits = (p.kblocks + p.kb_per_split - 1) / p.kb_per_split;  // every split non-empty
    p.bnc = width_for(plan, 2LL * p.tiles_m, K, 2);
    p.tile_cols = 2 * p.bnc;
    p.tiles_n = (K + p.tile_cols - 1) / p.tile_cols;
    p.out_rows = F;
    p.out_cols = K;
    p.found_inf = g->found_inf;
    p.health = g->health;
    float* part = reinterpret_cast<float*>(static_cast<char*>(g->workspace) + gate_bytes(plan));
    const bool out32 = p.splits > 1 || g->grad_weight_fp32;
    const CUtensorMapDataType out_type = out32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type;
    p.box_cols = out32 ? 32 : 64;
    const int granule = out32 ? 4 : 8;
    p.store_cols = p.splits > 1 ? K : K / granule * granule;
    p.out[0] = g->grad_gate;
    p.out[1] = g->grad_up;
    p.ld_out[0] = g->ld_grad_gate;
    p.ld_out[1] = g->ld_grad_up;
    p.scale = p.splits > 1 ? nullptr : g->grad_weight_scale;
    Maps maps;
    if (!make_block_map(&maps.a, type, g->workspace, hidden_blocks(plan, rows), p.row_blocks, 64, kBK, kBM / 64) ||
        !make_chunk_map(&maps.b0, &p.b_merged, "x", type, g->x, K, rows, g->ldx, p.bnc / 64))
        return -1;
    maps.b1 = maps.b0;
    if (p.splits > 1) {
        if (!make_map(&maps.d0, "partial weight gradients", out_type, part, K, F, 2LL * p.splits, ldp, ldp * F, 32, 32)) return -1;
        maps.d1 = maps.d0;
    } else if (!make_map(&maps.d0, "gate weight gradient", out_type, g->grad_gate, stored(K, granule), F, 1, g->ld_grad_gate,
                         g->ld_grad_gate * F, p.box_cols, 32) ||
               !make_map(&maps.d1, "up weight gradient", out_type, g->grad_up, stored(K, granule), F, 1, g->ld_grad_up,
                         g->ld_grad_up * F, p.box_cols, 32)) {
        return -1;
    }
    maps.in = maps.d0;
    if (launch(plan, kWeight, out32, p, maps, stream)) return -1;
    if (p.splits == 1) return 0;
    return reduce(plan, g->grad_weight_fp32, part, g->grad_weight_scale, p.splits, 2, F, K, static_cast<int>(ldp), g->grad_gate,
                  g->ld_grad_gate, g->grad_up, g->ld_grad_up, g->found_inf, g->health, stream);
}

}  // namespace gated
}  // namespace rl2

extern "C" void* rl2_gated_create(const rl2_gated_desc* d) {
    using namespace rl2;
    using namespace rl2::gated;
    clear_error();
    if (!d || d->rows < 1 || d->features < 1 || d->hidden < 1 || d->rows > (1 << 28) || d->features > (1 << 24) ||
        d->hidden > (1 << 24)) {
        set_error("gated MLP: rows (up to 2^28), features and hidden (up to 2^24) must be positive");
        return nullptr;
    }
    if ((d->dtype != 0 && d->dtype != 1) || d->activation < 0 || d->activation > 2) {
        set_error("gated MLP: dtype must be 0 (fp16) or 1 (bf16), activation 0 (SiLU), 1 (GELU) or 2 (ReLU)");
        return nullptr;
    }
    if (!encoder()) {
        set_error("cuTensorMapEncodeTiled is unavailable from the driver");
        return nullptr;
    }
    Plan* plan = new (std::nothrow) Plan{d->rows, d->features, d->hidden, d->dtype, d->activation, 0, 0};
    if (!plan) {
        set_error("out of host memory");
        return nullptr;
    }
    // pairs resident at once, asked (and the kernels' shared memory limits raised) once a device and kernel
    static std::atomic<int> resident[64][2][3][6];
    int sms = 0;
    bool ok = cudaGetDevice(&plan->device) == cudaSuccess &&
              cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, plan->device) == cudaSuccess;
    plan->pairs = sms / 2;
    for (int i = 0; ok && i < 6; ++i) {  // the four modes, then kInput and kWeight with fp32 outputs
        std::atomic<int>* known = plan->device < 64 ? &resident[plan->device][d->dtype][d->activation][i] : nullptr;
        int clusters = known ? known->load() : 0;
        if (clusters == 0) {
            const void* fn = reinterpret_cast<const void*>(kernel_of(plan, i < 4 ? i : i - 2, i >= 4));
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 2;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.gridDim = dim3(static_cast<unsigned>(2 * std::max(1, sms / 2)));
            cfg.blockDim = dim3(threads_of(i < 4 ? i : i - 2));
            cfg.dynamicSmemBytes = kMaxSmem - kStaticSmem;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            ok = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem - kStaticSmem) == cudaSuccess &&
                 cudaOccupancyMaxActiveClusters(&clusters, fn, &cfg) == cudaSuccess && clusters > 0;
            if (ok && known) known->store(clusters);
        }
        plan->pairs = std::min(plan->pairs, clusters);
    }
    if (!ok) {
        set_error("gated MLP: no pair of CTAs fits the current device (%s)", cudaGetErrorString(cudaGetLastError()));
        delete plan;
        return nullptr;
    }
    return plan;
}

extern "C" int rl2_gated_destroy(void* plan) {
    rl2::clear_error();
    delete static_cast<rl2::gated::Plan*>(plan);
    return 0;
}

extern "C" long long rl2_gated_workspace_bytes(void* opaque) {
    using namespace rl2::gated;
    const Plan* plan = static_cast<const Plan*>(opaque);
    return plan ? gate_bytes(plan) + part_bytes(plan) : -1;
}

extern "C" int rl2_gated_forward(void* opaque, const rl2_gated_forward_args* g, void* stream) {
    using namespace rl2;
    using namespace rl2::gated;
    clear_error();
    const Plan* plan = static_cast<const Plan*>(opaque);
    if (!g) {
        set_error("gated MLP: null arguments");
        return -1;
    }
    if (!ready(plan, g->rows)) return -1;
    if (g->rows == 0) return 0;
    if (!matrix_ok("x", g->x, g->ldx, plan->features, 2) ||
        !matrix_ok("gate weight", g->gate_weight, g->ld_gate, plan->features, 2) ||
        !matrix_ok("up weight", g->up_weight, g->ld_up, plan->features, 2) ||
        !matrix_ok("output", g->out, g->ld_out, plan->hidden, 2))
        return -1;
    const long long K = plan->features, F = plan->hidden;
    if (!apart("output", {g->out, g->rows, F * 2, g->ld_out * 2},
               {{g->x, g->rows, K * 2, g->ldx * 2}, {g->gate_weight, F, K * 2, g->ld_gate * 2}, {g->up_weight, F, K * 2, g->ld_up * 2}}))
        return -1;
    if (g->rows <= kFewRows) {
        const FewArgs few{static_cast<const uint16_t*>(g->x), static_cast<const uint16_t*>(g->gate_weight),
                          static_cast<const uint16_t*>(g->up_weight), static_cast<uint16_t*>(g->out), g->ldx, g->ld_gate, g->ld_up,
                          g->ld_out, g->rows, plan->features, plan->hidden, plan->act};
        return plan->bf16 ? launch_few<true>(few, as_stream(stream)) : launch_few<false>(few, as_stream(stream));
    }
    if (g->rows <= kStripRows) return launch_strip(plan, g, as_stream(stream));
    return project(plan, g->rows, g->x, g->ldx, g->gate_weight, g->ld_gate, g->up_weight, g->ld_up, nullptr, 0, g->out,
                   g->ld_out, nullptr, g->health, as_stream(stream));
}

extern "C" int rl2_gated_backward(void* opaque, const rl2_gated_backward_args* g, void* stream) {
    using namespace rl2;
    using namespace rl2::gated;
    clear_error();
    const Plan* plan = static_cast<const Plan*>(opaque);
    if (!g) {
        set_error("gated MLP: null arguments");
        return -1;
    }
    if (!ready(plan, g->rows)) return -1;
    const int K = plan->features, F = plan->hidden;
    const int elem = g->grad_weight_fp32 ? 4 : 2;
    const bool weights = g->grad_gate || g->grad_up;
    if (!weights && !g->grad_x) {
        set_error("gated MLP backward: no gradient asked for");
        return -1;
    }
    if (weights && (!matrix_ok("gate weight gradient", g->grad_gate, g->ld_grad_gate, K, elem) ||
                    !matrix_ok("up weight gradient", g->grad_up, g->ld_grad_up, K, elem)))
        return -1;
    cudaStream_t s = as_stream(stream);
    if (g->rows == 0) {
        if (weights && (cudaMemset2DAsync(g->grad_gate, g->ld_grad_gate * elem, 0, static_cast<size_t>(K) * elem, F, s) != cudaSuccess ||
                        cudaMemset2DAsync(g->grad_up, g->ld_grad_up * elem, 0, static_cast<size_t>(K) * elem, F, s) != cudaSuccess)) {
            set_error("gated MLP backward: clearing the weight gradients failed");
            return -1;
        }
        return 0;
    }
    if (!matrix_ok("x", g->x, g->ldx, K, 2) || !matrix_ok("gate weight", g->gate_weight, g->ld_gate, K, 2) ||
        !matrix_ok("up weight", g->up_weight, g->ld_up, K, 2) || !matrix_ok("output gradient", g->grad_out, g->ld_grad_out, F, 2) ||
        (g->grad_x && !matrix_ok("input gradient", g->grad_x, g->ld_grad_x, K, 2)))
        return -1;
    if (!g->workspace || !aligned(g->workspace, 256)) {
        set_error("gated MLP backward: the workspace must be non-null and 256-byte aligned");
        return -1;
    }
    if (g->grad_x == g->x) {
        set_error("gated MLP backward: grad_x may not be x (the weight gradients read x after it is written)");
        return -1;
    }
    // grad_out is done with before any gradient is written, the weights before theirs
    const Extent x{weights ? g->x : nullptr, g->rows, K * 2LL, g->ldx * 2}, dx{g->grad_x, g->rows, K * 2LL, g->ld_grad_x * 2};
    const Extent gate{g->gate_weight, F, K * 2LL, g->ld_gate * 2}, up{g->up_weight, F, K * 2LL, g->ld_up * 2};
    const Extent dgate{g->grad_gate, F, static_cast<long long>(K) * elem, g->ld_grad_gate * elem};
    const Extent dup{g->grad_up, F, static_cast<long long>(K) * elem, g->ld_grad_up * elem};
    if (!apart("grad_x", dx, {x, gate, up, dgate, dup}) || !apart("grad_gate", dgate, {x, dup}) || !apart("grad_up", dup, {x})) return -1;
    if (project(plan, g->rows, g->x, g->ldx, g->gate_weight, g->ld_gate, g->up_weight, g->ld_up, g->grad_out,
                g->ld_grad_out, g->workspace, 0, g->found_inf, g->health, s))
        return -1;
    if (g->grad_x && input_gradient(plan, g, s)) return -1;
    return weights ? weight_gradients(plan, g, s) : 0;
}
