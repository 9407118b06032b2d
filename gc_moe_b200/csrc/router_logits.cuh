// Router logits: logits[t][e] = sum_k x[t][k] * W[e][k], BF16 activations, f32 sums and result.
//
// W is kept as P BF16 planes [P][E][H] whose sum is the router's weight: one plane for a BF16
// weight, three for an f32 weight (8 + 8 + 8 significant bits), so that every product is an
// exact product of BF16 values and the result has the accuracy of f32 sums.
//
// Sums are added in an order that the sizes fix: no atomics.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "device_common.cuh"
#include "ptx.cuh"
#include "rms_norm.cuh"

namespace gcmoe {

constexpr uint32_t kLogitsThreads = 256;

struct LogitsParams {
    const __nv_bfloat16* x;       // [T][H]
    const __nv_bfloat16* weight;  // [P][E][H]
    float* out;                   // [T][E]
    uint64_t x_stride;            // elements between rows
    uint32_t num_tokens, num_experts, hidden;
};

// Few tokens: bound by the latency of the loads, so a thread has the loads of kRounds rounds
// of the loop in flight, and all CTAs should be resident at once.  A thread adds its channels
// in the same order in every variant.  The launch chooses one; with nine tokens, in four and
// on the tensor cores: 5120 x 384 5.1 and 4.2 us, FP32 weight 7.3 and 4.6; 4096 x 64 3.4 and 3.5.
constexpr uint32_t kFmaMaxTokens = 8;

// CTAs of an SM, the least that the compiler has to leave registers for.
template <int kTokens, int kPlanes>
constexpr uint32_t kFmaResident = kPlanes == 3 ? 2 : kTokens <= 2 ? 4 : 3;

template <int kTokens, int kPlanes, int kRounds>
__global__ void __launch_bounds__(kLogitsThreads, kFmaResident<kTokens, kPlanes>)
    logits_fma_kernel(const __grid_constant__ LogitsParams p) {
    constexpr int kExperts = 2, kSums = kTokens * kExperts;
    __shared__ float partial[kLogitsThreads / 32][kSums];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t e0 = blockIdx.x * kExperts, t0 = blockIdx.y * kTokens;
    const uint32_t chunks = p.hidden / 8;
    ptx::launch_dependents();
    ptx::grid_dependency_wait();

    // rows past the last are the last row again: loaded, never stored
    const uint4* x[kTokens];
    const uint4* w[kExperts];
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
        x[i] = reinterpret_cast<const uint4*>(p.x + min(t0 + i, p.num_tokens - 1) * p.x_stride);
#pragma unroll
    for (int e = 0; e < kExperts; ++e)
        w[e] = reinterpret_cast<const uint4*>(p.weight + uint64_t(min(e0 + e, p.num_experts - 1)) * p.hidden);
    const uint64_t plane = uint64_t(p.num_experts) * chunks;

    float acc[kTokens][kExperts] = {};
    for (uint32_t c0 = tid; c0 < chunks; c0 += kLogitsThreads * kRounds) {
        uint4 xr[kRounds][kTokens], wr[kRounds][kExperts][kPlanes];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const uint32_t c = c0 + r * kLogitsThreads;
            const bool in = c < chunks;
#pragma unroll
            for (int i = 0; i < kTokens; ++i) xr[r][i] = in ? __ldca(x[i] + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < kExperts; ++e)
#pragma unroll
                for (int q = 0; q < kPlanes; ++q) wr[r][e][q] = in ? __ldca(w[e] + q * plane + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < kRounds; ++r)
#pragma unroll
            for (int e = 0; e < kExperts; ++e) {
                float v[8];
                unpack_bf16x8(wr[r][e][0], v);
                if constexpr (kPlanes == 3) {              // exact: the planes are the bits of one f32
                    float mid[8], low[8];
                    unpack_bf16x8(wr[r][e][1], mid);
                    unpack_bf16x8(wr[r][e][2], low);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += mid[j] + low[j];
                }
#pragma unroll
                for (int i = 0; i < kTokens; ++i) {
                    float u[8];
                    unpack_bf16x8(xr[r][i], u);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[i][e] = fmaf(u[j], v[j], acc[i][e]);
                }
            }
    }
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
#pragma unroll
        for (int e = 0; e < kExperts; ++e) {
            float v = acc[i][e];
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
            if (lane == 0) partial[warp][i * kExperts + e] = v;
        }
    __syncthreads();
    if (tid < kSums) {
        const uint32_t t = t0 + tid / kExperts, e = e0 + tid % kExperts;
        float v = 0.f;
#pragma unroll
        for (uint32_t g = 0; g < kLogitsThreads / 32; ++g) v += partial[g][tid];
        if (t < p.num_tokens && e < p.num_experts) p.out[static_cast<uint64_t>(t) * p.num_experts + e] = v;
    }
}

// ---------------------------------------------------------------------------------------
// Tensor-core form, for more than a few tokens: tiles of kM tokens x kN experts, the K
// blocks (64 channels) of a tile split over CTAs of a cluster, whose partial tiles are added
// through distributed shared memory in rank order.
//
// The planes of an f32 weight are further columns of the tile's product: x is loaded once for
// all three, and an MMA of 96 columns takes the time of one of 32 (the x operand's way out of
// shared memory).  They are added to one sum when the accumulators are read.
//
// The tensor core truncates each addition to its f32 accumulator, always towards zero:
// measured, the result of a K = 7168 product is 6.7e-6 too small in magnitude (relative
// error 7.9e-6), growing with the number of MMAs in a chain.  So a chain ends after
// kChainBlocks K blocks (512 channels: 4.7e-7) and its accumulator is added to f32 sums in
// registers, rounded to nearest; two accumulators in TMEM keep the MMAs going meanwhile.
//
// Bound by launch, load latency and the partial tiles' exchange for up to a few hundred
// tokens (33 x 5120 x 384: 4.2 us, an empty launch 0.6), then by the MMAs (82
// cycles for 128 x 128, 64 at best) and the traffic from L2 to the SMs: 4096 x 7168 x 256 takes
// 18.7 us (21.8 after a second of it) with 235 MB brought to the SMs; the inputs need 10.2 us of HBM.  Tiles of 256
// experts, as one CTA or as a pair with 256 tokens, move half to two thirds of that but were
// no faster at any size (20.8 and 22 us here): their shared memory holds too few stages to
// cover the latency.  An MMA of 64 rows takes half the time of one of 128, and its smaller
// stages hold most of a CTA's K range at once.
//
// Warp 0: loads of x; warp 1: MMAs; warps 2-9: accumulators to registers, then the sums;
// warp 10: loads of W.
constexpr uint32_t kLogitsMmaThreads = 352;
constexpr uint32_t kLogitsBlockK = 64;
constexpr uint32_t kChainBlocks = 8;

// Where a wait of these launches gave up, for gcmoe_producer_status (they have no plan).
static __device__ uint32_t g_producer_status[kStatusWords];

template <int kM, int kN, int kPlanes>
struct LogitsTile {
    static constexpr uint32_t kColumns = kN * kPlanes;                    // of one accumulator
    static constexpr uint32_t kStageBlocks = kColumns < 128 ? 2 : 1;      // K blocks of a stage
    static constexpr uint32_t kStageBytes = kStageBlocks * (kM + kColumns) * 128;
    static constexpr uint32_t kChainStages = kChainBlocks / kStageBlocks;
    // The partial tile that a CTA receives, row by row from every rank: its own memory where
    // that leaves room for enough stages, else the stages' once they are done with.
    // Apart from the stages, tiles of 128 x 128 take 24.1 us instead of 18.9 (4096 x 7168 x
    // 256); in the stages' memory, small ones 4.39 instead of 4.23 (33 x 5120 x 384).
    static constexpr uint32_t kPitch = kN + 4;                 // floats per row: no bank conflicts
    static constexpr uint32_t kPartBytes = kM * kPitch * 4;
    static constexpr bool kApart = kN <= 64;
    static constexpr uint32_t kStages = (224 * 1024 - (kApart ? kPartBytes : 0)) / kStageBytes;
    static constexpr uint32_t kDataBytes = kStages * kStageBytes + (kApart ? kPartBytes : 0);
    static constexpr uint32_t kPartOffset = kApart ? kStages * kStageBytes : 0;
    static_assert(kPartOffset + kPartBytes <= kDataBytes, "the partial tile fits");
    // barriers: full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain; TMEM slot, abort word
    static constexpr uint32_t kSmemBytes = 1024 + kDataBytes + (2 * kStages + 5) * 8 + 8;
    static_assert(kSmemBytes <= 227 * 1024, "shared memory of an SM");
    static constexpr uint32_t kTmemStride = kColumns <= 32 ? 32 : kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : 256;
    static constexpr uint32_t kTmemColumns = 2 * kTmemStride;
};

struct LogitsMmaParams {
    CUtensorMap x_map;            // bf16 [T][H], box 64 x box_tokens, 128-byte swizzle
    CUtensorMap w_map;            // bf16 [P * E][H], box 64 x kN
    const __nv_bfloat16* x;       // the same memory, for rows with infinities
    const __nv_bfloat16* weight;
    float* out;                   // [T][E]
    uint64_t x_stride;            // elements between rows
    uint32_t num_tokens, num_experts, hidden;
    uint32_t k_stages;            // stages that cover H; channels past H are filled with zeros
    uint32_t box_tokens;          // rows a load of x brings: fewer than a tile when there are fewer tokens; the rest of
                                  // the tile's rows keep what shared memory held and end in rows that are not stored
    uint32_t split;               // CTAs of a cluster, over which a tile's K blocks are split: 1, 2, 4 or 8
};

// What a CTA that gave up sends: a NaN that no addition makes (those have all bits set).
constexpr uint32_t kGaveUpBits = 0x7fc0deadu;

// Four experts' logits of a row whose sums over three planes are not all numbers.  Infinity
// times a plane that is zero, or times planes of both signs, is NaN although infinity times the
// weight is an infinity; the FMA form, which adds the planes first, has none of this.  What
// the formula gives is decided by the row's infinite channels alone.  One thread reads the
// whole row, which only calls with such a row pay for (33 x 7168 x 256: 0.12 ms with one).
static __device__ __noinline__ float4 infinite_row_logits(const LogitsMmaParams& p, uint32_t t, uint32_t e, float4 sum) {
    const uint4* const row = reinterpret_cast<const uint4*>(p.x + t * p.x_stride);
    const uint64_t plane = uint64_t(p.num_experts) * p.hidden;
    const uint32_t chunks = p.hidden / 8;
    float acc[4] = {};
    bool infinite = false;
    for (uint32_t c0 = 0; c0 < chunks; c0 += 8) {
        uint4 raw[8];                                                     // eight loads in flight; past the end the last again
        bool numbers = true;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) raw[i] = row[min(c0 + i, chunks - 1)];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) numbers = numbers && (v[j] & 0x7f80u) != 0x7f80u && (v[j] & 0x7f800000u) != 0x7f800000u;
        }
        if (numbers) continue;
        for (uint32_t k = c0 * 8; k < min(c0 * 8 + 64, p.hidden); ++k) {
            const float v = __bfloat162float(p.x[t * p.x_stride + k]);
            if (isnan(v) || (isnan(acc[0]) && isnan(acc[1]) && isnan(acc[2]) && isnan(acc[3])))
                return make_float4(NAN, NAN, NAN, NAN);
            if (!isinf(v)) continue;
            infinite = true;
            for (uint32_t i = 0; i < 4 && e + i < p.num_experts; ++i) {
                const __nv_bfloat16* const w = p.weight + uint64_t(e + i) * p.hidden + k;
                acc[i] = fmaf(v, __bfloat162float(w[0]) + (__bfloat162float(w[plane]) + __bfloat162float(w[2 * plane])), acc[i]);
            }
        }
    }
    return infinite ? make_float4(acc[0], acc[1], acc[2], acc[3]) : sum;
}

template <int kM, int kN, int kPlanes>
__global__ void __launch_bounds__(kLogitsMmaThreads, 1) logits_mma_kernel(const __grid_constant__ LogitsMmaParams p) {
    using Tile = LogitsTile<kM, kN, kPlanes>;
    constexpr uint32_t kBlocks = Tile::kStageBlocks, kStages = Tile::kStages;
    extern __shared__ uint8_t raw_smem[];
    const uint32_t base = (ptx::smem_u32(raw_smem) + 1023u) & ~1023u;     // swizzle atoms start on 1 KiB
    uint8_t* const smem = raw_smem + (base - ptx::smem_u32(raw_smem));
    const uint32_t bars = base + Tile::kDataBytes;
    const uint32_t bar_full = bars, bar_empty = bars + 8 * kStages, bar_acc_full = bars + 16 * kStages;
    const uint32_t bar_acc_empty = bar_acc_full + 16, bar_drain = bar_acc_full + 32;
    volatile uint32_t* const tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + Tile::kDataBytes + (2 * kStages + 5) * 8);
    volatile uint32_t* const abort_word = tmem_slot + 1;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = blockIdx.x;                                     // of the cluster: the K range
    const uint32_t e0 = blockIdx.y * kN, t0 = blockIdx.z * kM;
    const uint32_t first = uint32_t(uint64_t(p.k_stages) * rank / p.split);
    const uint32_t count = uint32_t(uint64_t(p.k_stages) * (rank + 1) / p.split) - first;   // >= 1: split <= k_stages
    const uint32_t x_block = p.box_tokens * 128, x_bytes = kBlocks * x_block;   // W follows x in a stage, on a 1 KiB boundary

    WaitCtl ctl;
    ctl.status = g_producer_status;
    ctl.failed = nullptr;
    ctl.abort = abort_word;
    ctl.timeout_ns = 2000000000ull;
    ctl.kernel = kKernelLogits;

    if (tid == 0) {
        ptx::prefetch_tensormap(&p.x_map);
        ptx::prefetch_tensormap(&p.w_map);
        for (uint32_t i = 0; i < kStages; ++i) {
            ptx::mbar_init(bar_full + 8 * i, 2);
            ptx::mbar_init(bar_empty + 8 * i, 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            ptx::mbar_init(bar_acc_full + 8 * i, 1);
            ptx::mbar_init(bar_acc_empty + 8 * i, 8);
        }
        ptx::mbar_init(bar_drain, 1);
        *abort_word = 0;
        ptx::fence_mbar_init();
    }
    __syncthreads();
    // The first phase of the cluster's barrier ends before anyone writes to another CTA: by
    // then all of them have started and, where the parts lie in the stages, are done with them.
    if constexpr (Tile::kApart) ptx::cluster_arrive_relaxed();
    ptx::grid_dependency_wait();

    uint32_t tmem = 0;
    if (warp >= 1 && warp < 10) {
        // The loads start meanwhile.  TMEM only after the kernels before this one have ended and
        // before the ones behind it may start: one of those could hold TMEM of this SM until
        // this kernel ends, and the allocation, which has no limit, would wait for it.
        if (warp == 1) {
            ptx::tmem_alloc<false>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), Tile::kTmemColumns);
            ptx::tmem_relinquish<false>();
            ptx::tc_fence_before();
        }
        asm volatile("bar.sync 1, 288;" ::: "memory");
        ptx::tc_fence_after();
        tmem = *tmem_slot;
        ptx::launch_dependents();
    }

    float acc[kN / 2];                                                    // warps 2-9: one token, half of the experts
    if (warp == 0 || warp == 10) {
        if (ptx::elect_one()) {
            // Counters instead of divisions: the loop is a chain of one thread's instructions.
            uint32_t i = 0, stage = 0, parity = 1, k = first * kBlocks * kLogitsBlockK;
            for (; i < count; ++i) {
                if (i >= kStages && !mbar_wait(bar_empty + 8 * stage, parity, ctl, 1)) break;
                const uint32_t dst = base + stage * Tile::kStageBytes;
                const uint32_t bar = bar_full + 8 * stage;
                ptx::mbar_arrive_expect_tx(bar, warp == 0 ? x_bytes : kBlocks * Tile::kColumns * 128);
#pragma unroll
                for (uint32_t j = 0; j < kBlocks; ++j) {
                    if (warp == 0) {
                        ptx::tma_load_2d(dst + j * x_block, &p.x_map, bar, int(k), int(t0), ptx::kEvictNormal);
                    } else {
#pragma unroll
                        for (uint32_t q = 0; q < kPlanes; ++q)
                            ptx::tma_load_2d(dst + x_bytes + (j * kPlanes + q) * kN * 128, &p.w_map, bar, int(k),
                                             int(q * p.num_experts + e0), ptx::kEvictLast);
                    }
                    k += kLogitsBlockK;
                }
                if (++stage == kStages) { stage = 0; parity ^= 1; }
            }
            if (i < count) {
                // Gave up: the copies in flight land before shared memory is used again.
                const uint64_t start = ptx::globaltimer_ns();
                for (uint32_t j = i > kStages ? i - kStages : 0; j < i; ++j)
                    while (!ptx::mbar_try_wait(bar_full + 8 * (j % kStages), (j / kStages) & 1) &&
                           ptx::globaltimer_ns() - start < 2000000ull) {}
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            constexpr uint32_t idesc = ptx::instr_desc_bf16(kM, Tile::kColumns);
            const uint64_t a_desc = ptx::smem_desc(base, 1024, true), b_desc = ptx::smem_desc(base + x_bytes, 1024, true);
            uint32_t i = 0, stage = 0, parity = 0, chain = 0, step = 0;
            for (; i < count; ++i) {
                const uint32_t which = chain & 1;
                if (step == 0 && chain >= 2 && !mbar_wait(bar_acc_empty + 8 * which, ((chain >> 1) - 1) & 1, ctl, 2)) break;
                if (!mbar_wait(bar_full + 8 * stage, parity, ctl, 3)) break;
                ptx::tc_fence_after();
                const uint32_t at = stage * (Tile::kStageBytes >> 4);     // descriptors count 16-byte units
#pragma unroll
                for (uint32_t j = 0; j < kBlocks; ++j)
                    ptx::mma_bf16_k64(tmem + which * Tile::kTmemStride, a_desc + at + j * (x_block >> 4),
                                      b_desc + at + j * (Tile::kColumns * 128 >> 4), idesc, step + j != 0);
                ptx::tc_commit<false>(bar_empty + 8 * stage);
                if (++step == Tile::kChainStages || i == count - 1) {
                    ptx::tc_commit<false>(bar_acc_full + 8 * which);
                    step = 0;
                    ++chain;
                }
                if (++stage == kStages) { stage = 0; parity ^= 1; }
            }
            if (i < count) {
                // Gave up: the MMAs in flight end before TMEM is freed and shared memory reused.
                ptx::tc_commit<false>(bar_drain);
                const uint64_t start = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(bar_drain, 0) && ptx::globaltimer_ns() - start < 2000000ull) {}
            }
        }
        __syncwarp();
    } else {
        const uint32_t side = (warp - 2) >> 2;                            // half of the columns
        const uint32_t lanes = (warp & 3) << 21;                          // this warp's quarter of the TMEM lanes
        const uint32_t chains = (count + Tile::kChainStages - 1) / Tile::kChainStages;
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) acc[j] = 0.f;
        bool arrived = false;
        for (uint32_t chain = 0; chain < chains; ++chain) {
            // all lanes wait alike; a warp leaves as a whole
            const bool ready = mbar_wait(bar_acc_full + 8 * (chain & 1), (chain >> 1) & 1, ctl, 4);
            if (!__all_sync(0xffffffffu, ready)) break;
            ptx::tc_fence_after();
            if (!Tile::kApart && chain == chains - 1) { ptx::cluster_arrive(); arrived = true; }
            const uint32_t column = tmem + lanes + (chain & 1) * Tile::kTmemStride + side * (kN / 2);
#pragma unroll
            for (int c = 0; c < kN / 2; c += 16) {
                uint32_t r[kPlanes][16];
#pragma unroll
                for (int q = 0; q < kPlanes; ++q) ptx::tmem_ld16(column + q * kN + c, r[q]);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float v = __uint_as_float(r[0][j]);
                    if constexpr (kPlanes == 3) v += __uint_as_float(r[1][j]) + __uint_as_float(r[2][j]);
                    acc[c + j] += v;
                }
            }
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar_acc_empty + 8 * (chain & 1));
        }
        if (!Tile::kApart && !arrived) ptx::cluster_arrive();
    }
    if (!Tile::kApart && (warp < 2 || warp == 10)) ptx::cluster_arrive();
    ptx::tc_fence_before();
    __syncthreads();
    // Every load has been consumed and every MMA has ended (the last chain's barrier), or has
    // been drained above.  Row r of the tile belongs to rank r % split, at place r / split of
    // its part for each sender.  (Where the parts lie in the stages, the loading and MMA warps
    // have arrived at their end, the others when the last chain was complete.)
    ptx::cluster_wait();
    const uint32_t part = base + Tile::kPartOffset, owned = kM / p.split;
    if (warp >= 2 && warp < 10) {
        const bool failed = *abort_word != 0u;
        const float gave_up = __uint_as_float(kGaveUpBits);
        // an accumulator of 64 rows has 16 of them in the first half of each quarter of the lanes
        const uint32_t side = (warp - 2) >> 2, token = kM == 128 ? (warp & 3) * 32 + lane : (warp & 3) * 16 + (lane & 15);
        const uint32_t at = part + ((rank * owned + token / p.split) * Tile::kPitch + side * (kN / 2)) * 4;
        const uint32_t to = ptx::mapa(at, token % p.split);
        if (kM == 128 || lane < 16) {
#pragma unroll
            for (int j = 0; j < kN / 2; j += 4)
                ptx::st_cluster_f32x4(to + j * 4, failed ? make_float4(gave_up, gave_up, gave_up, gave_up)
                                                         : make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]));
        }
    } else if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc<false>(tmem, Tile::kTmemColumns);
    }
    __syncwarp();
    // After this no CTA touches another's memory.
    ptx::cluster_sync();
    const uint32_t rows = min(kM, p.num_tokens - t0);
    // `out` may start at any f32: whole vectors where every row starts on 16 bytes
    const bool vectors = p.num_experts % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    for (uint32_t i = tid; i < owned * (kN / 4); i += kLogitsMmaThreads) {
        const uint32_t place = i / (kN / 4), r = place * p.split + rank, c = i % (kN / 4) * 4;
        if (r >= rows || e0 + c >= p.num_experts) continue;
        const float* const from = reinterpret_cast<const float*>(smem + Tile::kPartOffset) + place * Tile::kPitch + c;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        bool complete = true;
        for (uint32_t s = 0; s < p.split; ++s) {                          // in rank order
            const float4 v = *reinterpret_cast<const float4*>(from + s * owned * Tile::kPitch);
            complete = complete && __float_as_uint(v.x) != kGaveUpBits;
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        if constexpr (kPlanes == 3) {
            if (complete && (isnan(sum.x) || isnan(sum.y) || isnan(sum.z) || isnan(sum.w)))
                sum = infinite_row_logits(p, t0 + r, e0 + c, sum);
        }
        float* const out = p.out + static_cast<uint64_t>(t0 + r) * p.num_experts + e0 + c;
        if (vectors) {
            *reinterpret_cast<float4*>(out) = sum;
        } else {
            const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (e0 + c + j < p.num_experts) out[j] = v[j];
        }
    }
}

}  // namespace gcmoe
