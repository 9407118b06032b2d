// Residual addition, RMS norm and the layer's input format in one pass over a row:
//
//   h = x + residual                       (f32; written back rounded to the residual's type)
//   v = h / sqrt(mean(h^2) + eps) * weight (f32)
//   x_q, x_sf = e4m3(v / 2^(code-127)), code = biased exponent of the smallest power of two
//               >= amax/448 over 32 channels: the format of stage_inputs.cuh
//   normed = bf16(v)                       (what the router's product and other users read)
//
// Both outputs are rounded once, from the f32 value: quantising the BF16 copy would round twice.
// The mean runs over the unrounded f32 sum h, not over the copy that is written back.
//
// Bound by HBM for many rows (9 + 1/32 bytes per element with a BF16 residual and both
// outputs: 4096 x 7168 in 42.5 us, 6.2 TB/s, 96% of a copy's rate), by load latency
// and the reduction for few (1 x 7168: 2.4 us, an empty launch 0.6).  One CTA per row keeps the
// row in registers between the reduction and the output, so every input is read once; a thread
// holds kChunks times 8 channels, four lanes share one scale, sixteen one scale word.
// Up to 16 channels a thread take 32 registers, so that 2048 threads fit an SM: with more
// registers and half of the rows in flight, 4096 x 7168 took 48 us.
//
// A group whose amax lies within f32's rounding of a border, 448 times a power of two, gets
// one of the two scales next to it; either holds the group.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_common.cuh"
#include "ptx.cuh"
#include "stage_inputs.cuh"

namespace gcmoe {

constexpr uint32_t kNormThreads = 1024;      // most threads of a CTA
constexpr uint32_t kNormMaxChunks = 4;       // most 8-channel chunks of a thread
enum NormResidual : int { kNoResidual = 0, kResidualBf16 = 1, kResidualF32 = 2 };

struct NormParams {
    const __nv_bfloat16* x;
    const void* residual;         // bf16 or f32, or null
    const void* weight;           // bf16 or f32 [H]
    uint2* x_q;                   // e4m3 [T][H]
    uint32_t* x_sf;               // int32 [T][ceil(H/128)]
    __nv_bfloat16* normed;        // or null
    void* residual_out;           // type of residual; may be residual itself
    uint32_t* shared_sf;          // MN-major int32 [shared_sf_rows][H/128] or null
    uint64_t x_stride, residual_stride, normed_stride, residual_out_stride;   // elements between rows
    uint32_t shared_sf_rows, block_m;
    uint32_t hidden;
    float eps;
};

__device__ __forceinline__ void unpack_bf16x8(const uint4& raw, float (&v)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ uint4 pack_bf16x8(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

template <int kChunks, int kResidual, bool kWeightF32>
__global__ void __launch_bounds__(kNormThreads, kChunks <= 2 ? 2 : 1) rms_norm_kernel(const NormParams p) {
    __shared__ float group_sums[kNormThreads / 32 * kChunks];      // a group: 32 consecutive chunks
    const uint32_t t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t chunks = p.hidden / 8;
    ptx::grid_dependency_wait();
    ptx::launch_dependents();     // before the wait, later launches crowd in: 256 x 4096 took 2.8 us instead of 2.3

    float h[kChunks][8];
    const __nv_bfloat16* row = p.x + t * p.x_stride;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const uint32_t c = tid + i * blockDim.x;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (c < chunks) raw = __ldcs(reinterpret_cast<const uint4*>(row) + c);
        unpack_bf16x8(raw, h[i]);
    }
    if constexpr (kResidual == kResidualBf16) {
        const uint4* res = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.residual) + t * p.residual_stride);
        uint4* out = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.residual_out) + t * p.residual_out_stride);
        uint4 raw[kChunks];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = tid + i * blockDim.x;
            raw[i] = make_uint4(0, 0, 0, 0);
            if (c < chunks) raw[i] = __ldcs(res + c);
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = tid + i * blockDim.x;
            float r[8];
            unpack_bf16x8(raw[i], r);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] += r[j];
            if (c < chunks) out[c] = pack_bf16x8(h[i]);
        }
    } else if constexpr (kResidual == kResidualF32) {
        const float4* res = reinterpret_cast<const float4*>(static_cast<const float*>(p.residual) + t * p.residual_stride);
        float4* out = reinterpret_cast<float4*>(static_cast<float*>(p.residual_out) + t * p.residual_out_stride);
        float4 raw[kChunks][2];
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = tid + i * blockDim.x;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                raw[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c < chunks) raw[i][j] = __ldcs(res + 2 * c + j);
            }
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = tid + i * blockDim.x;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                h[i][4 * j] += raw[i][j].x; h[i][4 * j + 1] += raw[i][j].y;
                h[i][4 * j + 2] += raw[i][j].z; h[i][4 * j + 3] += raw[i][j].w;
                if (c < chunks)
                    out[2 * c + j] = make_float4(h[i][4 * j], h[i][4 * j + 1], h[i][4 * j + 2], h[i][4 * j + 3]);
            }
        }
    }

    // The order of the additions depends on the row's length alone, not on the threads that
    // share the row: a row has the same bits in a batch of any size.  With several chunks a
    // thread that takes a shuffle for each (511 x 7168: 6.0 us instead of 5.9).
    float sum[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[i] = fmaf(h[i][j], h[i][j], sum[i]);
    }
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1)
#pragma unroll
        for (int i = 0; i < kChunks; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) group_sums[warp + i * (blockDim.x / 32)] = sum[i];
    }
    __syncthreads();
    // the CTA's warps hold all of the row's groups; up to two chunks a thread there are at most 32
    const uint32_t groups = (chunks + 31) / 32;
    float total = lane < groups ? group_sums[lane] : 0.f;
    if constexpr (kChunks > 2) {
#pragma unroll
        for (uint32_t g = 32; g < kNormThreads / 32 * kChunks; g += 32) total += lane + g < groups ? group_sums[lane + g] : 0.f;
    }
#pragma unroll
    for (uint32_t d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    const float scale = 1.0f / sqrtf(total / float(p.hidden) + p.eps);

    uint32_t shared_row = 0;
    if (p.shared_sf != nullptr) {
        const uint32_t block = t / p.block_m;
        shared_row = block * round_up_u32(p.block_m, 128) + sf_row_in_block(t - block * p.block_m);
    }
    const uint32_t words = (p.hidden + 127) / 128;
    uint2* q_row = p.x_q + static_cast<uint64_t>(t) * chunks;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const uint32_t c = tid + i * blockDim.x;
        const bool in = c < chunks;
        float w[8] = {};
        if (in) {
            if constexpr (kWeightF32) {
                const float4 a = __ldca(static_cast<const float4*>(p.weight) + 2 * c);
                const float4 b = __ldca(static_cast<const float4*>(p.weight) + 2 * c + 1);
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
                w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
            } else {
                unpack_bf16x8(__ldca(static_cast<const uint4*>(p.weight) + c), w);
            }
        }
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[i][j] = h[i][j] * scale * w[j];
            amax = fmaxf(amax, fabsf(h[i][j]));
        }
        if (in && p.normed != nullptr)
            reinterpret_cast<uint4*>(p.normed + t * p.normed_stride)[c] = pack_bf16x8(h[i]);
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // channels past the row have no scale: their bytes of the last word are 127 (one)
        const uint32_t code = in ? ue8m0_code_for_e4m3(amax) : 127u;
        const float inv = __uint_as_float((254u - code) << 23);    // 2^(127 - code)
        if (in)
            q_row[c] = make_uint2(
                uint32_t(ptx::cvt_e4m3x2(h[i][0] * inv, h[i][1] * inv)) | (uint32_t(ptx::cvt_e4m3x2(h[i][2] * inv, h[i][3] * inv)) << 16),
                uint32_t(ptx::cvt_e4m3x2(h[i][4] * inv, h[i][5] * inv)) | (uint32_t(ptx::cvt_e4m3x2(h[i][6] * inv, h[i][7] * inv)) << 16));
        const uint32_t base = lane & 16u;
        const uint32_t word = __shfl_sync(0xffffffffu, code, base) |
                              (__shfl_sync(0xffffffffu, code, base + 4) << 8) |
                              (__shfl_sync(0xffffffffu, code, base + 8) << 16) |
                              (__shfl_sync(0xffffffffu, code, base + 12) << 24);
        if (in && (lane & 15u) == 0) {
            const uint32_t wi = c >> 4;
            p.x_sf[static_cast<uint64_t>(t) * words + wi] = word;
            if (p.shared_sf != nullptr)
                p.shared_sf[static_cast<uint64_t>(wi) * p.shared_sf_rows + shared_row] = word;
        }
    }
}

}  // namespace gcmoe
