// dcq_kv_row.h — slots of the paged KV cache: where one is, and how a workgroup writes a token's row into it.
#pragma once

#include "dcq_common.h"

namespace dcq {

constexpr int kKvBlock = 16;

__device__ __forceinline__ const uint8_t* kv_slot(const uint8_t* arena, int blk, int n_layer, int layer, int slot,
                                                  int64_t sb) {
    return arena + (((int64_t)blk * n_layer + layer) * kKvBlock + slot) * sb;
}

// One token's row of row_elems fp32 values into its slot, by a whole workgroup. Units: a 32-element block
// (Q8_0), 2 elements (F16), 4 (F32). No fp contraction: the bytes are those of the CPU's quantizer.
__device__ __forceinline__ void kv_encode_row(int ct, uint8_t* dst, const float* x, int64_t row_elems) {
#pragma clang fp contract(off)
    if (ct == kTypeQ8_0) {
        for (int64_t b = threadIdx.x; b < row_elems / 32; b += blockDim.x) {
            const float4* xb = reinterpret_cast<const float4*>(x + b * 32);
            float v[32];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float4 f = xb[j];
                v[4 * j] = f.x, v[4 * j + 1] = f.y, v[4 * j + 2] = f.z, v[4 * j + 3] = f.w;
            }
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j) amax = fmaxf(amax, fabsf(v[j]));
            const float d = amax / 127.f;
            const float id = d != 0.0f ? 1.0f / d : 0.0f;
            uint16_t* p16 = reinterpret_cast<uint16_t*>(dst + b * 34);
            p16[0] = float_to_half_bits(d);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float q0 = fminf(fmaxf(roundf(v[j] * id), -128.f), 127.f);
                const float q1 = fminf(fmaxf(roundf(v[j + 1] * id), -128.f), 127.f);
                p16[1 + j / 2] =
                    (uint16_t)(((uint32_t)(int32_t)q0 & 0xFFu) | (((uint32_t)(int32_t)q1 & 0xFFu) << 8));
            }
        }
    } else if (ct == kTypeF16) {
        uint32_t* d32 = reinterpret_cast<uint32_t*>(dst);
        for (int64_t u = threadIdx.x; u < row_elems / 2; u += blockDim.x) {
            const float2 f = reinterpret_cast<const float2*>(x)[u];
            d32[u] = (uint32_t)float_to_half_bits(f.x) | ((uint32_t)float_to_half_bits(f.y) << 16);
        }
    } else {
        float4* d4 = reinterpret_cast<float4*>(dst);
        for (int64_t u = threadIdx.x; u < row_elems / 4; u += blockDim.x) d4[u] = reinterpret_cast<const float4*>(x)[u];
    }
}

}  // namespace dcq
