// dcq_attn.h — what the attention kernels (dcq_kv.hip, dcq_attn_prompt.hip, dcq_tree.hip) share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dcq {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The exponent field that normalises magnitudes up to m: m * pow2(268 - E) is in [2^14, 2^15).
__device__ __forceinline__ int norm_exp(uint32_t bits) {
    return max((int)(bits >> 23), 30);  // below 2^-97 (zeros too): the floor's exponent
}
__device__ __forceinline__ float pow2_bits(int e) { return __uint_as_float((uint32_t)e << 23); }

// four consecutive fp32 values (already scaled) -> the f16 pieces
__device__ __forceinline__ void split4(const float x0, const float x1, const float x2, const float x3, f16x4& h,
                                       f16x4& l) {
    const f16x2 h0 = __builtin_convertvector((f32x2){x0, x1}, f16x2);
    const f16x2 h1 = __builtin_convertvector((f32x2){x2, x3}, f16x2);
    const f16x2 l0 = __builtin_convertvector((f32x2){x0 - (float)h0[0], x1 - (float)h0[1]}, f16x2);
    const f16x2 l1 = __builtin_convertvector((f32x2){x2 - (float)h1[0], x3 - (float)h1[1]}, f16x2);
    h = __builtin_shufflevector(h0, h1, 0, 1, 2, 3);
    l = __builtin_shufflevector(l0, l1, 0, 1, 2, 3);
}

// Transposing LDS read, per 16 lanes: lane j gives the address of elements 4 (j % 4) .. + 3 of row j / 4
// of a 4 x 16 matrix and receives column j.
__device__ __forceinline__ f16x4 lds_transposed(const _Float16* src) {
    typedef short i16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
    return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)src));
}

struct AttnArgs {
    const uint8_t* k_arena;
    const uint8_t* v_arena;
    int n_blocks, n_layer, layer;
    int64_t sb;  // slot bytes
    const int32_t* table;
    int n_table;
    const float* q;
    int64_t q_stride;  // floats between query tokens
    const float* k_cur;
    const float* v_cur;
    int64_t kv_stride;  // floats between current K (V) rows
    float* out;
    int64_t out_stride;
    float* ws_o;  // [splits][N][n_head][HD]
    float* ws_ml;  // [splits][N][n_head][2]
    int n_tokens, n_past, n_head, n_head_kv, hpw, nq;
    int nch_hist, nch_total, cps;  // chunks of history, all chunks, chunks per split
    int splits, groups;
    float scale_log2e;
};

// dcq_attn_prompt.hip: many query rows, on f16 MFMA pieces of the fp32 operands. cps counts its key
// blocks of 32 per split; with splits > 1 the partial results go to ws_o / ws_ml.
hipError_t launch_attn_prompt(int ct, int hd, const AttnArgs& a, hipStream_t st);

}  // namespace dcq
