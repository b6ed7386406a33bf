// dcq_i8_tile.h — what the int8 products' kernels (dcq_i8_gemm.hip, dcq_i8_rows.hip) share.
#pragma once

#include "dcq_common.h"
#include "dcq_i8.h"
#include "dcq_lds_load.h"

namespace dcq {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// A plan's tile, and a place of its order.
__device__ __forceinline__ PlanTile plan_tile(const int32_t* plan, int n_expert, int64_t slots, int at, int height) {
    return tile_inside(reinterpret_cast<const PlanTile*>(plan + plan_tiles_at(n_expert, slots))[at], n_expert, slots, height);
}
__device__ __forceinline__ int plan_slot(const int32_t* order, int at, int64_t slots) { return slot_inside(order[at], slots); }

// All but the last N loads have landed: "dcq counted wait" tells the assembly's checks so. The clobber keeps the compiler's LDS reads
// and writes of what has landed behind it, which the builtin wait, as it touches no memory, does not promise.
template <int N>
__device__ __forceinline__ void counted_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\t;dcq counted wait" ::"n"(N) : "memory");
}
__device__ __forceinline__ const int8_t* uniform(const int8_t* p) {  // in scalar registers, as dma16's base is to be
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
    return (const int8_t*)((uint64_t)hi << 32 | lo);
}

// LDS rows of 128 bytes: piece p of 16 bytes of row r lies at p ^ key(r), so that 16 rows' pieces p are on all 64 banks.
__device__ __forceinline__ int piece_key(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// 16 bytes of outputs past the caches' usual places: products whose outputs flow through L2 lose the operands there
// (4099 x 14336 x 4096, F16 out: 251 -> 229 us; 4096 x 14336 x 2048, F32: 164 -> 141). Down products' rows of slots and the planes of
// split products go this way, too, though the next launch reads them.
__device__ __forceinline__ void store_through(void* y, const void* v16) {
    typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));
    i32x4 v;
    __builtin_memcpy(&v, v16, 16);
    __builtin_nontemporal_store(v, reinterpret_cast<i32x4*>(y));
}

// y = sum * ws * xs, the weight's scale first: sum * ws is the product of the row's own unit, so that neither a small
// ws * xs is lost nor a large one infinite, as long as sum * ws itself is within fp32's normal range (always for ws from 2^-126 to
// 2^96, as |sum| < 2^31).
__device__ __forceinline__ float i8_value(int sum, float ws, float xs) {
#pragma clang fp contract(off)
    return (float)sum * ws * xs;
}
// The addend, after the value's own rounding: not fused with it in one kernel and added in another.
__device__ __forceinline__ float i8_plus(float v, float r) {
#pragma clang fp contract(off)
    return v + r;
}

}  // namespace dcq
