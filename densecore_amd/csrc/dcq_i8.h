// dcq_i8.h — layers in 8-bit integers, dense and of experts: what dcq_norm.hip, dcq_i8_gemm.hip, dcq_i8_rows.hip and
// dcq_moe.hip compute. int8 rows have a scale each: element k of row r stands for q[r][k] * s[r]. Arguments are
// checked by the caller; expert numbers out of range, which only the device sees, are no expert's.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dcq {

// dcq_norm.hip: rows to int8, with or without the RMS norm and the residual's addition before it.
struct NormArgs {
    const void* x;  // F32 or F16 rows
    int64_t x_stride;  // elements between rows, as all strides here
    const float* r;  // or null
    int64_t r_stride;
    float* h;  // or null; may be r
    int64_t h_stride;
    const float* w;  // null: no norm, the row itself is quantized
    float eps;
    int64_t rows;
    int width;
    int8_t* q;  // or null
    int64_t q_stride;
    float* s;
    float* y;  // or null: the normed row in fp32
    int64_t y_stride;
};
hipError_t launch_norm_i8(int type, const NormArgs& a, hipStream_t st);

// Products of int8 rows: y[m][n] = (sum_k x[m][k] w[n][k]) * ws[n] * xs[m], the sum exact.
//   dense     rows 0 .. M - 1, one matrix, an addend R
//   kUp       the rows of a plan's slots, x row slot / top; w and w2 the expert's: silu(product) * product2 to row slot
//   kDown     the rows of a plan's slots, x row slot; w the expert's, to row slot
enum I8Mode { kI8Dense = 0, kI8Up = 1, kI8Down = 2 };
struct I8Args {
    const int8_t* x;
    const float* xs;
    int64_t x_stride;  // bytes
    int64_t M;         // rows, or slots
    const int8_t* w;
    const float* ws;
    const int8_t* w2;
    const float* ws2;
    int64_t w_stride, w_expert;  // bytes between rows, and between experts
    int N, K;
    const float* R;  // dense: or null
    int64_t r_stride;  // floats; 0: one row for all
    void* y;
    int64_t y_stride;  // elements
    const int32_t* plan;
    int n_expert, top;
    int tiles_n, tiles_m, splits, stps;  // from here on the launcher's
    bool y_wide;  // rows of y are of whole dwords
    bool banded;  // experts' tiles in bands of 8 row tiles, as a dense product's are
};
size_t i8_workspace_bytes(int64_t M, int64_t N, int64_t K);
// ws: i8_workspace_bytes bytes, or null
hipError_t launch_i8_product(int ytype, const I8Args& a, void* ws, hipStream_t st);
hipError_t launch_moe_gate_up(int htype, const I8Args& a, hipStream_t st);
struct CombineArgs;
hipError_t launch_moe_down(int ytype, I8Args a, const CombineArgs& c, hipStream_t st);
// dcq_i8_rows.hip: few rows (of an expert); dcq_i8_gemm.hip: many
hipError_t launch_i8_rows(I8Mode mode, int ytype, const I8Args& a, hipStream_t st);
hipError_t launch_i8_gemm(I8Mode mode, int ytype, I8Args a, void* ws, hipStream_t st);
bool i8_few_rows(int64_t M, int64_t N, int64_t K);  // whether a dense product is the former's

// dcq_moe.hip. A plan, in int32: offsets[n_expert + 2] (expert e's slots are places offsets[e] .. offsets[e + 1] - 1 of the
// order, those of no expert offsets[n_expert] ..); the order: slots sorted by expert; each slot's expert, or -1; and tiles of
// the order, `plan_height` places each: {expert, first place, places, 0}, -1 for a tile that is not used. Tiles do not cross
// experts: group g's begin at (its first place + g (height - 1)) / height, which leaves every group room for its last,
// partial one whatever the others' sizes, so that each group's place is known without the others' tiles.
struct PlanTile {
    int expert, begin, count, unused;
};
// What a plan of another call may hold, brought inside this call's arrays: a tile whose rows are places of the order, or -1
// for its expert (none), and a slot.
__host__ __device__ inline PlanTile tile_inside(PlanTile t, int n_expert, int64_t slots, int height) {
    if (t.expert < 0 || t.expert > n_expert || t.count <= 0 || t.begin < 0 || t.begin >= slots) return {-1, 0, 0, 0};
    const int left = (int)slots - t.begin, most = left < height ? left : height;
    t.count = t.count < most ? t.count : most;
    return t;
}
__host__ __device__ inline int slot_inside(int32_t slot, int64_t slots) {
    const uint32_t last = (uint32_t)slots - 1u;
    return (int)((uint32_t)slot < last ? (uint32_t)slot : last);
}
// Rows of a tile: what the products' kernels take at a time, by the rows that an expert has on average (us, gate and up + down
// products. 128 experts of 768 and 2048 rows, heights 16, 64, 128: mean 8 69 + 46, 76 + 46, 84 + 52; 16 84 + 57, 82 + 52; 48 136 + 107,
// 87 + 68, 97 + 74. Heights 64, 128, 256: mean 128 128 + 117, 125 + 119, 145 + 125; 512 339 + 393, 314 + 389, 323 + 357; 1024 628 +
// 773, 560 + 761, 545 + 674. 8 experts of 14336 and 4096 rows: mean 64 248 + 134, 251 + 153, 272 + 177; 128 312 + 180, 302 + 162, 332 +
// 187; 384 634 + 364, 554 + 288, 564 + 374; 1024 1486 + 808, 1242 + 644, 1135 + 619).
__host__ __device__ inline int plan_height(int64_t slots, int n_expert) {
    const int64_t mean = slots / n_expert;
    return mean <= 12 ? 16 : mean <= 144 ? 64 : mean <= 480 ? 128 : 256;
}
__host__ __device__ inline int64_t plan_tiles(int64_t slots, int n_expert, int height) {
    return (slots + (int64_t)(n_expert + 1) * (height - 1)) / height;
}
__host__ __device__ inline int64_t plan_order_at(int n_expert) { return (n_expert + 2 + 63) / 64 * 64; }
__host__ __device__ inline int64_t plan_expert_at(int n_expert, int64_t slots) {
    return plan_order_at(n_expert) + (slots + 63) / 64 * 64;
}
__host__ __device__ inline int64_t plan_tiles_at(int n_expert, int64_t slots) {
    return plan_expert_at(n_expert, slots) + (slots + 63) / 64 * 64;
}
__host__ __device__ inline int64_t plan_ints(int n_expert, int64_t slots) {
    return plan_tiles_at(n_expert, slots) + 4 * plan_tiles(slots, n_expert, plan_height(slots, n_expert));
}
struct RouteArgs {
    const void* x;
    int64_t stride;  // elements
    int64_t rows;
    int n_expert, sigmoid;
    const float* bias;  // or null
    int n_group, topk_group, group_best, k, renorm;
    float scale;
    int32_t* ids;
    float* weights;
};
hipError_t launch_moe_route(int type, const RouteArgs& a, hipStream_t st);
hipError_t launch_moe_plan(const int32_t* ids, int64_t slots, int n_expert, int32_t* plan, hipStream_t st);
// y[m] = (R[m] +) sum_j weights[m][j] * p[m * top + j], over the slots that have an expert, in the order of j
struct CombineArgs {
    const float* p;  // [rows * top][N]
    const int32_t* expert;  // the plan's expert of each slot
    const float* weights;
    int top, N;
    int64_t rows;
    const float* R;
    int64_t r_stride;
    void* y;
    int64_t y_stride;
};
hipError_t launch_moe_combine(int ytype, const CombineArgs& a, hipStream_t st);

}  // namespace dcq
