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
// Rows of a tile: what the products' kernels take at a time, by the rows that an expert has on average. A plan knows the ids and not
// the matrices, for which the borders differ; those here lie between them (us, gate and up + down products).
//   16, 64 rows, 128 experts of 768 x 2048: mean 8 69 + 46, 76 + 46; 16 84 + 57, 82 + 52. One expert with every token costs short tiles
//     nothing, their weights come from L2 again (96 tokens x 8, mean 6: 70 + 45 with and without it, by 64 rows 82 + 47).
//   64, 128 rows, gate and up and down together, means 80, 128, 160, 256: 128 experts of 768 x 2048 190, 197; 244, 244; 285, 283; 408, 393. 64 of
//     1408 x 2048 167, 168; 215, 211; 241, 237; 338, 326. 8 of 14336 x 4096 457, 395; 504, 459; 594, 597; 752, 705. 8 of 4096 x 4096
//     155, 147; 159, 153; 201, 207; 240, 226. 16 of 1024 x 1024 28, 30; 32, 34; 37, 40; 49, 51.
//   128, 256 rows, means 384, 480, 576, 768, the same matrices: 552, 536; 669, 640; 785, 742; 1025, 949. 440, 442; 532, 504; 616, 582; 800, 748. 856,
//     946; 1075, 1058; 1212, 1194; 1527, 1370. 280, 315; 339, 331; 385, 391; 480, 434. 60, 72; 78, 81; 86, 86; 104, 97.
// Slots of no expert count in the mean, so that a batch mostly of padding has taller tiles than its tokens need (512 tokens x 8 of 128 experts of
// 768 x 2048 of which 16, 64 or 256 are not padding, with its 64 rows 72 + 44, 87 + 55, 85 + 55; with 16 rows 69 + 37, 87 + 48, 93 + 59).
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
