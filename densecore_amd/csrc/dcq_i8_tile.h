// dcq_i8_tile.h — what the int8 products' kernels (dcq_i8_gemm.hip, dcq_i8_rows.hip) share: where an expert's tile of
// rows is, and how sums become outputs.
#pragma once

#include "dcq_common.h"
#include "dcq_i8.h"

namespace dcq {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// The tile_at-th tile of `rows` places of a plan's order: tiles do not cross experts, and those of no expert come last.
// Found by a wave, an equal share of the experts to each lane. expert = n_expert: of no expert; -1: past the last tile.
struct PlanTile {
    int expert, begin, count;
};
__device__ __forceinline__ PlanTile find_tile(const int32_t* offsets, int n_expert, int rows, int tile_at) {
    const int lane = threadIdx.x & 63;
    const int share = (n_expert + 64) / 64;  // of n_expert + 1 groups
    const int first = lane * share, last = min(first + share, n_expert + 1);
    int tiles = 0;
    for (int e = first; e < last; ++e) tiles += (offsets[e + 1] - offsets[e] + rows - 1) / rows;
    int before = tiles;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(before, d, 64);
        if (lane >= d) before += v;
    }
    before -= tiles;
    PlanTile t = {-1, 0, 0};
    const uint64_t mine = __ballot(tile_at >= before && tile_at < before + tiles);
    if (mine) {
        const int who = __ffsll((unsigned long long)mine) - 1;
        int left = tile_at - before;
        if (lane == who) {
            for (int e = first; e < last; ++e) {
                const int at = offsets[e], n = offsets[e + 1] - at, k = (n + rows - 1) / rows;
                if (left < k) {
                    t.expert = e, t.begin = at + left * rows, t.count = min(rows, n - left * rows);
                    break;
                }
                left -= k;
            }
        }
        t.expert = __shfl(t.expert, who, 64);
        t.begin = __shfl(t.begin, who, 64);
        t.count = __shfl(t.count, who, 64);
    }
    return t;
}
// No more tiles than this, whatever the experts' shares.
inline int64_t most_tiles(int64_t slots, int n_expert, int rows) {
    const int64_t groups = slots < n_expert + 1 ? slots : n_expert + 1;
    return slots / rows + groups;
}

// y = sum * ws * xs, the weight's scale first: sum * ws is the product of the row's own unit, so that neither a small
// ws * xs is lost nor a large one infinite where the value is not.
__device__ __forceinline__ float i8_value(int sum, float ws, float xs) { return (float)sum * ws * xs; }

}  // namespace dcq
