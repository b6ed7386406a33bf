// dcq_i8_rows.hip — products of few int8 rows (a decode step's, or those of an expert) on 16 x 16 int8 MFMA.
#include <algorithm>

#include "dcq_common.h"
#include "dcq_i8.h"
#include "dcq_i8_tile.h"
#include "dcq_kernels.h"

namespace dcq {

// 16 MT rows x 16 NT weight rows to a wave (kI8Up: 16 gate and 16 up rows, NT = 2); KW waves take a chunk of 256 k in
// turn and add their sums in LDS, NW such groups to a workgroup.
template <I8Mode MODE, int MT, int NT, int KW, int NW, class T>
__global__ void __launch_bounds__(64 * KW * NW) i8_rows_kernel(I8Args a) {
    constexpr bool UP = MODE == kI8Up, GROUPED = MODE != kI8Dense;
    constexpr int TILE_N = UP ? 8 * NT : 16 * NT;  // outputs of a wave group
    static_assert(!UP || NT == 2, "a gate and an up row to each output");
    __shared__ int part[NW][KW > 1 ? KW : 1][MT * NT * 4][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave % KW, nw = wave / KW;
    const int tile_m = (int)blockIdx.x / a.tiles_n, tile_n = (int)blockIdx.x % a.tiles_n;
    const int n0 = (tile_n * NW + nw) * TILE_N;
    int rows_here, expert = 0;
    const int32_t* order = nullptr;
    if constexpr (GROUPED) {
        const PlanTile t = find_tile(a.plan, a.n_expert, 16 * MT, tile_m);  // each wave for itself
        expert = __builtin_amdgcn_readfirstlane(t.expert);
        if (expert < 0) return;
        rows_here = __builtin_amdgcn_readfirstlane(t.count);
        order = a.plan + plan_order_at(a.n_expert) + __builtin_amdgcn_readfirstlane(t.begin);
        if (expert == a.n_expert) {  // slots of no expert
            if constexpr (UP) {
                if (kw == 0)
                    for (int i = lane; i < rows_here * TILE_N; i += 64)
                        if (n0 + i % TILE_N < a.N)
                            static_cast<T*>(a.y)[(int64_t)order[i / TILE_N] * a.y_stride + n0 + i % TILE_N] = (T)0.0f;
            }
            return;
        }
    } else {
        rows_here = (int)std::min<int64_t>(16 * MT, a.M - (int64_t)tile_m * 16 * MT);
    }

    const int8_t* xp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int r = min(16 * i + (lane & 15), rows_here - 1);
        int64_t src;
        if constexpr (GROUPED) src = UP ? order[r] / a.top : order[r];
        else src = (int64_t)tile_m * 16 * MT + r;
        xp[i] = a.x + src * a.x_stride + 16 * (lane >> 4);
    }
    const int8_t* wp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = min(UP ? n0 + (lane & 15) : n0 + 16 * j + (lane & 15), a.N - 1);
        wp[j] = (UP && j ? a.w2 : a.w) + (int64_t)expert * a.w_expert + (int64_t)n * a.w_stride + 16 * (lane >> 4);
    }
    v4i acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (v4i){0, 0, 0, 0};

    v4i fw[2][NT][4];
    auto load_w = [&](int c, int into) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = 256 * c + 64 * u;
            const int at = k + 16 * (lane >> 4) < a.K ? k : -16 * (lane >> 4);  // past K: the row's first piece
#pragma unroll
            for (int j = 0; j < NT; ++j) fw[into][j][u] = *reinterpret_cast<const v4i*>(wp[j] + at);
        }
    };
    auto multiply = [&](int c, int from) {
        v4i fx[MT][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = 256 * c + 64 * u;
            const bool in = k + 16 * (lane >> 4) < a.K;
            const int at = in ? k : -16 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                fx[i][u] = *reinterpret_cast<const v4i*>(xp[i] + at);
                if (!in) fx[i][u] = (v4i){0, 0, 0, 0};  // x is zero past K
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx[i][u], fw[from][j][u], acc[i][j], 0, 0, 0);
    };
    const int chunks = (a.K + 255) / 256;
    if (kw < chunks) load_w(kw, 0);
    for (int c = kw; c < chunks; c += 2 * KW) {
        if (c + KW < chunks) load_w(c + KW, 1);
        multiply(c, 0);
        if (c + KW < chunks) {
            if (c + 2 * KW < chunks) load_w(c + 2 * KW, 0);
            multiply(c + KW, 1);
        }
    }

    // ---- the waves' sums together; a lane's sums are column lane % 16 of rows 4 (lane / 16) + v ----
    auto out = [&](int i, int v, int ln, int sum0, int sum1, int j) {
        const int r = 16 * i + 4 * (ln >> 4) + v, n = n0 + (UP ? 0 : 16 * j) + (ln & 15);
        if (r >= rows_here || n >= a.N) return;
        const int64_t row = GROUPED ? (int64_t)order[r] : (int64_t)tile_m * 16 * MT + r;
        const float xs = a.xs[UP ? row / a.top : row];
        const int64_t ns = (int64_t)expert * a.N + n;
        float y = i8_value(sum0, a.ws[ns], xs);
        if constexpr (UP) y = silu(y) * i8_value(sum1, a.ws2[ns], xs);
        if (!GROUPED && a.R) y += a.R[row * a.r_stride + n];
        static_cast<T*>(a.y)[row * a.y_stride + n] = (T)y;
    };
    if constexpr (KW == 1) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int j = 0; j < (UP ? 1 : NT); ++j) out(i, v, lane, acc[i][j][v], acc[i][UP ? 1 : 0][v], j);
    } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) part[nw][kw][(i * NT + j) * 4 + v][lane] = acc[i][j][v];
        __syncthreads();
        // pieces of 64 sums to a wave
        for (int p = kw; p < MT * 4 * (UP ? 1 : NT); p += KW) {
            const int v = p % 4, j = UP ? 0 : p / 4 % NT, i = UP ? p / 4 : p / 4 / NT;
            int s0 = 0, s1 = 0;
#pragma unroll
            for (int q = 0; q < KW; ++q) {
                s0 += part[nw][q][(i * NT + j) * 4 + v][lane];
                if constexpr (UP) s1 += part[nw][q][(i * NT + 1) * 4 + v][lane];
            }
            out(i, v, lane, s0, s1, j);
        }
    }
}

namespace {

template <I8Mode MODE, int MT, int NT, int KW, int NW, class T>
hipError_t launch_one(I8Args a, hipStream_t st) {
    constexpr int tile_n = (MODE == kI8Up ? 8 * NT : 16 * NT) * NW;
    a.tiles_n = (a.N + tile_n - 1) / tile_n;
    a.tiles_m = (int)(MODE == kI8Dense ? (a.M + 16 * MT - 1) / (16 * MT) : most_tiles(a.M, a.n_expert, 16 * MT));
    i8_rows_kernel<MODE, MT, NT, KW, NW, T><<<dim3((unsigned)((int64_t)a.tiles_n * a.tiles_m)), 64 * KW * NW, 0, st>>>(a);
    return hipGetLastError();
}

template <I8Mode MODE, int MT, int NT, class T>
hipError_t launch_waves(const I8Args& a, hipStream_t st) {
    const int chunks = (a.K + 255) / 256;
    if (chunks >= 8) return launch_one<MODE, MT, NT, 8, 1, T>(a, st);
    if (chunks >= 4) return launch_one<MODE, MT, NT, 4, 1, T>(a, st);
    return launch_one<MODE, MT, NT, 2, 2, T>(a, st);
}

template <I8Mode MODE, class T>
hipError_t launch_rows_of(const I8Args& a, int64_t rows, hipStream_t st) {
    constexpr int NT = MODE == kI8Up ? 2 : 1;
    if (rows <= 16) return launch_waves<MODE, 1, NT, T>(a, st);
    if (rows <= 32) return launch_waves<MODE, 2, NT, T>(a, st);
    return launch_waves<MODE, 4, NT, T>(a, st);
}

}  // namespace

hipError_t launch_i8_rows(I8Mode mode, int ytype, I8Args a, hipStream_t st) {
    if (mode == kI8Dense)
        return ytype == kTypeF16 ? launch_rows_of<kI8Dense, _Float16>(a, a.M, st) : launch_rows_of<kI8Dense, float>(a, a.M, st);
    if (mode == kI8Up)
        return ytype == kTypeF16 ? launch_rows_of<kI8Up, _Float16>(a, 16, st) : launch_rows_of<kI8Up, float>(a, 16, st);
    return launch_rows_of<kI8Down, float>(a, 16, st);
}

hipError_t launch_i8_product(int ytype, I8Args a, void* ws, size_t ws_bytes, hipStream_t st) {
    const int most = knob(Knob::I8Rows) >= 0 ? knob(Knob::I8Rows) : 64;
    return a.M <= most ? launch_i8_rows(kI8Dense, ytype, a, st) : launch_i8_gemm(kI8Dense, ytype, a, ws, ws_bytes, st);
}

hipError_t launch_i8_experts(I8Mode mode, int ytype, I8Args a, hipStream_t st) {
    const int most = knob(Knob::I8Experts) >= 0 ? knob(Knob::I8Experts) : 12;
    a.splits = 1;
    return a.M <= (int64_t)most * a.n_expert ? launch_i8_rows(mode, ytype, a, st) : launch_i8_gemm(mode, ytype, a, nullptr, 0, st);
}

}  // namespace dcq
