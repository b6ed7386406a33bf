// dcq_i8_rows.hip — products of few int8 rows (a decode step's, or those of an expert) on 16 x 16 int8 MFMA.
//
// Weights are read once for a tile of 16 to 64 rows (33 to 64 rows are one such tile or two of 32, up to 256 rows of small matrices
// four or more), so the time of few rows is the weights' bytes over the rate of HBM, and what is left to do is to keep enough of
// them on their way; with more rows, what every workgroup takes of x from L2 counts, too (61 x 2560 x 9728: 148 MB of requests to L2, two
// thirds of them x, for 31 MB from memory). A wave owns 16 to 48 rows of W and a share of K; its operands come through a ring of
// two stages in LDS that no other wave touches, so that nothing waits for a barrier until the sums are added. Through LDS because
// an operand's consecutive lanes are in 16 different rows: loaded to registers, every lane's 16 bytes are a request of their own
// (61 rows x 2560 x 9728: 22.7 us that way, 11.0 with rows of 128 bytes to LDS, 15.2 with rows of 64; one row x 2560 x 9728:
// 8.1, 6.1 and 6.5).
#include <algorithm>

#include "dcq_common.h"
#include "dcq_i8.h"
#include "dcq_i8_tile.h"
#include "dcq_kernels.h"

namespace dcq {

namespace {

constexpr int kStages = 2;

// A wave's sums over its share of K: 16 MT rows of x (x_off: the rows' bytes of the lane's loads, 8 rows a load) times 16 NT
// rows of weights. Lane l gets column l % 16 of rows 4 (l / 16) + v.
template <int MT, int NT>
__device__ __forceinline__ void wave_sums(v4i (&acc)[MT][NT], int8_t* ring, const int8_t* xb, const uint32_t (&x_off)[2 * MT],
                                          const int8_t* const (&wb)[NT], const uint32_t (&w_off)[2 * NT], int K, int begin, int end) {
    constexpr int KB = 128, LX = 2 * MT, LW = 2 * NT, L = LX + LW;
    const int lane = threadIdx.x & 63, l_row = lane / 8;
    auto issue = [&](int s, int at) {
        int8_t* S = ring + at * (1024 * L);
        const int64_t k0 = (int64_t)s * KB;
        const int pieces = min(8, (K - s * KB) / 16);  // pieces past K are the row's first of the stage
#pragma unroll
        for (int i = 0; i < LW; ++i) {
            const int p = lane % 8 ^ piece_key(8 * i + l_row);
            dma16<true>(wb[i / 2] + k0, w_off[i] + (p < pieces ? 16 * p : 0), S + 1024 * i);
        }
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int p = lane % 8 ^ piece_key(8 * i + l_row);
            dma16<true>(xb + k0, x_off[i] + (p < pieces ? 16 * p : 0), S + 1024 * (LW + i));
        }
    };
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (v4i){0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kStages; ++i)
        if (begin + i < end) issue(begin + i, i);
    const int r16 = lane & 15, q = lane >> 4;
    for (int s = begin, at = 0; s < end; ++s) {
        if (s + 1 < end) counted_wait<L>();  // a wave's loads retire in order: all but the next stage's
        else counted_wait<0>();
        const int8_t* S = ring + at * (1024 * L);
        v4i fw[NT][2], fx[MT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int fo = r16 * KB + 16 * ((4 * u + q) ^ piece_key(r16));
#pragma unroll
            for (int j = 0; j < NT; ++j) fw[j][u] = *reinterpret_cast<const v4i*>(S + fo + j * 16 * KB);
#pragma unroll
            for (int i = 0; i < MT; ++i) fx[i][u] = *reinterpret_cast<const v4i*>(S + 1024 * LW + fo + i * 16 * KB);
        }
        if (s + kStages < end) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage is in registers, its room free
            issue(s + kStages, at);
        }
        at ^= 1;
        if ((s + 1) * KB > K) {  // x is zero past K
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (s * KB + 64 * u + 16 * q >= K)
#pragma unroll
                    for (int i = 0; i < MT; ++i) fx[i][u] = (v4i){0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fx[i][u], fw[j][u], acc[i][j], 0, 0, 0);
    }
}

// The lane's part of loads of 16 weight rows from n0 on; rows past N are the last one's again.
__device__ __forceinline__ void weight_rows(uint32_t* w_off, int n0, int N, int64_t w_stride) {
    const int l_row = (threadIdx.x & 63) / 8;
    for (int i = 0; i < 2; ++i) w_off[i] = (uint32_t)max(min(8 * i + l_row, N - 1 - n0), 0) * (uint32_t)w_stride;
}

}  // namespace

// 16 MT rows x 16 NB outputs to a wave (kI8Up: of 16 gate and 16 up rows). KW waves share K, an equal run of stages each, and add
// their sums in LDS; NW such groups to a workgroup.
template <I8Mode MODE, int MT, int NB, int KW, int NW, class T>
__global__ void __launch_bounds__(64 * KW * NW) i8_rows_kernel(I8Args a) {
    constexpr bool UP = MODE == kI8Up, GROUPED = MODE != kI8Dense;
    constexpr int NT = UP ? 2 : NB;
    extern __shared__ __align__(16) uint8_t smem[];
    int(*part)[KW][MT * NT * 4][64] = reinterpret_cast<int(*)[KW][MT * NT * 4][64]>(smem);  // when the stages are done
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave % KW, nw = wave / KW;
    const int tile_m = (int)blockIdx.x / a.tiles_n, tile_n = (int)blockIdx.x % a.tiles_n;
    const int n0 = (tile_n * NW + nw) * 16 * NB;
    int rows_here, expert = 0;
    const int32_t* order = nullptr;
    if constexpr (GROUPED) {
        const PlanTile t = plan_tile(a.plan, a.n_expert, a.M, tile_m, 16 * MT);
        if (t.expert < 0) return;
        expert = t.expert, rows_here = t.count;
        order = a.plan + plan_order_at(a.n_expert) + t.begin;
        if (expert == a.n_expert) {  // slots of no expert
            if constexpr (UP) {
                if (kw == 0)
                    for (int i = lane; i < rows_here * 16; i += 64)
                        if (n0 + i % 16 < a.N) static_cast<T*>(a.y)[(int64_t)plan_slot(order, i / 16, a.M) * a.y_stride + n0 + i % 16] = (T)0.0f;
            }
            return;
        }
    } else {
        rows_here = (int)std::min<int64_t>(16 * MT, a.M - (int64_t)tile_m * 16 * MT);
    }

    uint32_t x_off[2 * MT], w_off[2 * NT];
    const int8_t* wb[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int nj = UP ? n0 : n0 + 16 * j;
        wb[j] = uniform((UP && j ? a.w2 : a.w) + (int64_t)expert * a.w_expert + (int64_t)min(nj, a.N - 1) * a.w_stride);
        weight_rows(w_off + 2 * j, nj, a.N, a.w_stride);
    }
    const int8_t* xb = GROUPED ? a.x : a.x + (int64_t)tile_m * 16 * MT * a.x_stride;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        int src = min(8 * i + lane / 8, rows_here - 1);
        if constexpr (GROUPED) src = UP ? plan_slot(order, src, a.M) / a.top : plan_slot(order, src, a.M);
        x_off[i] = (uint32_t)src * (uint32_t)a.x_stride;
    }
    // What goes with the sums, on its way before the operands. Pieces of 64 sums, row 16 (p / (4 NB)) + 4 (lane / 16) + p % 4 of
    // column 16 (p / 4 % NB) + lane % 16, are shared among the KW waves.
    constexpr int PIECES = MT * NB * 4, OUT = (PIECES + KW - 1) / KW;
    float ws[NB], ws2 = 0.0f;
#pragma unroll
    for (int j = 0; j < NB; ++j) ws[j] = a.ws[(int64_t)expert * a.N + min(n0 + 16 * j + (lane & 15), a.N - 1)];
    if constexpr (UP) ws2 = a.ws2[(int64_t)expert * a.N + min(n0 + (lane & 15), a.N - 1)];
    float xs[OUT], add[OUT];
    int64_t row[OUT];
#pragma unroll
    for (int t = 0; t < OUT; ++t) {
        const int p = min(kw + KW * t, PIECES - 1), r = min(16 * (p / (4 * NB)) + 4 * (lane >> 4) + p % 4, rows_here - 1);
        row[t] = GROUPED ? (int64_t)plan_slot(order, r, a.M) : (int64_t)tile_m * 16 * MT + r;
        xs[t] = a.xs[UP ? row[t] / a.top : row[t]];
        add[t] = !GROUPED && a.R ? a.R[row[t] * a.r_stride + min(n0 + 16 * (p / 4 % NB) + (lane & 15), a.N - 1)] : 0.0f;
    }
    const int stages = (a.K + 127) / 128;
    v4i acc[MT][NT];
    wave_sums<MT, NT>(acc, reinterpret_cast<int8_t*>(smem) + wave * (kStages * 2048 * (MT + NT)), xb, x_off, wb, w_off, a.K,
                      stages * kw / KW, stages * (kw + 1) / KW);
    if constexpr (KW > 1) {
        __syncthreads();  // every wave's stages are done
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) part[nw][kw][(i * NT + j) * 4 + v][lane] = acc[i][j][v];
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < OUT; ++t) {
        const int p = kw + KW * t;
        if (p >= PIECES) continue;
        const int i = p / (4 * NB), j = p / 4 % NB, at = (i * NT + j) * 4 + p % 4;
        int s0 = 0, s1 = 0;
        if constexpr (KW > 1) {
#pragma unroll
            for (int q = 0; q < KW; ++q) {
                s0 += part[nw][q][at][lane];
                if constexpr (UP) s1 += part[nw][q][at + 4][lane];
            }
        } else {  // p is t
            s0 = acc[t / (4 * NB)][t / 4 % NB][t % 4], s1 = acc[t / (4 * NB)][NT - 1][t % 4];
        }
        const int n = n0 + 16 * j + (lane & 15);
        if (16 * i + 4 * (lane >> 4) + p % 4 >= rows_here || n >= a.N) continue;
        float scale = ws[0];
#pragma unroll
        for (int c = 1; c < NB; ++c) scale = j == c ? ws[c] : scale;
        float y = i8_value(s0, scale, xs[t]);
        if constexpr (UP) y = silu(y) * i8_value(s1, ws2, xs[t]);
        if (!GROUPED && a.R) y = i8_plus(y, add[t]);
        static_cast<T*>(a.y)[row[t] * a.y_stride + n] = (T)y;
    }
}

// A token's 16 outputs of the down products, a slot to a wave: y = R + sum of the slots' products by their weights, in one launch
// and without a plan's order.
template <class T>
__global__ void __launch_bounds__(1024) i8_token_kernel(I8Args a, CombineArgs c) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float part[16][16];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t token = blockIdx.x / a.tiles_n;
    const int n0 = (int)blockIdx.x % a.tiles_n * 16, n = n0 + (lane & 15);
    const int64_t slot = token * c.top + wave;
    const int expert = __builtin_amdgcn_readfirstlane(c.expert[slot]);
    if ((unsigned)expert < (unsigned)a.n_expert) {
        uint32_t x_off[2], w_off[2];
        weight_rows(w_off, n0, a.N, a.w_stride);
        x_off[0] = x_off[1] = 0;
        const int8_t* const wb[1] = {uniform(a.w + (int64_t)expert * a.w_expert + (int64_t)n0 * a.w_stride)};
        v4i acc[1][1];
        wave_sums<1, 1>(acc, reinterpret_cast<int8_t*>(smem) + wave * (kStages * 4096), uniform(a.x + slot * a.x_stride), x_off, wb,
                        w_off, a.K, 0, (a.K + 127) / 128);
        if (lane < 16)  // row 0; the others are the same
            part[wave][lane] = i8_value(acc[0][0][0], a.ws[(int64_t)expert * a.N + min(n, a.N - 1)], a.xs[slot]);
    }
    __syncthreads();
    if (threadIdx.x < 16 && n < a.N) {
        float y = 0.0f;
        for (int j = 0; j < c.top; ++j)
            if ((unsigned)c.expert[token * c.top + j] < (unsigned)a.n_expert) y = fmaf(c.weights[token * c.top + j], part[j][threadIdx.x], y);
        if (c.R) y += c.R[token * c.r_stride + n];
        static_cast<T*>(c.y)[token * c.y_stride + n] = (T)y;
    }
}

namespace {

template <I8Mode MODE, int MT, int NB, int KW, int NW, class T>
hipError_t launch_waves(I8Args a, hipStream_t st) {
    constexpr int NT = MODE == kI8Up ? 2 : NB;
    a.tiles_n = (a.N + 16 * NB * NW - 1) / (16 * NB * NW);
    a.tiles_m = (int)(MODE == kI8Dense ? (a.M + 16 * MT - 1) / (16 * MT) : plan_tiles(a.M, a.n_expert, 16 * MT));
    constexpr size_t lds = std::max<size_t>(KW * NW * kStages * (MT + NT) * 2048, KW * NW * MT * NT * 1024);
    i8_rows_kernel<MODE, MT, NB, KW, NW, T>
        <<<dim3((unsigned)((int64_t)a.tiles_n * a.tiles_m)), 64 * KW * NW, lds, st>>>(a);
    return hipGetLastError();
}

// Experts' tiles are many, and a wave's share of K short: 1, 2 or 4 waves by K (48 tokens x 8 of 128, gate and up of 768 rows, with
// 1, 2, 4: K 256 10.1, 11.7, 16.4 us; 1024 33.4, 31.6, 33.2; 2048 61.9, 59.4, 57.8, with 8 79.4; 4096 129.5, 114.1, 112.9; down
// products of 2048 rows: 512 26.9, 29.2, 40.7; 768 38.0, 38.3, 47.0; 1024 46.1, 44.7, 51.6), but two for the slots of one or two
// tokens, whose tiles are few (8 slots, K 2048: 9.2, 8.3, 8.7; 24 slots 16.1, 13.6, 13.3).
template <I8Mode MODE, class T>
hipError_t launch_expert_rows(const I8Args& a, hipStream_t st) {
    if (a.K < 1024) return launch_waves<MODE, 1, 1, 1, 2, T>(a, st);
    return a.K < 2048 || a.M < 16 ? launch_waves<MODE, 1, 1, 2, 1, T>(a, st) : launch_waves<MODE, 1, 1, 4, 1, T>(a, st);
}

template <int MT, class T>
hipError_t launch_dense_rows(const I8Args& a, int nb, hipStream_t st) {
    if (a.K < 512) return launch_waves<kI8Dense, MT, 1, 1, 4, T>(a, st);
    if (nb == 3) return launch_waves<kI8Dense, MT, 3, 4, 1, T>(a, st);
    if (nb == 2) return launch_waves<kI8Dense, MT, 2, 4, 1, T>(a, st);
    // 8 waves on K where no CU has a second workgroup and K is long or CUs are idle (us, 4 and 8: 1 x 4096 x 14336 12.7 and 10.6, 24 rows
    // 14.9 and 14.2; 1 x 2560 x 9728 9.2 and 6.9; 61 x 2048 x 2048 3.8 and 3.6; but 1 x 4096 x 4096 4.5 and 4.8)
    if constexpr (MT <= 2) {
        const int64_t groups = (int64_t)((a.N + 15) / 16) * ((a.M + 16 * MT - 1) / (16 * MT));
        if (groups <= 256 && (a.K >= 8192 || (a.K >= 2048 && a.N < 4096))) return launch_waves<kI8Dense, MT, 1, 8, 1, T>(a, st);
    }
    return launch_waves<kI8Dense, MT, 1, 4, 1, T>(a, st);
}

// 16 mt rows and 16 nb weight rows to a wave. Every workgroup takes its rows of x from L2: more weight rows beside them are fewer
// such trips, but also fewer workgroups. The least by rounds of a workgroup per CU, each of mt + nb pieces of operands; above 32
// rows tiles of 32 are a choice, too (us, nb = 1, 2, 3: 32 x 9728 x 2560 10.6, 10.7, 9.3; 32 x 14336 x 4096 17.7, 15.3, 17.9;
// 24 x 5120 x 8192 15.2, 12.2, 14.6; 61 x 9728 x 2560 14.5, 15.6, 11.5; 61 x 8192 x 2048 7.8, 7.2, 8.7; tiles of 32 for
// 61 x 3584 x 4096 6.3 -> 6.0, 61 x 4608 x 4096 10.4 -> 8.6).
template <class T>
hipError_t launch_dense(const I8Args& a, hipStream_t st) {
    const int all = (int)std::min<int64_t>(4, (a.M + 15) / 16);
    int mt = all, nb = 1;
    int64_t least = INT64_MAX;
    auto look = [&](int m, int most) {
        for (int n = 1; n <= most; ++n) {
            const int64_t groups = (a.N + 16 * n - 1) / (16 * n) * ((a.M + 16 * m - 1) / (16 * m)), cost = (groups + 255) / 256 * (m + n);
            if (cost < least) least = cost, mt = m, nb = n;
        }
    };
    // up to 8 rows HBM is what counts (1 x 9728 x 2560 6.8, 7.7, 6.9; 1 x 151936 x 2560 63.1, 64.2, 65.4), and two
    // workgroups of up to 32 rows with a short K share a CU well (16 x 8192 x 2048 4.8, 5.1; 24 x 7168 x 2048 5.1, 5.2)
    const bool one = a.M <= 8 || a.K < 512 || (a.M <= 32 && a.K < 4096 && a.N <= 512 * 16);
    look(all, one ? 1 : 3);
    if (all > 2 && a.K >= 512) {
        // Two tiles of 32 rows whose workgroups are up to a third more than CUs: the model counts the second round as a whole one, but a
        // CU that holds two of them takes little longer. The two read their weights once between them where they are on one XCD (a multiple
        // of 8 workgroups apart). us, so and by the model, weights from HBM: 48 x 2304 x 4096 7.0, 7.4; 61 x 2304 x 8192 11.4, 11.9; 33 x
        // 2560 x 9728 12.3, 12.1; 48 rows 12.6, 14.1; 61 rows 13.5, 14.4; 61 x 2688 x 4096 7.6, 7.9; x 12288 16.9, 18.6. But 61 x 2816 (352
        // workgroups) x 4096 8.7, 7.9; 48 x 2816 x 8192 13.2, 11.8; 61 x 2816 x 12288 20.6, 18.1; 36 x 2576 (322, on two XCDs) x 4096 7.4, 6.9;
        // x 12288 16.8, 15.8. At K 2048 and 1024 (48 x 2304 5.0, 5.2; 4.1, 4.1) the model stays.
        const int64_t weight_tiles = (a.N + 15) / 16;
        const bool shared = a.K >= 4096 && weight_tiles % 8 == 0 && weight_tiles * ((a.M + 31) / 32) <= 336;
        if (shared) least = INT64_MAX;
        look(2, shared ? 1 : 3);
    }
    if (mt == 1) return launch_dense_rows<1, T>(a, nb, st);
    if (mt == 2) return launch_dense_rows<2, T>(a, nb, st);
    if (mt == 3) return launch_dense_rows<3, T>(a, nb, st);
    return launch_dense_rows<4, T>(a, nb, st);
}

}  // namespace

// Experts' tiles here are of 16 rows (plan_height).
hipError_t launch_i8_rows(I8Mode mode, int ytype, const I8Args& a, hipStream_t st) {
    if (mode == kI8Dense) return ytype == kTypeF16 ? launch_dense<_Float16>(a, st) : launch_dense<float>(a, st);
    if (mode == kI8Up)
        return ytype == kTypeF16 ? launch_expert_rows<kI8Up, _Float16>(a, st) : launch_expert_rows<kI8Up, float>(a, st);
    return launch_expert_rows<kI8Down, float>(a, st);
}

// Up to 64 rows, but of tall matrices the 64 x 64 tiles share the weights' and the rows' way through LDS better (17 rows x
// 151936 x 2560: 81 us here, 78 there; 40 x 14336 x 4096 16.3 and 14.1; but 32 x 32000 x 4096 29.0 and 33.5, 40 x 11008 x 4096
// 11.5 and 13.2, 64 x 8192 x 2048 6.6 and 7.5); and up to 128 or 256 of small ones, which leave those CUs idle (100 x 4096 x 4096:
// 7.7 and 12.4, 256 x 2048 x 2048: 6.6 and 7.7; but 100 x 2560 x 9728 20.3 and 16.2, 150 x 4096 x 4096 13.1 and 12.3).
bool i8_few_rows(int64_t M, int64_t N, int64_t K) {
    if (knob(Knob::I8Rows) >= 0) return M <= knob(Knob::I8Rows);
    if (M <= 64) return M <= 16 || (N < 65536 && (M <= 32 || N < 12288));
    return K <= 4096 && ((M <= 128 && N <= 4096) || (M <= 256 && N <= 2048));
}

hipError_t launch_i8_product(int ytype, const I8Args& a, void* ws, hipStream_t st) {
    return i8_few_rows(a.M, a.N, a.K) ? launch_i8_rows(kI8Dense, ytype, a, st) : launch_i8_gemm(kI8Dense, ytype, a, ws, st);
}

static hipError_t launch_experts(I8Mode mode, int ytype, const I8Args& a, hipStream_t st) {
    return plan_height(a.M, a.n_expert) == 16 ? launch_i8_rows(mode, ytype, a, st) : launch_i8_gemm(mode, ytype, a, nullptr, st);
}

hipError_t launch_moe_gate_up(int htype, const I8Args& a, hipStream_t st) { return launch_experts(kI8Up, htype, a, st); }

hipError_t launch_moe_down(int ytype, I8Args a, const CombineArgs& c, hipStream_t st) {
    // One token, or so few slots that hardly two share an expert: no weight is read more often for it. Not where one wave on K
    // keeps too little on its way: a long K beside few slots (us, this way and by the plan with its launch of sums: one token x 8 of 128,
    // 2048 x 768 6.1 and 9.8; x 8 of 256, 7168 x 2048 24.3 and 42.4; x 4 of 16, 4096 x 4096 14.3 and 15.9; 3 x 6 of 64, 2048 x
    // 1408 11.5 and 13.5; but x 2 of 8, 4096 x 14336 40.1 and 29.2; x 2 of 4, 2048 x 4096 10.1 and 9.0; 5 x 8 of 128, 2048 x
    // 768 14.8 and 13.9; 16 x 8 of 256, 7168 x 2048 296 and 223).
    if (c.top <= 16 && a.M <= 32 && a.K <= 1280 * c.top && (c.rows == 1 || 2 * a.M <= a.n_expert)) {
        a.tiles_n = (a.N + 15) / 16;
        const dim3 grid((unsigned)(a.tiles_n * c.rows));
        const size_t lds = c.top * kStages * 4096;
        if (ytype == kTypeF16) i8_token_kernel<_Float16><<<grid, 64 * c.top, lds, st>>>(a, c);
        else i8_token_kernel<float><<<grid, 64 * c.top, lds, st>>>(a, c);
        return hipGetLastError();
    }
    const hipError_t e = launch_experts(kI8Down, kTypeF32, a, st);
    return e == hipSuccess ? launch_moe_combine(ytype, c, st) : e;
}

}  // namespace dcq
