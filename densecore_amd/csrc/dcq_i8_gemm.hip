// dcq_i8_gemm.hip — products of many int8 rows on gfx950 int8 MFMA: dense ones, and those of a plan's experts.
//
//   y[m][n] = (sum over k of x[m][k] w[n][k]) ws[n] xs[m] (+ R[m][n]);   experts' gate and up: silu(y_gate) y_up
//
// The sums are exact in 32 bits, so that tiles and splits of K are chosen by time alone and change no bit.
//
// Large products are bound by the matrix units and the power they draw: 32x32x32 products of random bytes held in registers
// reach 3.5 POPS (of zeros 4.9: the clock falls with the bits that switch); with their operands through LDS 2.3, at 1.85 GHz with
// the units busy 61 % of the time (8192 x 8192 x 8192: 479 us). Hence tiles of 256 x 256, each wave 128 x 64 of it, which read
// the fewest LDS bytes per product (waves of 128 x 128 leave no registers for operands read ahead, and are slower), and nothing
// else next to the products: loads go straight to LDS, two stages of 128 bytes of K ahead, outputs leave through LDS in
// 16-byte stores past the caches. Rings of 3 stages and more, stages of 64 bytes, two workgroups of half the size on a CU, raised
// priorities and fixed orders of reads and products: no faster.
// Small ones are bound by the weights' bytes and by rounds of workgroups: see plan_dense.
// Experts' products are bound by moving rows: for 1571 tokens x 8 of 128 experts the gate and up products of 768 x 2048 take 111 us,
// of which their loads to LDS alone, without products and outputs, take 92 (402 MB of weights, 39 of outputs); the down products
// of 2048 x 768 take 71 (201 MB of weights, 103 of partial rows: 4.3 TB/s). Tiles of 64 x 128, 128 x 128 or 256 x 256, as
// tall as the plan's; a run of tiles to each XCD, whose L2 then holds an expert's weights while its tiles last (tiles interleaved over XCDs,
// weights asked for ahead of their tile, 64 x 256 and 128 x 256: slower).
#include <algorithm>
#include <cmath>

#include "dcq_common.h"
#include "dcq_i8.h"
#include "dcq_i8_tile.h"
#include "dcq_kernels.h"

namespace dcq {

namespace {

constexpr int kXcds = 8;

template <class T>
__device__ __forceinline__ void put(void* y, int64_t at, float v) {
    static_cast<T*>(y)[at] = (T)v;
}

}  // namespace

// A tile of BM rows x BN weight rows per workgroup of WM x WN waves. kI8Up: half of a wave's columns are gate rows and
// half the same rows of the up matrix, so that a lane holds both products of an output.
// T: the output's type; int32_t: the sums themselves, to a plane of `splits`.
template <I8Mode MODE, int BM, int BN, int WM, int WN, int ST, class T>
__global__ void __launch_bounds__(64 * WM * WN, 2) i8_gemm_kernel(I8Args a) {
    constexpr int W = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 32, NJ = TN / 32;
    constexpr int KB = 128;  // bytes of an LDS row
    constexpr int P = KB / 16, LR = 64 / P;  // 16-byte pieces of an LDS row; rows of a 1 KB load
    constexpr int LA = BM / LR / W, LB = BN / LR / W;  // loads of a wave and stage
    constexpr int Q = KB / 32;  // products' steps of a stage
    constexpr bool UP = MODE == kI8Up, GROUPED = MODE != kI8Dense;
    constexpr int TILE_N = UP ? BN / 2 : BN;  // outputs
    struct __align__(16) Stage {
        int8_t a[BM * KB];
        int8_t b[BN * KB];
    };
    extern __shared__ __align__(16) uint8_t smem[];
    Stage* st = reinterpret_cast<Stage*>(smem);
    __shared__ __align__(16) float row_scale[BM], col_scale[BN];
    __shared__ int row_out[BM];  // grouped: the slot
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // ---- which tile: an XCD (workgroup id % 8) takes a run of tiles ----
    const int tiles = a.tiles_n * a.tiles_m;
    const int split = GROUPED ? 0 : (int)blockIdx.x / tiles;
    const int id = (int)blockIdx.x - split * tiles;
    const int xcd = id % kXcds;
    const int at = xcd * (tiles / kXcds) + min(xcd, tiles % kXcds) + id / kXcds;
    int tile_m, tile_n;
    if (GROUPED && !a.banded) {
        tile_m = at / a.tiles_n, tile_n = at % a.tiles_n;
    } else {  // bands of 8 row tiles, so that what an XCD's CUs hold at a time is 8 x 4 tiles
        const int band = at / (8 * a.tiles_n), high = min(8, a.tiles_m - 8 * band), in = at - band * 8 * a.tiles_n;
        tile_m = 8 * band + in % high, tile_n = in / high;
    }
    const int n0 = tile_n * TILE_N;
    int rows_here, expert = 0;
    const int32_t* order = nullptr;
    if constexpr (GROUPED) {
        const PlanTile t = plan_tile(a.plan, a.n_expert, a.M, tile_m, BM);
        if (t.expert < 0) return;
        expert = t.expert, rows_here = t.count;
        order = a.plan + plan_order_at(a.n_expert) + t.begin;
        if (expert == a.n_expert) {  // slots of no expert
            if constexpr (UP) {
                for (int i = tid; i < rows_here * TILE_N; i += 64 * W)
                    if (n0 + i % TILE_N < a.N) put<T>(a.y, (int64_t)plan_slot(order, i / TILE_N, a.M) * a.y_stride + n0 + i % TILE_N, 0.0f);
            }
            return;
        }
    } else {
        rows_here = (int)min((int64_t)BM, a.M - (int64_t)tile_m * BM);
    }

    // ---- loads of a stage: instruction i of a wave fills 8 tile rows, lane l piece l % 8 of row l / 8 ----
    const int8_t* xb = GROUPED ? a.x : a.x + (int64_t)tile_m * BM * a.x_stride;
    const int8_t* wb = a.w + (int64_t)expert * a.w_expert;
    const int8_t* wb2 = UP ? a.w2 + (int64_t)expert * a.w_expert : nullptr;
    uint32_t a_off[LA], b_off[LB];
    const int l_row = lane / P;
    const int8_t* wbase[LB];
#pragma unroll
    for (int i = 0; i < LB; ++i) {
        const int r0 = LR * (LB * wave + i), r = r0 + l_row;
        int n;
        if constexpr (UP) {  // 8 rows of one instruction are of one matrix (TN / 2 is a multiple of 8)
            const int in = r0 % TN;
            wbase[i] = in < TN / 2 ? wb : wb2;
            n = r0 / TN * (TN / 2) + in % (TN / 2) + l_row;
        } else {
            wbase[i] = wb;
            n = r;
        }
        // within the tile's rows: offsets of 32 bits from the tile's first row
        wbase[i] = uniform(wbase[i] + (int64_t)n0 * a.w_stride);
        b_off[i] = (uint32_t)min(n, a.N - 1 - n0) * (uint32_t)a.w_stride + 16u * (uint32_t)((lane % P) ^ piece_key(r));
    }
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int r = LR * (LA * wave + i) + l_row;
        int src = min(r, rows_here - 1);
        if constexpr (GROUPED) src = UP ? plan_slot(order, src, a.M) / a.top : plan_slot(order, src, a.M);
        a_off[i] = (uint32_t)src * (uint32_t)a.x_stride + 16u * (uint32_t)((lane % P) ^ piece_key(r));
    }
    const int stages = (a.K + KB - 1) / KB;
    const int s_begin = split * a.stps, s_end = min(stages, s_begin + a.stps);
    const int tail_pieces = (a.K % KB) / 16;  // 0: the last stage is whole

    auto issue = [&](int s, Stage& S) {  // the wave's LA + LB loads
        const bool tail = tail_pieces && s == stages - 1;
        const int64_t k0 = (int64_t)s * KB;
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const uint32_t piece = (lane % P) ^ piece_key(LR * (LA * wave + i) + l_row);
            dma16(xb + k0, tail && (int)piece >= tail_pieces ? a_off[i] - 16 * piece : a_off[i], S.a + 1024 * (LA * wave + i));
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            const uint32_t piece = (lane % P) ^ piece_key(LR * (LB * wave + i) + l_row);
            dma16(wbase[i] + k0, tail && (int)piece >= tail_pieces ? b_off[i] - 16 * piece : b_off[i],
                  S.b + 1024 * (LB * wave + i));
        }
    };
    // after the wait: pieces past K, which hold the row's first piece again, become zeros in x
    auto clear_tail = [&](int s, Stage& S) {
        if (!(tail_pieces && s == stages - 1)) return;
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const int piece = (lane % P) ^ piece_key(LR * (LA * wave + i) + l_row);
            if (piece >= tail_pieces) *reinterpret_cast<uint4*>(S.a + 1024 * (LA * wave + i) + 16 * lane) = make_uint4(0, 0, 0, 0);
        }
    };

    const int wm = wave / WN * TM, wn = wave % WN * TN;
    const int col = lane & 31, hl = lane >> 5;
    v16i acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;

    // The products run a quarter stage behind the operands' reads, over the stages' borders too: in front of a stage's last
    // quarter, whose operands are in registers, every wave waits for its part of the next stage; behind the barrier that
    // stage is whole and this one's room free for the stage after it.
    v4i fa[2][MI], fb[2][NJ];
    auto read = [&](const Stage& S, int kb, int into) {
        const int fo = col * KB + 16 * ((2 * kb + hl) ^ piece_key(col));
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[into][j] = *reinterpret_cast<const v4i*>(S.b + fo + (wn + 32 * j) * KB);
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[into][i] = *reinterpret_cast<const v4i*>(S.a + fo + (wm + 32 * i) * KB);
    };
    auto multiply = [&](int from) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[from][j], fa[from][i], acc[i][j], 0, 0, 0);
    };
    // the tile's scales, on their way before the stages, and to LDS after the products
    constexpr int RT = (BM + 64 * W - 1) / (64 * W), CT = (BN + 64 * W - 1) / (64 * W);
    float rs[RT], cs[CT];
    int slot[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = min(tid + 64 * W * t, rows_here - 1);
        if constexpr (GROUPED) {
            slot[t] = plan_slot(order, r, a.M);
            rs[t] = a.xs[UP ? slot[t] / a.top : slot[t]];
        } else {
            rs[t] = a.xs[(int64_t)tile_m * BM + r];
        }
    }
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int i = min(tid + 64 * W * t, BN - 1);
        int n = i;
        if constexpr (UP) n = i / TN * (TN / 2) + i % (TN / 2);
        cs[t] = (UP && i % TN >= TN / 2 ? a.ws2 : a.ws)[(int64_t)expert * a.N + min(n0 + n, a.N - 1)];
    }
    // A ring of ST stages. A wave's loads retire in order: all but the last n stages' have landed when no more than n (LA + LB)
    // are on their way.
    if (s_end - s_begin >= ST) {
#pragma unroll
        for (int i = 0; i < ST; ++i) issue(s_begin + i, st[i]);
        counted_wait<(ST - 1) * (LA + LB)>();
    } else {
#pragma unroll
        for (int i = 0; i < ST - 1; ++i)
            if (s_begin + i < s_end) issue(s_begin + i, st[i]);
        counted_wait<0>();
    }
    clear_tail(s_begin, st[0]);
    __syncthreads();
    read(st[0], 0, 0);
    int now = 0;
    for (int s = s_begin; s < s_end; ++s) {
        Stage& S = st[now];
        now = now + 1 == ST ? 0 : now + 1;
        Stage& next = st[now];
#pragma unroll
        for (int q = 1; q < Q; ++q) {
            read(S, q, q & 1);
            multiply((q - 1) & 1);
        }
        if (s + 1 < s_end) {
            counted_wait<(ST - 2) * (LA + LB)>();
            if (ST > 2 && s + ST > s_end) counted_wait<0>();  // fewer stages are on their way
            clear_tail(s + 1, next);
            __syncthreads();
            read(next, 0, 0);
            if (s + ST < s_end) issue(s + ST, S);
        }
        multiply(1);
    }

    // ---- out, 32 rows of a wave at a time: a lane holds row col, columns 32 j + 8 q + 4 hl .. + 3 in sums 4 q .. + 3. Through
    // LDS (the stages' room), so that a row's columns go out in wide stores ----
    constexpr bool SUMS = sizeof(T) == 4 && T(0.5f) == T(0);  // int32_t: a plane of sums
    constexpr int OUT = UP ? TN / 2 : TN, PITCH = OUT + 4, PER = 16 / sizeof(T);  // PER: elements of a store
    __builtin_amdgcn_s_waitcnt(0);  // every stage was waited for: this one makes that plain
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int i = tid + 64 * W * t;
        if (i < BM) {
            row_scale[i] = rs[t];
            if constexpr (GROUPED) row_out[i] = slot[t];
        }
    }
#pragma unroll
    for (int t = 0; t < CT; ++t)
        if (tid + 64 * W * t < BN) col_scale[tid + 64 * W * t] = cs[t];
    __syncthreads();  // and the stages' room is free
    float* mine = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
    const int nw = n0 + wn / (UP ? 2 : 1);  // the wave's first output
    float ws[NJ][16];
    if constexpr (!SUMS) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 f = *reinterpret_cast<const float4*>(col_scale + wn + 32 * j + 8 * q + 4 * hl);
                ws[j][4 * q] = f.x, ws[j][4 * q + 1] = f.y, ws[j][4 * q + 2] = f.z, ws[j][4 * q + 3] = f.w;
            }
    }
    const bool wide = a.y_wide;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        if (wm + 32 * i >= rows_here) break;
        const float xs = row_scale[wm + 32 * i + col];
#pragma unroll
        for (int j = 0; j < OUT / 32; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 4 * q + e;
                    if constexpr (SUMS) v[e] = __int_as_float(acc[i][j][at]);
                    else if constexpr (UP)
                        v[e] = silu(i8_value(acc[i][j][at], ws[j][at], xs)) *
                               i8_value(acc[i][j + NJ / 2][at], ws[j + NJ / 2][at], xs);
                    else v[e] = i8_value(acc[i][j][at], ws[j][at], xs);
                }
                *reinterpret_cast<float4*>(mine + col * PITCH + 32 * j + 8 * q + 4 * hl) = make_float4(v[0], v[1], v[2], v[3]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        constexpr int LANES = OUT / PER;  // of a row
#pragma unroll
        for (int t = 0; t < 32 * LANES / 64; ++t) {
            const int r = t * (64 / LANES) + lane / LANES, c = lane % LANES * PER, n = nw + c;
            if (wm + 32 * i + r >= rows_here || n >= a.N) continue;
            const int64_t row = SUMS ? (int64_t)tile_m * BM + wm + 32 * i + r
                                : GROUPED ? (int64_t)row_out[wm + 32 * i + r] : (int64_t)tile_m * BM + wm + 32 * i + r;
            float v[PER];
#pragma unroll
            for (int e = 0; e < PER; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(mine + r * PITCH + c + e);
                v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
            }
            const int left = min(PER, a.N - n);
            if (MODE == kI8Dense && !SUMS && a.R) {
                const float* add = a.R + row * a.r_stride + n;
                if (left == PER) {
                    float u[PER];
                    __builtin_memcpy(u, __builtin_assume_aligned(add, 4), 4 * PER);
#pragma unroll
                    for (int e = 0; e < PER; ++e) v[e] = i8_plus(v[e], u[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < PER; ++e)
                        if (e < left) v[e] = i8_plus(v[e], add[e]);
                }
            }
            T o[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                if constexpr (SUMS) o[e] = __float_as_int(v[e]);
                else o[e] = (T)v[e];
            }
            T* y = static_cast<T*>(a.y) + (SUMS ? (int64_t)split * a.M * a.N : 0) + row * a.y_stride + n;
            if (left == PER && wide) {
                store_through(y, o);
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (e < left) y[e] = o[e];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// y = the sum of the planes' int32 sums (exact, so that any split gives the same bits), scaled, plus R. A thread for V
// columns of a row.
template <class T, int V>
__global__ void __launch_bounds__(256) i8_join_kernel(I8Args a, const int32_t* planes) {
    const int blocks = (a.N + 256 * V - 1) / (256 * V);
    const int64_t row = blockIdx.x / blocks;
    const int n = ((int)blockIdx.x % blocks * 256 + (int)threadIdx.x) * V;
    if (n >= a.N) return;
    const int32_t* p = planes + row * a.N + n;
    int sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        int v[V];
        __builtin_memcpy(v, __builtin_assume_aligned(p + s * (a.M * a.N), 4 * V), 4 * V);
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += v[e];
    }
    const float xs = a.xs[row];
    T o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float y = i8_value(sum[e], a.ws[n + e], xs);
        if (a.R) y = i8_plus(y, a.R[row * a.r_stride + n + e]);
        o[e] = (T)y;
    }
    T* y = static_cast<T*>(a.y) + row * a.y_stride + n;
    if (V > 1 && a.y_wide) {
        __builtin_memcpy(__builtin_assume_aligned(y, 4), o, sizeof(o));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = o[e];
    }
}

namespace {

template <I8Mode MODE, int BM, int BN, int WM, int WN, int ST, class T>
hipError_t launch_tile(I8Args a, hipStream_t st) {
    constexpr int tile_n = MODE == kI8Up ? BN / 2 : BN;
    a.tiles_n = (a.N + tile_n - 1) / tile_n;
    a.tiles_m = (int)(MODE == kI8Dense ? (a.M + BM - 1) / BM : plan_tiles(a.M, a.n_expert, BM));
    constexpr int out = MODE == kI8Up ? BN / WN / 2 : BN / WN;
    const size_t lds = std::max<size_t>(ST * (size_t)(BM + BN) * 128, (size_t)WM * WN * 32 * (out + 4) * 4);
    const int64_t groups = (int64_t)a.tiles_n * a.tiles_m * a.splits;
    auto fn = i8_gemm_kernel<MODE, BM, BN, WM, WN, ST, T>;
    fn<<<dim3((unsigned)groups), 64 * WM * WN, lds, st>>>(a);
    return hipGetLastError();
}

template <I8Mode MODE, class T>
hipError_t launch_shape(I8Args a, int shape, hipStream_t st) {
    if constexpr (MODE == kI8Dense) {
        if (shape == 0) return launch_tile<MODE, 64, 64, 2, 2, 4, T>(a, st);
        if (shape == 3) return launch_tile<MODE, 256, 256, 2, 4, 2, T>(a, st);
    } else {
        if (shape == 1) return launch_tile<MODE, 64, 128, 2, 2, 2, T>(a, st);
        if (shape == 3) return launch_tile<MODE, 256, 256, 2, 4, 2, T>(a, st);
    }
    return launch_tile<MODE, 128, 128, 2, 2, 2, T>(a, st);
}

template <class T>
hipError_t launch_join(const I8Args& a, const void* planes, hipStream_t st) {
    const int per = a.N % 4 ? 256 : 1024;
    const dim3 grid((unsigned)((a.N + per - 1) / per * a.M));
    if (per == 1024) i8_join_kernel<T, 4><<<grid, 256, 0, st>>>(a, static_cast<const int32_t*>(planes));
    else i8_join_kernel<T, 1><<<grid, 256, 0, st>>>(a, static_cast<const int32_t*>(planes));
    return hipGetLastError();
}

}  // namespace

// Which tile, and into how many shares of K: the least of the times that the kernels take by their rounds of workgroups,
// fitted to 64 products of 40 to 1536 rows x 1024 .. 14336 x 1024 .. 14336 (the choice is never more than 13 % behind the
// best of them, and mostly the best). A round is a + b * stages us, less where its workgroups have a CU to themselves; a
// split adds a launch that reads its planes.
struct DensePlan {
    int shape, splits;
};
static DensePlan plan_dense(int64_t M, int64_t N, int64_t K, bool may_split) {
    static const struct {
        int shape, bm, bn, slots;
        double a, b, a_half, b_half;
    } kTiles[] = {{0, 64, 64, 512, 7.5, 0.27, 3.5, 0.28}, {2, 128, 128, 512, 8.0, 0.87, 8.0, 0.52}, {3, 256, 256, 256, 17.0, 1.38, 8.0, 1.2}};
    const int forced = knob(Knob::I8Tile), forced_split = knob(Knob::I8Split);
    const int64_t stages = (K + 127) / 128;
    DensePlan best = {2, 1};
    double least = INFINITY;
    for (const auto& t : kTiles) {
        if (forced >= 0 && forced != t.shape) continue;
        for (int splits : {1, 2, 3, 4, 6, 8}) {
            if (splits > 1 && (!may_split || stages / splits < 8 || M * N * splits > (int64_t)1 << 24)) break;
            if (forced_split > 0 && splits != forced_split) continue;
            const int64_t groups = (M + t.bm - 1) / t.bm * ((N + t.bn - 1) / t.bn) * splits, rest = groups % t.slots;
            const double st = (double)((stages + splits - 1) / splits);
            double us = (double)(groups / t.slots + (rest > t.slots / 2)) * (t.a + t.b * st);
            if (rest && rest <= t.slots / 2) us += t.a_half + t.b_half * st;
            if (splits > 1) us += 3.0 + (double)(8 * splits + 4) * (double)(M * N) / 9e6;
            if (us < least) least = us, best = {t.shape, splits};
        }
    }
    return best;
}

size_t i8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (i8_few_rows(M, N, K)) return 0;
    const DensePlan p = plan_dense(M, N, K, true);
    return p.splits > 1 ? (size_t)round_up(p.splits * M * N * 4, 256) : 0;
}

hipError_t launch_i8_gemm(I8Mode mode, int ytype, I8Args a, void* ws, hipStream_t st) {
    const int stages = (a.K + 127) / 128;
    a.splits = 1, a.stps = stages;
    // wide stores need whole dwords
    a.y_wide = ytype == kTypeF32 || (a.y_stride % 2 == 0 && (uintptr_t)a.y % 4 == 0);
    if (mode != kI8Dense) {
        // An expert's tiles of all columns for a row tile, then the next row tile's, while its weights stay in an XCD's L2
        // between the two; else bands (us: 4096 tokens x 8 of 128, gate and up of 768 x 2048 188 so and 209 in bands; but 4096 x 2 of 8,
        // 14336 x 4096 1671 and 1249).
        a.banded = (mode == kI8Up ? 2 : 1) * (int64_t)a.N * a.K > (int64_t)8 << 20;
        const int height = plan_height(a.M, a.n_expert), shape = height == 256 ? 3 : height == 128 ? 2 : 1;
        if (mode == kI8Up)
            return ytype == kTypeF16 ? launch_shape<kI8Up, _Float16>(a, shape, st) : launch_shape<kI8Up, float>(a, shape, st);
        return launch_shape<kI8Down, float>(a, shape, st);
    }
    const DensePlan plan = plan_dense(a.M, a.N, a.K, ws != nullptr);
    if (plan.splits <= 1)
        return ytype == kTypeF16 ? launch_shape<kI8Dense, _Float16>(a, plan.shape, st) : launch_shape<kI8Dense, float>(a, plan.shape, st);
    a.stps = (stages + plan.splits - 1) / plan.splits;
    a.splits = (stages + a.stps - 1) / a.stps;
    I8Args p = a;
    p.y = ws, p.y_stride = a.N, p.y_wide = true;
    const hipError_t e = launch_shape<kI8Dense, int32_t>(p, plan.shape, st);
    if (e != hipSuccess) return e;
    return ytype == kTypeF16 ? launch_join<_Float16>(a, ws, st) : launch_join<float>(a, ws, st);
}

}  // namespace dcq
