// dcq_i8_gemm.hip — products of many int8 rows on gfx950 int8 MFMA: dense ones, and those of a plan's experts.
#include <algorithm>

#include "dcq_common.h"
#include "dcq_i8.h"
#include "dcq_i8_tile.h"
#include "dcq_kernels.h"

#pragma clang diagnostic ignored "-Winline-asm"  // M0 in the clobber list (see dma16)

namespace dcq {

namespace {

constexpr int kRowB = 128;  // k per stage = bytes of an LDS row: 8 pieces of 16, piece p of row r at p ^ key(r)
constexpr int kXcds = 8;

__device__ __forceinline__ int piece_key(int row) { return (row & 7) ^ ((row >> 3) & 1); }

typedef __attribute__((address_space(3))) void* lds_ptr_t;

// 16 bytes per lane from a uniform base + per-lane offset to LDS at lds_base + 16 * lane (lds_base uniform, in M0). The
// compiler does not count these loads: an explicit wait comes before the barrier that publishes them.
__device__ __forceinline__ void dma16(const void* g, uint32_t off, const void* lds_base) {
    const uint32_t m0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds_base;
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(g), "s"(m0) : "memory", "m0");
}

template <class T>
__device__ __forceinline__ void put(void* y, int64_t at, float v) {
    static_cast<T*>(y)[at] = (T)v;
}

}  // namespace

// A tile of BM rows x BN weight rows per workgroup of WM x WN waves. kI8Up: half of a wave's columns are gate rows and
// half the same rows of the up matrix, so that a lane holds both products of an output.
// T: the output's type; int32_t: the sums themselves, to a plane of `splits`.
template <I8Mode MODE, int BM, int BN, int WM, int WN, class T>
__global__ void __launch_bounds__(64 * WM * WN, 2) i8_gemm_kernel(I8Args a) {
    constexpr int W = WM * WN, TM = BM / WM, TN = BN / WN, MI = TM / 32, NJ = TN / 32;
    constexpr int LA = BM / 8 / W, LB = BN / 8 / W;  // 1 KB loads of a wave and stage
    constexpr bool UP = MODE == kI8Up, GROUPED = MODE != kI8Dense;
    constexpr int TILE_N = UP ? BN / 2 : BN;  // outputs
    struct __align__(16) Stage {
        int8_t a[BM * kRowB];
        int8_t b[BN * kRowB];
    };
    extern __shared__ __align__(16) uint8_t smem[];
    Stage* st = reinterpret_cast<Stage*>(smem);
    __shared__ float row_scale[BM];
    __shared__ int row_out[BM];  // grouped: the slot
    __shared__ PlanTile found;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    // ---- which tile: an XCD (workgroup id % 8) takes a run of tiles, the row tiles of one band of weights ----
    const int tiles = a.tiles_n * a.tiles_m;
    const int split = GROUPED ? 0 : (int)blockIdx.x / tiles;
    const int id = (int)blockIdx.x - split * tiles;
    int at = id;
    if (tiles % kXcds == 0) at = id % kXcds * (tiles / kXcds) + id / kXcds;
    int tile_m, tile_n;
    if constexpr (GROUPED) tile_m = at / a.tiles_n, tile_n = at % a.tiles_n;
    else tile_n = at / a.tiles_m, tile_m = at % a.tiles_m;
    const int n0 = tile_n * TILE_N;
    int rows_here, expert = 0, begin = 0;
    if constexpr (GROUPED) {
        if (wave == 0) {
            const PlanTile t = find_tile(a.plan, a.n_expert, BM, tile_m);
            if (lane == 0) found = t;
        }
        __syncthreads();
        expert = __builtin_amdgcn_readfirstlane(found.expert);
        begin = __builtin_amdgcn_readfirstlane(found.begin);
        rows_here = __builtin_amdgcn_readfirstlane(found.count);
        if (expert < 0) return;
        const int32_t* order = a.plan + plan_order_at(a.n_expert) + begin;
        if (expert == a.n_expert) {  // slots of no expert
            if constexpr (UP) {
                for (int i = tid; i < rows_here * TILE_N; i += 64 * W)
                    if (n0 + i % TILE_N < a.N) put<T>(a.y, (int64_t)order[i / TILE_N] * a.y_stride + n0 + i % TILE_N, 0.0f);
            }
            return;
        }
        for (int i = tid; i < BM; i += 64 * W) {
            const int slot = order[min(i, rows_here - 1)];
            row_out[i] = slot;
            row_scale[i] = a.xs[UP ? slot / a.top : slot];
        }
        __syncthreads();
    } else {
        rows_here = (int)min((int64_t)BM, a.M - (int64_t)tile_m * BM);
        for (int i = tid; i < BM; i += 64 * W) row_scale[i] = a.xs[(int64_t)tile_m * BM + min(i, rows_here - 1)];
    }

    // ---- loads of a stage: instruction i of a wave fills 8 tile rows, lane l piece l % 8 of row l / 8 ----
    const int8_t* xb = GROUPED ? a.x : a.x + (int64_t)tile_m * BM * a.x_stride;
    const int8_t* wb = a.w + (int64_t)expert * a.w_expert;
    const int8_t* wb2 = UP ? a.w2 + (int64_t)expert * a.w_expert : nullptr;
    uint32_t a_off[LA], b_off[LB];
    const int l_row = lane >> 3;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int r = 8 * (LA * wave + i) + l_row;
        const int src = GROUPED ? (UP ? row_out[r] / a.top : row_out[r]) : min(r, rows_here - 1);
        a_off[i] = (uint32_t)src * (uint32_t)a.x_stride + 16u * (uint32_t)((lane & 7) ^ piece_key(r));
    }
    const int8_t* wbase[LB];
#pragma unroll
    for (int i = 0; i < LB; ++i) {
        const int r0 = 8 * (LB * wave + i), r = r0 + l_row;
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
        wbase[i] += (int64_t)n0 * a.w_stride;
        b_off[i] = (uint32_t)min(n, a.N - 1 - n0) * (uint32_t)a.w_stride + 16u * (uint32_t)((lane & 7) ^ piece_key(r));
    }
    const int stages = (a.K + kRowB - 1) / kRowB;
    const int s_begin = split * a.stps, s_end = min(stages, s_begin + a.stps);
    const int tail_pieces = (a.K % kRowB) / 16;  // 0: the last stage is whole

    // loads from .. to of the wave's LA + LB
    auto issue = [&](int s, Stage& S, int from, int to) {
        const bool tail = tail_pieces && s == stages - 1;
        const int64_t k0 = (int64_t)s * kRowB;
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            if (i < from || i >= to) continue;
            const uint32_t piece = (lane & 7) ^ piece_key(8 * (LA * wave + i) + l_row);
            dma16(xb + k0, tail && (int)piece >= tail_pieces ? a_off[i] - 16 * piece : a_off[i], S.a + 1024 * (LA * wave + i));
        }
#pragma unroll
        for (int i = 0; i < LB; ++i) {
            if (i + LA < from || i + LA >= to) continue;
            const uint32_t piece = (lane & 7) ^ piece_key(8 * (LB * wave + i) + l_row);
            dma16(wbase[i] + k0, tail && (int)piece >= tail_pieces ? b_off[i] - 16 * piece : b_off[i],
                  S.b + 1024 * (LB * wave + i));
        }
    };
    // after the wait: pieces past K, which hold the row's first piece again, become zeros in x
    auto clear_tail = [&](int s, Stage& S) {
        if (!(tail_pieces && s == stages - 1)) return;
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const int piece = (lane & 7) ^ piece_key(8 * (LA * wave + i) + l_row);
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

    issue(s_begin, st[0], 0, LA + LB);
    __builtin_amdgcn_s_waitcnt(0);
    clear_tail(s_begin, st[0]);
    __syncthreads();
    for (int s = s_begin; s < s_end; ++s) {
        const Stage& S = st[(s - s_begin) & 1];
        Stage& next = st[(s - s_begin + 1) & 1];
        const bool more = s + 1 < s_end;
        v4i fa[2][MI], fb[2][NJ];
        auto read = [&](int kb, int into) {
            const int fo = col * kRowB + 16 * ((2 * kb + hl) ^ piece_key(col));
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[into][i] = *reinterpret_cast<const v4i*>(S.a + fo + (wm + 32 * i) * kRowB);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[into][j] = *reinterpret_cast<const v4i*>(S.b + fo + (wn + 32 * j) * kRowB);
        };
        read(0, 0);
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            if (kb < 3) read(kb + 1, (kb + 1) & 1);
            if (kb < 2 && more) issue(s + 1, next, kb * (LA + LB) / 2, (kb + 1) * (LA + LB) / 2);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[kb & 1][j], fa[kb & 1][i], acc[i][j], 0, 0, 0);
        }
        if (more) {
            __builtin_amdgcn_s_waitcnt(0);
            clear_tail(s + 1, next);
            __syncthreads();
        }
    }

    // ---- out, 32 rows of a wave at a time: a lane holds row col, columns 32 j + 8 q + 4 hl .. + 3 in sums 4 q .. + 3. Through
    // LDS (the stages' room), so that a row's columns go out in wide stores ----
    constexpr bool SUMS = sizeof(T) == 4 && T(0.5f) == T(0);  // int32_t: a plane of sums
    constexpr int OUT = UP ? TN / 2 : TN, PITCH = OUT + 4, PER = 16 / sizeof(T);  // PER: elements of a store
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
    const int nw = n0 + wn / (UP ? 2 : 1);  // the wave's first output
    float ws[NJ][16];
    if constexpr (!SUMS) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const int n = nw + 32 * (UP ? j % (NJ / 2) : j) + 8 * (v >> 2) + 4 * hl + (v & 3);
                ws[j][v] = (UP && j >= NJ / 2 ? a.ws2 : a.ws)[(int64_t)expert * a.N + min(n, a.N - 1)];
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
                    for (int e = 0; e < PER; ++e) v[e] += u[e];
                } else {
#pragma unroll
                    for (int e = 0; e < PER; ++e)
                        if (e < left) v[e] += add[e];
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
                __builtin_memcpy(__builtin_assume_aligned(y, 4), o, 16);
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (e < left) y[e] = o[e];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// y = the sum of the planes' int32 sums (exact, so that any split gives the same bits), scaled, plus R.
template <class T>
__global__ void __launch_bounds__(256) i8_join_kernel(I8Args a, const int32_t* planes) {
    const int64_t n = a.N, plane = a.M * n;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < plane; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / n, c = i - row * n;
        int sum = 0;
        for (int s = 0; s < a.splits; ++s) sum += planes[s * plane + i];
        float y = i8_value(sum, a.ws[c], a.xs[row]);
        if (a.R) y += a.R[row * a.r_stride + c];
        put<T>(a.y, row * a.y_stride + c, y);
    }
}

namespace {

template <I8Mode MODE, int BM, int BN, int WM, int WN, class T>
hipError_t launch_tile(I8Args a, hipStream_t st) {
    constexpr int tile_n = MODE == kI8Up ? BN / 2 : BN;
    a.tiles_n = (a.N + tile_n - 1) / tile_n;
    a.tiles_m = (int)(MODE == kI8Dense ? (a.M + BM - 1) / BM : most_tiles(a.M, a.n_expert, BM));
    const size_t lds = 2 * (size_t)(BM + BN) * kRowB;
    const int64_t groups = (int64_t)a.tiles_n * a.tiles_m * a.splits;
    auto fn = i8_gemm_kernel<MODE, BM, BN, WM, WN, T>;
    fn<<<dim3((unsigned)groups), 64 * WM * WN, lds, st>>>(a);
    return hipGetLastError();
}

template <I8Mode MODE, class T>
hipError_t launch_shape(I8Args a, int shape, hipStream_t st) {
    switch (shape) {
        case 0: return launch_tile<MODE, 64, 128, 2, 2, T>(a, st);
        case 1: return launch_tile<MODE, 128, 128, 2, 2, T>(a, st);
        default: return launch_tile<MODE, 256, 256, 2, 4, T>(a, st);
    }
}

}  // namespace

hipError_t launch_i8_gemm(I8Mode mode, int ytype, I8Args a, void* ws, size_t ws_bytes, hipStream_t st) {
    const int stages = (a.K + kRowB - 1) / kRowB;
    a.splits = 1, a.stps = stages;
    // wide stores need whole dwords
    a.y_wide = ytype == kTypeF32 || (a.y_stride % 2 == 0 && (uintptr_t)a.y % 4 == 0);
    const int forced = knob(Knob::I8Tile);
    if (mode != kI8Dense) {
        const int64_t mean = a.M / a.n_expert;
        const int shape = forced >= 0 ? forced : mean >= 192 ? 2 : mean >= 48 ? 1 : 0;
        if (mode == kI8Up)
            return ytype == kTypeF16 ? launch_shape<kI8Up, _Float16>(a, shape, st) : launch_shape<kI8Up, float>(a, shape, st);
        return launch_shape<kI8Down, float>(a, shape, st);
    }
    auto tiles = [&](int bm, int bn) { return (a.M + bm - 1) / bm * ((a.N + bn - 1) / bn); };
    int shape = forced >= 0 ? forced : tiles(256, 256) >= 200 ? 2 : a.M > 64 ? 1 : 0;
    const int64_t count = shape == 2 ? tiles(256, 256) : shape == 1 ? tiles(128, 128) : tiles(64, 128);
    const int forced_split = knob(Knob::I8Split);
    int splits = 1;
    if (count < 256) {
        splits = (int)std::min<int64_t>({512 / count, stages / 4, (int64_t)(ws_bytes / 4) / (a.M * a.N)});
        splits = std::max(splits, 1);
    }
    if (forced_split > 0) splits = std::min<int64_t>(forced_split, std::max<int64_t>(1, (int64_t)(ws_bytes / 4) / (a.M * a.N)));
    if (splits == 1)
        return ytype == kTypeF16 ? launch_shape<kI8Dense, _Float16>(a, shape, st) : launch_shape<kI8Dense, float>(a, shape, st);
    a.stps = (stages + splits - 1) / splits;
    a.splits = (stages + a.stps - 1) / a.stps;
    I8Args p = a;
    p.y = ws, p.y_stride = a.N, p.y_wide = true;
    hipError_t e = launch_shape<kI8Dense, int32_t>(p, shape, st);
    if (e != hipSuccess) return e;
    const unsigned blocks = (unsigned)std::min<int64_t>((a.M * a.N + 255) / 256, 2048);
    if (ytype == kTypeF16) i8_join_kernel<_Float16><<<blocks, 256, 0, st>>>(a, static_cast<const int32_t*>(ws));
    else i8_join_kernel<float><<<blocks, 256, 0, st>>>(a, static_cast<const int32_t*>(ws));
    return hipGetLastError();
}

size_t i8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (K <= 1024 || M * N > (int64_t)1 << 24) return 0;
    return (size_t)std::min<int64_t>(16, K / 512) * M * N * 4 > ((size_t)64 << 20) ? (size_t)64 << 20
                                                                                   : (size_t)std::min<int64_t>(16, K / 512) * M * N * 4;
}

}  // namespace dcq
