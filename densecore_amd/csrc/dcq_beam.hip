// dcq_beam.hip — the best continuations of each request's beams over the vocabulary.
//
// Candidate (beam w, token t) scores  beam[w] + log softmax(x[w])[t] = beam[w] + (x[w][t] - lse(w)),
// lse(w) = log sum_t exp x[w][t]; the n_out best of a request, ties to the lower w, then the lower t.
//
//   beam_chunk_kernel  one pass over the logits, a chunk of a row per workgroup: the chunk's sum of exp x, as
//                      2^ref sum 2^(x log2 e - ref), and its n_out largest logits (their order is the scores')
//   beam_join_kernel   per request: lse of each row in 64 bits, and the n_out best of the chunks' candidates
//                      by their 64-bit scores
// A chunk's largest are found without sorting it: the n_out-th largest of the maxima of 64 groups of threads
// is a bound that n_out elements reach at least and few others do; those are ranked against each other.
#include <algorithm>

#include "dcq_common.h"
#include "dcq_kernels.h"
#include "dcq_search.h"

namespace dcq {

constexpr int kBeamThreads = 256;
constexpr int kBeamCap = 1024;  // candidates that are ranked; more (ties) are taken one by one
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);

// Order of logits, then of indices from the lowest: larger key first. 0 is no candidate's.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t idx) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 as 0
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

// The n-th largest (n <= 64) of the 64 values in a wave's lanes.
__device__ __forceinline__ float lanes_nth_largest(float v, int n) {
    const int lane = threadIdx.x & 63;
    int rank = 0;
#pragma unroll
    for (int k = 0; k < 64; ++k) {
        const float o = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), k));
        rank += o > v || (o == v && k < lane);
    }
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), __ffsll((unsigned long long)__ballot(rank == n - 1)) - 1));
}

template <class T, int EPT>
__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(BeamArgs a) {
    constexpr int V = 16 / sizeof(T), NV = EPT / V;
    __shared__ uint64_t keys[kBeamCap];
    __shared__ float wmax[4], gmax[64];
    __shared__ double wsum[4];
    __shared__ int count;
    __shared__ unsigned long long best;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row = blockIdx.y;
    const int chunk = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    // the same elements to a thread whatever the row's alignment: rows of equal logits have equal sums
    float e[NV][V];
    const int64_t v0 = (int64_t)chunk * kBeamThreads * NV + tid;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t i0 = (v0 + j * kBeamThreads) * V;
        if (i0 + V <= a.vocab) {
            uint32_t u[4];
            __builtin_memcpy(u, x + i0, 16);
#pragma unroll
            for (int k = 0; k < V; ++k)
                e[j][k] = sizeof(T) == 4 ? __uint_as_float(u[k % 4])
                                         : half_bits_to_float(k % 2 ? u[k / 2 % 4] >> 16 : u[k / 2 % 4] & 0xFFFFu);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) e[j][k] = i0 + k < a.vocab ? (float)x[i0 + k] : -INFINITY;
        }
    }
    float tmax = -INFINITY;
    bool any_nan = false;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            tmax = fmaxf(tmax, e[j][k]);
            any_nan |= e[j][k] != e[j][k];
        }
    const float qmax = lanes_max<4>(tmax);
    if (lane % 4 == 0) gmax[tid / 4] = qmax;
    const float wm = lanes_max<64>(tmax);
    if (lane == 0) wmax[wave] = wm;
    if (tid == 0) count = 0;
    __syncthreads();
    const float top = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    double ref = 0.0, part[2] = {0.0, 0.0};
    if (fabsf(top) < 65536.0f) {
#pragma clang fp contract(off)
        // 2^(x log2 e) = 2^n 2^f, n whole, x log2 e to 2^-24 in two parts, so that a term is the same number in
        // whatever chunk it is
        const float n_top = floorf(top * kLog2e), cut = top - 150.0f;
        ref = n_top;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float y = e[j][k], hi = y * kLog2e, lo = fmaf(y, kLog2eLow, fmaf(y, kLog2e, -hi));
                const float f = __builtin_amdgcn_fractf(hi), n = hi - f;
                const float p = __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f + lo), (int)(n - n_top));
                part[k % 2] += (double)(y < cut ? 0.0f : p);  // NaN stays
            }
    } else if (top != -INFINITY) {
        ref = (double)top * 1.4426950408889634;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) part[k % 2] += (double)__builtin_amdgcn_exp2f((e[j][k] - top) * kLog2e);
    } else if (__any(any_nan)) {
        part[0] = (double)NAN;
    }
    double sum = part[0] + part[1];
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s, 64);
    if (lane == 0) wsum[wave] = sum;

    // ---- elements no smaller than the n_out-th largest group maximum
    const float bound = lanes_nth_largest(gmax[lane], a.n_out);
    const int64_t list = row * a.chunks + chunk;
    auto index_of = [&](int j, int k) { return (uint32_t)((v0 + j * kBeamThreads) * V + k); };
    if (tmax >= bound && tmax > -INFINITY) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (e[j][k] >= bound && e[j][k] > -INFINITY) {
                    const int at = atomicAdd(&count, 1);
                    if (at < kBeamCap) keys[at] = beam_key(e[j][k], index_of(j, k));
                }
    }
    __syncthreads();
    if (tid == 0) {
        a.stat_sum[list] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
        a.stat_ref[list] = ref;
    }
    uint64_t* out = a.cand + list * a.n_out;
    const int n = count;
    if (n <= kBeamCap) {
        for (int i = tid; i < n; i += kBeamThreads) {
            const uint64_t key = keys[i];
            int rank = 0;
            for (int k = 0; k < n; ++k) rank += keys[k] > key;
            if (rank < a.n_out) out[rank] = key;
        }
        for (int i = n + tid; i < a.n_out; i += kBeamThreads) out[i] = 0;
    } else {
        uint64_t last = ~(uint64_t)0;
        for (int r = 0; r < a.n_out; ++r) {
            if (tid == 0) best = 0;
            __syncthreads();
            uint64_t mine = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (e[j][k] > -INFINITY) {
                        const uint64_t key = beam_key(e[j][k], index_of(j, k));
                        if (key < last && key > mine) mine = key;
                    }
            if (mine) atomicMax(&best, (unsigned long long)mine);
            __syncthreads();
            last = best;
            if (tid == 0) out[r] = last;
            __syncthreads();
        }
    }
}

// A candidate before another: the higher score, then the lower beam * vocab + token.
struct BeamPick {
    double score;
    int64_t at;
    __device__ __forceinline__ bool before(const BeamPick& o) const {
        return score > o.score || (score == o.score && at < o.at);
    }
};

__global__ void __launch_bounds__(kBeamThreads) beam_join_kernel(BeamArgs a) {
    __shared__ BeamPick picks[kBeamCap];
    __shared__ double lse[kBeamMaxBeams], base[kBeamMaxBeams];
    __shared__ float gmax[64];
    __shared__ BeamPick wbest[4];
    __shared__ int count;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t req = blockIdx.x, row0 = req * a.n_beams;
    // ---- lse of each row; base is NaN for a beam without continuations
    for (int w = wave; w < a.n_beams; w += 4) {
        const int64_t list = (row0 + w) * a.chunks;
        double m = -(double)INFINITY;
        for (int c = lane; c < a.chunks; c += 64)
            if (a.stat_sum[list + c] != 0.0) m = fmax(m, a.stat_ref[list + c]);
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) m = fmax(m, __shfl_xor(m, k, 64));
        double s = 0.0;
        for (int c = lane; c < a.chunks; c += 64) {
            const double sc = a.stat_sum[list + c];
            s += sc == 0.0 ? 0.0 : sc * exp2(a.stat_ref[list + c] - m);
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k, 64);
        if (lane == 0) {
            const float b = a.beam[row0 + w];
            // to a multiple of 2^-32, less than its error: the same logits in another order have the same lse
            lse[w] = rint((m + log2(s)) * (0.6931471805599453 * 0x1p32)) * 0x1p-32;
            base[w] = s > 0.0 && s < INFINITY && fabsf(b) < INFINITY ? (double)b : (double)NAN;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    const int lists = a.n_beams * a.chunks;
    const uint64_t* cand = a.cand + row0 * a.chunks * a.n_out;
    auto pick_of = [&](int w, uint64_t key) {
        return BeamPick{base[w] + ((double)key_logit(key) - lse[w]), (int64_t)w * a.vocab + key_index(key)};
    };
    // ---- a bound as in the chunks, on the lists' first candidates (rounded down to fp32: no higher)
    float tmax = -INFINITY;
    for (int i = tid; i < lists; i += kBeamThreads) {
        const uint64_t key = cand[(int64_t)i * a.n_out];
        if (key) tmax = fmaxf(tmax, __double2float_rd(pick_of(i / a.chunks, key).score));
    }
    const float qmax = lanes_max<4>(tmax);
    if (lane % 4 == 0) gmax[tid / 4] = qmax;
    __syncthreads();
    const double bound = lanes_nth_largest(gmax[lane], a.n_out);
    for (int i = tid; i < lists; i += kBeamThreads) {
        for (int r = 0; r < a.n_out; ++r) {
            const uint64_t key = cand[(int64_t)i * a.n_out + r];
            if (!key) break;
            const BeamPick p = pick_of(i / a.chunks, key);
            if (!(p.score >= bound)) break;  // a list is in order; NaN: a beam without continuations
            const int at = atomicAdd(&count, 1);
            if (at < kBeamCap) picks[at] = p;
        }
    }
    __syncthreads();
    auto put = [&](int r, const BeamPick& p) {
        const int64_t o = req * a.n_out + r;
        a.scores[o] = (float)p.score;
        a.parents[o] = (int32_t)(row0 + p.at / a.vocab);
        a.tokens[o] = (int32_t)(p.at % a.vocab);
    };
    auto put_none = [&](int r) {
        const int64_t o = req * a.n_out + r;
        a.scores[o] = -INFINITY, a.parents[o] = -1, a.tokens[o] = -1;
    };
    const int n = count;
    if (n <= kBeamCap) {
        for (int i = tid; i < n; i += kBeamThreads) {
            const BeamPick p = picks[i];
            int rank = 0;
            for (int k = 0; k < n; ++k) rank += picks[k].before(p);
            if (rank < a.n_out) put(rank, p);
        }
        for (int i = n + tid; i < a.n_out; i += kBeamThreads) put_none(i);
        return;
    }
    BeamPick last{INFINITY, -1};
    for (int r = 0; r < a.n_out; ++r) {
        BeamPick mine{-INFINITY, INT64_MAX};
        for (int64_t i = tid; i < (int64_t)lists * a.n_out; i += kBeamThreads) {
            const uint64_t key = cand[i];
            if (!key) continue;
            const BeamPick p = pick_of((int)(i / a.n_out / a.chunks), key);
            if (last.before(p) && p.before(mine)) mine = p;
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const BeamPick o{__shfl_xor(mine.score, k, 64), (int64_t)__shfl_xor((long long)mine.at, k, 64)};
            if (o.before(mine)) mine = o;
        }
        if (lane == 0) wbest[wave] = mine;
        __syncthreads();
        last = wbest[0];
        for (int k = 1; k < 4; ++k)
            if (wbest[k].before(last)) last = wbest[k];
        if (tid == 0) put(r, last);  // more than kBeamCap candidates: there is one in every round
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
// Elements of a thread: 32 where that makes two workgroups per CU or more, else 8.
struct BeamPlan {
    int ept, chunks;
};
static BeamPlan beam_plan(int64_t rows, int vocab) {
    const auto chunks = [&](int ept) { return (vocab + kBeamThreads * ept - 1) / (kBeamThreads * ept); };
    const int ept = rows * chunks(32) >= 2 * (int64_t)cu_count() ? 32 : 8;
    return {ept, chunks(ept)};
}

size_t beam_workspace_bytes(int64_t n_batch, int n_beams, int vocab, int n_out) {
    const int64_t lists = n_batch * n_beams * beam_plan(n_batch * n_beams, vocab).chunks;
    return (size_t)(2 * round_up(lists * 8, 256) + round_up(lists * n_out * 8, 256));
}

hipError_t launch_beam_select(int type, BeamArgs a, int64_t n_batch, void* ws, hipStream_t st) {
    const int64_t rows = n_batch * a.n_beams;
    const BeamPlan p = beam_plan(rows, a.vocab);
    a.chunks = p.chunks;
    const int64_t lists = rows * p.chunks;
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.stat_sum = reinterpret_cast<double*>(w);
    a.stat_ref = reinterpret_cast<double*>(w + round_up(lists * 8, 256));
    a.cand = reinterpret_cast<uint64_t*>(w + 2 * round_up(lists * 8, 256));
    const dim3 grid((unsigned)p.chunks, (unsigned)rows);
    if (type == kTypeF32 && p.ept == 32)
        hipLaunchKernelGGL((beam_chunk_kernel<float, 32>), grid, dim3(kBeamThreads), 0, st, a);
    else if (type == kTypeF32)
        hipLaunchKernelGGL((beam_chunk_kernel<float, 8>), grid, dim3(kBeamThreads), 0, st, a);
    else if (p.ept == 32)
        hipLaunchKernelGGL((beam_chunk_kernel<_Float16, 32>), grid, dim3(kBeamThreads), 0, st, a);
    else
        hipLaunchKernelGGL((beam_chunk_kernel<_Float16, 8>), grid, dim3(kBeamThreads), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)n_batch), dim3(kBeamThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace dcq
