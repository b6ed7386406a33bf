// dcq_beam.hip — the best continuations of each request's beams over the vocabulary.
//
// Candidate (beam w, token t) scores  beam[w] + log softmax(x[w])[t] = beam[w] + (x[w][t] - lse(w)),
// lse(w) = log sum_t exp x[w][t]; the n_out best of a request, ties to the lower w, then the lower t.
//
//   beam_chunk_kernel  one pass over the logits, a chunk of a row per workgroup: the chunk's sum of exp x, as
//                      e^ref sum e^(x - ref), and its n_out largest logits (their order is the scores')
//   beam_join_kernel   per request: lse of each row in 64 bits, and the n_out best of the chunks' candidates
//                      by their 64-bit scores
// A chunk's largest are found without sorting it: just below the n_out-th largest of the maxima of 64 or 256 groups of
// threads lies a bound that n_out elements reach at least and few others do; those are ranked against each other.
#include <algorithm>

#include "dcq_common.h"
#include "dcq_kernels.h"
#include "dcq_search.h"

namespace dcq {

constexpr int kBeamThreads = 256;
constexpr int kBeamCap = 1024;  // candidates that are ranked; more (ties) are taken one by one
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eLow = (float)(1.4426950408889634 - (double)kLog2e);

__device__ __forceinline__ uint32_t order_bits(float x) {  // larger for larger x; -0 below 0
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
// Order of logits, then of indices (beam << 24 | token) from the lowest: larger key first. 0 is no candidate's.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t idx) {
    return (uint64_t)order_bits(x + 0.0f) << 32 | (0xFFFFFFFFu - idx);  // -0 as 0
}
__device__ __forceinline__ float key_logit(uint64_t key) { return order_value((uint32_t)(key >> 32)); }
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

// A bound that n (<= 64) of the values in a wave's 64 lanes, G in each, reach: the n-th largest to 20 bits (its sign,
// exponent and 11 bits, the rest as low as can be), found bit by bit with one comparison each. No more exact: a
// bound a thousandth lower lets a few candidates more through.
template <int G>
__device__ __forceinline__ float lanes_bound(const float (&v)[G], int n) {
    uint32_t o[G], t = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) o[g] = order_bits(v[g]);
#pragma unroll
    for (int b = 31; b >= 12; --b) {
        const uint32_t with = t | 1u << b;
        int reach = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) reach += (int)__popcll(__ballot(o[g] >= with));
        if (reach >= n) t = with;
    }
    return t < 0x00800000u ? -INFINITY : order_value(t);  // below the finite ones
}
// The bound on the maxima of the workgroup's groups of threads: 64 of them up to 32 outputs, 256 beyond, where 64
// groups' maxima would all have to be reached (4 beams over 151936 tokens, 64 outputs: hundreds of elements of a
// chunk and more candidates than are ranked, 472 us).
constexpr int kFewGroups = 32;
__device__ __forceinline__ float groups_bound(const float* gmax, int lane, int n) {
    if (n <= kFewGroups) return lanes_bound<1>({gmax[lane]}, n);
    return lanes_bound<4>({gmax[lane], gmax[lane + 64], gmax[lane + 128], gmax[lane + 192]}, n);
}

// All of a thread's logits are loaded at once and stay in registers. 256 rows of 151936 F32: 34 us for 156 MB, 4.6 TB/s,
// 93 % of a copy's rate; VALU (the exponentials, and their sums in 64 bits) busy 73 % of it. 4 rows: 4.9 us, latency.
template <class T, int EPT>
__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(BeamArgs a) {
    constexpr int V = 16 / sizeof(T), NV = EPT / V;
    __shared__ uint64_t keys[kBeamCap];
    __shared__ float wmax[4], gmax[256];
    __shared__ double wsum[4];
    __shared__ int count;
    __shared__ unsigned long long best;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t row = blockIdx.y;
    const int chunk = blockIdx.x;
    const uint32_t beam = (uint32_t)(row % a.n_beams) << 24;
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
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) tmax = fmaxf(tmax, e[j][k]);
    if (a.n_out <= kFewGroups) {
        const float qmax = lanes_max<4>(tmax);
        if (lane % 4 == 0) gmax[tid / 4] = qmax;
    } else {
        gmax[tid] = tmax;
    }
    const float wm = lanes_max<64>(tmax);
    if (lane == 0) wmax[wave] = wm;
    if (tid == 0) count = 0;
    __syncthreads();
    const float top = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    // exp x = e^ref e^d, d = x - ref: the difference first, so that nothing overflows or rounds by the size of x
    // (finite logits go up to 3.4e38, and 2.4e38 times log2 e is infinite). e^d = 2^hi (1 + ln 2 low), the product
    // d log2 e rounded and what that left; of a term that counts |d| is below 200, and low below 2^-16. ref is 0 for
    // all logits but far ones, so that a term is the same number in whatever chunk it is, and then the multiple of 64
    // (of 2^30 on: the logit) next to the chunk's largest
    const float ref = fabsf(top) < 44.0f || top == -INFINITY ? 0.0f : 64.0f * rintf(top * (1.0f / 64.0f));
    double part[2] = {0.0, 0.0};
    {
#pragma clang fp contract(off)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = e[j][k] - ref, hi = d * kLog2e;
                // in bounds, and a number beside -infinity
                const float lo = __builtin_amdgcn_fmed3f(fmaf(d, kLog2eLow, fmaf(d, kLog2e, -hi)), -0.5f, 0.5f);
                const float t = __builtin_amdgcn_exp2f(hi);
                part[k % 2] += (double)fmaf(t * lo, 0.693147181f, t);
            }
    }
    double sum = part[0] + part[1];
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s, 64);
    if (lane == 0) wsum[wave] = sum;

    // ---- elements no smaller than the bound on the groups' maxima
    const float bound = groups_bound(gmax, lane, a.n_out);
    const int64_t list = row * a.chunks + chunk;
    auto index_of = [&](int j, int k) { return beam | (uint32_t)((v0 + j * kBeamThreads) * V + k); };
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

// A candidate before another: the higher score, then the lower beam << 24 | token.
struct BeamPick {
    double score;
    uint32_t at;
    __device__ __forceinline__ bool before(const BeamPick& o) const {
        return score > o.score || (score == o.score && at < o.at);
    }
};

constexpr int kJoinThreads = 1024, kJoinWaves = kJoinThreads / 64;
constexpr int kBeamBatch = 8;  // candidates of a thread that wait in registers
// A workgroup per request, bound by its latency: loads, the rows' sums, two barriers of bounds and ranks (4 rows of 75
// chunks, 8 outputs: 6.4 us; 8 rows of 19, 16 outputs: 9).
__global__ void __launch_bounds__(kJoinThreads) beam_join_kernel(BeamArgs a) {
    constexpr int NK = kBeamBatch;
    __shared__ BeamPick picks[kBeamCap];
    __shared__ double lse[kBeamMaxBeams], base[kBeamMaxBeams], from[kBeamMaxBeams];
    __shared__ float gmax[256];
    __shared__ BeamPick wbest[kJoinWaves];
    __shared__ int count;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t req = blockIdx.x, row0 = req * a.n_beams;
    const int lists = a.n_beams * a.chunks, total = lists * a.n_out;
    const uint64_t* cand = a.cand + row0 * a.chunks * a.n_out;
    // As they lie if all fit in registers and a list is no longer than a group of 16 threads; else the lists' first
    // ones, then the second ones, ...: the best are spread over the groups, and held (8 beams over 151936 tokens, 16
    // outputs, join 7.0 | 11.2 us; 4 beams, 64 outputs 45 | 21, 16 beams 416 | 18).
    constexpr int held = NK * kJoinThreads;
    const bool in_lists = total <= held && a.n_out <= 16;
    auto candidate = [&](int i) {
        return i >= total ? 0 : in_lists ? cand[i] : cand[(int64_t)(i % lists) * a.n_out + i / lists];
    };
    uint64_t mine[NK];
#pragma unroll
    for (int k = 0; k < NK; ++k) mine[k] = candidate(tid + k * kJoinThreads);
    // ---- lse of each row, from its largest chunk's reference; base is NaN for a beam without continuations
    for (int w = wave; w < a.n_beams; w += kJoinWaves) {
        const int64_t list = (row0 + w) * a.chunks;
        double m = -(double)INFINITY;
        for (int c = lane; c < a.chunks; c += 64)
            if (a.stat_sum[list + c] != 0.0) m = fmax(m, (double)a.stat_ref[list + c]);
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) m = fmax(m, __shfl_xor(m, k, 64));
        double s = 0.0;
        for (int c = lane; c < a.chunks; c += 64) {
            const double sc = a.stat_sum[list + c], r = a.stat_ref[list + c];
            s += sc == 0.0 ? 0.0 : r == m ? sc : sc * exp(r - m);
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k, 64);
        if (lane == 0) {
            const float b = a.beam[row0 + w];
            from[w] = m;
            // to a multiple of 2^-32, less than its error: the same logits in another order have the same lse
            lse[w] = rint(log(s) * 0x1p32) * 0x1p-32;
            base[w] = s > 0.0 && s < INFINITY && fabsf(b) < INFINITY ? (double)b : (double)NAN;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    auto pick_of = [&](uint64_t key) {
        const uint32_t at = key_index(key), w = at >> 24;
        return BeamPick{base[w] + (((double)key_logit(key) - from[w]) - lse[w]), at};
    };
    // ---- a bound as in the chunks, on the groups' largest scores among those in registers (rounded down to fp32: no
    // higher)
    float tmax = -INFINITY;
#pragma unroll
    for (int k = 0; k < NK; ++k)
        if (mine[k]) tmax = fmaxf(tmax, __double2float_rd(pick_of(mine[k]).score));
    if (a.n_out <= kFewGroups) {
        const float gm = lanes_max<16>(tmax);
        if (lane % 16 == 0) gmax[tid / 16] = gm;
    } else {
        const float gm = lanes_max<4>(tmax);
        if (lane % 4 == 0) gmax[tid / 4] = gm;
    }
    __syncthreads();
    const double bound = groups_bound(gmax, lane, a.n_out);
    auto take = [&](uint64_t key) {
        if (!key) return false;
        const BeamPick p = pick_of(key);
        if (!(p.score >= bound)) return false;  // NaN: of a beam without continuations
        const int at = atomicAdd(&count, 1);
        if (at < kBeamCap) picks[at] = p;
        return true;
    };
#pragma unroll
    for (int k = 0; k < NK; ++k) take(mine[k]);
    // the lists' other candidates, which fall: up to the first below the bound
    if (total > held)
        for (int i = tid; i < lists; i += kJoinThreads) {
            int r = i < held ? (held - i + lists - 1) / lists : 0;
            while (r < a.n_out && take(cand[(int64_t)i * a.n_out + r])) ++r;
        }
    __syncthreads();
    auto put = [&](int r, const BeamPick& p) {
        const int64_t o = req * a.n_out + r;
        a.scores[o] = (float)p.score;
        a.parents[o] = (int32_t)(row0 + (p.at >> 24));
        a.tokens[o] = (int32_t)(p.at & 0xFFFFFFu);
    };
    auto put_none = [&](int r) {
        const int64_t o = req * a.n_out + r;
        a.scores[o] = -INFINITY, a.parents[o] = -1, a.tokens[o] = -1;
    };
    const int n = count;
    if (n <= kBeamCap) {
        for (int i = tid; i < n; i += kJoinThreads) {
            const BeamPick p = picks[i];
            int rank = 0;
            for (int k = 0; k < n; ++k) rank += picks[k].before(p);
            if (rank < a.n_out) put(rank, p);
        }
        for (int i = n + tid; i < a.n_out; i += kJoinThreads) put_none(i);
        return;
    }
    BeamPick last{INFINITY, 0};
    for (int r = 0; r < a.n_out; ++r) {
        BeamPick best{-INFINITY, 0xFFFFFFFFu};
        for (int i = tid; i < total; i += kJoinThreads)
            if (const uint64_t key = candidate(i)) {
                const BeamPick p = pick_of(key);
                if (last.before(p) && p.before(best)) best = p;
            }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const BeamPick o{__shfl_xor(best.score, k, 64), (uint32_t)__shfl_xor((int)best.at, k, 64)};
            if (o.before(best)) best = o;
        }
        if (lane == 0) wbest[wave] = best;
        __syncthreads();
        last = wbest[0];
        for (int k = 1; k < kJoinWaves; ++k)
            if (wbest[k].before(last)) last = wbest[k];
        if (tid == 0) put(r, last);  // more than kBeamCap candidates: there is one in every round
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
// Elements of a thread: 32 where that makes two workgroups per CU or more, or where 8 make more candidates of a request
// than wait in the join's registers. Chunks + join, 8 | 32, us: 1 x 4 beams over 151936 F32 tokens, 8 outputs, 4.9 + 6.2 |
// 6.3 + 5.3; 8 x 4 over 32000 5.0 + 6.6 | 6.4 + 12.6; 32 x 8 over 151936, 16 outputs, 48 + 13 | 34 + 9; one request of 8
// beams over 151936, 16 outputs (9600 candidates | 2432), 5.7 + 11.1 | 7.0 + 6.9.
struct BeamPlan {
    int ept, chunks;
};
static BeamPlan beam_plan(int64_t n_batch, int n_beams, int vocab, int n_out) {
    const auto chunks = [&](int ept) { return (vocab + kBeamThreads * ept - 1) / (kBeamThreads * ept); };
    const bool fill = n_batch * n_beams * chunks(32) >= 2 * (int64_t)cu_count();
    const bool many = (int64_t)n_beams * chunks(8) * n_out > 4096;
    const int ept = fill || many ? 32 : 8;
    return {ept, chunks(ept)};
}

size_t beam_workspace_bytes(int64_t n_batch, int n_beams, int vocab, int n_out) {
    const int64_t lists = n_batch * n_beams * beam_plan(n_batch, n_beams, vocab, n_out).chunks;
    return (size_t)(round_up(lists * 8, 256) + round_up(lists * 4, 256) + round_up(lists * n_out * 8, 256));
}

hipError_t launch_beam_select(int type, BeamArgs a, int64_t n_batch, void* ws, hipStream_t st) {
    const int64_t rows = n_batch * a.n_beams;
    const BeamPlan p = beam_plan(n_batch, a.n_beams, a.vocab, a.n_out);
    a.chunks = p.chunks;
    const int64_t lists = rows * p.chunks;
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.stat_sum = reinterpret_cast<double*>(w);
    a.stat_ref = reinterpret_cast<float*>(w + round_up(lists * 8, 256));
    a.cand = reinterpret_cast<uint64_t*>(w + round_up(lists * 8, 256) + round_up(lists * 4, 256));
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
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)n_batch), dim3(kJoinThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace dcq
