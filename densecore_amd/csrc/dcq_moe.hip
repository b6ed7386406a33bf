// dcq_moe.hip — which experts a token goes to, the tokens' slots sorted by expert, and their results summed per token.
#include <algorithm>

#include "dcq_common.h"
#include "dcq_i8.h"

namespace dcq {

namespace {

// Order of doubles as integers: larger for larger, -infinity above 0 (no candidate).
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);  // -0 as 0
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
constexpr uint32_t kNoHigh = 0x000FFFFF;  // of order_key(-infinity)

// The largest of a wave's values, in a scalar register: by lanes within rows of 16, then of the four rows.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
    const uint32_t r0 = __builtin_amdgcn_readlane((int)v, 0), r1 = __builtin_amdgcn_readlane((int)v, 16),
                   r2 = __builtin_amdgcn_readlane((int)v, 32), r3 = __builtin_amdgcn_readlane((int)v, 48);
    return max(max(r0, r1), max(r2, r3));
}
__device__ __forceinline__ double lane_xor(double v, int d) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)u, d, 64), hi = (uint32_t)__shfl_xor((int)(u >> 32), d, 64);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += lane_xor(v, d);
    return v;
}
__device__ __forceinline__ double from_lane(double v, int lane) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane),
                   hi = (uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

}  // namespace

// A token per wave, expert lane + 64 i in register i. Scores in 64 bits, so that what is chosen is the definition's
// choice and not that of a rounding. The best are taken one at a time, by the upper half of their keys; the lower halves and
// the experts' numbers decide between the few that share one.
// 8192 tokens, 256 experts in 8 groups, best 8: 15.6 us, 0.5 TB/s. Bound by VALU, 842 instructions a token: 64-bit
// exponentials and quotients, the groups' best and the choices' steps (18.4 us with the scores' winners followed through every step
// in place of read back at the end). 5 tokens of 128 experts: 4.3 us, latency.
constexpr int kRouteWaves = 4;
template <class T, int EPL>
__global__ void __launch_bounds__(64 * kRouteWaves) moe_route_kernel(RouteArgs a) {
    __shared__ double shared[kRouteWaves][64 * EPL], scores[kRouteWaves][64 * EPL];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row_at = (int64_t)blockIdx.x * kRouteWaves + wave;
    const int64_t row = row_at < a.rows ? row_at : a.rows - 1;
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    float v[EPL];
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < a.n_expert ? (float)x[e] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        bad |= !(v[i] < INFINITY);
        top = fmaxf(top, v[i]);
    }
    bad = __ballot(bad) != 0;
    double score[EPL];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) score[i] = 1.0 / (1.0 + exp(-(double)v[i]));
    } else {
        top = lanes_max<64>(top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            score[i] = v[i] == -INFINITY ? 0.0 : exp((double)v[i] - (double)top);
            sum += score[i];
        }
        const double inv = 1.0 / wave_sum(sum);
#pragma unroll
        for (int i = 0; i < EPL; ++i) score[i] *= inv;
    }
    uint32_t high[EPL], low[EPL];  // order_key's halves
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane + 64 * i;
        double c = score[i];
        scores[wave][e] = c;
        bool out = bad || v[i] == -INFINITY;
        if (a.bias && e < a.n_expert) {
            const float b = a.bias[e];
            out |= !(fabsf(b) < INFINITY);
            c += (double)b;
        }
        c = out ? -INFINITY : c;
        const uint64_t key = order_key(c);
        high[i] = (uint32_t)(key >> 32), low[i] = (uint32_t)key;
        if (a.n_group > 1) shared[wave][e] = c;
    }
    __syncthreads();
    if (a.n_group > 1) {
        // `share` lanes to a group, each the best two of its part, then of each other's
        const int per = a.n_expert / a.n_group, bits = 31 - __clz(64 / a.n_group), share = 1 << bits;
        const int group = lane >> bits;
        double b1 = -INFINITY, b2 = -INFINITY;
        if (group < a.n_group)
            for (int e = lane & (share - 1); e < per; e += share) {
                const double c = shared[wave][group * per + e];
                b2 = fmax(b2, fmin(b1, c));
                b1 = fmax(b1, c);
            }
        for (int d = 1; d < share; d *= 2) {
            const double o1 = lane_xor(b1, d), o2 = lane_xor(b2, d);
            b2 = fmax(fmax(b2, o2), fmin(b1, o1));
            b1 = fmax(b1, o1);
        }
        const double worth = a.group_best == 2 && b2 > -INFINITY ? b1 + b2 : b1;
        int ahead = 0;
        for (int g = 0; g < a.n_group; ++g) {
            const double o = from_lane(worth, g << bits);
            ahead += o > worth || (o == worth && g < group);
        }
        const uint64_t kept = __ballot(group < a.n_group && ahead < a.topk_group);  // bit g * share: group g's
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane + 64 * i;
            if (e >= a.n_expert || !(kept >> (e / per << bits) & 1)) high[i] = 0;
        }
    }
    int my_id = -1;
    for (int j = 0; j < a.k; ++j) {
        uint32_t best = high[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i) best = max(best, high[i]);
        const uint32_t most = wave_max(best);
        if (most <= kNoHigh) break;
        // who has it: usually one lane in one register
        int e = 0, count = 0;
#pragma unroll
        for (int i = EPL - 1; i >= 0; --i) {
            const uint64_t who = __ballot(high[i] == most);
            count += (int)__popcll(who);
            if (who) e = 64 * i + (int)__builtin_ctzll(who);
        }
        if (count > 1) {  // the largest lower half, then the lowest expert
            uint32_t lower = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) lower = max(lower, high[i] == most ? low[i] : 0u);
            lower = wave_max(lower);
#pragma unroll
            for (int i = EPL - 1; i >= 0; --i) {
                const uint64_t who = __ballot(high[i] == most && low[i] == lower);
                if (who) e = 64 * i + (int)__builtin_ctzll(who);
            }
        }
        my_id = lane == j ? e : my_id;
#pragma unroll
        for (int i = 0; i < EPL; ++i) high[i] = lane + 64 * i == e ? 0u : high[i];
    }
    const double my_score = my_id >= 0 ? scores[wave][my_id] : 0.0;
    double w = my_id >= 0 ? (double)a.scale * my_score : 0.0;
    if (a.renorm) {
        const double sum = wave_sum(my_score);
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (row_at < a.rows && lane < a.k) {
        a.ids[row * a.k + lane] = my_id;
        a.weights[row * a.k + lane] = (float)w;
    }
}

template <class T>
hipError_t launch_route_type(const RouteArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((a.rows + kRouteWaves - 1) / kRouteWaves));
    if (a.n_expert <= 64) moe_route_kernel<T, 1><<<grid, 64 * kRouteWaves, 0, st>>>(a);
    else if (a.n_expert <= 128) moe_route_kernel<T, 2><<<grid, 64 * kRouteWaves, 0, st>>>(a);
    else if (a.n_expert <= 256) moe_route_kernel<T, 4><<<grid, 64 * kRouteWaves, 0, st>>>(a);
    else moe_route_kernel<T, 8><<<grid, 64 * kRouteWaves, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_moe_route(int type, const RouteArgs& a, hipStream_t st) {
    return type == kTypeF16 ? launch_route_type<_Float16>(a, st) : launch_route_type<float>(a, st);
}

// A workgroup per expert (and one for the slots of none) looks at all slots: those of lower experts give its place, its
// own go there in their order. No atomics and no second launch; the slots' numbers come from the caches, 16 loads of a wave
// on their way at a time. 40 slots of 128 experts 3.6 us, which is the launch and two trips to memory; 12568 slots 6.5 (13.2 with
// one load at a time); 65536 slots of 256 experts 22, by the instructions of every workgroup's look at every slot.
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads) moe_plan_kernel(const int32_t* ids, int slots, int n_expert, int32_t* plan) {
    constexpr int W = kPlanThreads / 64, G = 16;
    __shared__ int less[W], mine[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int me = blockIdx.x;  // n_expert: none
    int32_t* order = plan + plan_order_at(n_expert);
    int32_t* expert = plan + plan_expert_at(n_expert, slots);
    // a run of slots to each wave
    const int run = ((slots + W - 1) / W + 63) / 64 * 64, begin = min(wave * run, slots), end = min(begin + run, slots);
    int e[G];
    auto load = [&](int at) {  // numbers out of range, negative ones too, are the least that is too large
        const uint32_t none = n_expert;
        if (at + 64 * G <= end) {
#pragma unroll
            for (int g = 0; g < G; ++g) e[g] = ids[at + 64 * g + lane];
#pragma unroll
            for (int g = 0; g < G; ++g) e[g] = (int)min((uint32_t)e[g], none);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) e[g] = ids[min(at + 64 * g + lane, end - 1)];
#pragma unroll
            for (int g = 0; g < G; ++g) e[g] = at + 64 * g + lane < end ? (int)min((uint32_t)e[g], none) : 0x7FFFFFFF;
        }
    };
    const int shares = ((slots + 63) / 64 + n_expert) / (n_expert + 1);  // of the slots' experts to write, 64 at a time
    const int share = me * shares, share_end = share + shares;
    int below = 0, same = 0;
    for (int at = begin; at < end; at += 64 * G) {
        load(at);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (at + 64 * g >= end) break;
            below += (int)__popcll(__ballot(e[g] < me));
            same += (int)__popcll(__ballot(e[g] == me));
            const int i = at + 64 * g + lane;
            if (at / 64 + g >= share && at / 64 + g < share_end && i < end) expert[i] = e[g] < n_expert ? e[g] : -1;
        }
    }
    if (lane == 0) less[wave] = below, mine[wave] = same;
    __syncthreads();
    int first = 0, all = 0, before = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        first += less[w];
        all += mine[w];
        before += w < wave ? mine[w] : 0;
    }
    if (threadIdx.x == 0) {
        plan[me] = first;
        if (me == n_expert) plan[n_expert + 1] = slots;
    }
    const int height = plan_height(slots, n_expert);
    const int t0 = (first + me * (height - 1)) / height, t1 = (first + all + (me + 1) * (height - 1)) / height;
    PlanTile* tiles = reinterpret_cast<PlanTile*>(plan + plan_tiles_at(n_expert, slots));
    for (int t = t0 + (int)threadIdx.x; t < t1; t += kPlanThreads) {
        const int done = (t - t0) * height;
        tiles[t] = done < all ? PlanTile{me, first + done, min(height, all - done), 0} : PlanTile{-1, 0, 0, 0};
    }
    if (same == 0) return;
    first += before;
    for (int at = begin; at < end; at += 64 * G) {
        if (run > 64 * G) load(at);  // else what the first pass left
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (at + 64 * g >= end) break;
            const uint64_t hit = __ballot(e[g] == me);
            if (hit == 0) continue;
            const int ahead = __builtin_amdgcn_mbcnt_hi((uint32_t)(hit >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
            if (e[g] == me) order[first + ahead] = at + 64 * g + lane;
            first += (int)__popcll(hit);
        }
    }
}

hipError_t launch_moe_plan(const int32_t* ids, int64_t slots, int n_expert, int32_t* plan, hipStream_t st) {
    moe_plan_kernel<<<n_expert + 1, kPlanThreads, 0, st>>>(ids, (int)slots, n_expert, plan);
    return hipGetLastError();
}

// y[m] = (R[m] +) sum of the slots' rows by their weights, in the order of a token's slots, in fp32. A thread for V columns of a
// token. HBM: 1571 tokens x 8 slots x 2048 and the residual, 129 MB, 25.4 us: 5.1 TB/s.
template <class T, int V>
__global__ void __launch_bounds__(256) moe_combine_kernel(CombineArgs a) {
    const int blocks = (a.N + 256 * V - 1) / (256 * V);
    const int64_t row = blockIdx.x / blocks;
    const int n = ((int)blockIdx.x % blocks * 256 + (int)threadIdx.x) * V;
    if (n >= a.N) return;
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = 0.0f;
    for (int j0 = 0; j0 < a.top; j0 += 4) {  // four slots' loads on their way at a time; those of no expert do not count
        float v[4][V], w[4];
        bool in[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t slot = row * a.top + min(j0 + j, a.top - 1);
            in[j] = j0 + j < a.top && a.expert[slot] >= 0;
            w[j] = a.weights[slot];
            __builtin_memcpy(v[j], __builtin_assume_aligned(a.p + slot * a.N + n, 4 * V), 4 * V);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = in[j] ? fmaf(w[j], v[j][i], y[i]) : y[i];
    }
    if (a.R) {
        float v[V];
        __builtin_memcpy(v, __builtin_assume_aligned(a.R + row * a.r_stride + n, 4 * V), 4 * V);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] += v[i];
    }
    T* out = static_cast<T*>(a.y) + row * a.y_stride + n;
    T o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (T)y[i];
    __builtin_memcpy(__builtin_assume_aligned(out, sizeof(T) * V), o, sizeof(T) * V);
}

template <class T>
hipError_t launch_combine_type(const CombineArgs& a, hipStream_t st) {
    const bool wide = a.N % 4 == 0 && a.y_stride % 4 == 0 && (uintptr_t)a.y % (4 * sizeof(T)) == 0 &&
                      (!a.R || ((uintptr_t)a.R % 16 == 0 && a.r_stride % 4 == 0));
    const int per = wide ? 1024 : 256;
    const dim3 grid((unsigned)((a.N + per - 1) / per * a.rows));
    if (wide) moe_combine_kernel<T, 4><<<grid, 256, 0, st>>>(a);
    else moe_combine_kernel<T, 1><<<grid, 256, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_moe_combine(int ytype, const CombineArgs& a, hipStream_t st) {
    return ytype == kTypeF16 ? launch_combine_type<_Float16>(a, st) : launch_combine_type<float>(a, st);
}

}  // namespace dcq
