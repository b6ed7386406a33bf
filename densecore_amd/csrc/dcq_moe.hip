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
__device__ __forceinline__ uint64_t dpp64(uint64_t v, int ctrl_at) {
    const int lo = (int)(uint32_t)v, hi = (int)(uint32_t)(v >> 32);
    int l, h;
    switch (ctrl_at) {
        case 0: l = dpp_mov<0xB1>(lo), h = dpp_mov<0xB1>(hi); break;
        case 1: l = dpp_mov<0x4E>(lo), h = dpp_mov<0x4E>(hi); break;
        case 2: l = dpp_mov<0x141>(lo), h = dpp_mov<0x141>(hi); break;
        case 3: l = dpp_mov<0x140>(lo), h = dpp_mov<0x140>(hi); break;
        case 4: l = __shfl_xor(lo, 16, 64), h = __shfl_xor(hi, 16, 64); break;
        default: l = __shfl_xor(lo, 32, 64), h = __shfl_xor(hi, 32, 64); break;
    }
    return (uint64_t)(uint32_t)h << 32 | (uint32_t)l;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const uint64_t o = dpp64(v, i);
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int i = 0; i < 6; ++i) v += __longlong_as_double((long long)dpp64((uint64_t)__double_as_longlong(v), i));
    return v;
}

constexpr uint64_t kNoKey = 0x000FFFFFFFFFFFFFull;  // order_key(-infinity)

}  // namespace

// A token per wave, expert lane + 64 i in register i. Scores in 64 bits, so that what is chosen is the definition's
// choice and not that of a rounding; the best are taken one at a time.
constexpr int kRouteWaves = 4;
template <class T, int EPL>
__global__ void __launch_bounds__(64 * kRouteWaves) moe_route_kernel(RouteArgs a) {
    __shared__ double shared[kRouteWaves][64 * EPL];
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
        sum = wave_sum(sum);
#pragma unroll
        for (int i = 0; i < EPL; ++i) score[i] = score[i] / sum;
    }
    uint64_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane + 64 * i;
        double c = score[i];
        bool out = bad || v[i] == -INFINITY;
        if (a.bias && e < a.n_expert) {
            const float b = a.bias[e];
            out |= !(fabsf(b) < INFINITY);
            c += (double)b;
        }
        c = out ? -INFINITY : c;
        key[i] = order_key(c);
        if (a.n_group > 1) shared[wave][e] = c;
    }
    if (a.n_group > 1) {
        __syncthreads();
        const int per = a.n_expert / a.n_group;
        double b1 = -INFINITY, b2 = -INFINITY;
        if (lane < a.n_group)
            for (int e = 0; e < per; ++e) {
                const double c = shared[wave][lane * per + e];
                b2 = c > b1 ? b1 : c > b2 ? c : b2;
                b1 = c > b1 ? c : b1;
            }
        const double worth = a.group_best == 2 && b2 > -INFINITY ? b1 + b2 : b1;
        const uint64_t wk = order_key(worth);
        int ahead = 0;
        for (int g = 0; g < a.n_group; ++g) {
            const uint64_t o = (uint64_t)(uint32_t)__shfl((int)(uint32_t)(wk >> 32), g, 64) << 32 |
                               (uint32_t)__shfl((int)(uint32_t)wk, g, 64);
            ahead += o > wk || (o == wk && g < lane);
        }
        const uint64_t kept = __ballot(lane < a.n_group && ahead < a.topk_group);
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane + 64 * i;
            if (e >= a.n_expert || !(kept >> (e / per) & 1)) key[i] = kNoKey;
        }
    }
    int my_id = -1;
    double my_score = 0.0;
    for (int j = 0; j < a.k; ++j) {
        uint64_t best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < EPL; ++i)
            if (key[i] > best) best = key[i], at = i;
        const uint64_t most = wave_max(best);
        if (most <= kNoKey) break;
        uint64_t who = __ballot(best == most);
        int e = lane + 64 * at;
        if (who & (who - 1)) {  // equal scores: the lowest expert
            int low = best == most ? e : 0x7FFFFFFF;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) low = min(low, __shfl_xor(low, d, 64));
            who = __ballot(best == most && e == low);
        }
        const int from = __ffsll((unsigned long long)who) - 1;
        double s = score[0];
#pragma unroll
        for (int i = 1; i < EPL; ++i) s = at == i ? score[i] : s;
        e = __shfl(e, from, 64);
        s = __shfl(s, from, 64);
        if (lane == j) my_id = e, my_score = s;
        if (lane == from) {
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (at == i) key[i] = kNoKey;
        }
    }
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
// own go there in their order. No atomics and no second launch; the slots' numbers come from the caches.
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads) moe_plan_kernel(const int32_t* ids, int slots, int n_expert, int32_t* plan) {
    constexpr int W = kPlanThreads / 64;
    __shared__ int less[W], mine[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int me = blockIdx.x;  // n_expert: none
    int32_t* order = plan + plan_order_at(n_expert);
    int32_t* expert = plan + plan_expert_at(n_expert, slots);
    // a run of slots to each wave
    const int run = ((slots + W - 1) / W + 63) / 64 * 64, begin = min(wave * run, slots), end = min(begin + run, slots);
    int below = 0, same = 0;
    for (int at = begin; at < end; at += 64) {
        const int i = at + lane;
        int e = i < end ? ids[i] : 0x7FFFFFFF;
        const bool in = i < end;
        e = e < 0 || e >= n_expert ? n_expert : e;
        below += (int)__popcll(__ballot(in && e < me));
        same += (int)__popcll(__ballot(in && e == me));
        if (in && at / 64 % (int)gridDim.x == me) expert[i] = e < n_expert ? e : -1;
    }
    if (lane == 0) less[wave] = below, mine[wave] = same;
    __syncthreads();
    int first = 0;
    for (int w = 0; w < W; ++w) first += less[w];
    if (threadIdx.x == 0) {
        plan[me] = first;
        if (me == n_expert) plan[n_expert + 1] = slots;
    }
    int all = 0;
    for (int w = 0; w < W; ++w) all += mine[w];
    const int height = plan_height(slots, n_expert);
    const int t0 = (first + me * (height - 1)) / height, t1 = (first + all + (me + 1) * (height - 1)) / height;
    PlanTile* tiles = reinterpret_cast<PlanTile*>(plan + plan_tiles_at(n_expert, slots));
    for (int t = t0 + (int)threadIdx.x; t < t1; t += kPlanThreads) {
        const int done = (t - t0) * height;
        tiles[t] = done < all ? PlanTile{me, first + done, min(height, all - done), 0} : PlanTile{-1, 0, 0, 0};
    }
    for (int w = 0; w < wave; ++w) first += mine[w];
    if (same == 0) return;
    for (int at = begin; at < end; at += 64) {
        const int i = at + lane;
        int e = i < end ? ids[i] : 0x7FFFFFFF;
        e = e < 0 || e >= n_expert ? n_expert : e;
        const uint64_t hit = __ballot(i < end && e == me);
        if (hit >> lane & 1) order[first + (int)__popcll(hit & ((1ull << lane) - 1))] = i;
        first += (int)__popcll(hit);
    }
}

hipError_t launch_moe_plan(const int32_t* ids, int64_t slots, int n_expert, int32_t* plan, hipStream_t st) {
    moe_plan_kernel<<<n_expert + 1, kPlanThreads, 0, st>>>(ids, (int)slots, n_expert, plan);
    return hipGetLastError();
}

template <class T, int V>
__global__ void __launch_bounds__(256) moe_combine_kernel(CombineArgs a) {
    const int blocks = (a.N + 256 * V - 1) / (256 * V);
    const int64_t row = blockIdx.x / blocks;
    const int n = ((int)blockIdx.x % blocks * 256 + (int)threadIdx.x) * V;
    if (n >= a.N) return;
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = 0.0f;
    for (int j = 0; j < a.top; ++j) {
        const int64_t slot = row * a.top + j;
        if (a.expert[slot] < 0) continue;
        const float w = a.weights[slot];
        const float* p = a.p + slot * a.N + n;
        float v[V];
        __builtin_memcpy(v, __builtin_assume_aligned(p, 4 * V), 4 * V);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = fmaf(w, v[i], y[i]);
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
