// dcq_norm.hip — rows to int8 with a scale each, and before it the residual's addition and the RMS norm.
//
//   h = x + r (rounded to fp32: the residual stream),   y = h w / sqrt(mean h^2 + eps),
//   s = max |y| / 127,   q = rint(127 y / max |y|)
//
// The norm's factor cancels in q: with p = h w, exact in 64 bits, q = rint(p * (127 / max |p|)), so that no order of a sum
// decides which step a value next to a border rounds to, and the bytes are the definition's. All of it is 64-bit
// arithmetic, beside the loads (VALU busy 62 %): the kernel waits for memory (2048 x 4096, F16 x, fp32 r and h: 92 MB in 16.3 us, 5.7 TB/s,
// the writes past the caches; one row of 2560: 3.2 us with its launch, latency). Sums and the largest are found in one pass
// over a row that stays in registers, with one barrier. Largest values are compared as bit patterns, where a NaN is above
// infinity and infinity above all else: a row that holds either has q = 0 and s = NaN, so that what is made of it shows it.
#include "dcq_common.h"
#include "dcq_i8.h"

namespace dcq {

namespace {

// The value `from` lanes away, by the four DPP steps of a row of 16 lanes (see lanes_sum) and then across rows.
template <int STEP>
__device__ __forceinline__ uint64_t partner(uint64_t v) {
    const int lo = (int)(uint32_t)v, hi = (int)(uint32_t)(v >> 32);
    if constexpr (STEP < 4) {
        constexpr int ctrl = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140;
        return (uint64_t)(uint32_t)dpp_mov<ctrl>(hi) << 32 | (uint32_t)dpp_mov<ctrl>(lo);
    } else {
        return (uint64_t)(uint32_t)__shfl_xor(hi, STEP == 4 ? 16 : 32, 64) << 32 |
               (uint32_t)__shfl_xor(lo, STEP == 4 ? 16 : 32, 64);
    }
}
template <int STEP>
__device__ __forceinline__ void reduce_step(double& sum, uint64_t& top) {
    sum += __longlong_as_double((long long)partner<STEP>((uint64_t)__double_as_longlong(sum)));
    const uint64_t t = partner<STEP>(top);
    top = t > top ? t : top;
}
// Sum and largest over the workgroup, the same in every thread.
template <int THREADS>
__device__ __forceinline__ void reduce_row(double& sum, uint64_t& top) {
    reduce_step<0>(sum, top);
    reduce_step<1>(sum, top);
    reduce_step<2>(sum, top);
    reduce_step<3>(sum, top);
    reduce_step<4>(sum, top);
    reduce_step<5>(sum, top);
    if constexpr (THREADS > 64) {
        constexpr int W = THREADS / 64;
        __shared__ double sums[W];
        __shared__ uint64_t tops[W];
        if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum, tops[threadIdx.x / 64] = top;
        __syncthreads();
        sum = 0.0, top = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            sum += sums[i];
            top = tops[i] > top ? tops[i] : top;
        }
    }
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const _Float16* p, float (&v)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = half_bits_to_float(d[i / 2] >> (16 * (i % 2)) & 0xFFFFu);
}
// h goes past the caches' usual places: the layer's products come before it is read again (2048 x 4096, F16 x: 23.2 -> 17.8 us, before the shapes below).
__device__ __forceinline__ void store_h8(float* p, const float (&v)[8]) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store((f32x4){v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(p));
    __builtin_nontemporal_store((f32x4){v[4], v[5], v[6], v[7]}, reinterpret_cast<f32x4*>(p) + 1);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// What is left to do with a row when its sum and largest are known.
struct RowScale {
    double inv, rstd;
    float s;
    bool bad;
};
__device__ __forceinline__ RowScale row_scale(const NormArgs& a, double sum, uint64_t top_bits) {
    RowScale k;
    const double top = __longlong_as_double((long long)top_bits);
    const double root = a.w ? sqrt(sum / a.width + (double)a.eps) : 1.0;
    k.bad = top_bits >= 0x7FF0000000000000ull || !(sum < __longlong_as_double(0x7FF0000000000000ll));
    k.inv = top_bits && !k.bad ? 127.0 / top : 0.0;
    k.rstd = 1.0 / root;
    // (the norm of an all-zero row with eps = 0 is 0 / 0: the row has no value to scale)
    k.s = k.bad ? __uint_as_float(0x7FC00000u) : top_bits ? (float)(top / (127.0 * root)) : 0.0f;
    return k;
}
// rint of |v| <= 127.5 by adding 1.5 * 2^52: the integer is the sum's low bits.
__device__ __forceinline__ uint32_t rint_bits(double v) {
    return (uint32_t)__double_as_longlong(v + 6755399441055744.0);
}
__device__ __forceinline__ void store_q8(int8_t* dst, const double (&p)[8], const RowScale& k) {
#pragma clang fp contract(off)
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const double t = p[i] * k.inv;  // rounded by itself, as the definition's
        b[i] = rint_bits(t);
    }
    const uint2 v = make_uint2(pack_low_bytes(b[0], b[1], b[2], b[3]), pack_low_bytes(b[4], b[5], b[6], b[7]));
    *reinterpret_cast<uint2*>(dst) = k.bad ? make_uint2(0, 0) : v;
}
__device__ __forceinline__ void store_y8(float* dst, const double (&p)[8], double rstd) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(p[i] * rstd);
    store8(dst, v);
}

}  // namespace

// A row per workgroup, C pieces of 8 elements to a thread, all of them in registers.
template <class T, int THREADS, int C>
__global__ void __launch_bounds__(THREADS) norm_row_kernel(NormArgs a) {
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    float v[C][8], wv[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = 8 * (threadIdx.x + c * THREADS);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = 0.0f, wv[c][i] = 1.0f;
        if (at < a.width) {
            load8(x + at, v[c]);
            if (a.w) load8(a.w + at, wv[c]);
        }
    }
    if (a.r) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = 8 * (threadIdx.x + c * THREADS);
            if (at < a.width) {
                float rv[8];
                load8(a.r + row * a.r_stride + at, rv);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += rv[i];
            }
        }
    }
    double sum = 0.0;
    uint64_t top = 0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double h = v[c][i];
            sum = fma(h, h, sum);
            const uint64_t m = (uint64_t)__double_as_longlong(h * (double)wv[c][i]) & 0x7FFFFFFFFFFFFFFFull;
            top = m > top ? m : top;
        }
    reduce_row<THREADS>(sum, top);
    const RowScale k = row_scale(a, sum, top);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = 8 * (threadIdx.x + c * THREADS);
        if (at >= a.width) continue;
        if (a.h) store_h8(a.h + row * a.h_stride + at, v[c]);
        double p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (double)v[c][i] * (double)wv[c][i];
        if (a.q) store_q8(a.q + row * a.q_stride + at, p, k);
        if (a.y) store_y8(a.y + row * a.y_stride + at, p, k.rstd);
    }
    if (a.q && threadIdx.x == 0) a.s[row] = k.s;
}

// Rows that no workgroup's registers hold: h is written in the first pass and read again in the second, each element by
// the thread that wrote it.
template <class T>
__global__ void __launch_bounds__(1024) norm_long_kernel(NormArgs a) {
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const float* r = a.r ? a.r + row * a.r_stride : nullptr;
    float* h = a.h ? a.h + row * a.h_stride : nullptr;
    double sum = 0.0;
    uint64_t top = 0;
    for (int at = 8 * threadIdx.x; at < a.width; at += 8 * 1024) {
        float v[8], w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        load8(x + at, v);
        if (a.w) load8(a.w + at, w);
        if (r) {
            float rv[8];
            load8(r + at, rv);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += rv[i];
        }
        if (h) store8(h + at, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double d = v[i];
            sum = fma(d, d, sum);
            const uint64_t m = (uint64_t)__double_as_longlong(d * (double)w[i]) & 0x7FFFFFFFFFFFFFFFull;
            top = m > top ? m : top;
        }
    }
    reduce_row<1024>(sum, top);
    const RowScale k = row_scale(a, sum, top);
    for (int at = 8 * threadIdx.x; at < a.width; at += 8 * 1024) {
        float v[8], w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
        if (h) load8(h + at, v);
        else load8(x + at, v);
        if (a.w) load8(a.w + at, w);
        double p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = (double)v[i] * (double)w[i];
        if (a.q) store_q8(a.q + row * a.q_stride + at, p, k);
        if (a.y) store_y8(a.y + row * a.y_stride + at, p, k.rstd);
    }
    if (a.q && threadIdx.x == 0) a.s[row] = k.s;
}

template <class T>
hipError_t launch_norm_type(const NormArgs& a, hipStream_t st) {
    const int pieces = a.width / 8;
    const dim3 grid((unsigned)a.rows);
    // The narrowest workgroup that holds a row, a piece to a thread, until its barrier has more than 8 waves: then two pieces
    // (us, 2048 rows and one: width 2048 8.98 and 2.96, by two pieces 9.69 and 3.41; 4096 16.3 and 3.29, 17.6 and 3.59; but
    // 8192, where one piece takes 16 waves, 37.1 and 4.03, by one 44.0 and 4.46; 12288 62.9, by four pieces 68.6).
    if (pieces <= 64) norm_row_kernel<T, 64, 1><<<grid, 64, 0, st>>>(a);
    else if (pieces <= 128) norm_row_kernel<T, 128, 1><<<grid, 128, 0, st>>>(a);
    else if (pieces <= 256) norm_row_kernel<T, 256, 1><<<grid, 256, 0, st>>>(a);
    else if (pieces <= 512) norm_row_kernel<T, 512, 1><<<grid, 512, 0, st>>>(a);
    else if (pieces <= 1024) norm_row_kernel<T, 512, 2><<<grid, 512, 0, st>>>(a);
    else if (pieces <= 2048) norm_row_kernel<T, 1024, 2><<<grid, 1024, 0, st>>>(a);
    else norm_long_kernel<T><<<grid, 1024, 0, st>>>(a);
    return hipGetLastError();
}

hipError_t launch_norm_i8(int type, const NormArgs& a, hipStream_t st) {
    return type == kTypeF16 ? launch_norm_type<_Float16>(a, st) : launch_norm_type<float>(a, st);
}

}  // namespace dcq
