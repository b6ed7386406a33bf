// dcq_tree.hip — attention of drafted tokens over the paged KV cache, several sequences in one call.
//
// Sequence b has n_past(b) cached keys (pages tables[b]) and n_draft(b) drafted tokens with fp32 K / V rows of
// their own. Row (token j, query head h) attends every cached key, and drafted key i where bit i of mask[b][j]
// is set:  out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t).  The online softmax keeps a reference m
// (an integer in base 2, raised when a score passes it by 3), the sum l of p' = 2^(s - m), s = scale log2(e)
// q . k, and O = sum p' v.
//
// Query rows of a KV head are the (token, head of its group) pairs, token-major, in tiles of 16: a column of
// the matrix instructions, whatever the group size. S^T = K Q^T puts the keys 4 (lane / 16) + i of row
// lane % 16 into lane registers i, and O^T += V^T P^T takes its weights from the same lanes, so P never
// moves; K and V go from memory to the matrix registers without LDS (Q's operands wait there):
//   K: a lane holds 8 consecutive dims of key lane % 16 (fp32: 4), the A operand as it is.
//   V: a lane holds dims 64 u + 4 (lane % 16) + 0..3 of the keys whose weights it has; output tile (u, e) is
//      made of the dims 64 u + 4 m + e, so that its A operand is in the lane, one byte permute per two keys.
//
// Many query rows of a KV head (tree_block_kernel): as many rows as a workgroup has waves x 32 share the keys,
// which go through LDS in blocks, decoded once. 32 x 32 tiles, S^T and O^T as above; V^T comes by transposing
// LDS reads. Drafted keys, a small part, are the other kernel's work, in workgroups of the same launch.
//
// Arithmetic. F16 and Q8_0 slots are multiplied on the f16 matrix instructions (16 x the fp32 ones' rate):
// q and p', fp32, are split into two f16 pieces of 22 bits (q under an exponent per row, fewer bits below
// 2^-16 of its largest), an F16 slot is one exact piece, and a Q8_0 value d * q, a product of 11 and 7 bits, is
// exactly the two pieces f16(d q) and d q - f16(d q). F32 slots and the drafted rows use the fp32 matrix
// instructions. Sums are fp32.
// All weights keep 22 bits, however far below the row's largest one they are: a first key far above the others
// whose value is next to zero, as models make them, leaves the output to weights of 2^-20 and less. So the
// second piece is 2^11 times what the first one left, in a sum of its own, and scores more than 26 below the
// reference take another pass over the step's values, in units of 2^-26 (piece_weights). With both pieces in one
// unit and one sum, weights had 22 bits from 2^-10 on and none from 2^-32; that took, us a call, 24 tokens of 8
// sequences of 1500..4096 keys, 32/8 heads x 128, F16 44 where it now takes 48, 64 tokens over 32768 keys Q8_0
// 124 | 128, F16 91 | 101, 8 sequences x 64 dims 29 | 35. A unit of each step's own for one sum needs a second pass in
// about every seventh step of such scores: 68, 185, 152, 49.
// Infinities and NaN: what a 16-row tile shares can reach a row that does not see it, and an infinity in one
// piece has no second piece. A row whose m, l or O is not finite is therefore computed again one key at a
// time in fp32, of the keys it sees alone.
#include <algorithm>
#include <type_traits>

#include "dcq_attn.h"
#include "dcq_common.h"
#include "dcq_kernels.h"
#include "dcq_kv_row.h"
#include "dcq_search.h"

namespace dcq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 16;          // query rows of a tile
constexpr int kTreeWaves = 4;      // waves of a workgroup, a share of the keys each
constexpr int kRowsPerWave = 32;   // of the block kernel
// A row's reference is raised when a score passes it by kSlack; a weight counts kPieces in O, 2^15 at most. Its first
// f16 piece is a normal number, and both have their 11 bits, from 2^-kBandBits on.
constexpr float kSlack = 3.0f, kBandBits = 26.0f;
constexpr float kPieces = 0x1p12f, kLow = 0x1p11f;  // kLow: of the second piece

// No sum of the 16 x 16 matrix instructions is to be put over an operand, or half over the sum before it. TIED: an
// empty statement uses operands and sum once more when the new sum is there. That is free at head_dim 256; at 128 it
// has sums moved between register files (fp32, 256 rows: 118 -> 160 us), and operands kept to the end of a chain of
// instructions do.
template <bool TIED>
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
    f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    if constexpr (TIED) asm volatile("" : "+v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}
template <bool TIED>
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b) {
    f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
    if constexpr (TIED) asm volatile("" : "+v"(d) : "v"(a), "v"(b));
    return d;
}
template <bool TIED>
__device__ __forceinline__ f32x4 mfma16(float a, float b, f32x4 c) {
    f32x4 d = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
    if constexpr (TIED) asm volatile("" : "+v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}
__device__ __forceinline__ void keep(f32x4 x) { asm volatile("" ::"v"(x)); }

// Eight weights as f16 pieces.
__device__ __forceinline__ void split_weights(const float* p, f16x8& h, f16x8& l) {
    f16x2 hh[4], ll[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const f32x2 w = {p[2 * t] * kPieces, p[2 * t + 1] * kPieces};
        hh[t] = __builtin_convertvector(w, f16x2);
        ll[t] = __builtin_convertvector((f32x2){(w[0] - (float)hh[t][0]) * kLow, (w[1] - (float)hh[t][1]) * kLow}, f16x2);
    }
    h = __builtin_shufflevector(__builtin_shufflevector(hh[0], hh[1], 0, 1, 2, 3),
                                __builtin_shufflevector(hh[2], hh[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
    l = __builtin_shufflevector(__builtin_shufflevector(ll[0], ll[1], 0, 1, 2, 3),
                                __builtin_shufflevector(ll[2], ll[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}
// a + b f
__device__ __forceinline__ f32x4 plus_low(f32x4 a, f32x4 b, float f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = __builtin_fmaf(b[i], f, a[i]);
    return a;
}

template <int CT>
constexpr int tree_chunk() { return CT == kTypeF32 ? 16 : 32; }  // keys of a wave's step

// ---------------------------------------------------------------- cached keys of one step
__device__ __forceinline__ f16x2 as_f16x2(uint32_t w) { return __builtin_bit_cast(f16x2, w); }
__device__ __forceinline__ uint32_t as_u32(f16x2 h) { return __builtin_bit_cast(uint32_t, h); }
// bytes (b0, 0, b1, 0) of int8 values as two f16: 0x6400 | (b ^ 0x80) is 1024 + 128 + b
__device__ __forceinline__ f16x2 int8_pair(uint32_t t) {
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    return as_f16x2(t ^ 0x64806480u) - bias;
}
struct Pieces {
    f16x2 h, l;
};
__device__ __forceinline__ Pieces q8_pieces(f16x2 q, f16x2 d) {
    const f16x2 h = q * d;
    return {h, __builtin_elementwise_fma(q, d, -h)};
}
__device__ __forceinline__ f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(f16x8, (u32x4){a, b, c, d});
}
__device__ __forceinline__ f16x8 as_f16x8(const uint4& w) { return as_f16x8(w.x, w.y, w.z, w.w); }
__device__ __forceinline__ uint32_t ldu32(const uint8_t* p) {  // 2-byte aligned
    uint32_t w;
    __builtin_memcpy(&w, p, 4);
    return w;
}

// K and V of one step's keys in a lane's registers. Key (j, i) of a lane's V is 16 j + 4 (lane / 16) + i.
template <int CT, int HD>
struct TreeKeys;

template <int HD>
struct TreeKeys<kTypeF16, HD> {
    static constexpr int U = HD / 64, S = HD / 32;
    uint4 k[2][S];
    uint2 v[2][4][U];
    __device__ __forceinline__ void load_k(int j, const uint8_t* page, uint32_t off, int g) {
#pragma unroll
        for (int s = 0; s < S; ++s) k[j][s] = ld16(page + (off + 16 * g + 64 * s));
    }
    __device__ __forceinline__ void load_v(int j, const uint8_t* page, uint32_t off, uint32_t sb, int m) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[j][i][u] = *reinterpret_cast<const uint2*>(page + (off + i * sb + 8 * m + 128 * u));
    }
    __device__ __forceinline__ void zero_k(int j) {
#pragma unroll
        for (int s = 0; s < S; ++s) k[j][s] = make_uint4(0u, 0u, 0u, 0u);
    }
    __device__ __forceinline__ void zero_v(int j, int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[j][i][u] = make_uint2(0u, 0u);
    }
    // V's operands are made again in the next pass over a step's weights, not kept
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < U; ++u) asm volatile("" : "+v"(v[j][i][u].x), "+v"(v[j][i][u].y));
    }
    // q: the lane's operand of k-step 0; k-steps and pieces lie 64 apart
    __device__ __forceinline__ void scores(const uint4* q, f32x4 (&r)[2]) const {
        f32x4 lo[2], hi[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) lo[j] = hi[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const f16x8 qh = as_f16x8(q[128 * s]), ql = as_f16x8(q[128 * s + 64]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f16x8 f = as_f16x8(k[j][s]);
                lo[j] = mfma16<HD == 256>(f, ql, lo[j]);
                hi[j] = mfma16<HD == 256>(f, qh, hi[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) r[j] = hi[j] + lo[j];
    }
    // V^T P^T in units of `unit` into O. FIRST: the unit is 1, and the first piece's products go on from O
    template <bool FIRST>
    __device__ __forceinline__ void weigh(const f16x8 ph, const f16x8 pl, float unit, f32x4 (&o)[U][4]) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint2 a = v[t / 2][2 * (t % 2)][u], b = v[t / 2][2 * (t % 2) + 1][u];
                    w[t] = __builtin_amdgcn_perm(e < 2 ? b.x : b.y, e < 2 ? a.x : a.y,
                                                 e % 2 ? 0x07060302u : 0x05040100u);
                }
                const f16x8 f = as_f16x8(w[0], w[1], w[2], w[3]);
                const f32x4 low = mfma16<HD == 256>(f, pl);
                if constexpr (FIRST)
                    o[u][e] = plus_low(mfma16<HD == 256>(f, ph, o[u][e]), low, 1.0f / kLow);
                else
                    o[u][e] = plus_low(o[u][e], plus_low(mfma16<HD == 256>(f, ph), low, 1.0f / kLow), unit);
            }
    }
};

template <int HD>
struct TreeKeys<kTypeQ8_0, HD> {
    static constexpr int U = HD / 64, S = HD / 32;
    uint2 k[2][S];
    uint32_t kd[2][S];
    uint32_t v[2][4][U], vd[2][4][U];
    __device__ __forceinline__ void load_k(int j, const uint8_t* page, uint32_t off, int g) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const uint8_t* b = page + (off + 34 * s);
            kd[j][s] = ldu16(b);
            __builtin_memcpy(&k[j][s], b + (2 + 8 * g), 8);  // 2-byte aligned
        }
    }
    __device__ __forceinline__ void load_v(int j, const uint8_t* page, uint32_t off, uint32_t sb, int m) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint8_t* b = page + (off + i * sb + 34 * (2 * u + (m >> 3)));
                vd[j][i][u] = ldu16(b);
                v[j][i][u] = ldu32(b + (2 + 4 * (m & 7)));
            }
    }
    __device__ __forceinline__ void zero_k(int j) {
#pragma unroll
        for (int s = 0; s < S; ++s) kd[j][s] = 0u;
    }
    __device__ __forceinline__ void zero_v(int j, int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) vd[j][i][u] = 0u;
    }
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < U; ++u) asm volatile("" : "+v"(v[j][i][u]), "+v"(vd[j][i][u]));
    }
    __device__ __forceinline__ void scores(const uint4* q, f32x4 (&r)[2]) const {
        f32x4 lo[2], hi[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) lo[j] = hi[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const f16x8 qh = as_f16x8(q[128 * s]), ql = as_f16x8(q[128 * s + 64]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f16x2 d = as_f16x2(kd[j][s] | kd[j][s] << 16);
                const uint32_t w[2] = {k[j][s].x, k[j][s].y};
                Pieces p[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    p[t] = q8_pieces(int8_pair(__builtin_amdgcn_perm(0u, w[t / 2], t % 2 ? 0x0c030c02u : 0x0c010c00u)), d);
                const f16x8 fh = as_f16x8(as_u32(p[0].h), as_u32(p[1].h), as_u32(p[2].h), as_u32(p[3].h));
                const f16x8 fl = as_f16x8(as_u32(p[0].l), as_u32(p[1].l), as_u32(p[2].l), as_u32(p[3].l));
                lo[j] = mfma16<HD == 256>(fl, qh, lo[j]);
                lo[j] = mfma16<HD == 256>(fh, ql, lo[j]);
                hi[j] = mfma16<HD == 256>(fh, qh, hi[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) r[j] = hi[j] + lo[j];
    }
    template <bool FIRST>
    __device__ __forceinline__ void weigh(const f16x8 ph, const f16x8 pl, float unit, f32x4 (&o)[U][4]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f16x2 d[4];
#pragma unroll
            for (int t = 0; t < 4; ++t)
                d[t] = as_f16x2(vd[t / 2][2 * (t % 2)][u] | vd[t / 2][2 * (t % 2) + 1][u] << 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                Pieces p[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    p[t] = q8_pieces(int8_pair(__builtin_amdgcn_perm(v[t / 2][2 * (t % 2) + 1][u],
                                                                     v[t / 2][2 * (t % 2)][u],
                                                                     0x0c040c00u + 0x00010001u * e)), d[t]);
                const f16x8 fh = as_f16x8(as_u32(p[0].h), as_u32(p[1].h), as_u32(p[2].h), as_u32(p[3].h));
                const f16x8 fl = as_f16x8(as_u32(p[0].l), as_u32(p[1].l), as_u32(p[2].l), as_u32(p[3].l));
                const f32x4 low = mfma16<HD == 256>(fh, pl);
                if constexpr (FIRST)
                    o[u][e] = plus_low(mfma16<HD == 256>(fh, ph, mfma16<HD == 256>(fl, ph, o[u][e])), low, 1.0f / kLow);
                else
                    o[u][e] = plus_low(o[u][e], plus_low(mfma16<HD == 256>(fh, ph, mfma16<HD == 256>(fl, ph)), low, 1.0f / kLow),
                                       unit);
            }
        }
    }
};

// 16 keys of fp32: cached F32 slots, and the drafted rows of every cache type.
template <int HD>
struct TreeKeys<kTypeF32, HD> {
    static constexpr int U = HD / 64, S = HD / 16;
    f32x4 k[S];
    f32x4 v[4][U];
    f32x4 last_k, last_q;  // of the scores' last instructions
    __device__ __forceinline__ void load_k(int, const uint8_t* page, uint32_t off, int g) {
#pragma unroll
        for (int s = 0; s < S; ++s) k[s] = *reinterpret_cast<const f32x4*>(page + (off + 16 * g + 64 * s));
    }
    __device__ __forceinline__ void load_v(int, const uint8_t* page, uint32_t off, uint32_t sb, int m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load_v_key(i, page, off + i * sb, m);
    }
    __device__ __forceinline__ void load_v_key(int i, const uint8_t* page, uint32_t off, int m) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[i][u] = *reinterpret_cast<const f32x4*>(page + (off + 16 * m + 256 * u));
    }
    __device__ __forceinline__ void zero_k(int) {
#pragma unroll
        for (int s = 0; s < S; ++s) k[s] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void zero_v(int, int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[i][u] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void scores(const uint4* qs, f32x4 (&r)[1]) {
        f32x4 a[4];  // four sums: a quarter of the roundings in a row
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const f32x4 q = last_q = __builtin_bit_cast(f32x4, qs[64 * s]);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = mfma16<HD == 256>(k[s][e], q[e], a[e]);
            if (HD < 256) keep(q);
            if (HD == 256 && s % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more of q at once
        }
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (HD < 256) keep(k[s]);
        r[0] = (a[0] + a[1]) + (a[2] + a[3]);
        last_k = k[S - 1];
    }
    // keeps the last instructions' operands until the scores are there; after the loads that are issued meanwhile
    __device__ __forceinline__ void scored(f32x4 (&r)[1]) const {
        if constexpr (HD < 256) asm volatile("" : "+v"(r[0]) : "v"(last_k), "v"(last_q));
    }
    __device__ __forceinline__ void weigh(const float (&p)[4], f32x4 (&o)[U][4]) const {
        const f32x4 w = (f32x4){p[0], p[1], p[2], p[3]} * kPieces;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[u][e] = mfma16<HD == 256>(v[i][u][e], w[i], o[u][e]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (HD < 256) keep(v[i][u]);
        if (HD < 256) keep(w);
    }
};

// The row's reference raised where the largest score of a step asks for it (the lane has N keys of it; -inf: not seen).
template <int N, int U>
__device__ __forceinline__ void raise_reference(const float (&s)[N], float& m, float& l, f32x4 (&o)[U][4]) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__any(mx > m + kSlack)) {
        const float m_new = mx > m + kSlack ? __builtin_ceilf(mx) : m;
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        l *= alpha;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[u][e] *= alpha;
        m = m_new;
    }
}

// One step of the online softmax: scores to weights.
template <int N, int U>
__device__ __forceinline__ void softmax_step(float (&s)[N], float& m, float& l, f32x4 (&o)[U][4]) {
    raise_reference<N, U>(s, m, l, o);
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
        l += s[i];
    }
}

// The same for weights that go into f16 pieces, of scores s qsc: the weights of a pass, those below 2^(-kBandBits pass)
// and not below 2^(-kBandBits (pass + 1)), in units of the former (all from there up in pass 0). `again`, in the
// whole wave, if keys are left whose weight is above 2^-126: five passes at the most.
__device__ __forceinline__ float band_unit(int pass) { return __builtin_amdgcn_exp2f(-kBandBits * (float)pass); }
template <int N>
__device__ __forceinline__ void piece_weights(float (&s)[N], float qsc, float m, float& l, int pass, bool& again) {
    const float ref = m == -INFINITY ? 0.0f : m - kBandBits * (float)pass;
    if (pass)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = s[i] * qsc < ref ? s[i] : -INFINITY;
    float low = s[0], sum = 0.0f;
#pragma unroll
    for (int i = 1; i < N; ++i) low = fminf(low, s[i]);
    again = false;
    if (__any(low * qsc < ref - kBandBits)) {  // such keys, or some that are not seen
        const float cut = ref < INFINITY ? ref - kBandBits : -INFINITY;  // an infinite reference: NaN, not keys left out
        bool left = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool below = s[i] * qsc < cut;  // not a NaN
            left |= below && s[i] * qsc > m - 126.0f;
            s[i] = below ? -INFINITY : s[i];
        }
        again = pass < 4 && __any(left);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], qsc, -ref));
#pragma unroll
    for (int i = 0; i < N; i += 4) sum += (s[i] + s[i + 1]) + (s[i + 2] + s[i + 3]);
    l = pass ? __builtin_fmaf(sum, band_unit(pass), l) : l + sum;
}

// The factor that takes sums in units of 2^m to units of 2^mx: 0 for sums of no key (l == 0, m = -inf), 1
// where m = -inf beside a NaN, which then stays.
__device__ __forceinline__ float ref_factor(float m, float l, float mx) {
    return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - mx);
}

// One element of a cached row of one KV head, as fp32.
template <int CT>
__device__ __forceinline__ float slot_value(const uint8_t* head, int e) {
    if constexpr (CT == kTypeQ8_0) {
        const uint8_t* b = head + (e / 32) * 34;
        return half_bits_to_float(ldu16(b)) * (float)(int8_t)b[2 + e % 32];
    } else if constexpr (CT == kTypeF16) {
        return half_bits_to_float(ldu16(head + 2 * e));
    } else {
        return reinterpret_cast<const float*>(head)[e];
    }
}

template <int W>
struct __align__(16) TreeSmem {
    union {
        float o[W][kTile][68];  // 64 dims of the waves' sums; pitch: 16-byte aligned, 4 banks apart
        struct {                // before: the tile's queries as operands, [k-step][lane]
            uint4 qf[16][64];   // fp32
            uint4 q[16][64];    // f16 pieces, [k-step * 2 + piece]
        };
    };
    float m[W][kTile], l[W][kTile];
    uint32_t again;  // rows to compute again
};

// What a workgroup of a sequence works on (uniform).
struct TreeJob {
    int seq, h_kv, row0, n_rows, n_draft, past;
    int k_begin, k_end;  // cached keys
    bool drafts;         // and the drafted ones
    int slot;            // of the partial results
    int first[2];        // the pages of this wave's first step
};

// The page of a sequence's logical block (uniform), negative where there is none. A scalar load: its wait is
// not the vector loads', which are in flight beside it.
__device__ __forceinline__ int page_of(const TreeArgs& a, int seq, int lb) {
    if (a.n_table <= 0) return -1;
    typedef __attribute__((address_space(4))) const int32_t* ScalarPtr;
    lb = __builtin_amdgcn_readfirstlane(lb);
    const int blk = *(ScalarPtr)(a.tables + ((int64_t)seq * a.table_stride + min(lb, a.n_table - 1)));
    return lb < a.n_table && blk < a.n_blocks ? blk : -1;
}

__device__ __forceinline__ bool draft_seen(const TreeArgs& a, int seq, int tok, int i) {
    if (!a.mask) return i <= tok;
    return (a.mask[((int64_t)seq * a.n_tokens + tok) * a.words + i / 64] >> (i % 64)) & 1;
}

// One row again, key by key in fp32, by the whole workgroup of W waves: each takes every W-th key, its lanes dims
// lane + 64 u. The result goes to the output or the partial results.
template <int CT, int HD, int W>
__device__ __forceinline__ void tree_row_again(const TreeArgs& a, const TreeJob& w, TreeSmem<W>& sm, int row) {
    constexpr int U = HD / 64;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int tok = row / a.rep, h = w.h_kv * a.rep + row % a.rep;
    const int64_t hb = (int64_t)a.sb / a.n_head_kv * w.h_kv;
    const float* qp = a.q + ((int64_t)w.seq * a.n_tokens + tok) * a.q_stride + (int64_t)h * HD;
    float q[U], acc[U], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = qp[lane + 64 * u] * a.scale_log2e, acc[u] = 0.0f;
    auto add = [&](const float (&k)[U], const float (&v)[U]) {
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) s = fmaf(q[u], k[u], s);
        s = lanes_sum<64>(s);
        if (s == -INFINITY) return;  // no weight
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : exp2f(m - mn), p = exp2f(s - mn);
        l = l * c + p;
#pragma unroll
        for (int u = 0; u < U; ++u) acc[u] = fmaf(p, v[u], acc[u] * c);
        m = mn;
    };
    for (int t = w.k_begin + wave; t < w.k_end; t += W) {
        const int blk = page_of(a, w.seq, t / kKvBlock);
        float k[U], v[U];
        const int64_t off = (((int64_t)max(blk, 0) * a.n_layer + a.layer) * kKvBlock + t % kKvBlock) * a.sb + hb;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = blk >= 0 ? slot_value<CT>(a.k_arena + off, lane + 64 * u) : 0.0f;
            v[u] = blk >= 0 ? slot_value<CT>(a.v_arena + off, lane + 64 * u) : 0.0f;
        }
        add(k, v);
    }
    for (int t = wave; w.drafts && t < w.n_draft; t += W) {
        if (!draft_seen(a, w.seq, tok, t)) continue;
        const int64_t off = ((int64_t)w.seq * a.n_tokens + t) * a.kv_stride + (int64_t)w.h_kv * HD;
        float k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = a.k_cur[off + lane + 64 * u], v[u] = a.v_cur[off + lane + 64 * u];
        add(k, v);
    }
    float* so = &sm.o[0][0][0];  // [wave][HD]
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) so[wave * HD + lane + 64 * u] = acc[u];
    if (lane == 0) sm.m[wave][0] = m, sm.l[wave][0] = l;
    __syncthreads();
    float mx = -INFINITY, ls = 0.0f, o = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) mx = fmaxf(mx, sm.m[k][0]);
#pragma unroll
    for (int k = 0; k < W; ++k) {
        const float c = ref_factor(sm.m[k][0], sm.l[k][0], mx);
        ls += sm.l[k][0] * c;
        if (tid < HD) o += so[k * HD + tid] * c;
    }
    const int64_t tr = (int64_t)w.seq * a.n_tokens + tok, wr = (int64_t)w.slot * a.rows + tr * a.n_head + h;
    if (tid < HD) {
        if (a.splits == 1)
            a.out[tr * a.out_stride + (int64_t)h * HD + tid] = ls != 0.0f ? o / ls : 0.0f;
        else
            a.ws_o[wr * HD + tid] = o;
    }
    if (a.splits > 1 && tid == 0) a.ws_ml[2 * wr] = mx, a.ws_ml[2 * wr + 1] = ls;
    __syncthreads();
}

// A tile of 16 rows over a share of the keys, by a workgroup of W waves (HIST: cached keys too). EARLY: the first
// drafted keys are loaded before all else and taken before the cached ones, whose loads are in flight meanwhile:
// for calls without key splits, where a workgroup is a chain of latencies (on the device, 7 tokens over 100 keys 9.8 ->
// 9.4 us, one over one 8.0 -> 7.7). With splits few workgroups have drafted keys, and all pay for the registers (us a
// call: 8 sequences of 1500..4096 keys, 16 rows x 128, F16 25.9 -> 26.6, 64 dims 19.6 -> 20.5; 256 rows over 4096 F32 keys of
// two sequences 115 -> 139); at head_dim 256 they do not fit.
template <int CT, int HD, int W, bool HIST, bool EARLY>
__device__ __forceinline__ void tree_tile(const TreeArgs& a, const TreeJob& w, TreeSmem<W>& sm) {
    constexpr int U = HD / 64, CK = tree_chunk<CT>(), NP = CK / kKvBlock;
    // When a step's V is loaded and the next one's K: with K and after the scores, so that both have a step's time
    // to come, or (head_dim 256) after the scores and at the next step's start, for fewer registers and two waves
    // on a SIMD in place of one: 37 beams over 301..1501 F32 keys 39.8 -> 26.1 us, 16 over 1000..4096 59 -> 44
    // (F16 39 -> 34, Q8_0 46 -> 33); the next K after the products, where their registers meet, spills: a call 31.7 where
    // it now takes 27.3 (F16), 33.2 | 30.5 (Q8_0), the beams 28.2 | 27.2
    constexpr bool LATE = HD == 256;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, n = lane & 15;

    // ---- the lane's query row
    const int row = w.row0 + n;
    const bool q_ok = row < w.n_rows;
    const int tok = q_ok ? row / a.rep : 0, h = w.h_kv * a.rep + (q_ok ? row % a.rep : 0);
    const float* qp = a.q + ((int64_t)w.seq * a.n_tokens + tok) * a.q_stride + (int64_t)h * HD;
    auto load_q = [&](int d) {
        f32x4 t = *reinterpret_cast<const f32x4*>(qp + d);
        return q_ok ? t * a.scale_log2e : (f32x4){0.f, 0.f, 0.f, 0.f};
    };
    // ---- drafted keys, 16 at a time: the waves from the last on, which have the fewest cached keys
    const uint32_t rs = (uint32_t)(a.kv_stride * 4);
    uint64_t seen = 0;  // the row's mask word of the drafted keys in td, from the lane's first one
    auto load_drafts = [&](TreeKeys<kTypeF32, HD>& t, int k0) {
        const int left = w.n_draft - k0;
        const int64_t base = ((int64_t)w.seq * a.n_tokens + k0) * a.kv_stride + (int64_t)w.h_kv * HD;
        t.load_k(0, reinterpret_cast<const uint8_t*>(a.k_cur + base), min(n, left - 1) * rs, g);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            t.load_v_key(i, reinterpret_cast<const uint8_t*>(a.v_cur + base), min(4 * g + i, left - 1) * rs, n);
        if (a.mask)
            seen = a.mask[((int64_t)w.seq * a.n_tokens + tok) * a.words + k0 / 64] >> (k0 % 64 + 4 * g);
        else
            seen = (1u << min(max(tok + 1 - k0 - 4 * g, 0), 4)) - 1u;
    };
    const int d0 = w.drafts ? 16 * (W - 1 - wave) : w.n_draft;
    TreeKeys<kTypeF32, HD> early;
    if (EARLY && d0 < w.n_draft) load_drafts(early, d0);

    // ---- cached keys: the waves take steps of CK keys in turn. The first step's loads come before the queries
    const uint32_t head = (uint32_t)(a.sb / a.n_head_kv) * w.h_kv;
    const uint32_t sb = (uint32_t)a.sb, off_k = n * sb + head, off_v = 4 * g * sb + head;
    const int c0 = w.k_begin / CK + wave, c1 = HIST ? (w.k_end + CK - 1) / CK : 0;
    TreeKeys<CT, HD> t;
    int pages[NP], next[NP];
    auto pages_of = [&](int c, int (&p)[NP]) {
#pragma unroll
        for (int j = 0; j < NP; ++j) p[j] = page_of(a, w.seq, c * NP + j);
    };
    auto page_bytes = [&](int blk) {  // a missing page's loads read page 0; what they bring is cleared
        return ((int64_t)max(blk, 0) * a.n_layer + a.layer) * kKvBlock * a.sb;
    };
    if (c0 < c1) {
#pragma unroll
        for (int j = 0; j < NP; ++j) pages[j] = w.first[j];
        if constexpr (!LATE) {
#pragma unroll
            for (int j = 0; j < NP; ++j) t.load_k(j, a.k_arena + page_bytes(pages[j]), off_k, g);
#pragma unroll
            for (int j = 0; j < NP; ++j) t.load_v(j, a.v_arena + page_bytes(pages[j]), off_v, sb, n);
        }
    }

    // ---- the queries as operands, in LDS: a wave makes every W-th k-step's
    float qsc = 1.0f;
    if (CT == kTypeF32 || w.drafts)
        for (int s = wave; s < HD / 16; s += W) sm.qf[s][lane] = __builtin_bit_cast(uint4, load_q(16 * s + 4 * g));
    if constexpr (CT != kTypeF32) {
        constexpr int S = HD / 32;
        f32x4 x[S][2];
        float mx = 0.0f;  // of the whole row
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                x[s][k] = load_q(32 * s + 8 * g + 4 * k);
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[s][k][e]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const int ex = norm_exp(__float_as_uint(mx));
        const float f = pow2_bits(268 - ex);
        qsc = pow2_bits(ex - 14);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (s % W != wave) continue;
            f16x4 h0, l0, h1, l1;
            split4(x[s][0][0] * f, x[s][0][1] * f, x[s][0][2] * f, x[s][0][3] * f, h0, l0);
            split4(x[s][1][0] * f, x[s][1][1] * f, x[s][1][2] * f, x[s][1][3] * f, h1, l1);
            sm.q[2 * s][lane] = __builtin_bit_cast(uint4, __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7));
            sm.q[2 * s + 1][lane] = __builtin_bit_cast(uint4, __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    f32x4 o[U][4];
    float m = -INFINITY, l = 0.0f;  // l: of this lane's keys
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][e] = (f32x4){0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    // read again in every step: kept over the loop they would take as many registers as the keys
    auto operands = [&](const uint4(&q)[16][64]) {
        int at = lane;
        asm volatile("" : "+v"(at));
        return &q[0][at];
    };

    auto add_drafts = [&](TreeKeys<kTypeF32, HD>& t, int k0) {
        f32x4 r[1];
        t.scores(operands(sm.qf), r);
        t.scored(r);
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = 4 * g + i < w.n_draft - k0;
            s[i] = in && (seen >> i & 1) ? r[0][i] : -INFINITY;
            if (!in) t.zero_v(0, i);
        }
        softmax_step<4, U>(s, m, l, o);
        t.weigh(s, o);
    };
    if (EARLY && d0 < w.n_draft) add_drafts(early, d0);

    if (c0 < c1) {
        int pass = 0;
        bool again = false;
        for (int c = c0; c < c1;) {
            const bool more = c + W < c1;
            if (more) pages_of(c + W, next);
            if constexpr (LATE)
#pragma unroll
                for (int j = 0; j < NP; ++j) t.load_k(j, a.k_arena + page_bytes(pages[j]), off_k, g);
            const int left = w.k_end - c * CK;  // keys of the step, if fewer than CK
            bool whole = left >= CK;
#pragma unroll
            for (int j = 0; j < NP; ++j) whole &= pages[j] >= 0;
            if (!whole)  // zero rows for missing pages
#pragma unroll
                for (int j = 0; j < NP; ++j)
                    if (pages[j] < 0) t.zero_k(j);
            f32x4 r[NP];
            if constexpr (CT == kTypeF32)
                t.scores(operands(sm.qf), r);
            else
                t.scores(operands(sm.q), r);
            if constexpr (LATE) {
                __builtin_amdgcn_sched_barrier(0);  // not over the scores' registers
#pragma unroll
                for (int j = 0; j < NP; ++j) t.load_v(j, a.v_arena + page_bytes(pages[j]), off_v, sb, n);
            } else if (more) {
#pragma unroll
                for (int j = 0; j < NP; ++j) t.load_k(j, a.k_arena + page_bytes(next[j]), off_k, g);
            }
            if constexpr (CT == kTypeF32) t.scored(r);
            float s[4 * NP];
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[4 * j + i] = left >= CK || 16 * j + 4 * g + i < left ? r[j][i] * qsc : -INFINITY;
            if (!whole)  // no rows past the last key
#pragma unroll
                for (int j = 0; j < NP; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (pages[j] < 0 || 16 * j + 4 * g + i >= left) t.zero_v(j, i);
            if constexpr (CT == kTypeF32) {
                softmax_step<4 * NP, U>(s, m, l, o);
                t.weigh(s, o);
            } else {
                if constexpr (LATE) {
                    f16x8 ph, pl;
                    if (!again) raise_reference<4 * NP, U>(s, m, l, o);
                    pass = again ? pass + 1 : 0;
                    piece_weights<4 * NP>(s, 1.0f, m, l, pass, again);
                    split_weights(s, ph, pl);
                    t.template weigh<false>(ph, pl, band_unit(pass), o);
                    __builtin_amdgcn_sched_barrier(0);  // the next keys' loads no earlier than that
                } else {
                    float p[4 * NP];
                    f16x8 ph, pl;
#pragma unroll
                    for (int i = 0; i < 4 * NP; ++i) p[i] = s[i];
                    raise_reference<4 * NP, U>(p, m, l, o);
                    piece_weights<4 * NP>(p, 1.0f, m, l, 0, again);
                    split_weights(p, ph, pl);
                    t.template weigh<true>(ph, pl, 1.0f, o);
#pragma unroll 1
                    for (pass = 1; again; ++pass) {
#pragma unroll
                        for (int i = 0; i < 4 * NP; ++i) p[i] = s[i];
                        piece_weights<4 * NP>(p, 1.0f, m, l, pass, again);
                        split_weights(p, ph, pl);
                        t.again();
                        t.template weigh<false>(ph, pl, band_unit(pass), o);
                    }
                }
            }
            if (LATE && again) continue;  // the step once more: there is no room to keep its scores
            c += W;
            if (more) {
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    if constexpr (!LATE) t.load_v(j, a.v_arena + page_bytes(next[j]), off_v, sb, n);
                    pages[j] = next[j];
                }
            }
        }
    }

    for (int k0 = EARLY ? d0 + 16 * W : d0; k0 < w.n_draft; k0 += 16 * W) {
        TreeKeys<kTypeF32, HD> t;
        load_drafts(t, k0);
        add_drafts(t, k0);
    }

    // ---- the waves' sums together, 64 dims at a time: thread (of the first 256) -> row tid / 16, 4 dims
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < kTile) sm.m[wave][lane] = m, sm.l[wave][lane] = l;
    if (tid == 0) sm.again = 0u;
    __syncthreads();
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < W; ++k) mx = fmaxf(mx, sm.m[k][n]);
    const float c = ref_factor(m, l, mx) * (1.0f / kPieces);
    const int r = (tid >> 4) % kTile, d4 = 4 * (tid & 15), orow = w.row0 + r;
    float rm = -INFINITY, rl = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) rm = fmaxf(rm, sm.m[k][r]);
#pragma unroll
    for (int k = 0; k < W; ++k) rl += sm.l[k][r] * ref_factor(sm.m[k][r], sm.l[k][r], rm);
    const bool live = tid < 16 * kTile && orow < w.n_rows, direct = a.splits == 1;
    const int otok = orow / a.rep, oh = w.h_kv * a.rep + orow % a.rep;
    const int64_t trow = (int64_t)w.seq * a.n_tokens + otok, wrow = (int64_t)w.slot * a.rows + trow * a.n_head + oh;
    auto store4 = [&](int d, f32x4 v) {
        if (direct) {
            if (tid < 16 * kTile && otok < a.n_tokens) {
                float* out = a.out + trow * a.out_stride + (int64_t)oh * HD + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = live && rl != 0.0f ? v[e] / rl : 0.0f;
            }
        } else if (live) {
            *reinterpret_cast<f32x4*>(a.ws_o + wrow * HD + d) = v;
        }
    };
    bool bad = !(rl < INFINITY);
    for (int u = 0; u < U; ++u) {
        if (u) __syncthreads();
#pragma unroll
        for (int uu = 0; uu < U; ++uu)
            if (uu == u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4*>(&sm.o[wave][n][16 * g + 4 * i]) =
                        (f32x4){o[uu][0][i], o[uu][1][i], o[uu][2][i], o[uu][3][i]} * c;
        __syncthreads();
        f32x4 v = *reinterpret_cast<const f32x4*>(&sm.o[0][r][d4]);
#pragma unroll
        for (int k = 1; k < W; ++k) v += *reinterpret_cast<const f32x4*>(&sm.o[k][r][d4]);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= !(fabsf(v[e]) < INFINITY);
        store4(64 * u + d4, v);
    }
    if (!direct && live && d4 == 0) a.ws_ml[2 * wrow] = rm, a.ws_ml[2 * wrow + 1] = rl;
    if (bad && live) atomicOr(&sm.again, 1u << r);
    __syncthreads();
    for (uint32_t again = sm.again; again; again &= again - 1)
        tree_row_again<CT, HD, W>(a, w, sm, w.row0 + __builtin_ctz(again));
}

__device__ __forceinline__ void tree_job(const TreeArgs& a, TreeJob& w, int seq) {
    w.seq = seq;
    w.past = min(max(a.past[seq], 0), a.max_past);
    w.n_draft = a.n_draft ? min(max(a.n_draft[seq], 0), a.n_tokens) : a.n_tokens;
    w.n_rows = w.n_draft * a.rep;
}

// Grid: (unit, tile) pairs with the tiles of a unit on one XCD (workgroup id % 8) one after another, as they
// read the same keys; unit = (sequence, split, KV head).
// Few keys: a chain of latencies, lengths and page numbers, K and V, the queries, then scores, softmax and products
// once or twice, the waves' sums (7 tokens over 100 keys, 16/8 heads x 128 F16: 10 us, of which the memory is 0.4 MB).
// Many: the keys' loads, one step ahead (37 beams over 301..1501 F32 keys, 8/1 x 256: 24.6 us, 69 MB, 2.8 TB/s; matrix
// instructions busy 27 %), and under many rows of F32 the fp32 matrix instructions and what a wave does between
// them (256 rows over 4096 F32 keys, two sequences: 116 us, 58 of the 150 TFLOP/s of a large product; half the reads of
// a key, by two tiles to a wave, 121).
template <int CT, int HD, bool EARLY>
__global__ void __launch_bounds__(64 * kTreeWaves, HD == 256 ? 2 : 1) tree_attn_kernel(TreeArgs a) {
    __shared__ TreeSmem<kTreeWaves> sm;
    TreeJob w;
    const int id = blockIdx.x, turn = id / (8 * a.tiles), rest = id % (8 * a.tiles), unit = turn * 8 + rest % 8;
    if (unit >= a.units) return;
    w.h_kv = unit % a.n_head_kv;
    w.slot = unit / a.n_head_kv % a.splits;
    w.k_begin = w.slot * a.kps;
    w.row0 = rest / 8 * kTile;
    const int seq = unit / a.n_head_kv / a.splits, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int CK = tree_chunk<CT>();
#pragma unroll
    for (int j = 0; j < CK / kKvBlock; ++j)  // beside the loads of the lengths, not after them
        w.first[j] = page_of(a, seq, (w.k_begin / CK + wave) * (CK / kKvBlock) + j);
    tree_job(a, w, seq);
    const int n_split = max((w.past + a.kps - 1) / a.kps, 1);
    if (w.slot >= n_split || (w.row0 >= w.n_rows && a.splits > 1)) return;  // the merge writes such rows' zeros
    w.k_end = w.row0 < w.n_rows ? min(w.past, w.k_begin + a.kps) : 0;
    w.drafts = w.slot == n_split - 1 && w.row0 < w.n_rows;
    tree_tile<CT, HD, kTreeWaves, true, EARLY>(a, w, sm);
}

// ---------------------------------------------------------------- many rows
// Blocks of keys in LDS, two buffers of them, as f16 pieces. Q8_0: 8 W keys, decoded on the way into two pieces.
// F16: 64 keys, by direct loads, in rows without padding (8 sequences of 1500..4096 keys, 96 rows x 128: 51 -> 49 us a
// call, against a ring of four blocks of 32, when weights had one sum).
template <int CT, int HD, int W>
struct __align__(16) TreeBlock {
    static constexpr bool DMA = CT == kTypeF16;
    static constexpr int NPC = DMA ? 1 : 2, NBUF = 2, BK = DMA ? 64 : 8 * W;
    // K rows are read 16 bytes per lane down a column of 32 rows, V rows four at a time, 64 bytes each. Padded
    // rows lie 4 and 16 banks apart for that; in rows without padding the 16-byte pieces are permuted instead,
    // piece c of row r at c ^ swizzle(r).
    static constexpr int KP = DMA ? HD : HD + 8, VP = DMA ? HD : HD + 32;
    _Float16 k[NBUF][NPC][BK][KP];  // [buffer][piece][key][dim]
    _Float16 v[NBUF][NPC][BK][VP];
    static __device__ __forceinline__ int k_swizzle(int r) { return DMA ? r & (HD / 8 - 1) & 15 : 0; }
    static __device__ __forceinline__ int v_swizzle(int r) { return DMA ? (r & 3) << 1 : 0; }
};

// 16 bytes per lane from global memory (uniform base + per-lane byte offset) into LDS at lds_base + 16 lane.
// Inline asm: the compiler's builtin form makes LDS reads of any buffer wait for it. Not counted by the compiler;
// counted_wait below comes before the barrier that publishes the block. M0 is read one instruction after its write
// at the earliest.
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t off, const void* lds_base) {
    typedef __attribute__((address_space(3))) const void* LdsPtr;
    const uint32_t m0 = (uint32_t)(uintptr_t)(LdsPtr)lds_base;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m0)
                 : "memory", "m0");
}
// All loads but the N issued last have landed.
template <int N>
__device__ __forceinline__ void counted_wait() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);  // vmcnt(N) alone
    asm volatile(";dcq counted wait" ::: "memory");
}

// E elements of a Q8_0 slot's head piece from element e0, as loaded, and their way into LDS.
template <int E>
struct TreeRaw {
    uint32_t w[E / 4], d;
    __device__ __forceinline__ void load(const uint8_t* head, int e0) {
        const uint8_t* b = head + e0 / 32 * 34;
        d = ldu16(b);
        __builtin_memcpy(w, b + 2 + e0 % 32, E);  // 2-byte aligned
    }
    __device__ __forceinline__ void clear() { d = 0u; }
    __device__ __forceinline__ void store(_Float16* h, _Float16* l) const {
        const f16x2 dd = as_f16x2(d | d << 16);
#pragma unroll
        for (int j = 0; j < E / 8; ++j) {
            Pieces p[4];
#pragma unroll
            for (int t = 0; t < 4; ++t)
                p[t] = q8_pieces(int8_pair(__builtin_amdgcn_perm(0u, w[2 * j + t / 2], t % 2 ? 0x0c030c02u : 0x0c010c00u)), dd);
            *reinterpret_cast<f16x8*>(h + 8 * j) = as_f16x8(as_u32(p[0].h), as_u32(p[1].h), as_u32(p[2].h), as_u32(p[3].h));
            *reinterpret_cast<f16x8*>(l + 8 * j) = as_f16x8(as_u32(p[0].l), as_u32(p[1].l), as_u32(p[2].l), as_u32(p[3].l));
        }
    }
};

// What the unit-th workgroups (of every KV head and tile) work on: split `split` of kps keys of a sequence.
struct TreeShare {
    int seq, split, kps;  // seq -1: nothing
};
// Up to 64 sequences share the units by their lengths, which the host does not know: the fewest keys per unit
// (a.kps or more, in steps of an eighth) that a.share units suffice for. 8 sequences of 1500..4096 keys on 64
// units: 384 keys, where their longest alone would ask for 512 and leave a quarter of the units without work;
// 24 tokens of 32/8 heads x 128, F16: 40.7 -> 38.5 us as it was taken. More sequences even out by themselves.
__device__ __forceinline__ TreeShare tree_share(const TreeArgs& a, int unit) {
    const int per_seq = a.splits - 1;
    if (!a.share) return {unit / per_seq, unit % per_seq, a.kps};
    const int lane = threadIdx.x & 63;
    const int past = lane < a.n_seqs ? min(max(a.past[lane], 0), a.max_past) : 0;
    int sum = past;  // below 2^30
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k, 64);
    int kps = max(a.kps, (int)(((uint32_t)sum + a.share - 1) / a.share + 31) & ~31), n, upto;
    for (;; kps += max(kps / 8 & ~31, 32)) {
        n = ((uint32_t)past + kps - 1) / (uint32_t)kps;
        upto = n;  // units up to this lane's sequence
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const int o = __shfl_up(upto, k, 64);
            upto += lane >= k ? o : 0;
        }
        if (__builtin_amdgcn_readlane(upto, 63) <= a.share || kps >= a.max_past) break;
    }
    const uint64_t after = __ballot(upto > unit);
    if (!after) return {-1, 0, kps};
    const int seq = __ffsll((unsigned long long)after) - 1;
    return {seq, unit - __builtin_amdgcn_readlane(upto - n, seq), kps};
}

// 32 W rows of a KV head over a share of its cached keys (slots 1 ..), or 16 rows over the drafted keys (slot 0:
// the workgroups from hist_wgs on, which fill the end of the launch).
// A wave's block is a chain: 32 to 48 matrix instructions of scores, the softmax, as many of values and their sums into
// O; two waves a SIMD cover each other's. 24 tokens of 8 sequences of 1500..4096 keys, 32/8 heads x 128, F16: 41 us; by
// a timeline 2 for the share, 2.7 for the queries, 2 for the first block, 22 for 384 keys (3.7 a block of 64, 2.8 alone on
// a SIMD), 2 for the results, and 6 of drafted keys at the end, in part beside the others. 64 tokens over 32768 keys,
// Q8_0: 120 us for 34.4 GFLOP, three products each: 0.86 PFLOP/s of f16 where a large library product reaches 1.42; matrix
// instructions busy 47 % of the cycles, VALU 36 %. In it 99 us of the shares' loops, 7 before and 6 for drafted keys after
// them.
template <int CT, int HD, int W>
__global__ void __launch_bounds__(64 * W, HD == 256 ? 1 : 2) tree_block_kernel(TreeArgs a) {
    using Block = TreeBlock<CT, HD, W>;
    constexpr int E = HD / 8;    // elements per staging thread of Q8_0: key tid / 8 of the block
    constexpr int KS = HD / 16;  // k-steps of the score product
    constexpr int NT = HD / 32;  // 32-dim tiles of the output
    constexpr int NPC = Block::NPC;
    __shared__ union {
        Block b;
        TreeSmem<W> t;
    } sm;
    __shared__ uint32_t again[W];
    TreeJob w;
    int id = (int)blockIdx.x - a.hist_wgs;
    if (id >= 0) {
        const int per_seq = a.n_head_kv * a.tiles16;
        tree_job(a, w, id / per_seq);
        w.h_kv = id % per_seq / a.tiles16;
        w.row0 = id % a.tiles16 * kTile;
        w.k_begin = w.k_end = 0;
        w.drafts = true;
        w.slot = 0;
        if (w.row0 < w.n_rows) tree_tile<kTypeF32, HD, W, false, false>(a, w, sm.t);
        return;
    }
    id = blockIdx.x;
    const int turn = id / (8 * a.tiles), rest = id % (8 * a.tiles), unit = turn * 8 + rest % 8;
    if (unit >= a.units) return;
    w.h_kv = unit % a.n_head_kv;
    w.row0 = rest / 8 * (kRowsPerWave * W);
    TreeShare share = tree_share(a, unit / a.n_head_kv);
    share.seq = __builtin_amdgcn_readfirstlane(share.seq);
    share.split = __builtin_amdgcn_readfirstlane(share.split);
    share.kps = __builtin_amdgcn_readfirstlane(share.kps);
    if (id == 0 && threadIdx.x == 0 && a.ws_kps) *a.ws_kps = share.kps;
    if (share.seq < 0) return;
    tree_job(a, w, share.seq);
    w.slot = share.split + 1;
    w.k_begin = share.split * share.kps;
    w.k_end = min(w.past, w.k_begin + share.kps);
    w.drafts = false;
    if (w.k_begin >= w.k_end || w.row0 >= w.n_rows) return;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int p = lane >> 5, c32 = lane & 31;

    // ---- the lane's query row: pieces of q * scale * log2(e) at dims 16 s + 8 p .. + 7
    const int r0 = w.row0 + kRowsPerWave * wave, row = r0 + c32;
    const bool q_ok = row < w.n_rows;
    const int tok = q_ok ? row / a.rep : 0, h = w.h_kv * a.rep + (q_ok ? row % a.rep : 0);
    const int64_t trow = (int64_t)w.seq * a.n_tokens + tok;
    f16x8 qh[KS], ql[KS];
    float qsc;
    {
        const float* qp = a.q + trow * a.q_stride + (int64_t)h * HD + 8 * p;
        f32x4 t[KS][2];
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                t[s][k] = *reinterpret_cast<const f32x4*>(qp + 16 * s + 4 * k) * (q_ok ? a.scale_log2e : 0.0f);
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(t[s][k][e]));
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const int ex = norm_exp(__float_as_uint(mx));
        const float f = pow2_bits(268 - ex);
        qsc = pow2_bits(ex - 14);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            f16x4 h0, l0, h1, l1;
            split4(t[s][0][0] * f, t[s][0][1] * f, t[s][0][2] * f, t[s][0][3] * f, h0, l0);
            split4(t[s][1][0] * f, t[s][1][1] * f, t[s][1][2] * f, t[s][1][3] * f, h1, l1);
            qh[s] = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
            ql[s] = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }

    constexpr int BK = Block::BK, RW = BK / W;  // keys of a block, and of them a wave's
    constexpr int NH = BK / 32;                 // 32-key parts of a block
    constexpr bool DMA = Block::DMA;
    constexpr int NBUF = Block::NBUF;
    const int64_t head = a.sb / a.n_head_kv * w.h_kv;
    // ---- staging, Q8_0: a block's loads are issued before the products of the block before, and stored after them
    const int skey = tid >> 3, se0 = E * (tid & 7);
    TreeRaw<E> rk, rv;
    // the page of the wave's rows 8 w .. + 7
    auto wave_page = [&](int kb) { return kb < w.k_end ? page_of(a, w.seq, (kb + RW * wave) / kKvBlock) : -1; };
    auto load_block = [&](int kb, int blk) {  // zeros for missing pages and past the last key
        if (blk >= 0 && kb + skey < w.k_end) {
            const int64_t off = (((int64_t)blk * a.n_layer + a.layer) * kKvBlock + (kb + skey) % kKvBlock) * a.sb + head;
            rk.load(a.k_arena + off, se0);
            rv.load(a.v_arena + off, se0);
        } else {
            rk.clear();
            rv.clear();
        }
    };
    auto store_block = [&](int buf) {
        rk.store(&sm.b.k[buf][0][skey][se0], &sm.b.k[buf][NPC - 1][skey][se0]);
        rv.store(&sm.b.v[buf][0][skey][se0], &sm.b.v[buf][NPC - 1][skey][se0]);
    };
    // ---- staging, F16: NI loads of RI rows each for K and for V
    constexpr int RI = 512 / HD, NI = RW / RI;
    uint32_t k_off[NI], v_off[NI];
    bool partial = false;  // of the block issued last this wave has rows to clear
    int page_next = 0;
    if constexpr (DMA) {
        const int c = lane % (HD / 8);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = RW * wave + i * RI + lane / (HD / 8);
            const uint32_t at = (uint32_t)(r % kKvBlock) * (uint32_t)a.sb + (uint32_t)head;
            k_off[i] = at + 16 * (c ^ Block::k_swizzle(r));
            v_off[i] = at + 16 * (c ^ Block::v_swizzle(r));
        }
    }
    auto issue = [&](int kb, int blk, int buf) {  // a missing page's loads read page 0; their rows are cleared
        const int64_t page = ((int64_t)max(blk, 0) * a.n_layer + a.layer) * kKvBlock * a.sb;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            dma16(a.k_arena + page, k_off[i], &sm.b.k[buf][0][RW * wave + i * RI][0]);
            dma16(a.v_arena + page, v_off[i], &sm.b.v[buf][0][RW * wave + i * RI][0]);
        }
        partial = blk < 0 || kb + RW * (wave + 1) > w.k_end;
    };
    auto clear_rows = [&](int kb, int buf) {  // rows of a missing page, and past the last key
        const int from = wave_page(kb) < 0 ? 0 : max(w.k_end - kb - RW * wave, 0);
        for (int i = from * (HD / 8) + lane; i < RW * HD / 8; i += 64) {  // RW rows of HD / 8 pieces
            *reinterpret_cast<uint4*>(&sm.b.k[buf][0][RW * wave][8 * i]) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(&sm.b.v[buf][0][RW * wave][8 * i]) = make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto landed = [&](int kb, int buf) {  // the wave's rows of block kb, the last one issued
        counted_wait<0>();
        if (partial && kb < w.k_end) clear_rows(kb, buf);
    };

    f32x16 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // l: this lane's keys only, until the end

    // ---- S^T = K Q^T of the 32 keys from row `sub` of a block, the small products in a sum of their own
    auto scores = [&](int buf, int sub, f32x16& sc) {
        f32x16 hi;
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] = 0.0f, hi[v] = 0.0f;
        const _Float16* kh = &sm.b.k[buf][0][sub + c32][0];
        const _Float16* kl = &sm.b.k[buf][NPC - 1][sub + c32][0];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int at = 8 * ((2 * s + p) ^ Block::k_swizzle(c32));
            const f16x8 fh = *reinterpret_cast<const f16x8*>(kh + at);
            if constexpr (NPC == 2) {
                const f16x8 fl = *reinterpret_cast<const f16x8*>(kl + at);
                sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fl, qh[s], sc, 0, 0, 0);
            }
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(fh, ql[s], sc, 0, 0, 0);
            hi = __builtin_amdgcn_mfma_f32_32x32x16_f16(fh, qh[s], hi, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] += hi[v];
    };
    // the lane's keys are 8 (i / 4) + 4 p + i % 4
    auto mask = [&](f32x16& sc, int left) {
        if (left < 32) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i >> 2) + 4 * p + (i & 3) >= left) sc[i] = -INFINITY;
        }
    };
    // a new reference where the largest of a block's scores asks for one
    auto raise = [&](const float (&s)[16 * NH]) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16 * NH; ++i) mx = fmaxf(mx, s[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * qsc;
        if (!__any(mx > m + kSlack)) return;
        const float m_new = mx > m + kSlack ? __builtin_ceilf(mx) : m;
        const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[t][v] *= alpha;
    };
    // O^T += V^T P^T of a block, the weights in units of `unit`: as pieces, operand s takes i = 8 s .. + 7, keys
    // 16 s + 4 p + 0..3 and 16 s + 8 + 4 p + 0..3. first: the unit is 1, and the first pieces' products go on from O
    auto values = [&](auto first, int buf, const float (&pw)[16 * NH], float unit) {
        f16x8 ph[2 * NH], pl[2 * NH];
#pragma unroll
        for (int s = 0; s < 2 * NH; ++s) split_weights(pw + 8 * s, ph[s], pl[s]);
        const int vrow = 4 * p + ((lane & 15) >> 2);
        // of tile t the 16-byte piece 4 t + vc of the row, its half lane % 2
        const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vx = Block::v_swizzle(lane >> 2);
        f32x16 low[2];
        auto add_low = [&](int t) {
#pragma unroll
            for (int v = 0; v < 16; ++v) o[t][v] = __builtin_fmaf(low[t % 2][v], 1.0f / kLow, o[t][v]);
        };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x16 &lo = low[t % 2], high;
#pragma unroll
            for (int v = 0; v < 16; ++v) lo[v] = 0.0f, high[v] = first ? o[t][v] : 0.0f;
#pragma unroll
            for (int s = 0; s < 2 * NH; ++s) {
                f16x8 f[NPC];
#pragma unroll
                for (int u = 0; u < NPC; ++u) {
                    const int at = 8 * ((4 * t + vc) ^ vx) + 4 * (lane & 1);
                    const f16x4 a0 = lds_transposed(&sm.b.v[buf][u][16 * s + vrow][at]);
                    const f16x4 a1 = lds_transposed(&sm.b.v[buf][u][16 * s + 8 + vrow][at]);
                    f[u] = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
                }
                lo = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[0], pl[s], lo, 0, 0, 0);
                if constexpr (NPC == 2) high = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[1], ph[s], high, 0, 0, 0);
                high = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[0], ph[s], high, 0, 0, 0);
            }
            if constexpr (first) {
                o[t] = high;
                if (t) add_low(t - 1);
            } else {
#pragma unroll
                for (int v = 0; v < 16; ++v)
                    o[t][v] = __builtin_fmaf(__builtin_fmaf(lo[v], 1.0f / kLow, high[v]), unit, o[t][v]);
                // O where the VALU takes it, the queries (below) in the other half of the registers: Q8_0, 32 tokens of 8
                // sequences of 1500..4096 keys, 16/4 heads, 132 -> 124 us a call
                if constexpr (HD == 256) asm volatile("" : "+v"(o[t]));
            }
        }
        if constexpr (first) add_low(NT - 1);
    };

    int blk_next = -1;
    if constexpr (DMA) {
        issue(w.k_begin, wave_page(w.k_begin), 0);
        page_next = wave_page(w.k_begin + BK);
        landed(w.k_begin, 0);
    } else {
        load_block(w.k_begin, wave_page(w.k_begin));
        blk_next = wave_page(w.k_begin + BK);
        store_block(0);
    }
    __syncthreads();
    int buf = 0;
    for (int kb = w.k_begin; kb < w.k_end; kb += BK, buf ^= 1) {
        const bool more = kb + BK < w.k_end;
        if constexpr (DMA) {
            if (more) {
                issue(kb + BK, page_next, buf ^ 1);
                page_next = wave_page(kb + 2 * BK);
            }
        } else if (more) {
            load_block(kb + BK, blk_next);
            blk_next = wave_page(kb + 2 * BK);
        }
        if (r0 < w.n_rows) {
            if constexpr (HD == 256) {
#pragma unroll
                for (int k = 0; k < KS; ++k) asm volatile("" : "+a"(qh[k]), "+a"(ql[k]));
            }
            float s[16 * NH];
            auto all_scores = [&](int b) {
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    f32x16 sc;
                    scores(b, 32 * h, sc);
                    mask(sc, w.k_end - kb - 32 * h);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[16 * h + i] = sc[i];
                }
            };
            // head_dim 256 has one form of the products for all passes: two spill (F16 139 us where this takes 97)
            bool again = true;
            if constexpr (HD < 256) {
                all_scores(buf);
                raise(s);
                piece_weights<16 * NH>(s, qsc, m, l, 0, again);
                values(std::true_type{}, buf, s, 1.0f);
            }
#pragma unroll 1
            for (int pass = HD < 256; again; ++pass) {
                int b = buf;
                asm volatile("" : "+s"(b));  // read anew, not kept from pass to pass
                all_scores(b);
                if (HD == 256 && pass == 0) raise(s);
                piece_weights<16 * NH>(s, qsc, m, l, pass, again);
                values(std::false_type{}, b, s, band_unit(pass));
            }
        }
        if constexpr (DMA)
            landed(kb + BK, buf ^ 1);
        else if (more)
            store_block(buf ^ 1);
        __syncthreads();
    }
    l += __shfl_xor(l, 32, 64);

    // ---- partial results: dims 32t + 8j + 4p + 0..3 of the lane's row
    bool bad = !(l < INFINITY);
    const int64_t wrow = (int64_t)w.slot * a.rows + trow * a.n_head + h;
    float* orow = a.ws_o + wrow * HD;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 x = {o[t][4 * j], o[t][4 * j + 1], o[t][4 * j + 2], o[t][4 * j + 3]};
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= !(fabsf(x[e]) < INFINITY);
            if (q_ok) *reinterpret_cast<f32x4*>(orow + 32 * t + 8 * j + 4 * p) = x * (1.0f / kPieces);
        }
    if (q_ok && p == 0) a.ws_ml[2 * wrow] = m, a.ws_ml[2 * wrow + 1] = l;
    const uint64_t set = __ballot(bad && q_ok);
    if (lane == 0) again[wave] = (uint32_t)set | (uint32_t)(set >> 32);
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < W; ++k)
        for (uint32_t x = again[k]; x; x &= x - 1)
            tree_row_again<CT, HD, W>(a, w, sm.t, w.row0 + kRowsPerWave * k + __builtin_ctz(x));
}

// The merge of a sequence's splits (6144 rows x 128 of up to 12 splits: 7.2 us, 2048 of 33: 9.3; the partial results
// come from L2 at 4 to 5 TB/s): M = max m, L = sum l 2^(m - M), out = sum o 2^(m - M) / L, zeros for a row
// that saw no key or has no drafted token. P lanes share 4 outputs, lane p the splits p, p + P, ...
template <int HD, int P>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a) {
    constexpr int NS = 8;  // splits of a lane whose loads are issued together
    constexpr int QP = HD / 4 * P;  // threads of a row
    const int p = threadIdx.x % P, d = threadIdx.x / P % (HD / 4) * 4;
    const int row = (int)blockIdx.x * (256 / QP) + threadIdx.x / QP;  // below 2^27
    if (row >= a.rows) return;
    const int trow = row / a.n_head, h = row % a.n_head, seq = trow / a.n_tokens, tok = trow % a.n_tokens;
    const int past = min(max(a.past[seq], 0), a.max_past);
    const int n_draft = a.n_draft ? min(max(a.n_draft[seq], 0), a.n_tokens) : a.n_tokens;
    const int kps = a.ws_kps ? *a.ws_kps : a.kps, n_hist = (past + kps - 1) / kps;
    const int n_split = tok < n_draft ? (a.draft_wgs ? n_hist + 1 : max(n_hist, 1)) : 0;
    float m = -INFINITY, l = 0.0f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = p; s0 < n_split; s0 += P * NS) {
        float2 ml[NS];
        f32x4 ov[NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            const int s = s0 + P * k;
            const int64_t r = (int64_t)s * a.rows + row;
            ml[k] = s < n_split ? *reinterpret_cast<const float2*>(a.ws_ml + 2 * r) : make_float2(-INFINITY, 0.0f);
            ov[k] = s < n_split ? *reinterpret_cast<const f32x4*>(a.ws_o + r * HD + d) : (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        float mn = m;
#pragma unroll
        for (int k = 0; k < NS; ++k) mn = fmaxf(mn, ml[k].x);
        const float c = ref_factor(m, l, mn);
        l *= c;
        acc *= c;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            const float f = ref_factor(ml[k].x, ml[k].y, mn);
            l = fmaf(ml[k].y, f, l);
            acc += ov[k] * f;
        }
        m = mn;
    }
    const float mx = lanes_max<P>(m), f = ref_factor(m, l, mx);
    l = lanes_sum<P>(l * f);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = lanes_sum<P>(acc[e] * f);
    if (p != 0) return;
    float* out = a.out + (int64_t)trow * a.out_stride + (int64_t)h * HD + d;
    const float inv = 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = l != 0.0f ? acc[e] * inv : 0.0f;
}

// ---------------------------------------------------------------- host side
struct TreePlan {
    int block_waves;  // 0: the 16-row kernel
    int tiles, splits, kps;
    int share, units;  // of the block kernel: see tree_share; units: of all KV heads
};

// Key splits: workgroups until about three per CU have work, 128 keys (a step of each wave) at the least. Two, three,
// four, five, six per CU, 16 sequences of 1000..4096 keys, us a call: F16, 16/4 heads x 128, 24.9, 23.8, 29.8, 29.8, 29.5;
// x 64 17.4, 18.6, 20.8, 20.8, 21.6; 8/2 x 256 26.9, 27.1, 35.1, 35.2, 35.2; Q8_0 x 128 31, 27.2, 36.5, 36.6, 36.7; F32 x 256
// 43.5, 39.4, 48.7, 48.6, 48.8.
static TreePlan tree_plan16(int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past) {
    TreePlan p{};
    p.tiles = (n_tokens * (n_head / n_head_kv) + kTile - 1) / kTile;
    const int64_t base = (int64_t)p.tiles * n_head_kv * n_seqs, want = std::max<int64_t>(1, (3 * cu_count() + base - 1) / base);
    p.kps = (int)std::max<int64_t>(128, round_up((max_past + want - 1) / want, 64));
    p.splits = std::max(1, (max_past + p.kps - 1) / p.kps);
    return p;
}

// The block kernel's rows share the keys that the 16-row kernel reads once per tile, but its workgroups need more of
// both to be worth their start. From which number of rows on it is the faster (16-row kernel | block kernel, us a call;
// 16/4 heads at head_dim 256, else 32/8):
//   8 sequences of 1500..4096 keys, head_dim 128: 16 rows F16 26 | 33, Q8_0 30 | 41; 20 rows 42 | 32, 61 | 44
//   the same, head_dim 64: 64 rows F16 32 | 34, Q8_0 43 | 37; 80 rows 37 | 34, 50 | 39; 32 of 1000..2048 keys 64 rows
//   59 | 61, 74 | 75; 80 rows 69 | 65, 91 | 81
//   the same, head_dim 256: 80 rows F16 86 | 89, Q8_0 122 | 116; 96 rows 98 | 91, 144 | 119; 128 rows 110 | 97, 143 | 126;
//   32 of 1000..2048 keys 96 rows 173 | 170, 241 | 222; one of 32768 96 rows 97 | 109, 135 | 137; 128 rows 119 | 115, 168 | 146
//   one sequence of 4096 keys, where the block kernel's 256 keys per workgroup leave CUs without one: head_dim 128
//   32 rows F16 18 | 20, Q8_0 21 | 27; 40 rows 25 | 21, 29 | 28; head_dim 64 128 rows 19 | 23, 23 | 24; 256 rows 23 | 25,
//   30 | 26; head_dim 256 192 rows 44 | 47, 55 | 64; 256 rows 48 | 50, 63 | 65
//   fewer than 256 keys: never (8 sequences of 100..255 keys: 64 rows F16 18 | 24, Q8_0 22 | 30, 256 rows 37 | 36, 45 | 40)
static bool tree_in_blocks(int ct, int hd, int n_head_kv, int n_seqs, int rows, int max_past) {
    if (ct == kTypeF32 || max_past < 256) return false;
    const int from = hd == 128 ? 16 : hd == 64 ? 64 : ct == kTypeF16 ? 96 : 80;
    const bool idle = (int64_t)n_head_kv * n_seqs * ((max_past + 255) / 256) < cu_count();
    return rows > (idle ? (hd == 128 ? 2 : 3) * from : from);
}

static TreePlan tree_plan(int ct, int hd, int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past) {
    const int rows = n_tokens * (n_head / n_head_kv), bk = 64;
    if (!tree_in_blocks(ct, hd, n_head_kv, n_seqs, rows, max_past))
        return tree_plan16(n_head, n_head_kv, n_seqs, n_tokens, max_past);
    TreePlan p{};
    int share;
    int64_t kps;
    auto plan_of = [&](int waves) {  // as many workgroups as there is room for at once
        p.block_waves = waves;
        p.tiles = (rows + kRowsPerWave * waves - 1) / (kRowsPerWave * waves);
        const int64_t base = (int64_t)p.tiles * n_head_kv, wgs = waves == 8 ? cu_count() : 2 * cu_count();
        share = (int)std::max<int64_t>((wgs + base - 1) / base, n_seqs);
        kps = std::max<int64_t>(256, round_up(((int64_t)max_past * n_seqs + share - 1) / share, bk));
    };
    // Eight waves decode a Q8_0 block for twice the rows, four start and end sooner: eight for long shares of long
    // histories. 256 rows x 128, four | eight, us a call: one sequence of 4096 keys 38 | 43, of 16384 (512 keys a share)
    // 80 | 76, of 32768 131 | 121, of 65536 255 | 242, 64 dims 178 | 172; four of 16384 267 | 257, 16 of 4096 258 | 263.
    // F16, which is not decoded, with one sum for both pieces of the weights: 16 of 500..2048 89 | 114, one of 4096
    // 22 | 28, of 65536 143 | 142.
    if (ct == kTypeQ8_0 && rows > 128 && hd <= 128 && max_past >= 8192) plan_of(8);
    if (p.block_waves == 0 || kps < 1024) plan_of(4);
    // kps: keys of a split were all sequences as long as the longest; up to 64 sequences share out by their lengths,
    // of no fewer than half as many keys (which bounds the partial results)
    p.share = n_seqs > 1 && n_seqs <= 64 ? share : 0;
    p.kps = (int)(p.share ? std::max<int64_t>(256, round_up(kps / 2, bk)) : kps);
    p.splits = 1 + (max_past + p.kps - 1) / p.kps;
    p.units = (p.share ? p.share : n_seqs * (p.splits - 1)) * n_head_kv;
    return p;
}

static size_t tree_partial_bytes(const TreePlan& p, int hd, int64_t rows) {
    return p.splits <= 1 ? 0 : (size_t)(round_up(p.splits * rows * hd * 4, 256) + round_up(p.splits * rows * 2 * 4, 256) + 256);
}

// Of the largest plan: the query does not know the cache type.
size_t tree_workspace_bytes(int hd, int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past) {
    const int64_t rows = (int64_t)n_seqs * n_tokens * n_head;
    size_t most = 0;
    for (int ct : {kTypeF32, kTypeF16, kTypeQ8_0})
        most = std::max(most, tree_partial_bytes(tree_plan(ct, hd, n_head, n_head_kv, n_seqs, n_tokens, max_past), hd, rows));
    return most;
}

template <int HD, int P>
static void launch_tree_merge_t(const TreeArgs& a, hipStream_t st) {
    constexpr int rows = 256 / (HD / 4 * P);
    hipLaunchKernelGGL((tree_merge_kernel<HD, P>), dim3((unsigned)((a.rows + rows - 1) / rows)), dim3(256), 0, st, a);
}

// Lanes that share an output: one where a lane takes all splits in one step or there are outputs for half the
// CUs' waves (2048 rows x 128, 33 splits: 9.2 us, four lanes 11.8; 6144 rows, 9 splits 6.0 and 9.4), else a
// workgroup a row.
template <int HD>
static void launch_tree_merge(const TreeArgs& a, hipStream_t st) {
    if (a.splits <= 8 || a.rows * (HD / 4) >= 32768)
        launch_tree_merge_t<HD, 1>(a, st);
    else
        launch_tree_merge_t<HD, 1024 / HD>(a, st);
}

template <int CT, int HD>
static void launch_tree_t(const TreeArgs& a, int block_waves, int wgs, hipStream_t st) {
    if constexpr (CT == kTypeQ8_0 && HD <= 128) {
        if (block_waves == 8) {
            hipLaunchKernelGGL((tree_block_kernel<CT, HD, 8>), dim3(wgs), dim3(512), 0, st, a);
            return;
        }
    }
    if constexpr (CT != kTypeF32) {
        if (block_waves == 4) {
            hipLaunchKernelGGL((tree_block_kernel<CT, HD, 4>), dim3(wgs), dim3(256), 0, st, a);
            return;
        }
    }
    if constexpr (HD < 256) {
        if (a.splits == 1) {
            hipLaunchKernelGGL((tree_attn_kernel<CT, HD, true>), dim3(wgs), dim3(64 * kTreeWaves), 0, st, a);
            return;
        }
    }
    hipLaunchKernelGGL((tree_attn_kernel<CT, HD, false>), dim3(wgs), dim3(64 * kTreeWaves), 0, st, a);
}

// A call's workgroups: of the shares of the cached keys, and of drafted keys alone.
struct TreeGrid {
    int64_t units, drafts, wgs;
};
static TreeGrid tree_grid(const TreePlan& p, int n_head, int n_head_kv, int n_seqs, int n_tokens) {
    const int tiles16 = (n_tokens * (n_head / n_head_kv) + kTile - 1) / kTile;
    TreeGrid g;
    g.drafts = p.block_waves ? (int64_t)n_seqs * n_head_kv * tiles16 : 0;
    g.units = p.block_waves ? p.units : (int64_t)n_seqs * p.splits * n_head_kv;
    g.wgs = g.drafts + (g.units + 7) / 8 * 8 * p.tiles;
    return g;
}

bool tree_fits(int ct, int hd, int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past) {
    const TreePlan p = tree_plan(ct, hd, n_head, n_head_kv, n_seqs, n_tokens, max_past);
    const int threads = 64 * (p.block_waves ? p.block_waves : kTreeWaves);
    return tree_grid(p, n_head, n_head_kv, n_seqs, n_tokens).wgs * threads <= UINT32_MAX;
}

hipError_t launch_tree_attention(int ct, int hd, TreeArgs a, void* ws, hipStream_t st) {
    const TreePlan p = tree_plan(ct, hd, a.n_head, a.n_head_kv, a.n_seqs, a.n_tokens, a.max_past);
    a.rep = a.n_head / a.n_head_kv;
    a.tiles = p.tiles, a.splits = p.splits, a.kps = p.kps;
    a.rows = (int64_t)a.n_seqs * a.n_tokens * a.n_head;
    a.tiles16 = (a.n_tokens * a.rep + kTile - 1) / kTile;
    const TreeGrid g = tree_grid(p, a.n_head, a.n_head_kv, a.n_seqs, a.n_tokens);
    const int wgs = (int)g.wgs;
    a.units = (int)g.units, a.draft_wgs = (int)g.drafts, a.hist_wgs = (int)(g.wgs - g.drafts);
    a.share = p.share;
    if (p.splits > 1) {  // O, (m, l), and the keys per split where the device chooses them
        uint8_t* w = static_cast<uint8_t*>(ws);
        a.ws_o = reinterpret_cast<float*>(w), w += round_up(p.splits * a.rows * hd * 4, 256);
        a.ws_ml = reinterpret_cast<float*>(w), w += round_up(p.splits * a.rows * 2 * 4, 256);
        if (p.share) a.ws_kps = reinterpret_cast<int*>(w);
    }
#define DCQ_TREE_CASE(C, H)                                         \
    if (ct == C && hd == H) {                                       \
        launch_tree_t<C, H>(a, p.block_waves, wgs, st);             \
    } else
    DCQ_TREE_CASE(kTypeQ8_0, 128)
    DCQ_TREE_CASE(kTypeQ8_0, 64)
    DCQ_TREE_CASE(kTypeQ8_0, 256)
    DCQ_TREE_CASE(kTypeF16, 128)
    DCQ_TREE_CASE(kTypeF16, 64)
    DCQ_TREE_CASE(kTypeF16, 256)
    DCQ_TREE_CASE(kTypeF32, 128)
    DCQ_TREE_CASE(kTypeF32, 64)
    DCQ_TREE_CASE(kTypeF32, 256)
    return hipErrorNotSupported;
#undef DCQ_TREE_CASE
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits <= 1) return e;
    if (hd == 64)
        launch_tree_merge<64>(a, st);
    else if (hd == 128)
        launch_tree_merge<128>(a, st);
    else
        launch_tree_merge<256>(a, st);
    return hipGetLastError();
}

}  // namespace dcq
