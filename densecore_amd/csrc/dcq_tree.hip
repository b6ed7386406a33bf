// dcq_tree.hip — attention of drafted tokens over the paged KV cache, several sequences in one call.
//
// Sequence b has n_past(b) cached keys (pages tables[b]) and n_draft(b) drafted tokens with fp32 K / V rows of
// their own. Row (token j, query head h) attends every cached key, and drafted key i where bit i of mask[b][j]
// is set:  out = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t).  The online softmax keeps a reference m
// (an integer in base 2, raised when a score passes it by 8), the sum l of p' = 2^(s - m), s = scale log2(e)
// q . k, and O = sum p' v.
//
// Query rows of a KV head are the (token, head of its group) pairs, token-major, in tiles of 16: a column of
// the matrix instructions, whatever the group size. S^T = K Q^T puts the keys 4 (lane / 16) + i of row
// lane % 16 into lane registers i, and O^T += V^T P^T takes its weights from the same lanes, so P never
// moves; K, V and Q go from memory to the matrix registers without LDS:
//   K: a lane holds 8 consecutive dims of key lane % 16 (fp32: 4), the A operand as it is.
//   V: a lane holds dims 64 u + 4 (lane % 16) + 0..3 of the keys whose weights it has; output tile (u, e) is
//      made of the dims 64 u + 4 m + e, so that its A operand is in the lane, one byte permute per two keys.
//
// Arithmetic. F16 and Q8_0 slots are multiplied on the f16 matrix instructions (16 x the fp32 ones' rate):
// q and p', fp32, are split into two f16 pieces of 22 bits (q under an exponent per row, p' times 2^7), an
// F16 slot is one exact piece, and a Q8_0 value d * q, a product of 11 and 7 bits, is exactly the two pieces
// f16(d q) and d q - f16(d q). F32 slots and the drafted rows use the fp32 matrix instructions. Sums are fp32.
// Infinities and NaN: what a 16-row tile shares can reach a row that does not see it, and an infinity in one
// piece has no second piece. A row whose m, l or O is not finite is therefore computed again one key at a
// time in fp32, of the keys it sees alone.
#include <algorithm>

#include "dcq_attn.h"
#include "dcq_common.h"
#include "dcq_kernels.h"
#include "dcq_kv_row.h"
#include "dcq_search.h"

namespace dcq {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 16;          // query rows of a tile
constexpr int kTreeWaves = 4;      // waves of a workgroup, a share of the keys each
constexpr float kPieces = 128.0f;  // of the weights in O: 2^15 at most before the reference is raised

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
    __device__ __forceinline__ f32x4 scores(int j, const f16x8 (&qh)[S], const f16x8 (&ql)[S]) const {
        f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const f16x8 f = as_f16x8(k[j][s].x, k[j][s].y, k[j][s].z, k[j][s].w);
            lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, ql[s], lo, 0, 0, 0);
            hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, qh[s], hi, 0, 0, 0);
        }
        return hi + lo;
    }
    __device__ __forceinline__ void weigh(const f16x8 ph, const f16x8 pl, f32x4 (&o)[U][4]) const {
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
                o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, pl, o[u][e], 0, 0, 0);
                o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, ph, o[u][e], 0, 0, 0);
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
    __device__ __forceinline__ f32x4 scores(int j, const f16x8 (&qh)[S], const f16x8 (&ql)[S]) const {
        f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const f16x2 d = as_f16x2(kd[j][s] | kd[j][s] << 16);
            const uint32_t w[2] = {k[j][s].x, k[j][s].y};
            Pieces p[4];
#pragma unroll
            for (int t = 0; t < 4; ++t)
                p[t] = q8_pieces(int8_pair(__builtin_amdgcn_perm(0u, w[t / 2], t % 2 ? 0x0c030c02u : 0x0c010c00u)), d);
            const f16x8 fh = as_f16x8(as_u32(p[0].h), as_u32(p[1].h), as_u32(p[2].h), as_u32(p[3].h));
            const f16x8 fl = as_f16x8(as_u32(p[0].l), as_u32(p[1].l), as_u32(p[2].l), as_u32(p[3].l));
            lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl, qh[s], lo, 0, 0, 0);
            lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh, ql[s], lo, 0, 0, 0);
            hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh, qh[s], hi, 0, 0, 0);
        }
        return hi + lo;
    }
    __device__ __forceinline__ void weigh(const f16x8 ph, const f16x8 pl, f32x4 (&o)[U][4]) const {
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
                o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fl, ph, o[u][e], 0, 0, 0);
                o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh, pl, o[u][e], 0, 0, 0);
                o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fh, ph, o[u][e], 0, 0, 0);
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
    __device__ __forceinline__ f32x4 scores(const f32x4 (&q)[S]) const {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;  // two sums: half the roundings in a row
#pragma unroll
        for (int s = 0; s < S; ++s) {
            a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][0], q[s][0], a, 0, 0, 0);
            b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][1], q[s][1], b, 0, 0, 0);
            a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][2], q[s][2], a, 0, 0, 0);
            b = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][3], q[s][3], b, 0, 0, 0);
        }
        return a + b;
    }
    __device__ __forceinline__ void weigh(const float (&p)[4], f32x4 (&o)[U][4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[u][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][u][e], p[i] * kPieces, o[u][e], 0, 0, 0);
    }
};

// One step of the online softmax: scores of the lane's N keys of its row (-inf: not seen) to weights.
template <int N, int U>
__device__ __forceinline__ void softmax_step(float (&s)[N], float& m, float& l, f32x4 (&o)[U][4]) {
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__any(mx > m + 8.0f)) {
        const float m_new = mx > m + 8.0f ? __builtin_ceilf(mx) : m;
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        l *= alpha;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[u][e] *= alpha;
        m = m_new;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
        l += s[i];
    }
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

struct TreeSmem {
    float o[kTreeWaves][kTile][68];  // 64 dims of the waves' sums; pitch: 16-byte aligned, 4 banks apart
    float m[kTreeWaves][kTile], l[kTreeWaves][kTile];
    uint32_t again;  // rows to compute again
};

// What a workgroup of a sequence works on (uniform).
struct TreeJob {
    int seq, h_kv, row0, n_rows, n_draft, past;
    int k_begin, k_end;  // cached keys
    bool drafts;         // and the drafted ones
};

__device__ __forceinline__ int page_of(const TreeArgs& a, int seq, int lb) {
    if (a.n_table <= 0) return -1;
    const int blk = a.tables[(int64_t)seq * a.table_stride + min(lb, a.n_table - 1)];
    return lb < a.n_table && blk < a.n_blocks ? blk : -1;
}

__device__ __forceinline__ bool draft_seen(const TreeArgs& a, int seq, int tok, int i) {
    if (!a.mask) return i <= tok;
    return (a.mask[((int64_t)seq * a.n_tokens + tok) * a.words + i / 64] >> (i % 64)) & 1;
}

// One row again, key by key in fp32, by the whole workgroup: each wave takes every fourth key, its lanes dims
// lane + 64 u. Leaves the row's m and l in sm.m[0][0], sm.l[0][0] and returns the thread's dim of O (tid < HD).
template <int CT, int HD>
__device__ __forceinline__ float tree_row_again(const TreeArgs& a, const TreeJob& w, TreeSmem& sm, int row) {
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
    for (int t = w.k_begin + wave; t < w.k_end; t += kTreeWaves) {
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
    for (int t = wave; w.drafts && t < w.n_draft; t += kTreeWaves) {
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
    for (int k = 0; k < kTreeWaves; ++k) mx = fmaxf(mx, sm.m[k][0]);
#pragma unroll
    for (int k = 0; k < kTreeWaves; ++k) {
        const float c = ref_factor(sm.m[k][0], sm.l[k][0], mx);
        ls += sm.l[k][0] * c;
        if (tid < HD) o += so[k * HD + tid] * c;
    }
    __syncthreads();
    if (tid == 0) sm.m[0][0] = mx, sm.l[0][0] = ls;
    __syncthreads();
    return o;
}

// A tile of 16 rows over a share of the keys. Grid: (unit, tile) pairs with the tiles of a unit on one XCD
// (workgroup id % 8) one after another, as they read the same keys; unit = (sequence, split, KV head).
template <int CT, int HD>
__global__ void __launch_bounds__(64 * kTreeWaves) tree_attn_kernel(TreeArgs a) {
    constexpr int U = HD / 64, CK = tree_chunk<CT>(), NP = CK / kKvBlock;
    __shared__ TreeSmem sm;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, n = lane & 15;
    TreeJob w;
    int split, tile;
    {
        const int id = blockIdx.x, turn = id / (8 * a.tiles), rest = id % (8 * a.tiles);
        const int unit = turn * 8 + rest % 8;
        tile = rest / 8;
        if (unit >= a.units) return;
        w.h_kv = unit % a.n_head_kv;
        split = unit / a.n_head_kv % a.splits;
        w.seq = unit / a.n_head_kv / a.splits;
    }
    w.past = min(max(a.past[w.seq], 0), a.max_past);
    w.n_draft = a.n_draft ? min(max(a.n_draft[w.seq], 0), a.n_tokens) : a.n_tokens;
    w.n_rows = w.n_draft * a.rep;
    w.row0 = tile * kTile;
    const int n_split = max((w.past + a.kps - 1) / a.kps, 1);
    if (split >= n_split || (w.row0 >= w.n_rows && a.splits > 1)) return;  // the merge writes such rows' zeros
    w.k_begin = split * a.kps;
    w.k_end = w.row0 < w.n_rows ? min(w.past, w.k_begin + a.kps) : 0;
    w.drafts = split == n_split - 1 && w.row0 < w.n_rows;

    // ---- the lane's query row
    const int row = w.row0 + n;
    const bool q_ok = row < w.n_rows;
    const int tok = q_ok ? row / a.rep : 0, h = w.h_kv * a.rep + (q_ok ? row % a.rep : 0);
    const float* qp = a.q + ((int64_t)w.seq * a.n_tokens + tok) * a.q_stride + (int64_t)h * HD;
    auto load_q = [&](int d) {
        f32x4 t = *reinterpret_cast<const f32x4*>(qp + d);
        return q_ok ? t * a.scale_log2e : (f32x4){0.f, 0.f, 0.f, 0.f};
    };
    f32x4 o[U][4];
    float m = -INFINITY, l = 0.0f;  // l: of this lane's keys
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][e] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // ---- cached keys: the waves take steps of CK keys in turn
    const uint32_t head = (uint32_t)(a.sb / a.n_head_kv) * w.h_kv;
    const uint32_t sb = (uint32_t)a.sb, off_k = n * sb + head, off_v = 4 * g * sb + head;
    const int c0 = w.k_begin / CK + wave, c1 = (w.k_end + CK - 1) / CK;
    if (c0 < c1) {
        constexpr int S = CT == kTypeF32 ? HD / 16 : HD / 32;
        f16x8 qh[CT == kTypeF32 ? 1 : S], ql[CT == kTypeF32 ? 1 : S];
        f32x4 qf[CT == kTypeF32 ? S : 1];
        float qsc = 1.0f;
        if constexpr (CT == kTypeF32) {
#pragma unroll
            for (int s = 0; s < S; ++s) qf[s] = load_q(16 * s + 4 * g);
        } else {
            f32x4 t[S][2];
            float mx = 0.0f;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    t[s][k] = load_q(32 * s + 8 * g + 4 * k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(t[s][k][e]));
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const int ex = norm_exp(__float_as_uint(mx));
            const float f = pow2_bits(268 - ex);
            qsc = pow2_bits(ex - 14);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                f16x4 h0, l0, h1, l1;
                split4(t[s][0][0] * f, t[s][0][1] * f, t[s][0][2] * f, t[s][0][3] * f, h0, l0);
                split4(t[s][1][0] * f, t[s][1][1] * f, t[s][1][2] * f, t[s][1][3] * f, h1, l1);
                qh[s] = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
                ql[s] = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
        TreeKeys<CT, HD> t;
        int pages[NP], next[NP];
        auto pages_of = [&](int c, int (&p)[NP]) {
#pragma unroll
            for (int j = 0; j < NP; ++j) p[j] = __builtin_amdgcn_readfirstlane(page_of(a, w.seq, c * NP + j));
        };
        auto page_bytes = [&](int blk) {  // a missing page's loads read page 0; what they bring is cleared
            return ((int64_t)max(blk, 0) * a.n_layer + a.layer) * kKvBlock * a.sb;
        };
        pages_of(c0, pages);
#pragma unroll
        for (int j = 0; j < NP; ++j) t.load_k(j, a.k_arena + page_bytes(pages[j]), off_k, g);
#pragma unroll
        for (int j = 0; j < NP; ++j) t.load_v(j, a.v_arena + page_bytes(pages[j]), off_v, sb, n);
        for (int c = c0; c < c1; c += kTreeWaves) {
            const bool more = c + kTreeWaves < c1;
            if (more) pages_of(c + kTreeWaves, next);
            const int left = w.k_end - c * CK;  // keys of the step, if fewer than CK
            bool whole = left >= CK;
#pragma unroll
            for (int j = 0; j < NP; ++j) whole &= pages[j] >= 0;
            if (!whole) {  // zero rows for missing pages; no rows past the last key
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    if (pages[j] < 0) t.zero_k(j);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (pages[j] < 0 || 16 * j + 4 * g + i >= left) t.zero_v(j, i);
                }
            }
            float s[4 * NP];
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                f32x4 r;
                if constexpr (CT == kTypeF32)
                    r = t.scores(qf);
                else
                    r = t.scores(j, qh, ql) * qsc;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * j + i] = left >= CK || 16 * j + 4 * g + i < left ? r[i] : -INFINITY;
            }
            if (more) {
#pragma unroll
                for (int j = 0; j < NP; ++j) t.load_k(j, a.k_arena + page_bytes(next[j]), off_k, g);
            }
            softmax_step<4 * NP, U>(s, m, l, o);
            if constexpr (CT == kTypeF32) {
                t.weigh(s, o);
            } else {
                f16x4 h0, l0, h1, l1;
                split4(s[0] * kPieces, s[1] * kPieces, s[2] * kPieces, s[3] * kPieces, h0, l0);
                split4(s[4] * kPieces, s[5] * kPieces, s[6] * kPieces, s[7] * kPieces, h1, l1);
                t.weigh(__builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7),
                        __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7), o);
            }
            if (more) {
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    t.load_v(j, a.v_arena + page_bytes(next[j]), off_v, sb, n);
                    pages[j] = next[j];
                }
            }
        }
    }

    // ---- drafted keys, 16 at a time
    if (w.drafts && 16 * wave < w.n_draft) {
        constexpr int S = HD / 16;
        f32x4 qf[S];
#pragma unroll
        for (int s = 0; s < S; ++s) qf[s] = load_q(16 * s + 4 * g);
        const uint32_t rs = (uint32_t)(a.kv_stride * 4);
        for (int k0 = 16 * wave; k0 < w.n_draft; k0 += 16 * kTreeWaves) {
            const int left = w.n_draft - k0;
            const int64_t base = ((int64_t)w.seq * a.n_tokens + k0) * a.kv_stride + (int64_t)w.h_kv * HD;
            TreeKeys<kTypeF32, HD> t;
            t.load_k(0, reinterpret_cast<const uint8_t*>(a.k_cur + base), min(n, left - 1) * rs, g);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                t.load_v_key(i, reinterpret_cast<const uint8_t*>(a.v_cur + base), min(4 * g + i, left - 1) * rs, n);
            uint32_t seen;  // bit i: key 4 g + i
            if (a.mask)
                seen = (uint32_t)(a.mask[((int64_t)w.seq * a.n_tokens + tok) * a.words + k0 / 64] >> (k0 % 64 + 4 * g));
            else
                seen = (1u << min(max(tok + 1 - k0 - 4 * g, 0), 4)) - 1u;
            const f32x4 r = t.scores(qf);
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = 4 * g + i < left;
                s[i] = in && (seen >> i & 1) ? r[i] : -INFINITY;
                if (!in) t.zero_v(0, i);
            }
            softmax_step<4, U>(s, m, l, o);
            t.weigh(s, o);
        }
    }

    // ---- the waves' sums together, 64 dims at a time: thread -> row tid / 16, 4 dims
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (lane < kTile) sm.m[wave][lane] = m, sm.l[wave][lane] = l;
    if (tid == 0) sm.again = 0u;
    __syncthreads();
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kTreeWaves; ++k) mx = fmaxf(mx, sm.m[k][n]);
    const float c = ref_factor(m, l, mx) * (1.0f / kPieces);
    const int r = tid >> 4, d4 = 4 * (tid & 15), orow = w.row0 + r;
    float rm = -INFINITY, rl = 0.0f;
#pragma unroll
    for (int k = 0; k < kTreeWaves; ++k) rm = fmaxf(rm, sm.m[k][r]);
#pragma unroll
    for (int k = 0; k < kTreeWaves; ++k) rl += sm.l[k][r] * ref_factor(sm.m[k][r], sm.l[k][r], rm);
    const bool live = orow < w.n_rows, direct = a.splits == 1;
    const int otok = orow / a.rep, oh = w.h_kv * a.rep + orow % a.rep;
    const int64_t trow = (int64_t)w.seq * a.n_tokens + otok, wrow = (int64_t)split * a.rows + trow * a.n_head + oh;
    auto store4 = [&](int d, f32x4 v) {
        if (direct) {
            if (otok < a.n_tokens) {
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
        for (int k = 1; k < kTreeWaves; ++k) v += *reinterpret_cast<const f32x4*>(&sm.o[k][r][d4]);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= !(fabsf(v[e]) < INFINITY);
        store4(64 * u + d4, v);
    }
    if (!direct && live && d4 == 0) a.ws_ml[2 * wrow] = rm, a.ws_ml[2 * wrow + 1] = rl;
    if (bad && live) atomicOr(&sm.again, 1u << r);
    __syncthreads();
    for (uint32_t again = sm.again; again; again &= again - 1) {
        const int rr = __builtin_ctz(again), arow = w.row0 + rr;
        const float v = tree_row_again<CT, HD>(a, w, sm, arow);
        const float am = sm.m[0][0], al = sm.l[0][0];
        const int at = arow / a.rep, ah = w.h_kv * a.rep + arow % a.rep;
        const int64_t tr = (int64_t)w.seq * a.n_tokens + at, wr = (int64_t)split * a.rows + tr * a.n_head + ah;
        if (tid < HD) {
            if (direct)
                a.out[tr * a.out_stride + (int64_t)ah * HD + tid] = al != 0.0f ? v / al : 0.0f;
            else
                a.ws_o[wr * HD + tid] = v;
        }
        if (!direct && tid == 0) a.ws_ml[2 * wr] = am, a.ws_ml[2 * wr + 1] = al;
        __syncthreads();
    }
}

// The merge of a sequence's splits: M = max m, L = sum l 2^(m - M), out = sum o 2^(m - M) / L, zeros for a row
// that saw no key or has no drafted token. P lanes share 4 outputs, lane p the splits p, p + P, ...
template <int P>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a, int hd) {
    constexpr int NS = 4;  // splits of a lane whose loads are issued together
    const int q4 = hd / 4;
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / P;
    const int p = threadIdx.x & (P - 1);
    const bool in = unit < a.rows * q4;
    const int64_t row = in ? unit / q4 : 0;
    const int d = in ? (int)(unit % q4) * 4 : 0;
    const int64_t trow = row / a.n_head;
    const int h = (int)(row % a.n_head), seq = (int)(trow / a.n_tokens), tok = (int)(trow % a.n_tokens);
    const int past = min(max(a.past[seq], 0), a.max_past);
    const int n_draft = a.n_draft ? min(max(a.n_draft[seq], 0), a.n_tokens) : a.n_tokens;
    const int n_split = tok < n_draft ? max((past + a.kps - 1) / a.kps, 1) : 0;
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
            ov[k] = s < n_split ? *reinterpret_cast<const f32x4*>(a.ws_o + r * hd + d) : (f32x4){0.f, 0.f, 0.f, 0.f};
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
    if (!in || p != 0) return;
    float* out = a.out + trow * a.out_stride + (int64_t)h * hd + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = l != 0.0f ? acc[e] / l : 0.0f;
}

// ---------------------------------------------------------------- host side
struct TreePlan {
    int tiles, splits, kps;
};

// Key splits: workgroups until about three per CU have work, 128 keys (a step of each wave) at the least.
static TreePlan tree_plan(int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past) {
    TreePlan p{};
    p.tiles = (n_tokens * (n_head / n_head_kv) + kTile - 1) / kTile;
    const int64_t base = (int64_t)p.tiles * n_head_kv * n_seqs, want = std::max<int64_t>(1, (3 * cu_count() + base - 1) / base);
    p.kps = (int)std::max<int64_t>(128, round_up((max_past + want - 1) / want, 128));
    p.splits = std::max(1, (max_past + p.kps - 1) / p.kps);
    return p;
}

size_t tree_workspace_bytes(int hd, int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past) {
    const TreePlan p = tree_plan(n_head, n_head_kv, n_seqs, n_tokens, max_past);
    if (p.splits <= 1) return 0;
    const int64_t rows = (int64_t)p.splits * n_seqs * n_tokens * n_head;
    return round_up(rows * hd * 4, 256) + round_up(rows * 2 * 4, 256);
}

template <int P>
static void launch_tree_merge(const TreeArgs& a, int hd, hipStream_t st) {
    const int64_t threads = a.rows * (hd / 4) * P;
    hipLaunchKernelGGL((tree_merge_kernel<P>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a, hd);
}

hipError_t launch_tree_attention(int ct, int hd, TreeArgs a, void* ws, hipStream_t st) {
    const TreePlan p = tree_plan(a.n_head, a.n_head_kv, a.n_seqs, a.n_tokens, a.max_past);
    a.rep = a.n_head / a.n_head_kv;
    a.tiles = p.tiles, a.splits = p.splits, a.kps = p.kps;
    a.rows = (int64_t)a.n_seqs * a.n_tokens * a.n_head;
    const int64_t units = (int64_t)a.n_seqs * p.splits * a.n_head_kv;
    const int64_t wgs = (units + 7) / 8 * 8 * p.tiles;
    if (wgs > INT32_MAX || a.rows * (hd / 4) * 32 > (int64_t)INT32_MAX * 256) return hipErrorInvalidValue;
    a.units = (int)units;
    if (p.splits > 1) {
        a.ws_o = static_cast<float*>(ws);
        a.ws_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + round_up(p.splits * a.rows * hd * 4, 256));
    }
    const dim3 grid((unsigned)wgs);
#define DCQ_TREE_CASE(C, H)                                                                           \
    if (ct == C && hd == H) {                                                                         \
        hipLaunchKernelGGL((tree_attn_kernel<C, H>), grid, dim3(64 * kTreeWaves), 0, st, a);          \
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
    if (p.splits <= 4)
        launch_tree_merge<1>(a, hd, st);
    else if (p.splits <= 32)
        launch_tree_merge<8>(a, hd, st);
    else
        launch_tree_merge<32>(a, hd, st);
    return hipGetLastError();
}

}  // namespace dcq
