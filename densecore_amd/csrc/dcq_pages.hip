// dcq_pages.hip — the pages of the paged KV cache between two steps of a search: the accepted path's rows
// into their slots, forks of sequences, and compaction. All of it moves bytes; the plans are whole numbers.
//
// A page is block b of both arenas: n_layer * 16 slots in a row, a multiple of 16 bytes. refs[b] counts the
// sequences (of this call or not) that hold page b; a page is free where refs[b] <= 0 and, in a fork, no child
// holds it (counts that are too low must not make it the source and the target of copies). Sequence i holds the
// first ceil(length / 16) entries of its table row; entries outside [0, n_blocks) hold nothing.
//
// Kernels:
//   path_write_kernel    accepted token rows of every layer into their sequences' slots (bytes of kv_write)
//   fork_count_kernel    the children's tables, and the counts without the parents' and with the children's
//   fork_plan_kernel     who keeps a partial last page, who gets a copy and where, and a few pages' copies
//   compact_kernel       a small compaction: holes, moving pages, tables, counts and copies
//   compact_plan_kernel  the holes among the first n_live pages and the pages that move there; one workgroup
//   copy_pages_kernel    whole pages (from, to) of both arenas, and the tables and counts after a compaction
#include <algorithm>

#include "dcq_common.h"
#include "dcq_kernels.h"
#include "dcq_kv_row.h"
#include "dcq_search.h"

namespace dcq {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

__device__ __forceinline__ int pages_of_length(int length, int n_table) {
    return min((int)(((int64_t)max(length, 0) + kKvBlock - 1) / kKvBlock), n_table);
}

// ---------------------------------------------------------------- accepted paths
// One workgroup per (accepted token, layer, arena): a row is read and written once, all of it in flight together, and a
// launch is the whole cost (16 sequences, 5 tokens, 36 layers x 1024 F32: 11.4 us for 47 MB, 4.1 TB/s; one sequence of
// 28 layers 3.1 us).
__global__ void __launch_bounds__(256) path_write_kernel(PathArgs a) {
    const int seq = blockIdx.x / a.max_path, j = blockIdx.x % a.max_path, layer = blockIdx.y;
    const int n = a.n_path ? a.n_path[seq] : a.max_path;
    const int tok = a.path[(int64_t)seq * a.path_stride + j];
    const int past = a.past[seq];
    if (j >= n || tok < 0 || tok >= a.n_tokens || past < 0) return;
    const int64_t pos = (int64_t)past + j;
    if (pos / kKvBlock >= a.n_table) return;
    const int blk = a.tables[(int64_t)seq * a.table_stride + pos / kKvBlock];
    if (blk < 0 || blk >= a.n_blocks) return;
    uint8_t* arena = blockIdx.z ? a.v_arena : a.k_arena;
    const float* cur = blockIdx.z ? a.v_cur : a.k_cur;
    const float* x = cur + (int64_t)layer * a.layer_stride + ((int64_t)seq * a.n_tokens + tok) * a.kv_stride;
    uint8_t* dst = const_cast<uint8_t*>(kv_slot(arena, blk, a.n_layer, layer, (int)(pos % kKvBlock), a.sb));
    kv_encode_row(a.ct, dst, x, a.row_elems);
}

hipError_t launch_path_write(const PathArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(path_write_kernel, dim3((unsigned)(a.n_seqs * a.max_path), (unsigned)a.n_layer, 2), dim3(256), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- whole pages
// A compaction's tables and counts after the move, the items first, first + step, ...; target(page): where a page at
// `live` or above goes.
template <class Target>
__device__ __forceinline__ void compact_map(const CompactArgs& a, int live, int first, int step, Target target) {
    const int64_t entries = (int64_t)a.n_seqs * a.n_table;
    for (int64_t i = first; i < entries + a.n_blocks; i += step) {
        if (i < entries) {
            const int row = (int)(i / a.n_table), at = (int)(i % a.n_table);
            int page = a.tables[(int64_t)row * a.table_stride + at];
            if (at < pages_of_length(a.lengths[row], a.n_table) && page >= live && page < a.n_blocks && a.refs[page] > 0)
                page = target(page);
            a.tables_out[(int64_t)row * a.tables_out_stride + at] = page;
        } else {
            const int page = (int)(i - entries), n = a.refs[page];
            if (page < live ? n > 0 : n <= 0) {
                a.refs_out[page] = n;
            } else if (page >= live) {  // moves: the pair's counts; a hole's comes from its pair
                a.refs_out[target(page)] = n;
                a.refs_out[page] = 0;
            }
        }
    }
}

// Pages of both arenas, pair(i) = {from, to} for i < n, in pieces of 16 KB dealt in turn to `of` groups of 256 threads:
// the part of group `group`, thread `lane` of it. Bound by HBM (501 pages of 36 layers x 512 F32, half of them moved:
// 108 us for 552 MB, 5.1 TB/s; four groups a CU instead of eight 112).
constexpr int kPiece = 16384;
template <class Pair>
__device__ __forceinline__ void copy_pages(uint8_t* k_arena, uint8_t* v_arena, int64_t page_bytes, int n, int group, int of,
                                           int lane, Pair pair) {
    const uint32_t per_page = (uint32_t)((page_bytes + kPiece - 1) / kPiece), pieces = 2 * per_page * n;
    for (uint32_t i = group; i < pieces; i += of) {
        const uint32_t unit = i / per_page;
        const int64_t at = (int64_t)(i - unit * per_page) * kPiece, left = page_bytes - at;
        const int2 p = pair(unit / 2);
        uint8_t* arena = unit % 2 ? v_arena : k_arena;
        const uint8_t* src = arena + p.x * page_bytes + at;
        uint8_t* dst = arena + p.y * page_bytes + at;
        uint4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int o = 16 * (lane + 256 * u);
            if (o < left) w[u] = ld16(src + o);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int o = 16 * (lane + 256 * u);
            if (o < left) *reinterpret_cast<uint4*>(dst + o) = w[u];
        }
    }
}

// plan[0] pairs (from, to) at plan[2 + 2 i].
template <bool MAP>
__global__ void __launch_bounds__(256) copy_pages_kernel(uint8_t* k_arena, uint8_t* v_arena, const int32_t* plan,
                                                         int64_t page_bytes, int map_wgs, CompactArgs c) {
    if (MAP && (int)blockIdx.x < map_wgs) {
        compact_map(c, c.plan[1], (int)blockIdx.x * 256 + (int)threadIdx.x, map_wgs * 256,
                    [&](int page) { return c.plan[3 + 2 * c.rank[page]]; });
        return;
    }
    const int wg = blockIdx.x - (MAP ? map_wgs : 0), wgs = gridDim.x - (MAP ? map_wgs : 0);
    copy_pages(k_arena, v_arena, page_bytes, plan[0], wg, wgs, threadIdx.x,
               [&](int i) { return make_int2(plan[2 + 2 * i], plan[3 + 2 * i]); });
}

static int64_t copy_pieces(int64_t max_pages, int64_t page_bytes) {
    return 2 * max_pages * ((page_bytes + kPiece - 1) / kPiece);
}
bool copies_fit(int64_t max_pages, int64_t page_bytes) { return copy_pieces(max_pages, page_bytes) <= INT32_MAX; }

// Groups of 256 threads that copy up to max_pages pages while they make the plan themselves, one launch for all: as
// many as pieces, at most eight per CU; 0 where there are more pieces and the plan has a launch before the copies'.
// One launch | two, us a call: 4 beams of 28 layers x 1024 F16 12.2 | 15.3, 120 pages of 16 layers x 512 F16 11.1 |
// 14.5; 128 beams of 36 layers x 1024 F16 52 | 50.5, 501 pages of 36 layers x 512 F32 114.4 | 113.7: 512 workgroups
// then wait for their own plans with nothing in flight, and longer than one does.
static int copies_beside_plan(int64_t max_pages, int64_t page_bytes) {
    const int64_t pieces = copy_pieces(max_pages, page_bytes);
    return pieces > 8 * (int64_t)cu_count() ? 0 : (int)std::max<int64_t>(pieces, 1);
}

// map: a compaction's tables and counts, in workgroups before the copying ones.
static hipError_t launch_copy_pages(void* k_arena, void* v_arena, const int32_t* plan, int64_t max_pages,
                                    int64_t page_bytes, const CompactArgs* map, hipStream_t st) {
    const int wgs = (int)std::min<int64_t>(std::max<int64_t>(copy_pieces(max_pages, page_bytes), 1), 8 * (int64_t)cu_count());
    uint8_t *k = static_cast<uint8_t*>(k_arena), *v = static_cast<uint8_t*>(v_arena);
    if (map) {
        const int64_t items = (int64_t)map->n_seqs * map->n_table + map->n_blocks;
        const int map_wgs = (int)std::min<int64_t>((items + 255) / 256, 2 * (int64_t)cu_count());
        hipLaunchKernelGGL((copy_pages_kernel<true>), dim3((unsigned)(map_wgs + wgs)), dim3(256), 0, st, k, v, plan,
                           page_bytes, map_wgs, *map);
    } else {
        hipLaunchKernelGGL((copy_pages_kernel<false>), dim3((unsigned)wgs), dim3(256), 0, st, k, v, plan, page_bytes, 0,
                           CompactArgs{});
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------- scans of a plan's workgroup
// The thread's offset among the flags of the workgroup's threads, in thread order, and their number.
struct Scan {
    int before, total;
};
__device__ __forceinline__ Scan block_scan(bool flag, int* counts /* kPlanWaves */) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint64_t set = __ballot(flag);
    __syncthreads();  // counts of the scan before are read
    if (lane == 0) counts[wave] = __popcll(set);
    __syncthreads();
    Scan s{(int)__popcll(set & ((1ull << lane) - 1)), 0};
#pragma unroll
    for (int k = 0; k < kPlanWaves; ++k) {
        const int c = counts[k];
        s.before += k < wave ? c : 0;
        s.total += c;
    }
    return s;
}

// ---------------------------------------------------------------- forks
// The counts: refs_out = refs - one for each page a sequence holds + one for each page a child takes over, and
// the children's tables and lengths. The part of one (sequence or child, table entry). length_of(i): sequence i's,
// 0 .. 16 n_table; parent_of(i): child i's, or -1; tail(i, page): the partial last page of child i; users: see
// fork_count_tail. write: tables and lengths.
constexpr int kHeld = 1 << 30;
template <class Length, class Parent, class Tail>
__device__ __forceinline__ void fork_count_entry(const ForkArgs& a, int row, int at, bool write, int32_t* refs, int32_t* users,
                                                 Length length_of, Parent parent_of, Tail tail) {
    const bool child = row >= a.n_seqs;
    const int i = child ? row - a.n_seqs : row, from = child ? parent_of(i) : i;
    const int length = from >= 0 ? length_of(from) : 0;
    int page = -1;
    if (at < pages_of_length(length, a.n_table)) {
        page = a.tables[(int64_t)from * a.table_stride + at];
        const bool real = page >= 0 && page < a.n_blocks;
        if (real) atomicAdd(refs + page, child ? 1 : -1);
        if (real && child) atomicOr(users + page, kHeld);
        if (child && real && at == length / kKvBlock) tail(i, page);
    }
    if (!child || !write) return;
    a.tables_out[(int64_t)i * a.tables_out_stride + at] = page;
    if (at == 0) a.lengths_out[i] = length;
}
__device__ __forceinline__ int fork_length(const ForkArgs& a, int i) {
    return min(max(a.lengths[i], 0), a.n_table * kKvBlock);
}
__device__ __forceinline__ int fork_parent(const ForkArgs& a, int i) {
    const int p = a.parents[i];
    return p >= 0 && p < a.n_seqs ? p : -1;
}

// Of a partial last page: the children that would write into it (beside kHeld, of all pages that a child holds), and
// the first of them.
__device__ __forceinline__ void fork_count_tail(int32_t* users, int32_t* first, int child, int page) {
    atomicAdd(users + page, 1);
    atomicMin(first + page, child);
}

__global__ void __launch_bounds__(256) fork_refs_kernel(ForkArgs a) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < a.n_blocks) a.refs_out[i] = a.refs[i], a.users[i] = 0, a.first[i] = INT32_MAX;
}

__global__ void __launch_bounds__(256) fork_count_kernel(ForkArgs a) {
    const int64_t entries = (int64_t)(a.n_seqs + a.n_children) * a.n_table;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256)
        fork_count_entry(
            a, (int)(i / a.n_table), (int)(i % a.n_table), true, a.refs_out, a.users,
            [&](int k) { return fork_length(a, k); }, [&](int k) { return fork_parent(a, k); },
            [&](int k, int page) { fork_count_tail(a.users, a.first, k, page); });
}

// LDS: the counts are in LDS. With arenas, every workgroup makes the whole plan for itself, the first one writes what
// the caller gets, and all copy the pages; without, one workgroup, and the plan goes to the workspace. Not LDS: that
// too, and refs_out, users and first hold the counts already.
template <bool LDS>
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(ForkArgs a, uint8_t* k_arena, uint8_t* v_arena,
                                                                 int64_t page_bytes) {
    extern __shared__ int32_t lds[];
    __shared__ int counts[kPlanWaves];
    const int tid = threadIdx.x;
    const bool lead = !LDS || blockIdx.x == 0;
    int32_t* tails = lds;                                        // [n_children]: partial last page, or -1
    int32_t* fresh = tails + a.n_children;                       // [n_children]: the copy's page, by its rank
    int32_t* from = fresh + a.n_children;                        // [n_children]: and the page it is of (LDS)
    int32_t* ranks = LDS ? from + a.n_children : a.rank;         // [n_children]
    int32_t* refs = LDS ? ranks + a.n_children : a.refs_out;     // [n_blocks]
    int32_t* users = LDS ? refs + a.n_blocks : a.users;          // [n_blocks]
    int32_t* first = LDS ? users + a.n_blocks : a.first;         // [n_blocks]
    if (LDS) {
        int32_t* parents = first + a.n_blocks;       // [n_children]
        int32_t* lengths = parents + a.n_children;  // [n_seqs]
        for (int i = tid; i < a.n_blocks; i += kPlanThreads) refs[i] = a.refs[i], users[i] = 0, first[i] = INT32_MAX;
        for (int i = tid; i < a.n_seqs; i += kPlanThreads) lengths[i] = fork_length(a, i);
        for (int i = tid; i < a.n_children; i += kPlanThreads) parents[i] = fork_parent(a, i), tails[i] = -1;
        __syncthreads();
        const int entries = (a.n_seqs + a.n_children) * a.n_table;
        for (int i = tid; i < entries; i += kPlanThreads)
            fork_count_entry(
                a, i / a.n_table, i % a.n_table, lead, refs, users, [&](int k) { return lengths[k]; },
                [&](int k) { return parents[k]; },
                [&](int k, int page) {
                    tails[k] = page;
                    fork_count_tail(users, first, k, page);
                });
    } else {
        for (int i = tid; i < a.n_children; i += kPlanThreads) {
            const int parent = fork_parent(a, i), length = parent >= 0 ? fork_length(a, parent) : 0;
            const int tail = length % kKvBlock ? a.tables[(int64_t)parent * a.table_stride + length / kKvBlock] : -1;
            tails[i] = tail < a.n_blocks ? tail : -1;
        }
    }
    __syncthreads();
    // ---- a child keeps its partial page if all who hold it are children that would write into it, and it is
    // the first of them; the others get copies, ranked in the children's order
    int copies = 0;
    for (int i0 = 0; i0 < a.n_children; i0 += kPlanThreads) {
        const int i = i0 + tid, tail = i < a.n_children ? tails[i] : -1;
        const bool copy = tail >= 0 && !(first[tail] == i && refs[tail] == (users[tail] & ~kHeld));
        const Scan s = block_scan(copy, counts);
        if (i < a.n_children) ranks[i] = copy ? copies + s.before : -1;
        copies += s.total;
    }
    // ---- as many free pages, the lowest first
    int found = 0;
    for (int i0 = 0; i0 < a.n_blocks && found < copies; i0 += kPlanThreads) {
        const int i = i0 + tid;
        const bool free = i < a.n_blocks && refs[i] <= 0 && users[i] == 0;
        const Scan s = block_scan(free, counts);
        if (free && found + s.before < copies) fresh[found + s.before] = i;
        found += s.total;
    }
    found = min(found, copies);
    __syncthreads();
    // ---- the copies' pages into tables, counts and the copy list
    for (int i = tid; i < a.n_children; i += kPlanThreads) {
        const int rank = ranks[i];
        if (rank < 0) continue;
        const int page = rank < found ? fresh[rank] : -1;
        if (lead) a.tables_out[(int64_t)i * a.tables_out_stride + a.lengths[a.parents[i]] / kKvBlock] = page;
        atomicAdd(refs + tails[i], -1);
        if (page >= 0) {
            refs[page] = 1;
            if (LDS) from[rank] = tails[i];
            if (!k_arena) {
                a.plan[2 + 2 * rank] = tails[i];
                a.plan[3 + 2 * rank] = page;
            }
        }
    }
    if (lead && tid == 0) {
        if (!k_arena) a.plan[0] = found;
        a.missing[0] = copies - found;
    }
    if (LDS) {
        __syncthreads();
        if (lead)
            for (int i = tid; i < a.n_blocks; i += kPlanThreads) a.refs_out[i] = refs[i];
        if (!k_arena) return;
        constexpr int groups = kPlanThreads / 256;
        copy_pages(k_arena, v_arena, page_bytes, found, (int)blockIdx.x * groups + tid / 256, (int)gridDim.x * groups,
                   tid % 256, [&](int i) { return make_int2(from[i], fresh[i]); });
    }
}

// Workspace: rank [n_children], the plan (its length, a spare word, the pairs), users and first [n_blocks].
size_t fork_workspace_bytes(int64_t n_blocks, int64_t n_children) {
    return (size_t)(round_up(n_children * 4, 256) + round_up((2 + 2 * n_children) * 4, 256) + 2 * round_up(n_blocks * 4, 256));
}

hipError_t launch_fork(ForkArgs a, void* k_arena, void* v_arena, int64_t page_bytes, void* ws, hipStream_t st) {
    uint8_t* w = static_cast<uint8_t*>(ws);
    a.rank = reinterpret_cast<int32_t*>(w), w += round_up((int64_t)a.n_children * 4, 256);
    a.plan = reinterpret_cast<int32_t*>(w), w += round_up((2 + 2 * (int64_t)a.n_children) * 4, 256);
    a.users = reinterpret_cast<int32_t*>(w), w += round_up((int64_t)a.n_blocks * 4, 256);
    a.first = reinterpret_cast<int32_t*>(w);
    const int64_t entries = (int64_t)(a.n_seqs + a.n_children) * a.n_table;
    // The counts in LDS (64 KB with the scans') while a workgroup's threads have few entries to see; beyond, the
    // counting alone takes longer than the launches it then gets. Plan in LDS | in three launches: 128 beams of 15 pages
    // 7.5 | 14.0 us on the device; 96 beams of 200 pages, 38912 entries, 12.9 in three.
    const int64_t words = 5 * (int64_t)a.n_children + 3 * (int64_t)a.n_blocks + a.n_seqs;
    uint8_t *k = static_cast<uint8_t*>(k_arena), *v = static_cast<uint8_t*>(v_arena);
    if (words <= 16000 && entries <= 32768) {
        const int groups = copies_beside_plan(a.n_children, page_bytes);
        hipLaunchKernelGGL((fork_plan_kernel<true>), dim3((unsigned)(groups ? (groups + 3) / 4 : 1)), dim3(kPlanThreads),
                           (size_t)words * 4, st, a, groups ? k : nullptr, groups ? v : nullptr, page_bytes);
        if (groups) return hipGetLastError();
    } else {
        hipLaunchKernelGGL(fork_refs_kernel, dim3((unsigned)((a.n_blocks + 255) / 256)), dim3(256), 0, st, a);
        const int64_t wgs = std::min<int64_t>((entries + 255) / 256, 4 * (int64_t)cu_count());
        hipLaunchKernelGGL(fork_count_kernel, dim3((unsigned)wgs), dim3(256), 0, st, a);
        hipLaunchKernelGGL((fork_plan_kernel<false>), dim3(1), dim3(kPlanThreads), 2 * (size_t)a.n_children * 4, st, a,
                           nullptr, nullptr, page_bytes);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_copy_pages(k_arena, v_arena, a.plan, a.n_children, page_bytes, nullptr, st);
}

// ---------------------------------------------------------------- compaction
// The plan, by a workgroup: hole(i, page), mover(i, page): the i-th hole below n_live, and the i-th page that moves.
struct CompactCounts {
    int live, movers;
};
template <class Hole, class Mover>
__device__ __forceinline__ CompactCounts compact_plan(const CompactArgs& a, int* counts, Hole set_hole, Mover set_mover) {
    const int tid = threadIdx.x;
    int live = 0;
    for (int i = tid; i < a.n_blocks; i += kPlanThreads) live += a.refs[i] > 0;
    live = (int)lanes_sum<64>((float)live);  // below 2^24
    if ((tid & 63) == 0) counts[tid >> 6] = live;
    __syncthreads();
    live = 0;
#pragma unroll
    for (int k = 0; k < kPlanWaves; ++k) live += counts[k];
    int holes = 0, movers = 0;
    for (int i0 = 0; i0 < a.n_blocks; i0 += kPlanThreads) {
        const int i = i0 + tid;
        const bool used = i < a.n_blocks && a.refs[i] > 0;
        const bool hole = i < live && !used, moves = used && i >= live;
        // a step's pages are below live, above, or (one step) on both sides
        if (i0 < live) {
            const Scan s = block_scan(hole, counts);
            if (hole) set_hole(holes + s.before, i);
            holes += s.total;
        }
        if (i0 + kPlanThreads > live) {
            const Scan s = block_scan(moves, counts);
            if (moves) set_mover(movers + s.before, i);
            movers += s.total;
        }
    }
    return {live, movers};
}

// rank [n_blocks]: of a page that moves, its place in the plan.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(CompactArgs a) {
    __shared__ int counts[kPlanWaves];
    const CompactCounts n = compact_plan(
        a, counts, [&](int i, int page) { a.plan[3 + 2 * i] = page; },
        [&](int i, int page) { a.plan[2 + 2 * i] = page, a.rank[page] = i; });
    if (threadIdx.x == 0) a.plan[0] = n.movers, a.plan[1] = n.live, a.n_live[0] = n.live;
}

// All in one launch: every workgroup makes the plan for itself, in LDS, and takes its part of the tables, counts and
// pages.
__global__ void __launch_bounds__(kPlanThreads) compact_kernel(CompactArgs a, uint8_t* k_arena, uint8_t* v_arena,
                                                               int64_t page_bytes) {
    extern __shared__ int32_t lds[];
    __shared__ int counts[kPlanWaves];
    int32_t *from = lds, *to = lds + a.n_blocks / 2;  // as many pages move as there are holes, half of all at the most
    const CompactCounts n = compact_plan(
        a, counts, [&](int i, int page) { to[i] = page; }, [&](int i, int page) { from[i] = page; });
    __syncthreads();
    const int tid = threadIdx.x, wg = blockIdx.x;
    if (wg == 0 && tid == 0) a.n_live[0] = n.live;
    compact_map(a, n.live, wg * kPlanThreads + tid, (int)gridDim.x * kPlanThreads, [&](int page) {
        int lo = 0, hi = n.movers - 1;  // from is in rising order
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (from[mid] < page)
                lo = mid + 1;
            else
                hi = mid;
        }
        return to[lo];
    });
    constexpr int groups = kPlanThreads / 256;
    copy_pages(k_arena, v_arena, page_bytes, n.movers, wg * groups + tid / 256, (int)gridDim.x * groups, tid % 256,
               [&](int i) { return make_int2(from[i], to[i]); });
}

size_t compact_workspace_bytes(int64_t n_blocks) {
    return (size_t)round_up(n_blocks * 4, 256) + (size_t)round_up((2 + n_blocks) * 4, 256);
}

hipError_t launch_compact(CompactArgs a, void* k_arena, void* v_arena, int64_t page_bytes, void* ws, hipStream_t st) {
    const int groups = copies_beside_plan(a.n_blocks / 2, page_bytes);
    if (groups) {  // at most nine pages per CU: the plan fits in LDS
        hipLaunchKernelGGL(compact_kernel, dim3((unsigned)((groups + 3) / 4)), dim3(kPlanThreads), (size_t)a.n_blocks * 4,
                           st, a, static_cast<uint8_t*>(k_arena), static_cast<uint8_t*>(v_arena), page_bytes);
        return hipGetLastError();
    }
    a.rank = static_cast<int32_t*>(ws);
    a.plan = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(ws) + round_up((int64_t)a.n_blocks * 4, 256));
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return launch_copy_pages(k_arena, v_arena, a.plan, a.n_blocks / 2, page_bytes, &a, st);
}

}  // namespace dcq
