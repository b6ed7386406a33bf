// dcq_search.h — search over the paged KV cache: what dcq_tree.hip, dcq_pages.hip and dcq_beam.hip compute.
// Arguments are checked by the caller; entries of device arrays that are out of their range are clamped or
// skipped by the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dcq {

// dcq_tree.hip: drafted tokens of several sequences over their cached keys. rep .. units and what follows is
// the launcher's.
struct TreeArgs {
    const uint8_t* k_arena;
    const uint8_t* v_arena;
    int n_blocks, n_layer, layer;
    int64_t sb;  // slot bytes
    const int32_t* tables;  // [n_seqs][n_table]
    int64_t table_stride;
    int n_table;
    const int32_t* past;     // [n_seqs], no more than max_past
    const int32_t* n_draft;  // [n_seqs], or null: n_tokens each
    const uint64_t* mask;    // [n_seqs][n_tokens][words], or null: token j sees drafted tokens 0 .. j
    int max_past, words;
    const float* q;
    int64_t q_stride;  // floats between rows
    const float* k_cur;
    const float* v_cur;
    int64_t kv_stride;
    float* out;
    int64_t out_stride;
    int n_seqs, n_tokens, n_head, n_head_kv;
    float scale_log2e;
    int rep, tiles, tiles16, splits, kps, units, share, hist_wgs, draft_wgs;
    int64_t rows;  // n_seqs * n_tokens * n_head
    float* ws_o;   // [splits][rows][HD]
    float* ws_ml;  // [splits][rows][2]
    int* ws_kps;   // keys per split, where the device chooses them
};
size_t tree_workspace_bytes(int hd, int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past);
// Whether a launch holds the call's workgroups.
bool tree_fits(int ct, int hd, int n_head, int n_head_kv, int n_seqs, int n_tokens, int max_past);
hipError_t launch_tree_attention(int ct, int hd, TreeArgs a, void* ws, hipStream_t st);

// dcq_pages.hip
struct PathArgs {
    int ct;
    uint8_t* k_arena;
    uint8_t* v_arena;
    int n_blocks, n_layer;
    int64_t row_elems, sb;
    const int32_t* tables;
    int64_t table_stride;
    int n_table;
    const int32_t* past;
    const int32_t* path;  // [n_seqs][max_path]: drafted token of each accepted place
    int64_t path_stride;
    const int32_t* n_path;  // or null: max_path each
    int max_path;
    const float* k_cur;  // [n_layer][n_seqs * n_tokens][row_elems]
    const float* v_cur;
    int64_t layer_stride, kv_stride;  // floats
    int n_seqs, n_tokens;
};
hipError_t launch_path_write(const PathArgs& a, hipStream_t st);

// Whether a launch counts the pieces of that many pages' copies.
bool copies_fit(int64_t max_pages, int64_t page_bytes);

struct ForkArgs {
    const int32_t* tables;
    int64_t table_stride;
    int n_table;
    const int32_t* lengths;
    int n_seqs;
    const int32_t* parents;
    int n_children;
    const int32_t* refs;
    int n_blocks;
    int32_t* tables_out;
    int64_t tables_out_stride;
    int32_t* lengths_out;
    int32_t* refs_out;
    int32_t* missing;
    int32_t* rank;  // from here on the launcher's, in the workspace
    int32_t* plan;
    int32_t* users;
    int32_t* first;
};
size_t fork_workspace_bytes(int64_t n_blocks, int64_t n_children);
hipError_t launch_fork(ForkArgs a, void* k_arena, void* v_arena, int64_t page_bytes, void* ws, hipStream_t st);

struct CompactArgs {
    const int32_t* tables;
    int64_t table_stride;
    int n_table;
    const int32_t* lengths;
    int n_seqs;
    const int32_t* refs;
    int n_blocks;
    int32_t* tables_out;
    int64_t tables_out_stride;
    int32_t* refs_out;
    int32_t* n_live;
    int32_t* rank;
    int32_t* plan;
};
size_t compact_workspace_bytes(int64_t n_blocks);
hipError_t launch_compact(CompactArgs a, void* k_arena, void* v_arena, int64_t page_bytes, void* ws, hipStream_t st);

// The best continuations of beams (dcq_beam.hip): logits F32 or F16.
constexpr int kBeamMaxBeams = 256;
struct BeamArgs {
    const void* x;
    int64_t stride;  // elements between rows
    int n_beams, vocab;
    const float* beam;
    int n_out;
    float* scores;
    int32_t* parents;
    int32_t* tokens;
    int chunks;  // from here on the launcher's
    double* stat_sum;
    float* stat_ref;
    uint64_t* cand;  // [rows][chunks][n_out]
};
size_t beam_workspace_bytes(int64_t n_batch, int n_beams, int vocab, int n_out);
hipError_t launch_beam_select(int type, BeamArgs a, int64_t n_batch, void* ws, hipStream_t st);

}  // namespace dcq
