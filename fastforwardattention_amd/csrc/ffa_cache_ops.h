// Host-side declarations of the operators next to the decode step: attention of a group of new
// tokens, the weight-summing decode step, and the moves of cache slots (path commit, eviction).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "ffa_host.h"

namespace ffa {

// ---------------------------------------------------------------------------------------
// Attention of a group of tokens.  The rows of a (sample, cache head) pair -- its tokens times
// its G query heads, row = token * G + head -- are cut into blocks of row_tiles * 16; a workgroup
// takes one row block over one piece of the keys, its waves every n-th tile of them.

// 16-key matrix tiles of a wave tile: 32 keys (16 in fp32) are what one product over keys takes; with
// one row tile and narrow heads the registers hold twice that, and a wave has twice the loads in flight.
constexpr int tree_tile_units(int elem_bytes, int head_dim, int row_tiles) {
    return (elem_bytes == 2 ? 2 : 1) * (row_tiles == 1 && head_dim <= 80 ? 2 : 1);
}

// Most 16-row matrix tiles a wave's registers hold.
constexpr int tree_row_tiles(int head_dim) { return head_dim == 256 ? 2 : 4; }

// Whether two waves a SIMD fit the registers.
constexpr bool tree_two_waves(int head_dim, int row_tiles) { return head_dim <= 128 && head_dim * row_tiles <= 256; }
// Whether there is a kernel of 8 waves beside the one of 4: where a wave's loads are too few for 4 of
// them to keep a CU's share of the memory busy.
constexpr bool tree_wide(int head_dim, int row_tiles) { return tree_two_waves(head_dim, row_tiles) && !(head_dim == 128 && row_tiles == 2); }

struct TreePlan {
    int row_tiles;        // 16-row matrix tiles a wave holds: 1 .. 4
    int row_blocks;       // workgroups a piece of keys is read by
    int waves;            // of a workgroup: 4, or 8 (tree_wide)
    int n_splits;         // pieces of the cached keys
    int tiles_per_split;  // wave tiles a piece holds
    int score_lds;        // weight-summing step: words of a row of scores held in LDS, 0 = in the workspace
};

struct TreeParams {
    const void *q, *k, *v;
    void *k_cache, *v_cache, *out;
    const int *parents, *first_keys, *lengths, *counts;
    long long q_stride[3], k_stride[3], v_stride[3], out_stride[3];  // (sample, head, token), elements
    float* ws_acc;       // [pairs, n_splits, rows, Dh], or unused with one piece
    float* ws_ml;        // [pairs, n_splits, rows, 2]: reference exponent and sum
    float* ws_scores;    // weight-summing step: [pairs, rows, score_stride], else nullptr
    float* key_weights;  // weight-summing step: [pairs, Lmax], else nullptr
    int score_stride;
    int score_lds;       // as in the plan
    int B, H, G, tokens, rows, Lmax, t;
    float scale_log2e;  // |softmax_scale| * log2(e), never zero
    int zero_rest;      // rows past a sample's count are set to zero
    int q_sign;         // sign of softmax_scale: Q enters with it
    int n_splits, tiles_per_split, row_blocks;
    unsigned splits_magic, H_magic, G_magic;  // tree_magic() of n_splits, H and G
};

// n / d = (n * tree_magic(d)) >> 32 while n * d < 2^32 (d > 1).
inline unsigned tree_magic(int d) { return d > 1 ? (unsigned)(0x100000000ull / (unsigned)d) + 1u : 0u; }

TreePlan plan_tree(int precision, int pairs, int rows, int head_dim, int t, bool weights, int cus);
int launch_tree(int precision, int head_dim, const TreeParams& P, const TreePlan& plan, void* stream);
int launch_tree_f16(const TreeParams& P, int head_dim, const TreePlan& plan, void* stream);
int launch_tree_bf16(const TreeParams& P, int head_dim, const TreePlan& plan, void* stream);
int launch_tree_f32(const TreeParams& P, int head_dim, const TreePlan& plan, void* stream);

// ---------------------------------------------------------------------------------------
// Moves of cache slots.  Pointers of up to kSlotCaches caches travel in the kernel arguments.
constexpr int kSlotCaches = 32;

struct CommitParams {
    void* k[kSlotCaches];
    void* v[kSlotCaches];
    const int *path, *accepted, *lengths;
    int path_len, n_caches, B, H, Lmax, t;
};
int launch_commit(const CommitParams& P, int head_dim, int elem_bytes, void* stream);

struct EvictParams {
    const void *k_src[kSlotCaches], *v_src[kSlotCaches];
    const float* w_src[kSlotCaches];
    void *k_dst[kSlotCaches], *v_dst[kSlotCaches];
    float* w_dst[kSlotCaches];
    const int *first_keys, *lengths;
    int* kept;  // [n_caches, B, H, keep]
    int n_caches, B, H, src_len, dst_len, t, keep, recent;
    int segment_batches;  // batches of a wave's walk through the kept slots
};
int launch_evict(const EvictParams& P, int head_dim, int elem_bytes, void* stream);

}  // namespace ffa
