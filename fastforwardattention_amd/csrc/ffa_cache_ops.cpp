// C ABI of the operators next to the decode step (attention of a group of tokens, the
// weight-summing step, path commit, eviction): argument validation, planning, workspace carving.
// Pure host C++; the kernels live in ffa_tree_kernels.h and ffa_slots.hip.
#include <stdint.h>

#include <algorithm>

#include "ffa_c_api.h"
#include "ffa_cache_ops.h"

using namespace ffa;

namespace {

// Most heads of a cache, and most query heads that share one of them.
constexpr int kTreeHeads = 4096;

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int ceil_div(int a, int b) { return (a + b - 1) / b; }

int compute_units() {
    const int cus = query_compute_units();
    return cus > 0 ? cus : 256;
}

int check_cache_shape(int precision, int B, int H, int Dh, int Lmax) {
    if (elem_bytes(precision) == 0) return FFA_ERR_DTYPE;
    if (Dh != 64 && Dh != 80 && Dh != 128 && Dh != 256) return FFA_ERR_HEAD_DIM;
    if (B <= 0 || H <= 0 || Lmax <= 0) return FFA_ERR_SHAPE;
    // Four chunk rows of a K cache are addressed with 32 bits from their first byte; pairs, heads and rows
    // are divided by multiplication with 32-bit factors (tree_magic), and pairs / 8 is a grid's y.
    if ((long long)B * H > (1ll << 18) || H > kTreeHeads || Lmax > (1 << 25)) return FFA_ERR_SHAPE;
    return FFA_OK;
}

// Weight-summing step: scores of the cached keys in whole wave tiles, the new token's behind them.
int score_stride_of(int t) { return (int)align_up((size_t)t, 64) + 64; }

struct TreeSizes {
    size_t acc = 0, ml = 0, scores = 0;
    size_t total() const { return acc + ml + scores; }
};

// With n_splits the most pieces the plan takes up to this t, which grows with t.
TreeSizes tree_sizes(int pairs, int rows, int head_dim, int n_splits, bool scores, int t) {
    TreeSizes s;
    if (n_splits > 1) s.acc = align_up((size_t)pairs * n_splits * rows * head_dim * sizeof(float), 256);
    if (n_splits > 1 || scores) s.ml = align_up((size_t)pairs * n_splits * rows * 2 * sizeof(float), 256);
    if (scores) s.scores = align_up((size_t)pairs * rows * score_stride_of(t) * sizeof(float), 256);
    return s;
}

// Scores of a piece are held in LDS, next to the merge buffer, up to this many words.
constexpr int kScoreLdsWords = 16384;

// Joining pieces costs a kernel, about 4 us: what 12 tiles take a workgroup (0.3 us a tile).
constexpr int kJoinTiles = 12;

struct TreeShape {
    int row_tiles, row_blocks, tile_keys, most_splits;
};

// 16-row tiles a workgroup may hold: more read the keys less often, but leave fewer waves a SIMD and cost more
// before the first key and after the last.  Measured, us in fp16 / bf16 / fp32, 64 rows (B x H x Dh):
//   one, where all workgroups of one tile run at once on few keys, against two: 1x32x128 t 500 12 and 16 / 12 and 14 /
//   19 and 22, t 1000 15 and 18 / 15 and 16 / 26 and 29; 1x32x256 t 1000 26 and 34 / 26 and 33 / 47 and 49; 1x32x80
//   t 100, 32 rows 8.5 and 10.6 / 8.3 and 11.0 / 10.4 and 12.2 (64 rows from t 500 on alike or up to 20 % the other way);
//   two up to 1280 keys, against four: 8x32x128 t 512 27 and 28 / 24 and 29 / 58 and 64, t 1280 43 and 43 / 39 and 45 /
//   121 and 123, but t 4000 137 and 110 / 129 and 112 / 337 and 338 (about 1500 to 2500 keys two are still 5 to 15 %
//   ahead); fp32 8x32x64 t 500 33 and 35, 11x32x64 t 800 59 and 77 (16x32x64 t 800 81 and 80);
//   four of 16-bit Dh 64, two of whose workgroups fit a CU, where there are more, against two: 16x32x64 t 0 14 and 18 /
//   14 and 18, t 600 28 and 33 / 28 and 33, t 4000 108 and 144 / 108 and 139 (8x32x64 t 0 10.9 and 9.6 / 11.5 and 9.9);
//   two of Dh 80, whose tiles take as many registers as Dh 96 would, against four: 16x32x80 t 1000 51 and 68 / 52 and
//   71 / 133 and 139, t 4000 166 and 164 / 163 and 169 / 450 and 444; 2x8(64) t 4000 35 and 46 / 36 and 48 / 108 and
//   122.  With fewer tiles two win on 64 rows (1x32x80 t 4000 21 and 25 / 22 and 26 / 40 and 44) and lose on 33 to 48,
//   which four read once (t 16000, 40 rows 41 and 39 / 41 and 40 / 114 and 88): four stay.
int most_row_tiles(int precision, int head_dim, int t, long long tiles, int cus) {
    const int most = tree_row_tiles(head_dim);
    if (head_dim == 64 && elem_bytes(precision) == 2 && tiles > 4 * cus) return most;
    if (t <= 1280) return tiles <= cus ? 1 : 2;
    return head_dim == 80 && tiles > cus ? 2 : most;
}

// What does not depend on the cut of the keys.  most_splits grows with t.
TreeShape tree_shape(int precision, int pairs, int rows, int head_dim, int t, int cus) {
    TreeShape s;
    const int row_tiles = ceil_div(rows, 16);
    s.row_blocks = ceil_div(row_tiles, most_row_tiles(precision, head_dim, t, (long long)pairs * row_tiles, cus));
    s.row_tiles = ceil_div(row_tiles, s.row_blocks);
    s.tile_keys = 16 * tree_tile_units(elem_bytes(precision), head_dim, s.row_tiles);
    const int tiles = ceil_div(t, s.tile_keys);
    const long long groups = (long long)pairs * s.row_blocks;
    // One workgroup a CU streams at the memory's rate (measured from 1/4 to 16 a CU: 8 heads x 20000 keys
    // 167, 95, 63, 84, 117 us at 1/4, 1/2, 1, 2, 4), more only add partial results to join.
    const int most = std::max(1, std::min({(int)((cus + groups - 1) / groups), tiles / 2, 128}));
    s.most_splits = tiles - tiles / most < kJoinTiles ? 1 : most;
    return s;
}

int run_tree(int precision, int head_dim, TreeParams& P, void* workspace, size_t workspace_bytes, void* stream) {
    const int pairs = P.B * P.H;
    const bool scores = P.key_weights != nullptr;
    const int cus = compute_units();
    const TreePlan plan = plan_tree(precision, pairs, P.rows, head_dim, P.t, scores, cus);
    const int most = tree_shape(precision, pairs, P.rows, head_dim, P.t, cus).most_splits;
    const TreeSizes s = tree_sizes(pairs, P.rows, head_dim, most, scores, P.t);
    if (s.total() > 0) {
        if (workspace == nullptr || workspace_bytes < s.total()) return FFA_ERR_WORKSPACE;
        if (!aligned(workspace, 16)) return FFA_ERR_ALIGNMENT;
    }
    char* base = static_cast<char*>(workspace);
    P.ws_acc = reinterpret_cast<float*>(base);
    P.ws_ml = reinterpret_cast<float*>(base + s.acc);
    P.ws_scores = scores ? reinterpret_cast<float*>(base + s.acc + s.ml) : nullptr;
    P.score_stride = score_stride_of(P.t);
    P.score_lds = plan.score_lds;
    P.n_splits = plan.n_splits;
    P.tiles_per_split = plan.tiles_per_split;
    P.row_blocks = plan.row_blocks;
    P.splits_magic = tree_magic(P.n_splits);
    P.H_magic = tree_magic(P.H);
    P.G_magic = tree_magic(P.G);
    return launch_tree(precision, head_dim, P, plan, stream);
}

// A positive factor for the kernel, so that the largest product is the largest score and a masked
// -inf stays -inf.  A scale of zero (or one that vanishes in fp32) makes all scores 0: Q is taken as 0.
void set_scale(TreeParams& P, float softmax_scale) {
    const float c = softmax_scale * 1.4426950408889634f;
    P.q_sign = c < 0.f ? -1 : 1;
    P.scale_log2e = c < 0.f ? -c : c;
    if (P.scale_log2e < 1.17549435e-38f) {
        P.q_sign = 0;
        P.scale_log2e = 1.f;
    }
}

size_t tree_workspace(int precision, int B, int H, int Hq, int Dh, int tokens, int t, bool scores) {
    if (check_cache_shape(precision, B, H, Dh, 1) != FFA_OK || Hq <= 0 || Hq % H != 0 || tokens < 1 ||
        tokens > FFA_MAX_TREE_TOKENS || t < 0)
        return 0;
    const long long rows = (long long)(Hq / H) * tokens;
    if (rows > (1 << 20)) return 0;
    const int n = tree_shape(precision, B * H, (int)rows, Dh, t, compute_units()).most_splits;
    return tree_sizes(B * H, (int)rows, Dh, n, scores, t).total();
}

// Caches of a launch: a grid has fewer than 2^32 threads in x, and its workgroups up to 1024 a pair and cache.
int launch_caches(long long pairs) { return (int)std::min<long long>(kSlotCaches, (1ll << 21) / pairs); }

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

}  // namespace

namespace ffa {

TreePlan plan_tree(int precision, int pairs, int rows, int head_dim, int t, bool weights, int cus) {
    const TreeShape shape = tree_shape(precision, pairs, rows, head_dim, t, cus);
    TreePlan p;
    p.row_tiles = shape.row_tiles;
    p.row_blocks = shape.row_blocks;
    const int tile = shape.tile_keys, tiles = ceil_div(t, tile);
    p.tiles_per_split = std::max(1, ceil_div(tiles, shape.most_splits));
    p.n_splits = std::max(1, ceil_div(tiles, p.tiles_per_split));
    // With one workgroup a CU at most, 8 waves where they have two tiles each (256 pairs, 8000 keys, 32 rows
    // 109 -> 81 us, 64 rows 123 -> 102 us); more workgroups share the CUs, and 8 waves would not fit twice
    // (320 pairs, 1128 keys, 32 rows 27 -> 33 us).
    p.waves = tree_wide(head_dim, p.row_tiles) && pairs * p.row_blocks * p.n_splits <= cus && p.tiles_per_split >= 16 ? 8 : 4;
    const long long words = (long long)p.tiles_per_split * tile + 64;
    p.score_lds = weights && rows <= 16 && words * rows <= kScoreLdsWords ? (int)words : 0;
    return p;
}

}  // namespace ffa

extern "C" {

size_t ffa_tree_workspace_bytes(int precision, int batch_size, int head_num, int q_head_num, int head_dim, int tokens,
                                int t) {
    return tree_workspace(precision, batch_size, head_num, q_head_num, head_dim, tokens, t, false);
}

size_t ffa_weights_workspace_bytes(int precision, int batch_size, int head_num, int q_head_num, int head_dim, int t) {
    return tree_workspace(precision, batch_size, head_num, q_head_num, head_dim, 1, t, true);
}

int ffa_attention_tree(int precision, int batch_size, int head_num, int head_dim, int max_seq_len, float softmax_scale,
                       int t, const ffa_tree_tokens* tokens, const void* q, const void* k, const void* v, void* k_cache,
                       void* v_cache, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check_cache_shape(precision, batch_size, head_num, head_dim, max_seq_len);
    if (st != FFA_OK) return st;
    if (t < 0 || t >= max_seq_len) return FFA_ERR_TIMESTEP;
    if (!tokens || !q || !k || !v || !k_cache || !v_cache || !out) return FFA_ERR_NULL_POINTER;
    const int n = tokens->tokens, Hq = tokens->q_head_num;
    if (n < 1 || n > FFA_MAX_TREE_TOKENS || n > max_seq_len - t || Hq <= 0 || Hq % head_num != 0) return FFA_ERR_TREE;
    if ((long long)batch_size * Hq * n > (1ll << 24) || Hq / head_num > kTreeHeads) return FFA_ERR_SHAPE;
    const int unit = 16 / elem_bytes(precision);
    for (int i = 0; i < 3; ++i)
        if (tokens->q_stride[i] % unit || tokens->k_stride[i] % unit || tokens->v_stride[i] % unit ||
            tokens->out_stride[i] % unit)
            return FFA_ERR_TREE;
    for (long long step : {tokens->k_stride[2], tokens->v_stride[2]})  // lanes count rows in 32 bits
        if (step < 0 || step >= (1 << 26) / elem_bytes(precision)) return FFA_ERR_TREE;
    for (const void* p : {q, k, v, (const void*)k_cache, (const void*)v_cache, (const void*)out})
        if (!aligned(p, 16)) return FFA_ERR_ALIGNMENT;
    for (const int32_t* p : {tokens->parents, tokens->first_keys, tokens->lengths, tokens->counts})
        if (!aligned(p, 4)) return FFA_ERR_ALIGNMENT;
    TreeParams P = {};
    P.q = q; P.k = k; P.v = v;
    P.k_cache = k_cache; P.v_cache = v_cache; P.out = out;
    P.parents = tokens->parents; P.first_keys = tokens->first_keys;
    P.lengths = tokens->lengths; P.counts = tokens->counts;
    P.zero_rest = tokens->zero_rest;
    for (int i = 0; i < 3; ++i) {
        P.q_stride[i] = tokens->q_stride[i]; P.k_stride[i] = tokens->k_stride[i];
        P.v_stride[i] = tokens->v_stride[i]; P.out_stride[i] = tokens->out_stride[i];
    }
    P.B = batch_size; P.H = head_num; P.G = Hq / head_num; P.tokens = n; P.rows = P.G * n;
    P.Lmax = max_seq_len; P.t = t;
    set_scale(P, softmax_scale);
    return run_tree(precision, head_dim, P, workspace, workspace_bytes, stream);
}

int ffa_attention_weights(int precision, int batch_size, int head_num, int q_head_num, int head_dim, int max_seq_len,
                          float softmax_scale, int t, const void* q, const void* k, const void* v, void* k_cache,
                          void* v_cache, void* out, float* key_weights, const int32_t* first_keys,
                          const int32_t* lengths, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = check_cache_shape(precision, batch_size, head_num, head_dim, max_seq_len);
    if (st != FFA_OK) return st;
    if (t < 0 || t >= max_seq_len) return FFA_ERR_TIMESTEP;
    if (!q || !k || !v || !k_cache || !v_cache || !out || !key_weights) return FFA_ERR_NULL_POINTER;
    if (q_head_num <= 0 || q_head_num % head_num != 0) return FFA_ERR_TREE;
    if ((long long)batch_size * q_head_num > (1ll << 24) || q_head_num / head_num > kTreeHeads) return FFA_ERR_SHAPE;
    for (const void* p : {q, k, v, (const void*)k_cache, (const void*)v_cache, (const void*)out})
        if (!aligned(p, 16)) return FFA_ERR_ALIGNMENT;
    if (!aligned(key_weights, 4) || !aligned(first_keys, 4) || !aligned(lengths, 4)) return FFA_ERR_ALIGNMENT;
    TreeParams P = {};
    P.q = q; P.k = k; P.v = v;
    P.k_cache = k_cache; P.v_cache = v_cache; P.out = out;
    P.first_keys = first_keys; P.lengths = lengths;
    P.key_weights = key_weights;
    const long long qs[3] = {(long long)q_head_num * head_dim, head_dim, 0};
    const long long ks[3] = {(long long)head_num * head_dim, head_dim, 0};
    for (int i = 0; i < 3; ++i) {
        P.q_stride[i] = P.out_stride[i] = qs[i];
        P.k_stride[i] = P.v_stride[i] = ks[i];
    }
    P.B = batch_size; P.H = head_num; P.G = q_head_num / head_num; P.tokens = 1; P.rows = P.G;
    P.Lmax = max_seq_len; P.t = t;
    set_scale(P, softmax_scale);
    return run_tree(precision, head_dim, P, workspace, workspace_bytes, stream);
}

int ffa_commit_tree(int precision, int n_caches, void* const* k_caches, void* const* v_caches, int batch_size,
                    int head_num, int head_dim, int max_seq_len, int t, const int32_t* path, int path_len,
                    const int32_t* accepted, const int32_t* lengths, void* stream) {
    const int st = check_cache_shape(precision, batch_size, head_num, head_dim, max_seq_len);
    if (st != FFA_OK) return st;
    if (n_caches < 0) return FFA_ERR_SHAPE;
    if (t < 0 || t >= max_seq_len) return FFA_ERR_TIMESTEP;
    if (path_len < 1 || path_len > FFA_MAX_TREE_TOKENS || path_len > max_seq_len - t) return FFA_ERR_TREE;
    if (!path || !accepted || (n_caches > 0 && (!k_caches || !v_caches))) return FFA_ERR_NULL_POINTER;
    if (!aligned(path, 4) || !aligned(accepted, 4) || !aligned(lengths, 4)) return FFA_ERR_ALIGNMENT;
    for (int i = 0; i < n_caches; ++i) {
        if (!k_caches[i] || !v_caches[i]) return FFA_ERR_NULL_POINTER;
        if (!aligned(k_caches[i], 16) || !aligned(v_caches[i], 16)) return FFA_ERR_ALIGNMENT;
    }
    // A cache that is moved twice at once would be read behind its own writes.
    const size_t bytes = (size_t)batch_size * head_num * max_seq_len * head_dim * elem_bytes(precision);
    for (int i = 0; i < n_caches; ++i) {
        if (overlap(k_caches[i], bytes, v_caches[i], bytes)) return FFA_ERR_OVERLAP;
        for (int j = 0; j < i; ++j)
            for (const void* a : {(const void*)k_caches[i], (const void*)v_caches[i]})
                if (overlap(a, bytes, k_caches[j], bytes) || overlap(a, bytes, v_caches[j], bytes)) return FFA_ERR_OVERLAP;
    }
    const int most = launch_caches((long long)batch_size * head_num);
    for (int i0 = 0; i0 < n_caches; i0 += most) {
        CommitParams P = {};
        P.n_caches = std::min(most, n_caches - i0);
        for (int i = 0; i < P.n_caches; ++i) {
            P.k[i] = k_caches[i0 + i];
            P.v[i] = v_caches[i0 + i];
        }
        P.path = path; P.accepted = accepted; P.lengths = lengths;
        P.path_len = path_len; P.B = batch_size; P.H = head_num; P.Lmax = max_seq_len; P.t = t;
        const int rc = launch_commit(P, head_dim, elem_bytes(precision), stream);
        if (rc != FFA_OK) return rc;
    }
    return FFA_OK;
}

int ffa_evict(int precision, int n_caches, const void* const* k_src, const void* const* v_src,
              const float* const* w_src, void* const* k_dst, void* const* v_dst, float* const* w_dst, int batch_size,
              int head_num, int head_dim, int src_max_seq_len, int dst_max_seq_len, int t, int keep, int recent,
              const int32_t* first_keys, const int32_t* lengths, int32_t* kept, void* stream) {
    int st = check_cache_shape(precision, batch_size, head_num, head_dim, src_max_seq_len);
    if (st == FFA_OK) st = check_cache_shape(precision, batch_size, head_num, head_dim, dst_max_seq_len);
    if (st != FFA_OK) return st;
    if (n_caches < 0) return FFA_ERR_SHAPE;
    if (t < 0 || t > src_max_seq_len) return FFA_ERR_TIMESTEP;
    if (keep < 1 || keep > dst_max_seq_len || recent < 0 || recent > keep) return FFA_ERR_EVICT;
    if (n_caches == 0) return FFA_OK;
    if (!k_src || !v_src || !w_src || !k_dst || !v_dst || !w_dst || !kept) return FFA_ERR_NULL_POINTER;
    if (!aligned(first_keys, 4) || !aligned(lengths, 4) || !aligned(kept, 4)) return FFA_ERR_ALIGNMENT;
    const size_t pairs = (size_t)batch_size * head_num;
    const size_t src_kv = pairs * src_max_seq_len * head_dim * elem_bytes(precision), src_w = pairs * src_max_seq_len * 4;
    const size_t dst_kv = pairs * dst_max_seq_len * head_dim * elem_bytes(precision), dst_w = pairs * dst_max_seq_len * 4;
    for (int i = 0; i < n_caches; ++i) {
        if (!k_src[i] || !v_src[i] || !w_src[i] || !k_dst[i] || !v_dst[i] || !w_dst[i]) return FFA_ERR_NULL_POINTER;
        for (const void* p : {k_src[i], v_src[i], (const void*)k_dst[i], (const void*)v_dst[i]})
            if (!aligned(p, 16)) return FFA_ERR_ALIGNMENT;
        if (!aligned(w_src[i], 4) || !aligned(w_dst[i], 4)) return FFA_ERR_ALIGNMENT;
    }
    // Every target against every other buffer of the call: its own source may be the same buffer of the same shape.
    const bool same_shape = src_max_seq_len == dst_max_seq_len;
    const size_t kept_bytes = (size_t)n_caches * pairs * keep * 4;
    for (int i = 0; i < n_caches; ++i) {
        // The list of kept slots is written while other pairs' weights are still read.
        if (overlap(k_src[i], src_kv, kept, kept_bytes) || overlap(v_src[i], src_kv, kept, kept_bytes) ||
            overlap(w_src[i], src_w, kept, kept_bytes))
            return FFA_ERR_OVERLAP;
        const void* dst[3] = {k_dst[i], v_dst[i], w_dst[i]};
        for (int a = 0; a < 3; ++a) {
            const size_t na = a == 2 ? dst_w : dst_kv;
            for (int j = 0; j < n_caches; ++j) {
                const void* src2[3] = {k_src[j], v_src[j], w_src[j]};
                const void* dst2[3] = {k_dst[j], v_dst[j], w_dst[j]};
                for (int b = 0; b < 3; ++b) {
                    const bool own = i == j && a == b;
                    if (!(own && same_shape && src2[b] == dst[a]) && overlap(dst[a], na, src2[b], b == 2 ? src_w : src_kv))
                        return FFA_ERR_OVERLAP;
                    if (!own && overlap(dst[a], na, dst2[b], b == 2 ? dst_w : dst_kv)) return FFA_ERR_OVERLAP;
                }
            }
            if (overlap(dst[a], na, kept, kept_bytes)) return FFA_ERR_OVERLAP;
        }
    }
    const int most = launch_caches((long long)pairs);
    for (int i0 = 0; i0 < n_caches; i0 += most) {
        EvictParams P = {};
        P.n_caches = std::min(most, n_caches - i0);
        for (int i = 0; i < P.n_caches; ++i) {
            P.k_src[i] = k_src[i0 + i]; P.v_src[i] = v_src[i0 + i]; P.w_src[i] = w_src[i0 + i];
            P.k_dst[i] = k_dst[i0 + i]; P.v_dst[i] = v_dst[i0 + i]; P.w_dst[i] = w_dst[i0 + i];
        }
        P.first_keys = first_keys; P.lengths = lengths;
        P.kept = kept + (size_t)i0 * pairs * keep;
        P.B = batch_size; P.H = head_num; P.src_len = src_max_seq_len; P.dst_len = dst_max_seq_len;
        P.t = t; P.keep = keep; P.recent = recent;
        const int rc = launch_evict(P, head_dim, elem_bytes(precision), stream);
        if (rc != FFA_OK) return rc;
    }
    return FFA_OK;
}

}  // extern "C"
