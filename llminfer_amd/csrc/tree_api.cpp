// C ABI of the calls for drafted tokens (include/llmi_hip.h, "a tree of them through the model in one pass"): argument
// validation and the split rule of the tree attention. The kernels live in mha_tree.hip, verify_tree.hip and qk_norm_rope.hip.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "llmi_hip.h"
#include "llmi_internal.h"

namespace llmi {
namespace {

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int validate_tree(const llmi_mha_tree_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    if (int rc = validate_mha(&a->mha)) return rc;
    if (a->node_num < 1 || a->node_num > LLMI_TREE_MAX_NODES) return LLMI_ERR_INVALID_ARG;
    if (a->mha.pos > a->mha.max_seq_len - a->node_num) return LLMI_ERR_POS_RANGE;
    if (a->mha.force_path != LLMI_PATH_AUTO || a->mha.waves_per_group != 0) return LLMI_ERR_INVALID_ARG;
    if (a->tree_mask && !aligned(a->tree_mask, 8)) return LLMI_ERR_ALIGNMENT;
    return LLMI_OK;
}

// Contexts of up to so many tiles run as one split: a second launch joins the others.
constexpr int kSingleTiles = 8;
constexpr int kSmallGroups = 1024;

// The rows' blocks. Sixteen rows where a KV head has no more, and up to a length that leaves each of the chip's 1024 SIMDs four tiles for
// sixteen rows or fewer: short calls wait for a tile's arithmetic, which is half as long. us, 32 : 16 rows, 8 KV heads: 8 nodes of 32 heads 8.9 : 7.4 at 250
// positions, 10.0 : 8.8 at 2000, 11.1 : 10.2 at 4099, 13.6 : 13.9 at 8192; 16 nodes 10.0 : 9.2 at 2000, 12.7 : 15.8 at 6000; 61 nodes 12.2 : 10.4
// at 500, 12.5 : 13.5 at 1000.
TreeForm tree_blocks(int rows, int n_kv, int64_t tiles) {
    const int small = (rows + 15) / 16;
    if (small == 1 || (int64_t)n_kv * small * ((tiles + 3) / 4) <= kSmallGroups) return {16, small, 1, 1};
    const int blocks = (rows + 31) / 32;
    return {32, blocks, blocks <= 1 ? 1 : blocks <= 2 ? 2 : 4, 1};
}

// Splits that a KV head's tiles are dealt to where nothing else limits them: a workgroup for each of 256 compute units, two from 64 tiles a
// workgroup on (one : two, us: 26 nodes of 32 heads, 8 KV heads 16.1 : 19.8 at 6007 positions, 25.8 : 30.2 at 16000, 61 nodes 20.6 : 24.0 at 6000,
// 62.7 : 60.2 at 32768, 64 nodes of 64 heads 451 : 358 at 131000: the parts of twice the splits have to be written and read).
int tree_splits(const TreeForm& f, int n_kv, int64_t tiles) {
    if (tiles <= kSingleTiles) return 1;
    const int row_groups = (f.blocks + f.row_waves - 1) / f.row_waves;
    const int groups = f.row_waves == 4 && tiles * n_kv * row_groups >= 256 * 64 ? 512 : 256;
    // No more than a tile for each wavefront; and beyond 32, with few KV heads, only as many as have four iterations (six of single tiles): us by
    // splits, 5 nodes of 8 heads, one KV head 10.3 : 9.7 : 11.5 with 32 : 64 : 70 at 9000 positions, 22.3 : 15.6 : 20.6 with 32 : 64 : 128 at 40000, 43.4 : 29.2
    // : 26.8 with 64 : 128 : 256 at 131000; 16 nodes of 16 heads, two 17.0 : 16.4 : 17.7 : 19.6 with 48 : 64 : 94 : 128 at 12000; 26 nodes, one
    // 16.3 : 17.9 : 24.5 with 32 : 64 : 128 at 9000.
    const int64_t most = std::max<int64_t>(32, tiles / (f.row_waves == 4 ? 6 : 16 / f.row_waves));
    const int64_t splits = std::min({(int64_t)std::min(groups / (n_kv * row_groups), kMaxSplits), tiles * f.row_waves / 4, most});
    return splits < 2 ? 1 : (int)splits;
}

// (64 bits: a bound near the type's largest position has more keys than that with its nodes' tile filled up)
int64_t tiles_of(const llmi_mha_tree_args* a) { return ((int64_t)a->mha.pos + a->node_num + kTreeKeys - 1) / kTreeKeys; }

int make_form(const llmi_mha_tree_args* a, TreeForm* f) {
    if (int rc = validate_tree(a)) return rc;
    const llmi_mha_args& m = a->mha;
    const int n_kv = m.kv_dim / m.head_dim;
    const int64_t tiles = tiles_of(a);
    *f = tree_blocks(a->node_num * m.kv_mul, n_kv, tiles);
    const size_t room = m.workspace ? m.workspace_bytes / ((size_t)n_kv * f->blocks * tree_split_bytes(*f)) : 0;
    f->splits = m.num_splits ? (int)std::min<int64_t>(m.num_splits, tiles) : (int)std::min<size_t>(tree_splits(*f, n_kv, tiles), room);
    if (f->splits < 2) f->splits = 1;
    return f->splits > 1 && (size_t)f->splits > room ? LLMI_ERR_WORKSPACE : LLMI_OK;
}

}  // namespace
}  // namespace llmi

using namespace llmi;

extern "C" {

int llmi_hip_mha_tree_plan(const llmi_mha_tree_args* args, llmi_mha_plan* plan) {
    if (!plan) return LLMI_ERR_NULL_POINTER;
    TreeForm f;
    if (int rc = make_form(args, &f)) return rc;
    const int64_t tiles = tiles_of(args);
    *plan = llmi_mha_plan{};
    plan->path = f.splits > 1 ? LLMI_PATH_SPLIT : LLMI_PATH_SINGLE_PASS;
    plan->num_splits = f.splits;
    plan->rows_per_split = (int32_t)std::min<int64_t>((tiles + f.splits - 1) / f.splits * kTreeKeys, INT32_MAX);
    plan->waves_per_group = 4;
    plan->group_pad = f.rows * f.row_waves;
    plan->workspace_needed = f.splits > 1 ? (size_t)(args->mha.kv_dim / 128) * f.blocks * f.splits * tree_split_bytes(f) : 0;
    return LLMI_OK;
}

int llmi_hip_mha_decode_tree(const llmi_mha_tree_args* args) {
    TreeForm f;
    if (int rc = make_form(args, &f)) return rc;
    return launch_mha_tree(*args, f);
}

size_t llmi_hip_mha_tree_workspace_bytes(int32_t head_num, int32_t head_dim, int32_t node_num) {
    if (head_num <= 0 || head_dim <= 0 || node_num <= 0 || node_num > LLMI_TREE_MAX_NODES) return 0;
    // (how many KV heads share the query heads is not said, nor the length: whatever needs most. Sixteen rows by length: a workgroup
    // takes one block)
    size_t most = 16;
    for (int group = 1; group <= kMaxGroup; ++group) {
        if (head_num % group != 0) continue;
        const int n_kv = head_num / group;
        const TreeForm f = tree_blocks(node_num * group, n_kv, INT32_MAX);
        most = std::max(most, (size_t)tree_splits(f, n_kv, INT32_MAX) * n_kv * f.blocks * tree_split_bytes(f));
    }
    return std::max(most, 256 * tree_split_bytes({16, 1, 1, 1}));
}

int llmi_hip_qk_norm_rope_append_tree(const llmi_qk_norm_rope_tree_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    const llmi_qk_norm_rope_args& r = a->row;
    if (!r.query || !r.key_new || !r.value_new || !r.key_cache || !r.value_cache || !r.norm_weight || !r.sin_cache || !r.cos_cache)
        return LLMI_ERR_NULL_POINTER;
    if (r.head_dim != 128) return LLMI_ERR_HEAD_DIM;
    if (r.kv_dim <= 0 || r.kv_dim % r.head_dim != 0) return LLMI_ERR_KV_DIM;
    if (r.head_num <= 0 || r.max_seq_len <= 0 || r.layer_id < 0) return LLMI_ERR_INVALID_ARG;
    if (a->node_num < 1 || a->node_num > LLMI_TREE_MAX_NODES) return LLMI_ERR_INVALID_ARG;
    if (r.pos < 0 || r.pos > r.max_seq_len - a->node_num) return LLMI_ERR_POS_RANGE;
    if (r.kv_layout != LLMI_KV_LAYOUT_POS_MAJOR && r.kv_layout != LLMI_KV_LAYOUT_HEAD_MAJOR) return LLMI_ERR_LAYOUT;
    const void* rows[] = {r.query, r.query_src, r.key_new, r.value_new, r.key_cache, r.value_cache, r.norm_weight, r.sin_cache, r.cos_cache};
    for (const void* q : rows)
        if (!aligned(q, 16)) return LLMI_ERR_ALIGNMENT;
    const int64_t strides[] = {a->query_stride, a->query_src_stride, a->key_new_stride, a->value_new_stride};
    const int64_t least[] = {(int64_t)r.head_num * 128, (int64_t)r.head_num * 128, r.kv_dim, r.kv_dim};
    for (int i = 0; i < 4; ++i) {
        if (strides[i] == 0) continue;
        if (strides[i] % 8 != 0) return LLMI_ERR_ALIGNMENT;
        if (strides[i] < least[i] && a->node_num > 1) return LLMI_ERR_INVALID_ARG;
    }
    if ((a->depth && !aligned(a->depth, 4)) || (a->pos_device && !aligned(a->pos_device, 4))) return LLMI_ERR_ALIGNMENT;
    if (!(r.eps >= 0.0f)) return LLMI_ERR_INVALID_ARG;
    return launch_qk_norm_rope_append_tree(*a);
}

int llmi_hip_verify_tree(const llmi_verify_tree_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    const bool greedy = a->temperature == 0.0f;
    if (!a->target_logits || !a->tokens || !a->path || !a->result || !a->workspace || (!greedy && !a->uniform)) return LLMI_ERR_NULL_POINTER;
    if (a->node_num < 1 || a->node_num > LLMI_TREE_MAX_NODES || a->vocab < 1) return LLMI_ERR_INVALID_ARG;
    if (a->logits_type != LLMI_LOGITS_F32 && a->logits_type != LLMI_LOGITS_BF16) return LLMI_ERR_INVALID_ARG;
    // (below 1e-5 the sampled token is the likeliest but for equals, and 1 / temperature would leave fp32's range further down)
    if (!greedy && !(a->temperature >= 1e-5f && std::isfinite(a->temperature))) return LLMI_ERR_INVALID_ARG;
    if (a->draft_logits && (a->parents || greedy)) return LLMI_ERR_INVALID_ARG;
    if ((a->target_stride != 0 && a->target_stride < a->vocab && a->node_num > 1) || a->target_stride < 0 ||
        (a->draft_stride != 0 && a->draft_stride < a->vocab && a->node_num > 1) || a->draft_stride < 0)
        return LLMI_ERR_INVALID_ARG;
    const uintptr_t item = a->logits_type == LLMI_LOGITS_F32 ? 4 : 2;
    if (!aligned(a->target_logits, item) || !aligned(a->draft_logits, item) || !aligned(a->tokens, 4) || !aligned(a->parents, 4) ||
        !aligned(a->uniform, 4) || !aligned(a->path, 4) || !aligned(a->result, 4) || !aligned(a->workspace, 16))
        return LLMI_ERR_ALIGNMENT;
    if (a->workspace_bytes < verify_tree_workspace_bytes(a->node_num, a->vocab)) return LLMI_ERR_WORKSPACE;
    return launch_verify_tree(*a);
}

size_t llmi_hip_verify_tree_workspace_bytes(int32_t node_num, int32_t vocab) {
    return node_num < 1 || vocab < 1 ? 0 : verify_tree_workspace_bytes(node_num, vocab);
}

int llmi_hip_kv_commit_tree(const llmi_kv_commit_tree_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    if (!a->key_cache || !a->value_cache || !a->path || !a->result) return LLMI_ERR_NULL_POINTER;
    if (a->head_dim != 128) return LLMI_ERR_HEAD_DIM;
    if (a->kv_dim <= 0 || a->kv_dim % a->head_dim != 0) return LLMI_ERR_KV_DIM;
    if (a->layer_num <= 0 || a->max_seq_len <= 0) return LLMI_ERR_INVALID_ARG;
    if (a->node_num < 1 || a->node_num > LLMI_TREE_MAX_NODES) return LLMI_ERR_INVALID_ARG;
    if (a->pos < 0 || a->pos > a->max_seq_len - a->node_num) return LLMI_ERR_POS_RANGE;
    if (a->kv_layout != LLMI_KV_LAYOUT_POS_MAJOR && a->kv_layout != LLMI_KV_LAYOUT_HEAD_MAJOR) return LLMI_ERR_LAYOUT;
    if (!aligned(a->key_cache, 16) || !aligned(a->value_cache, 16) || !aligned(a->path, 4) || !aligned(a->result, 4) || !aligned(a->pos_device, 4))
        return LLMI_ERR_ALIGNMENT;
    return launch_kv_commit_tree(*a);
}

}  // extern "C"
