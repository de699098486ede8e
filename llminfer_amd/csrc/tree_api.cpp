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

// Workgroups the splits aim for.
int tree_groups(const TreeForm& f) { return f.row_waves == 1 ? 256 : 512; }
// Contexts of up to so many tiles run as one split: a second launch joins the others.
constexpr int kTreeSingleTiles = 8;

int make_tree_plan(const llmi_mha_tree_args* a, llmi_mha_plan* p) {
    if (int rc = validate_tree(a)) return rc;
    const int n_kv = a->mha.kv_dim / a->mha.head_dim;
    const TreeForm form = tree_form(a->node_num * a->mha.kv_mul);
    const int wm = form.row_waves, row_groups = (form.blocks + wm - 1) / wm;
    const int tiles = (a->mha.pos + a->node_num + kTreeKeys - 1) / kTreeKeys;
    const size_t per_split = (size_t)n_kv * form.blocks * tree_split_bytes(form);
    const size_t room = a->mha.workspace ? a->mha.workspace_bytes / per_split : 0;
    int splits = a->mha.num_splits;
    if (splits == 0) {
        splits = tiles <= kTreeSingleTiles ? 1 : std::max(1, tree_groups(form) / (n_kv * row_groups));
        splits = std::min(splits, kMaxSplits);
        if (splits > 1) splits = std::max(1, std::min(splits, tiles / (4 / wm)));
        if ((size_t)splits > room) splits = (int)room;
    } else {
        splits = std::min(splits, tiles);
        if (splits > 1 && (size_t)splits > room) return LLMI_ERR_WORKSPACE;
    }
    if (splits < 2) splits = 1;
    *p = llmi_mha_plan{};
    p->path = splits > 1 ? LLMI_PATH_SPLIT : LLMI_PATH_SINGLE_PASS;
    p->num_splits = splits;
    p->rows_per_split = (tiles + splits - 1) / splits * kTreeKeys;
    p->waves_per_group = 4;
    p->group_pad = form.rows * wm;
    p->workspace_needed = splits > 1 ? per_split * splits : 0;
    return LLMI_OK;
}

}  // namespace
}  // namespace llmi

using namespace llmi;

extern "C" {

int llmi_hip_mha_tree_plan(const llmi_mha_tree_args* args, llmi_mha_plan* plan) {
    if (!plan) return LLMI_ERR_NULL_POINTER;
    return make_tree_plan(args, plan);
}

int llmi_hip_mha_decode_tree(const llmi_mha_tree_args* args) {
    llmi_mha_plan plan;
    if (int rc = make_tree_plan(args, &plan)) return rc;
    return launch_mha_tree(*args, plan);
}

size_t llmi_hip_mha_tree_workspace_bytes(int32_t head_num, int32_t head_dim, int32_t node_num) {
    if (head_num <= 0 || head_dim <= 0 || node_num <= 0) return 0;
    if (node_num > LLMI_TREE_MAX_NODES) return 0;
    // (how many KV heads share the query heads is not said: whatever needs most)
    size_t most = 16;
    for (int group = 1; group <= kMaxGroup; ++group) {
        if (head_num % group != 0) continue;
        const TreeForm form = tree_form(node_num * group);
        const int n_kv = head_num / group, row_groups = (form.blocks + form.row_waves - 1) / form.row_waves;
        const int splits = std::min(tree_groups(form) / (n_kv * row_groups), kMaxSplits);
        if (splits > 1) most = std::max(most, (size_t)splits * n_kv * form.blocks * tree_split_bytes(form));
    }
    return most;
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
