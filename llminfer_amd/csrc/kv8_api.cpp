// C ABI of the calls for an 8-bit KV cache (include/llmi_hip.h): argument validation and the split rule of its attention. The kernels
// live in mha_kv8.hip and kv8_rows.hip.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>

#include "llmi_hip.h"
#include "llmi_internal.h"

namespace llmi {
namespace {

// KV heads are a grid dimension.
constexpr int kMostKvHeads = 65535;

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

bool is_format(int32_t f) { return f == LLMI_KV8_E4M3 || f == LLMI_KV8_INT8; }

int validate_dims(int32_t head_dim, int32_t kv_dim, int32_t max_seq_len, int32_t format) {
    if (head_dim != 128) return LLMI_ERR_HEAD_DIM;
    if (kv_dim <= 0 || kv_dim % head_dim != 0) return LLMI_ERR_KV_DIM;
    if (kv_dim / head_dim > kMostKvHeads || max_seq_len <= 0 || !is_format(format)) return LLMI_ERR_INVALID_ARG;
    return LLMI_OK;
}

// Bytes of memory from an address on (none: nowhere), up to the end of the address space at most.
struct Range {
    uintptr_t from, to;
};
Range range(const void* p, size_t bytes) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(p);
    return p ? Range{from, bytes > UINTPTR_MAX - from ? UINTPTR_MAX : from + bytes} : Range{0, 0};
}
bool apart(Range a, Range b) { return a.to <= b.from || b.to <= a.from; }

// The 8-bit cache up to and with a layer (later layers' place is not known to be the cache's). No memory is as large as one whose size passes 64 bits.
Range cache_range(const void* cache8, int32_t layers, int32_t max_seq_len, int32_t kv_dim) {
    const size_t n = llmi_hip_kv8_bytes(layers, max_seq_len, kv_dim, 128);
    return range(cache8, n ? n : SIZE_MAX);
}

int validate(const llmi_mha_kv8_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    if (!a->query || !a->cache8 || !a->output) return LLMI_ERR_NULL_POINTER;
    if (int rc = validate_dims(a->head_dim, a->kv_dim, a->max_seq_len, a->format)) return rc;
    if (a->kv_mul < 1 || a->kv_mul > kMaxGroup || a->head_num != a->kv_mul * (a->kv_dim / a->head_dim)) return LLMI_ERR_HEAD_GROUP;
    if (a->layer_id < 0 || a->num_splits < 0 || a->num_splits > kMaxSplits) return LLMI_ERR_INVALID_ARG;
    if (a->pos < 0 || a->pos >= a->max_seq_len) return LLMI_ERR_POS_RANGE;
    if (!aligned(a->query, 16) || !aligned(a->cache8, 16) || !aligned(a->output, 16) || !aligned(a->workspace, 16) || !aligned(a->output_f32, 4) ||
        !aligned(a->pos_device, 4))
        return LLMI_ERR_ALIGNMENT;
    const Range query = range(a->query, (size_t)a->head_num * 256);
    if (!apart(query, range(a->output, (size_t)a->head_num * 256)) || !apart(query, range(a->output_f32, (size_t)a->head_num * 512))) return LLMI_ERR_INVALID_ARG;
    return LLMI_OK;
}

size_t split_bytes(const llmi_mha_kv8_args* a) { return (size_t)a->head_num * (128 * sizeof(float) + 2 * sizeof(unsigned long long)); }

// A KV head's query heads are joined by different workgroups where those, which wait for each other, fit the chip with room to spare.
constexpr int kMostJoining = 128;
// Records up to which a KV head is not split, and KV heads up to which four workgroups have 32 of its columns and all positions each there: K's codes are read and multiplied
// four times, V's once, and there is nothing to join. us, splits by the rule below : so, 32 Q / 8 KV heads E4M3: 2.69 : 2.45 at 21 positions, 2.94 : 2.56 at 128, 4.16 : 3.39 at 256, 4.54 : 3.83
// at 320, 4.66 : 4.25 at 401, 4.67 : 4.35 at 512, 4.66 : 4.64 at 601, 4.73 : 5.19 at 701; with the new token 3.89 : 3.36 at 57, 5.06 : 4.47 at 300 (16 Q), 5.51 : 4.98
// at 511. Whole numbers, whose conversion takes three times the instructions: 4.97 : 4.18 at 320, 4.86 : 5.08 at 401. (Sixteen wavefronts beyond eight records
// 0.2 - 0.65 slower.) Other KV heads, a record each : slices : one workgroup, at 58, 301 and 576 positions: 1 (16 Q) 8.40 : 2.71 : 3.34, 8.58 : 4.06 : 5.21, 5.54 : 4.95 : 6.49; 3 4.36 : 2.45 : 2.73,
// 4.24 : 3.77 : 4.37, 4.66 : 4.65 : 5.66; 32 4.57 : 2.78 : 3.10, 4.77 : 3.95 : 4.83, 5.03 : 5.47 : 6.06; 64 4.73 : 2.95 : 3.24, 5.23 : 4.65 : 4.96, 6.68 : 5.89 : 6.23. With more there are more slices than compute
// units, and one workgroup reads K once: 80 4.77 : 3.33 : 3.27, 5.51 : 5.87 : 5.02, 6.50 : 7.50 : 6.34; 128 4.87 : 3.47 : 3.36, 6.83 : 6.21 : 5.13, 7.45 : 8.88 : 6.67; 512 slices : one workgroup 6.71 : 4.55, 18.1 : 9.7, 30.3 : 14.5.
constexpr int kMostSingle = 18, kMostSingleWhole = 12;
constexpr int kMostSlicedHeads = 64;

// The workgroups a KV head's records are dealt to beyond that: a record each up to 32, then three records each, up to one workgroup per compute unit. us by
// splits, 32 Q / 8 KV heads, E4M3: 4.90 : 4.75 with 16 : 32 at 1024 positions, 5.68 : 6.55 with 32 : 64 at 4096, 7.31 : 7.96 at 8192, 14.2 : 15.9 at 32768, 42.7 : 45.6 at 131001.
constexpr int kRecordEach = 32;
// Eight wavefronts a workgroup where four would have more than a record each alone, more than five in a split (each wavefront has one record on
// its way; more in flight on a compute unit are slower: two a wavefront 43.9 : 42.4 us at 131001, 15.3 : 14.2 at 32768, three 18.6). us with 4 : 8: slices 3.10 : 3.15 at
// 160 positions, 3.53 : 3.48 at 256, 4.35 : 3.96 at 301, 5.79 : 4.68 at 576, whole numbers 4.76 : 4.20 at 301, with the new token 3.74 : 3.71 at 160 (16 Q 3.74 : 3.62), 4.84 : 4.38 at 300; one workgroup 3.08 : 3.16 at
// 128, 4.61 : 4.19 at 256, 5.48 : 4.54 at 301; splits 5.73 : 5.81 at 4096, 7.02 : 6.64 at 6008, 15.7 : 14.3 at 32768, 46.2 : 42.4 at 131001, whole
// numbers, 64 Q heads 6.16 : 6.33 at 4096, 7.59 : 7.25 at 6008, 51.8 : 44.0 at 131001.
int make_form(const llmi_mha_kv8_args* a, int new_rows, Kv8Form* form) {
    if (int rc = validate(a)) return rc;
    const int64_t keys = (int64_t)a->pos + 1 - new_rows, tiles = (keys + 31) / 32;
    // (partial outputs are addressed with 31 bits)
    const size_t room = a->workspace ? std::min(a->workspace_bytes > 16 ? a->workspace_bytes - 16 : 0, (size_t)INT32_MAX) / split_bytes(a) : 0;
    // (a chosen number: a record each)
    const bool chosen = a->num_splits > 0;
    form->single = chosen ? 1 : a->format == LLMI_KV8_E4M3 ? kMostSingle : kMostSingleWhole;
    form->each = chosen ? INT32_MAX : kRecordEach;
    form->sliced = !chosen && a->kv_dim / 128 <= kMostSlicedHeads && (a->pos_device || tiles <= form->single);
    const int most = chosen ? a->num_splits : (int)std::max<size_t>(std::min<size_t>({(size_t)std::max(256 / (a->kv_dim / 128), 1), (size_t)kMaxSplits, room}), 1);
    form->splits = kv8_active_splits((int)tiles, most, form->single, form->each);
    if (form->splits > 1 && (size_t)form->splits > room) return LLMI_ERR_WORKSPACE;
    // (with slices at some lengths up to the bound their workgroup size is all lengths')
    form->waves = tiles > (form->sliced || form->splits == 1 ? 4 : 5 * (int64_t)form->splits) ? 8 : 4;
    // (the new token's query heads, half a wavefront each, all but one wavefront's: six in one pass with four. us with 4 : 8, 64 Q heads: 3.70 : 3.46 at 127
    // positions, 5.74 : 5.95 at 1024, 6.15 : 6.17 at 2000, 7.61 : 7.05 at 4099)
    if (new_rows && a->kv_mul > 6 && (form->sliced || tiles >= 3 * (int64_t)form->splits)) form->waves = 8;
    form->spread_min = a->head_num <= kMostJoining ? 2 : INT32_MAX;
    return LLMI_OK;
}

// Whether what a call writes is apart from what it reads, and each thing written from the others: workgroups write while others still read.
bool writes_apart(const llmi_mha_kv8_args* a, const llmi_mha_kv8_append_args* append, int splits) {
    if (a->layer_id == INT32_MAX) return false;
    const size_t heads = (size_t)a->head_num * 256, new_row = (size_t)a->kv_dim * 2, table = ((size_t)a->pos + 1) * 256;
    const Range none{0, 0}, cache = cache_range(a->cache8, a->layer_id + 1, a->max_seq_len, a->kv_dim);
    const Range writes[] = {range(a->output, heads), range(a->output_f32, 2 * heads), splits > 1 ? range(a->workspace, split_bytes(a) * (size_t)splits) : none, append ? cache : none};
    const Range reads[] = {range(a->query, heads),
                           range(a->pos_device, 4),
                           append ? none : cache,
                           append ? range(append->key_new, new_row) : none,
                           append ? range(append->value_new, new_row) : none,
                           append ? range(append->norm_weight, 512) : none,
                           append ? range(append->sin_cache, table) : none,
                           append ? range(append->cos_cache, table) : none};
    for (const Range& w : writes) {
        for (const Range& r : reads)
            if (!apart(w, r)) return false;
        for (const Range* x = writes; x != &w; ++x)
            if (!apart(w, *x)) return false;
    }
    return true;
}

// Rows of the same length, `stride` bytes from one to the next: tokens' slices of a projection's result, or (one of them) anything.
struct Rows {
    const void* first;
    size_t width, stride;
    int32_t count;
};
Range span(const Rows& r) {
    size_t n;
    return range(r.first, __builtin_mul_overflow((size_t)(r.count - 1), r.stride, &n) || __builtin_add_overflow(n, r.width, &n) ? SIZE_MAX : n);
}
// Exact for rows of the same stride, as many of each, and for one row against others; rows of different strides are apart if their spans are.
bool apart(const Rows& a, const Rows& b) {
    const Range x = span(a), y = span(b);
    if (apart(x, y)) return true;
    if (a.count == 1 || (b.count == 1 ? y.from < x.from : a.stride != b.stride)) return false;
    const size_t behind = y.from >= x.from ? (y.from - x.from) % a.stride : (a.stride - (x.from - y.from) % a.stride) % a.stride;
    return behind >= a.width && b.width <= a.stride && behind <= a.stride - b.width;
}

// Whether what the rows' call writes, queries and cache, is apart from what it reads. (Queries in their raw rows' place are not: a row is read and written by the same lanes.)
bool writes_apart(const llmi_qk_norm_rope_kv8_args* a) {
    if (a->layer_id == INT32_MAX) return false;
    const size_t heads = (size_t)a->head_num * 256, kv = (size_t)a->kv_dim * 2, table = ((size_t)a->pos + (size_t)a->row_num) * 256;
    const auto rows = [&](const void* p, size_t width, int64_t stride) { return Rows{p, width, a->row_num > 1 && stride ? (size_t)stride * 2 : width, a->row_num}; };
    const auto whole = [](Range r) { return Rows{reinterpret_cast<const void*>(r.from), r.to - r.from, r.to - r.from, 1}; };
    const Rows query = rows(a->query, heads, a->query_stride), src = rows(a->query_src, heads, a->query_src_stride);
    const Rows cache = whole(cache_range(a->cache8, a->layer_id + 1, a->max_seq_len, a->kv_dim));
    const Rows reads[] = {rows(a->key_new, kv, a->key_new_stride), rows(a->value_new, kv, a->value_new_stride), whole(range(a->norm_weight, 512)), whole(range(a->sin_cache, table)),
                          whole(range(a->cos_cache, table))};
    for (const Rows& r : {query, src, reads[0], reads[1]})
        if (span(r).to == UINTPTR_MAX) return false;  // (no memory holds them)
    for (const Rows& r : reads)
        if (!apart(query, r) || !apart(r, cache)) return false;
    if (a->query_src && !(a->query_src == a->query && src.stride == query.stride) && !apart(query, src)) return false;
    if (a->query_src && !apart(src, cache)) return false;
    if (a->pos_device && (!apart(query, whole(range(a->pos_device, 4))) || !apart(span(cache), range(a->pos_device, 4)))) return false;
    return apart(query, cache);
}

int validate_copy(const llmi_kv8_copy_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    if (!a->key_cache || !a->value_cache || !a->cache8) return LLMI_ERR_NULL_POINTER;
    if (int rc = validate_dims(a->head_dim, a->kv_dim, a->max_seq_len, a->format)) return rc;
    if (a->layer_num < 0) return LLMI_ERR_INVALID_ARG;
    if (a->first_pos < 0 || a->num_pos < 0 || a->first_pos > a->max_seq_len || a->num_pos > a->max_seq_len - a->first_pos) return LLMI_ERR_POS_RANGE;
    if (a->kv_layout != LLMI_KV_LAYOUT_POS_MAJOR && a->kv_layout != LLMI_KV_LAYOUT_HEAD_MAJOR) return LLMI_ERR_LAYOUT;
    // (a workgroup per record and KV head: no layer of a bf16 cache that fits a GPU has more)
    if (kv8_records(a->max_seq_len) * (a->kv_dim / 128) > kKv8MostGroups) return LLMI_ERR_INVALID_ARG;
    if (!aligned(a->key_cache, 16) || !aligned(a->value_cache, 16) || !aligned(a->cache8, 16)) return LLMI_ERR_ALIGNMENT;
    return LLMI_OK;
}

// Whether the three caches of a copy are apart (the two that are read may be one).
bool caches_apart(const llmi_kv8_copy_args* a, bool load) {
    size_t rows = (size_t)a->max_seq_len * (size_t)a->kv_dim * 2;
    if (__builtin_mul_overflow(rows, (size_t)a->layer_num, &rows)) return false;
    const Range k = range(a->key_cache, rows), v = range(a->value_cache, rows), cache = cache_range(a->cache8, a->layer_num, a->max_seq_len, a->kv_dim);
    return apart(k, cache) && apart(v, cache) && (!load || apart(k, v));
}

}  // namespace
}  // namespace llmi

using namespace llmi;

extern "C" {

size_t llmi_hip_kv8_bytes(int32_t layer_num, int32_t max_seq_len, int32_t kv_dim, int32_t head_dim) {
    if (layer_num <= 0 || max_seq_len <= 0 || head_dim != 128 || kv_dim <= 0 || kv_dim % 128 != 0) return 0;
    size_t n = (size_t)kv8_records(max_seq_len) * kKv8Record;
    if (__builtin_mul_overflow(n, (size_t)(kv_dim / 128), &n) || __builtin_mul_overflow(n, (size_t)layer_num, &n)) return 0;
    return n;
}

int llmi_hip_kv8_store(const llmi_kv8_copy_args* args) {
    if (int rc = validate_copy(args)) return rc;
    if (args->layer_num == 0 || args->num_pos == 0) return LLMI_OK;
    if (!caches_apart(args, false)) return LLMI_ERR_INVALID_ARG;
    return launch_kv8_store(*args);
}

int llmi_hip_kv8_load(const llmi_kv8_copy_args* args) {
    if (int rc = validate_copy(args)) return rc;
    if (args->layer_num == 0 || args->num_pos == 0) return LLMI_OK;
    if (!caches_apart(args, true)) return LLMI_ERR_INVALID_ARG;
    return launch_kv8_load(*args);
}

int llmi_hip_qk_norm_rope_append_kv8(const llmi_qk_norm_rope_kv8_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    if (!a->query || !a->key_new || !a->value_new || !a->cache8 || !a->norm_weight || !a->sin_cache || !a->cos_cache) return LLMI_ERR_NULL_POINTER;
    if (int rc = validate_dims(a->head_dim, a->kv_dim, a->max_seq_len, a->format)) return rc;
    if (a->head_num <= 0 || a->head_num > kMaxGroup * kMostKvHeads || a->layer_id < 0 || a->row_num < 1 || !(a->eps >= 0.0f)) return LLMI_ERR_INVALID_ARG;
    if (a->pos < 0 || a->row_num > a->max_seq_len || a->pos > a->max_seq_len - a->row_num) return LLMI_ERR_POS_RANGE;
    const void* rows[] = {a->query, a->query_src, a->key_new, a->value_new, a->cache8, a->norm_weight, a->sin_cache, a->cos_cache};
    for (const void* q : rows)
        if (!aligned(q, 16)) return LLMI_ERR_ALIGNMENT;
    const int64_t strides[] = {a->query_stride, a->query_src_stride, a->key_new_stride, a->value_new_stride};
    const int64_t least[] = {(int64_t)a->head_num * 128, (int64_t)a->head_num * 128, a->kv_dim, a->kv_dim};
    for (int i = 0; i < 4; ++i) {
        if (strides[i] == 0) continue;
        if (strides[i] % 8 != 0) return LLMI_ERR_ALIGNMENT;
        if (strides[i] < least[i] && a->row_num > 1) return LLMI_ERR_INVALID_ARG;
    }
    if (!aligned(a->pos_device, 4)) return LLMI_ERR_ALIGNMENT;
    if (!writes_apart(a)) return LLMI_ERR_INVALID_ARG;
    return launch_qk_norm_rope_append_kv8(*a);
}

int llmi_hip_mha_kv8_plan(const llmi_mha_kv8_args* args, llmi_mha_plan* plan) {
    if (!plan) return LLMI_ERR_NULL_POINTER;
    Kv8Form form;
    if (int rc = make_form(args, 0, &form)) return rc;
    const int splits = form.splits;
    const int64_t tiles = ((int64_t)args->pos + 32) / 32, per = (tiles + splits - 1) / splits;
    *plan = llmi_mha_plan{};
    plan->path = splits > 1 ? LLMI_PATH_SPLIT_FUSED : LLMI_PATH_SINGLE_PASS;
    plan->num_splits = splits;
    plan->rows_per_split = (int32_t)std::min<int64_t>(per * 32, INT32_MAX);
    plan->waves_per_group = form.waves;
    plan->group_pad = 16;
    plan->workspace_needed = splits > 1 ? split_bytes(args) * (size_t)splits + 16 : 0;
    return LLMI_OK;
}

int llmi_hip_mha_decode_kv8(const llmi_mha_kv8_args* args) {
    Kv8Form form;
    if (int rc = make_form(args, 0, &form)) return rc;
    if (!writes_apart(args, nullptr, form.splits)) return LLMI_ERR_INVALID_ARG;
    return launch_mha_kv8(*args, nullptr, form);
}

int llmi_hip_mha_decode_append_kv8(const llmi_mha_kv8_append_args* a) {
    if (!a) return LLMI_ERR_NULL_POINTER;
    Kv8Form form;
    if (int rc = make_form(&a->mha, 1, &form)) return rc;
    if (!a->key_new || !a->value_new || !a->norm_weight || !a->sin_cache || !a->cos_cache) return LLMI_ERR_NULL_POINTER;
    if (!aligned(a->key_new, 16) || !aligned(a->value_new, 16) || !aligned(a->norm_weight, 16) || !aligned(a->sin_cache, 16) || !aligned(a->cos_cache, 16))
        return LLMI_ERR_ALIGNMENT;
    if (!(a->eps >= 0.0f)) return LLMI_ERR_INVALID_ARG;
    if (!writes_apart(&a->mha, a, form.splits)) return LLMI_ERR_INVALID_ARG;
    return launch_mha_kv8(a->mha, a, form);
}

}  // extern "C"
