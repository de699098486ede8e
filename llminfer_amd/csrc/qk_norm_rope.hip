// The per-token writers that feed decode attention on gfx950:
//   * fused per-head RMSNorm * weight + half-rotation RoPE on the query (in
//     place) and on the new K row, which lands in its cache slot in either
//     layout together with the new V row
//     (role of fused_qk_norm_rope_kernel, code/source/op/kernel/cuda/rmsnorm_kernel.cu:205-290,
//     plus the slot addressing of Model::slice_kv_cache, code/source/model/model.cpp:90-107);
//   * the sin/cos table (role of sin_cos_cache_kernel, code/source/op/kernel/cuda/rope_kernel.cu:6-21);
//   * a position-major -> head-major cache copy.
// One wavefront per head: lane i owns the rotation pair (i, i+64), the sum of
// squares is folded across the 64 lanes with DPP row steps and scalar reads, no LDS.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "llmi_internal.h"
#include "wave_ops.h"

namespace llmi {
namespace {

constexpr int kHeadDim = 128;
constexpr int kHalf = 64;

__device__ __forceinline__ float bf16_to_f32(uint16_t h) {
    return __builtin_bit_cast(float, (uint32_t)h << 16);
}

__device__ __forceinline__ uint16_t f32_to_bf16(float x) {
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    if (x != x) return 0x7fc0;
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

struct AppendArgs {
    uint16_t* query;
    const uint16_t* query_src;
    const uint16_t* key_new;
    const uint16_t* value_new;
    uint16_t* key_slot;    // cache address of (layer, pos, kv_head 0)
    uint16_t* value_slot;
    const uint16_t* weight;
    const float* sin_row;
    const float* cos_row;
    int64_t slot_head_stride;  // elements between KV heads inside the slot
    int32_t head_num;
    int32_t n_kv;
    float eps;
};

// One row on one wavefront: lane i owns the rotation pair (i, i + 64).
__device__ __forceinline__ void norm_rope_row(const uint16_t* src, const uint16_t* w, const float* sin_row, const float* cos_row, float eps,
                                              int i, uint16_t* dst) {
    const float x0 = bf16_to_f32(src[i]);
    const float x1 = bf16_to_f32(src[i + kHalf]);
    float ss = x0 * x0 + x1 * x1;
    ss = wave_sum(ss);
    const float r = 1.0f / sqrtf(ss / (float)kHeadDim + eps);
    const float av = x0 * bf16_to_f32(w[i]) * r;
    const float bv = x1 * bf16_to_f32(w[i + kHalf]) * r;
    const float sn = sin_row[i];
    const float cs = cos_row[i];
    dst[i] = f32_to_bf16(av * cs - bv * sn);
    dst[i + kHalf] = f32_to_bf16(av * sn + bv * cs);
}

__global__ __launch_bounds__(kHalf) void qk_norm_rope_append_kernel(AppendArgs a) {
    const int b = blockIdx.x;
    const int i = threadIdx.x;
    if (b >= a.head_num + a.n_kv) {
        // V row: plain copy into the slot, 4 bytes per lane.
        const int kh = b - a.head_num - a.n_kv;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.value_new + kh * kHeadDim);
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.value_slot + kh * a.slot_head_stride);
        dst[i] = src[i];
        return;
    }
    const uint16_t* src;
    uint16_t* dst;
    const uint16_t* w;
    if (b < a.head_num) {
        src = a.query_src + b * kHeadDim;
        dst = a.query + b * kHeadDim;
        w = a.weight;
    } else {
        const int kh = b - a.head_num;
        src = a.key_new + kh * kHeadDim;
        dst = a.key_slot + kh * a.slot_head_stride;
        w = a.weight + kHeadDim;
    }
    norm_rope_row(src, w, a.sin_row, a.cos_row, a.eps, i, dst);
}

// The same for the nodes of a tree: node i's rows to slot pos + i, rotated for position pos + depth[i].
struct AppendTreeArgs {
    uint16_t* query;
    const uint16_t* query_src;
    const uint16_t* key_new;
    const uint16_t* value_new;
    int64_t query_stride, query_src_stride, key_new_stride, value_new_stride;  // elements between nodes
    uint16_t* key_layer;
    uint16_t* value_layer;
    const uint16_t* weight;
    const float* sin_cache;
    const float* cos_cache;
    const int32_t* depth;    // optional
    const int32_t* pos_dev;  // optional
    int64_t row_stride, head_stride;  // elements between positions / KV heads of the caches
    int32_t pos, max_seq_len, head_num, n_kv;
    float eps;
};

__global__ __launch_bounds__(kHalf) void qk_norm_rope_append_tree_kernel(AppendTreeArgs a) {
    const int b = blockIdx.x, node = blockIdx.y, i = threadIdx.x;
    const int pos = a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos;
    const int kh = b < a.head_num ? 0 : (b - a.head_num) % a.n_kv;
    const int64_t slot = (int64_t)(pos + node) * a.row_stride + kh * a.head_stride;
    if (b >= a.head_num + a.n_kv) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.value_new + node * a.value_new_stride + kh * kHeadDim);
        reinterpret_cast<uint32_t*>(a.value_layer + slot)[i] = src[i];
        return;
    }
    const int64_t at = (int64_t)pos + (a.depth ? a.depth[node] : node);
    const int64_t table = (at < 0 ? 0 : at < a.max_seq_len ? at : a.max_seq_len - 1) * kHalf;
    const bool is_query = b < a.head_num;
    norm_rope_row(is_query ? a.query_src + node * a.query_src_stride + b * kHeadDim : a.key_new + node * a.key_new_stride + kh * kHeadDim,
                  a.weight + (is_query ? 0 : kHeadDim), a.sin_cache + table, a.cos_cache + table, a.eps, i,
                  is_query ? a.query + node * a.query_stride + b * kHeadDim : a.key_layer + slot);
}

// Rows of accepted nodes, slot pos + path[i] to slot pos + i. A workgroup has a KV head of a layer's keys or values: sixteen threads a row, all rows
// read before the first is written. (A thread for a chunk of all rows, one after the other : eight at a time : this, us: 4 rows of 36 layers of 8
// KV heads 2.6 : 2.9 : 2.3, 11 of 64 layers 3.8 : 3.9 : 2.6, 32 10.5 : 7.5 : 3.9.)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct CommitArgs {
    u32x4* cache[2];
    const int32_t* path;
    const int32_t* result;
    const int32_t* pos_dev;  // optional
    int64_t layer_chunks, row_chunks, head_chunks;
    int32_t pos, nodes, n_kv;
};

constexpr int kCommitThreads = 256;
__global__ __launch_bounds__(kCommitThreads) void kv_commit_tree_kernel(CommitArgs a) {
    constexpr int kRows = kCommitThreads / 16, kEach = LLMI_TREE_MAX_NODES / kRows;
    const int pos = a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos;
    const int count = min(a.result[0], a.nodes);
    u32x4* base = a.cache[blockIdx.z] + blockIdx.y * a.layer_chunks + pos * a.row_chunks + blockIdx.x * a.head_chunks + (threadIdx.x & 15);
    u32x4 row[kEach];
    bool moves[kEach];
#pragma unroll
    for (int x = 0; x < kEach; ++x) {
        const int i = x * kRows + (int)(threadIdx.x >> 4);
        const int from = i < count ? a.path[i] : 0;
        moves[x] = i > 0 && from > i && from < a.nodes;  // (row 0: the root is in its place)
        if (moves[x]) row[x] = base[from * a.row_chunks];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (every row is in registers, not just on its way, when the barrier lets go)
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kEach; ++x)
        if (moves[x]) base[(x * kRows + (int)(threadIdx.x >> 4)) * a.row_chunks] = row[x];
}

__global__ void sincos_table_kernel(float* __restrict__ sin_cache, float* __restrict__ cos_cache, int32_t half,
                                    int64_t total, float inv_head_dim, float ln_base) {
    const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= total) return;
    const int32_t i = (int32_t)(idx % half);
    const int32_t pos = (int32_t)(idx / half);
    // Same expression as the reference's host table (cpu/rope_kernel.cpp:12):
    // the exponent is formed in double and the frequency stored as float.
    const float freq = (float)exp(-2.0 * i * (double)inv_head_dim * (double)ln_base);
    const float theta = (float)pos * freq;
    float s, c;
    sincosf(theta, &s, &c);
    sin_cache[idx] = s;
    cos_cache[idx] = c;
}

// Memory-bound, reading and writing in equal parts: 16 head rows (256 bytes each) per workgroup, contiguous in the source, a
// 16-byte chunk per thread, both ways past the caches (each byte is touched once). K and V, 8 KV heads, cached accesses and a 64-bit
// division for each of layer, position and head : this, us: 36 layers of 3777 positions 184.5 : 177.7 (6.3 TB/s; a copy by torch of the
// same bytes 207), 8 of 12000 135.6 : 128.7, 28 of 500 23.7 : 23.0, 60 of 100 14.6 : 12.8; a first pass on new buffers 223 : 191 and
// 169 : 142. Where both caches fit the 256 MB memory-side cache a conversion of the same buffers over again is slower for going past it (36 layers of 1000
// 21.9 : 24.1, 28 of 2000 32.8 : 36.7, 28 of 500 level) and so is a reader of the result right behind it (copy included, 36 of 1000 49 : 53, but 28 of 2000 92 : 79); with the
// source just written it is faster (30 : 23, 50 : 34). A prompt is converted once, out of buffers that its prefill wrote. Cached reads with such stores 180 (first pass 230); two, four and eight chunks per thread 181, 187 and 280; positions of one KV
// head per workgroup (whole runs on the writing side) 184 ... 215.
constexpr int kRestrideThreads = 256;
__global__ __launch_bounds__(kRestrideThreads) void kv_restride_kernel(const uint4* __restrict__ src, uint4* __restrict__ dst,
                                                                       int32_t max_seq_len, int32_t n_kv, int32_t num_pos, int32_t layers) {
    const uint32_t row = blockIdx.x * (kRestrideThreads / 16) + (threadIdx.x >> 4);
    const uint32_t t = row / (uint32_t)n_kv, kh = row - t * (uint32_t)n_kv;
    if (t >= (uint32_t)num_pos) return;
    const int c = (int)(threadIdx.x & 15);
    const int64_t layer_chunks = (int64_t)max_seq_len * n_kv * 16;
    const int64_t from = (int64_t)row * 16 + c, to = ((int64_t)kh * max_seq_len + t) * 16 + c;
    for (int64_t layer = blockIdx.y; layer < layers; layer += gridDim.y) {
        const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src) + layer * layer_chunks + from);
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(dst) + layer * layer_chunks + to);
    }
}

}  // namespace

int launch_qk_norm_rope_append(const llmi_qk_norm_rope_args& args) {
    const int n_kv = args.kv_dim / args.head_dim;
    const int64_t layer_off = (int64_t)args.layer_id * args.max_seq_len * args.kv_dim;
    int64_t slot_off, slot_head_stride;
    if (args.kv_layout == LLMI_KV_LAYOUT_POS_MAJOR) {
        slot_off = layer_off + (int64_t)args.pos * args.kv_dim;
        slot_head_stride = args.head_dim;
    } else {
        slot_off = layer_off + (int64_t)args.pos * args.head_dim;
        slot_head_stride = (int64_t)args.max_seq_len * args.head_dim;
    }
    AppendArgs a;
    a.query = static_cast<uint16_t*>(args.query);
    a.query_src = args.query_src ? static_cast<const uint16_t*>(args.query_src) : a.query;
    a.key_new = static_cast<const uint16_t*>(args.key_new);
    a.value_new = static_cast<const uint16_t*>(args.value_new);
    a.key_slot = static_cast<uint16_t*>(args.key_cache) + slot_off;
    a.value_slot = args.value_cache ? static_cast<uint16_t*>(args.value_cache) + slot_off : nullptr;
    a.weight = static_cast<const uint16_t*>(args.norm_weight);
    a.sin_row = args.sin_cache + (int64_t)args.pos * (args.head_dim / 2);
    a.cos_row = args.cos_cache + (int64_t)args.pos * (args.head_dim / 2);
    a.slot_head_stride = slot_head_stride;
    a.head_num = args.head_num;
    a.n_kv = n_kv;
    a.eps = args.eps;
    const int blocks = args.head_num + n_kv + (args.value_new ? n_kv : 0);
    hipLaunchKernelGGL(qk_norm_rope_append_kernel, dim3(blocks), dim3(kHalf), 0,
                       static_cast<hipStream_t>(args.stream), a);
    return check_launch();
}

int launch_qk_norm_rope_append_tree(const llmi_qk_norm_rope_tree_args& args) {
    const llmi_qk_norm_rope_args& r = args.row;
    const bool by_head = r.kv_layout == LLMI_KV_LAYOUT_HEAD_MAJOR;
    const int64_t layer = (int64_t)r.layer_id * r.max_seq_len * r.kv_dim, q_row = (int64_t)r.head_num * kHeadDim;
    AppendTreeArgs a;
    a.query = static_cast<uint16_t*>(r.query);
    a.query_src = r.query_src ? static_cast<const uint16_t*>(r.query_src) : a.query;
    a.key_new = static_cast<const uint16_t*>(r.key_new);
    a.value_new = static_cast<const uint16_t*>(r.value_new);
    a.query_stride = args.query_stride ? args.query_stride : q_row;
    a.query_src_stride = !r.query_src ? a.query_stride : args.query_src_stride ? args.query_src_stride : q_row;
    a.key_new_stride = args.key_new_stride ? args.key_new_stride : r.kv_dim;
    a.value_new_stride = args.value_new_stride ? args.value_new_stride : r.kv_dim;
    a.key_layer = static_cast<uint16_t*>(r.key_cache) + layer;
    a.value_layer = static_cast<uint16_t*>(r.value_cache) + layer;
    a.weight = static_cast<const uint16_t*>(r.norm_weight);
    a.sin_cache = r.sin_cache;
    a.cos_cache = r.cos_cache;
    a.depth = args.depth;
    a.pos_dev = args.pos_device;
    a.row_stride = by_head ? kHeadDim : r.kv_dim;
    a.head_stride = by_head ? (int64_t)r.max_seq_len * kHeadDim : kHeadDim;
    a.pos = r.pos;
    a.max_seq_len = r.max_seq_len;
    a.head_num = r.head_num;
    a.n_kv = r.kv_dim / kHeadDim;
    a.eps = r.eps;
    hipLaunchKernelGGL(qk_norm_rope_append_tree_kernel, dim3(a.head_num + 2 * a.n_kv, args.node_num), dim3(kHalf), 0,
                       static_cast<hipStream_t>(r.stream), a);
    return check_launch();
}

int launch_kv_commit_tree(const llmi_kv_commit_tree_args& args) {
    if (args.node_num == 1) return LLMI_OK;  // (the root is in its place)
    const bool by_head = args.kv_layout == LLMI_KV_LAYOUT_HEAD_MAJOR;
    CommitArgs a;
    a.cache[0] = static_cast<u32x4*>(args.key_cache);
    a.cache[1] = static_cast<u32x4*>(args.value_cache);
    a.path = args.path;
    a.result = args.result;
    a.pos_dev = args.pos_device;
    a.n_kv = args.kv_dim / kHeadDim;
    a.layer_chunks = (int64_t)args.max_seq_len * a.n_kv * 16;
    a.row_chunks = by_head ? 16 : (int64_t)a.n_kv * 16;
    a.head_chunks = by_head ? (int64_t)args.max_seq_len * 16 : 16;
    a.pos = args.pos;
    a.nodes = args.node_num;
    hipLaunchKernelGGL(kv_commit_tree_kernel, dim3(a.n_kv, args.layer_num, 2), dim3(kCommitThreads), 0,
                       static_cast<hipStream_t>(args.stream), a);
    return check_launch();
}

int launch_sincos_table(float* sin_cache, float* cos_cache, int32_t head_dim, int32_t max_seq_len,
                        hipStream_t stream) {
    const int32_t half = head_dim / 2;
    const int64_t total = (int64_t)half * max_seq_len;
    const int threads = 256;
    const int64_t blocks = (total + threads - 1) / threads;
    hipLaunchKernelGGL(sincos_table_kernel, dim3((unsigned)blocks), dim3(threads), 0, stream, sin_cache, cos_cache,
                       half, total, 1.0f / (float)head_dim, logf(1000000.0f));
    return check_launch();
}

int launch_kv_restride(const void* src, void* dst, int32_t layer_num, int32_t max_seq_len, int32_t kv_dim,
                       int32_t head_dim, int32_t num_pos, hipStream_t stream) {
    const int n_kv = kv_dim / head_dim;
    if (layer_num == 0 || num_pos == 0) return LLMI_OK;
    constexpr int rows = kRestrideThreads / 16;
    const int64_t blocks = ((int64_t)num_pos * n_kv + rows - 1) / rows;
    const dim3 grid((unsigned)blocks, (unsigned)(layer_num < 65535 ? layer_num : 65535));
    hipLaunchKernelGGL(kv_restride_kernel, grid, dim3(kRestrideThreads), 0, stream, static_cast<const uint4*>(src), static_cast<uint4*>(dst),
                       max_seq_len, n_kv, num_pos, layer_num);
    return check_launch();
}

}  // namespace llmi
