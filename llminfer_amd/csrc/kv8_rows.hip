// What fills an 8-bit KV cache and reads it back (layout and codes: kv8.h): the rows of new tokens, normalised, rotated and quantised as
// they are filed; ranges of a bf16 cache of either layout, all layers, quantised and back.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv8.h"
#include "llmi_internal.h"

namespace llmi {
namespace {

struct RowsArgs {
    uint16_t* query;
    const uint16_t* query_src;
    const uint16_t* key_new;
    const uint16_t* value_new;
    int64_t query_stride, query_src_stride, key_new_stride, value_new_stride;  // elements between tokens
    char* cache;       // the layer's records
    const uint16_t* weight;
    const float* sin_cache;
    const float* cos_cache;
    const int32_t* pos_dev;  // optional
    int64_t records;   // per KV head
    int32_t pos, rows, head_num, n_kv;
    float eps;
};

// Half a wavefront a row: the token's query heads, K rows, V rows.
constexpr int kRowThreads = 256;
template <int FORMAT>
__global__ __launch_bounds__(kRowThreads) void kv8_append_kernel(RowsArgs a) {
    const int p = threadIdx.x & 31;
    const int b = blockIdx.x * (kRowThreads / 32) + (int)(threadIdx.x >> 5);
    if (b >= a.head_num + 2 * a.n_kv) return;
    const int base = a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos;
    for (int row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const int pos = base + row;
        const int kh = b < a.head_num ? 0 : (b - a.head_num) % a.n_kv;
        const bool is_query = b < a.head_num, is_v = b >= a.head_num + a.n_kv;
        const uint16_t* src = is_query ? a.query_src + row * a.query_src_stride + b * kHeadDim
                              : is_v   ? a.value_new + row * a.value_new_stride + kh * kHeadDim
                                       : a.key_new + row * a.key_new_stride + kh * kHeadDim;
        NewRow y;
        load_row32(y, reinterpret_cast<uint64_t>(src), reinterpret_cast<uint64_t>(a.weight + (is_query ? 0 : kHeadDim)), p);
        load_tables32(y, a.sin_cache + (int64_t)pos * 64, a.cos_cache + (int64_t)pos * 64, p);
        uint32_t lo, hi;
        norm_rope_regs32(y, p, a.eps, lo, hi);
        if (is_query) {
            uint32_t* dst = reinterpret_cast<uint32_t*>(a.query + row * a.query_stride + b * kHeadDim);
            dst[p] = lo;
            dst[p + 32] = hi;
            continue;
        }
        if (is_v) {
            lo = y.x[0];
            hi = y.x[1];
        }
        float s;
        const uint32_t codes = quantise_row32<FORMAT>(lo, hi, s);
        file_row32(a.cache + (kh * a.records + (pos >> 5)) * kKv8Record, pos & 31, is_v, p, codes, s);
    }
}

struct CopyArgs {
    char* cache;
    uint16_t* rows[2];   // K, V of the bf16 cache
    int64_t layer_elems, row_stride, head_stride;  // elements
    int64_t records;     // per KV head
    int32_t first, count, n_kv, layers;
};

// A workgroup per record of a KV head, K in the first half of the threads' turns, V in the second: sixteen lanes a row of 256 bytes.
constexpr int kCopyThreads = 256;
template <int FORMAT>
__global__ __launch_bounds__(kCopyThreads) void kv8_store_kernel(CopyArgs a) {
    __shared__ __attribute__((aligned(16))) char rec[kKv8Record];
    const int kh = blockIdx.y;
    const int record = (a.first >> 5) + (int)blockIdx.x;
    const int p0 = record * 32;
    const int from = max(a.first - p0, 0), to = (int)min((int64_t)a.first + a.count - p0, (int64_t)32);  // its positions that are filed
    const int lane16 = threadIdx.x & 15;
    for (int layer = blockIdx.z; layer < a.layers; layer += gridDim.z) {
        __syncthreads();
#pragma unroll
        for (int turn = 0; turn < 4; ++turn) {
            const int which = turn >> 1;
            const int p = (turn & 1) * 16 + (int)(threadIdx.x >> 4);
            const int pc = max(from, min(p, to - 1));  // (rows that are not filed repeat one that is)
            const u32x4 w = *reinterpret_cast<const u32x4*>(a.rows[which] + layer * a.layer_elems + (p0 + (int64_t)pc) * a.row_stride + kh * a.head_stride + lane16 * 8);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max_u32(top, pair_magnitude(w[e]));
            const float s = kv8_scale<FORMAT>(row16_max(top));
            uint32_t c[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t w0 = w[2 * e], w1 = w[2 * e + 1];
                c[e] = kv8_codes<FORMAT>(bf16_lo(w0), bf16_hi(w0), bf16_lo(w1), bf16_hi(w1), s);
            }
            if (which == 0) {
                *reinterpret_cast<u32x2*>(rec + k_byte(p, lane16 * 8)) = u32x2{c[0], c[1]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) rec[v_byte(p, lane16 * 8 + e)] = (char)(c[e >> 2] >> (8 * (e & 3)));
            }
            if (lane16 == 0) *reinterpret_cast<uint16_t*>(rec + k_scale_byte(p) + 64 * which) = (uint16_t)(__builtin_bit_cast(uint32_t, s) >> 16);
        }
        __syncthreads();
        char* dst = a.cache + (((int64_t)layer * a.n_kv + kh) * a.records + record) * kKv8Record;
        if (from == 0 && to == 32) {
            for (int i = threadIdx.x; i < kKv8Record / 16; i += kCopyThreads) reinterpret_cast<u32x4*>(dst)[i] = reinterpret_cast<const u32x4*>(rec)[i];
            continue;
        }
        // A record that is filed in part: what belongs to its other positions stays as it is.
        for (int i = threadIdx.x; i < (to - from) * kHeadDim; i += kCopyThreads) {
            const int p = from + i / kHeadDim, c = i % kHeadDim;
            dst[k_byte(p, c)] = rec[k_byte(p, c)];
            dst[v_byte(p, c)] = rec[v_byte(p, c)];
            if (c < 2) {
                const int at = k_scale_byte(p) + 64 * c;
                *reinterpret_cast<uint16_t*>(dst + at) = *reinterpret_cast<const uint16_t*>(rec + at);
            }
        }
    }
}

template <int FORMAT>
__global__ __launch_bounds__(kCopyThreads) void kv8_load_kernel(CopyArgs a) {
    __shared__ __attribute__((aligned(16))) char rec[kKv8Record];
    const int kh = blockIdx.y;
    const int record = (a.first >> 5) + (int)blockIdx.x;
    const int p0 = record * 32;
    const int from = max(a.first - p0, 0), to = (int)min((int64_t)a.first + a.count - p0, (int64_t)32);
    const int lane16 = threadIdx.x & 15;
    for (int layer = blockIdx.z; layer < a.layers; layer += gridDim.z) {
        __syncthreads();
        const char* src = a.cache + (((int64_t)layer * a.n_kv + kh) * a.records + record) * kKv8Record;
        for (int i = threadIdx.x; i < kKv8Record / 16; i += kCopyThreads) reinterpret_cast<u32x4*>(rec)[i] = reinterpret_cast<const u32x4*>(src)[i];
        __syncthreads();
#pragma unroll
        for (int turn = 0; turn < 4; ++turn) {
            const int which = turn >> 1;
            const int p = (turn & 1) * 16 + (int)(threadIdx.x >> 4);
            uint32_t c[2] = {0u, 0u};
            if (which == 0) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(rec + k_byte(p, lane16 * 8));
                c[0] = w[0];
                c[1] = w[1];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) c[e >> 2] |= (uint32_t)(uint8_t)rec[v_byte(p, lane16 * 8 + e)] << (8 * (e & 3));
            }
            const float s = __builtin_bit_cast(float, (uint32_t)*reinterpret_cast<const uint16_t*>(rec + k_scale_byte(p) + 64 * which) << 16);
            u32x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t pair = (e & 1) ? kv8_pair<FORMAT, true>(c[e >> 1]) : kv8_pair<FORMAT, false>(c[e >> 1]);
                y[e] = pack_bf16(bf16_lo(pair) * s, bf16_hi(pair) * s);
            }
            if (p >= from && p < to)
                *reinterpret_cast<u32x4*>(a.rows[which] + layer * a.layer_elems + (p0 + (int64_t)p) * a.row_stride + kh * a.head_stride + lane16 * 8) = y;
        }
    }
}

CopyArgs copy_args(const llmi_kv8_copy_args& args) {
    CopyArgs a;
    const bool by_head = args.kv_layout == LLMI_KV_LAYOUT_HEAD_MAJOR;
    a.cache = static_cast<char*>(args.cache8);
    a.rows[0] = static_cast<uint16_t*>(args.key_cache);
    a.rows[1] = static_cast<uint16_t*>(args.value_cache);
    a.layer_elems = (int64_t)args.max_seq_len * args.kv_dim;
    a.row_stride = by_head ? kHeadDim : args.kv_dim;
    a.head_stride = by_head ? (int64_t)args.max_seq_len * kHeadDim : kHeadDim;
    a.records = kv8_records(args.max_seq_len);
    a.first = args.first_pos;
    a.count = args.num_pos;
    a.n_kv = args.kv_dim / kHeadDim;
    a.layers = args.layer_num;
    return a;
}

dim3 copy_grid(const llmi_kv8_copy_args& args) {
    const unsigned records = (unsigned)(((int64_t)args.first_pos + args.num_pos - 1) / 32 - args.first_pos / 32 + 1);
    return dim3(records, (unsigned)(args.kv_dim / kHeadDim), (unsigned)(args.layer_num < 65535 ? args.layer_num : 65535));
}

}  // namespace

int launch_kv8_store(const llmi_kv8_copy_args& args) {
    if (args.layer_num == 0 || args.num_pos == 0) return LLMI_OK;
    const CopyArgs a = copy_args(args);
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    if (args.format == LLMI_KV8_E4M3) hipLaunchKernelGGL((kv8_store_kernel<LLMI_KV8_E4M3>), copy_grid(args), dim3(kCopyThreads), 0, stream, a);
    else hipLaunchKernelGGL((kv8_store_kernel<LLMI_KV8_INT8>), copy_grid(args), dim3(kCopyThreads), 0, stream, a);
    return check_launch();
}

int launch_kv8_load(const llmi_kv8_copy_args& args) {
    if (args.layer_num == 0 || args.num_pos == 0) return LLMI_OK;
    const CopyArgs a = copy_args(args);
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    if (args.format == LLMI_KV8_E4M3) hipLaunchKernelGGL((kv8_load_kernel<LLMI_KV8_E4M3>), copy_grid(args), dim3(kCopyThreads), 0, stream, a);
    else hipLaunchKernelGGL((kv8_load_kernel<LLMI_KV8_INT8>), copy_grid(args), dim3(kCopyThreads), 0, stream, a);
    return check_launch();
}

int launch_qk_norm_rope_append_kv8(const llmi_qk_norm_rope_kv8_args& args) {
    const int64_t q_row = (int64_t)args.head_num * kHeadDim;
    RowsArgs a;
    a.query = static_cast<uint16_t*>(args.query);
    a.query_src = args.query_src ? static_cast<const uint16_t*>(args.query_src) : a.query;
    a.key_new = static_cast<const uint16_t*>(args.key_new);
    a.value_new = static_cast<const uint16_t*>(args.value_new);
    a.query_stride = args.query_stride ? args.query_stride : q_row;
    a.query_src_stride = !args.query_src ? a.query_stride : args.query_src_stride ? args.query_src_stride : q_row;
    a.key_new_stride = args.key_new_stride ? args.key_new_stride : args.kv_dim;
    a.value_new_stride = args.value_new_stride ? args.value_new_stride : args.kv_dim;
    a.n_kv = args.kv_dim / kHeadDim;
    a.records = kv8_records(args.max_seq_len);
    a.cache = static_cast<char*>(args.cache8) + (int64_t)args.layer_id * a.n_kv * a.records * kKv8Record;
    a.weight = static_cast<const uint16_t*>(args.norm_weight);
    a.sin_cache = args.sin_cache;
    a.cos_cache = args.cos_cache;
    a.pos_dev = args.pos_device;
    a.pos = args.pos;
    a.rows = args.row_num;
    a.head_num = args.head_num;
    a.eps = args.eps;
    const int per = kRowThreads / 32;
    const dim3 grid((unsigned)((args.head_num + 2 * a.n_kv + per - 1) / per), (unsigned)(args.row_num < 65535 ? args.row_num : 65535));
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    if (args.format == LLMI_KV8_E4M3) hipLaunchKernelGGL((kv8_append_kernel<LLMI_KV8_E4M3>), grid, dim3(kRowThreads), 0, stream, a);
    else hipLaunchKernelGGL((kv8_append_kernel<LLMI_KV8_INT8>), grid, dim3(kRowThreads), 0, stream, a);
    return check_launch();
}

}  // namespace llmi
