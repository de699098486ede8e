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
    uint32_t record_groups;  // many rows: workgroups that have a record
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
    int32_t touched;     // records of a KV head that have positions of the call
    bool by_head;
};

// A workgroup per record of a KV head. Wavefront w has sixteen positions, 16 (w % 2) and on, of K (w < 2) or V; lane L of it the channels 8 (L % 16) .. + 7
// of four of them, 4 (L / 16) .. + 3: rows are read (written) whole, 256 bytes over sixteen lanes, a lane's four positions are the bytes of V's words (two
// rounds of v_perm), and what a row needs once (scale, reciprocal) is worked out for one row a lane and handed round the four neighbours. The record
// passes through LDS, where its blocks of 256 bytes are 272 apart: eight times fewer bank conflicts. Both ways past the caches, as in kv_restride.
constexpr int kCopyThreads = 256;
template <bool STREAM>
__device__ __forceinline__ u32x4 load_chunk(const u32x4* p) {
    return STREAM ? __builtin_nontemporal_load(p) : *p;
}
constexpr int kLdsScales = 32 * 272;
__device__ __forceinline__ int in_lds(int byte) { return byte + (byte >> 8) * 16; }  // (of codes)
// A record from LDS to where it belongs, positions from .. to - 1 of it.
__device__ __forceinline__ void write_record(char* dst, const char* rec, int from, int to) {
    const auto chunk = [&](int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const u32x4*>(rec + (i < 512 ? in_lds(16 * i) : kLdsScales - kScaleBytes + 16 * i));
    };
    if (from == 0 && to == 32) {
        for (int i = threadIdx.x; i < kKv8Record / 16; i += kCopyThreads) __builtin_nontemporal_store(chunk(i), reinterpret_cast<u32x4*>(dst) + i);
        return;
    }
    // In part: what belongs to its other positions stays as it is. Sixteen bytes of K are a position's, words of V belong to four, halfwords of
    // scales to one.
    const auto filed = [&](int p) __attribute__((always_inline)) { return p >= from && p < to; };
    for (int i = threadIdx.x; i < kKv8Record / 16; i += kCopyThreads) {
        const u32x4 x = chunk(i);
        if (i < 256) {
            if (filed(16 * (i >> 7) + (i & 15))) reinterpret_cast<u32x4*>(dst)[i] = x;
        } else if (i < 512) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = 16 * (e & 1) + 4 * ((i >> 4) & 3);
                char* word = dst + 16 * i + 4 * e;
                if (p >= from && p + 3 < to) {
                    *reinterpret_cast<uint32_t*>(word) = x[e];
                    continue;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (filed(p + j)) word[j] = (char)(x[e] >> (8 * j));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (filed(16 * (e >> 2) + 4 * (i & 3) + (e & 3))) reinterpret_cast<uint16_t*>(dst)[8 * i + e] = (uint16_t)(x[e >> 1] >> (16 * (e & 1)));
        }
    }
}

struct CopyPlace {
    int kh, record, from, to;     // positions from .. to - 1 of the record are the call's
    int which, p0, c0;            // the lane's first position and channel
};
__device__ __forceinline__ CopyPlace copy_place(const CopyArgs& a) {
    CopyPlace x;
    // (neighbours where the bf16 cache has its rows side by side)
    const uint32_t b = blockIdx.x, along = a.by_head ? (uint32_t)a.touched : (uint32_t)a.n_kv, far = b / along, near = b - far * along;
    x.kh = (int)(a.by_head ? far : near);
    x.record = (a.first >> 5) + (int)(a.by_head ? near : far);
    x.from = max(a.first - x.record * 32, 0);
    x.to = (int)min((int64_t)a.first + a.count - (int64_t)x.record * 32, (int64_t)32);
    const int wave = (int)(threadIdx.x >> 6), lane = (int)(threadIdx.x & 63);
    x.which = wave >> 1;
    x.p0 = 16 * (wave & 1) + 4 * (lane >> 4);
    x.c0 = 8 * (lane & 15);
    return x;
}

template <int FORMAT, bool STREAM>
__global__ __launch_bounds__(kCopyThreads) void kv8_store_kernel(CopyArgs a) {
    __shared__ __attribute__((aligned(16))) char rec[kLdsScales + 128];
    const CopyPlace at = copy_place(a);
    const int kh = at.kh;
    const int l4 = (int)(threadIdx.x & 3);
    const uint16_t* src = (at.which ? a.rows[1] : a.rows[0]) + (int64_t)at.record * 32 * a.row_stride + kh * a.head_stride + at.c0;
    int32_t row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = max(at.from, min(at.p0 + i, at.to - 1));  // (rows that are not filed repeat one that is)
    for (int layer = blockIdx.y; layer < a.layers; layer += gridDim.y) {
        if (layer != (int)blockIdx.y) __syncthreads();
        u32x4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = load_chunk<STREAM>(reinterpret_cast<const u32x4*>(src + layer * a.layer_elems + (int64_t)row[i] * a.row_stride));
        uint32_t top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            top[i] = row16_max(max_u32(max_u32(pair_magnitude(w[i][0]), pair_magnitude(w[i][1])), max_u32(pair_magnitude(w[i][2]), pair_magnitude(w[i][3]))));
        const float s_mine = kv8_scale<FORMAT>(l4 < 2 ? (l4 == 0 ? top[0] : top[1]) : (l4 == 2 ? top[2] : top[3])), r_mine = 1.0f / s_mine;
        const float s[4] = {quad_lane<0>(s_mine), quad_lane<1>(s_mine), quad_lane<2>(s_mine), quad_lane<3>(s_mine)};
        const float r[4] = {quad_lane<0>(r_mine), quad_lane<1>(r_mine), quad_lane<2>(r_mine), quad_lane<3>(r_mine)};
        uint32_t c[2][4];  // four channels' codes of the four rows
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t w0 = w[i][2 * e], w1 = w[i][2 * e + 1];
                c[e][i] = kv8_codes<FORMAT>(bf16_lo(w0), bf16_hi(w0), bf16_lo(w1), bf16_hi(w1), s[i], r[i]);
            }
        if (at.which == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x2*>(rec + in_lds(k_byte(at.p0 + i, at.c0))) = u32x2{c[0][i], c[1][i]};
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t v[4];
                transpose_bytes(c[e], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(rec + in_lds(v_byte(at.p0, at.c0 + 4 * e + j))) = v[j];
            }
        }
        if ((threadIdx.x & 12) == 0)
            *reinterpret_cast<uint16_t*>(rec + kLdsScales - kScaleBytes + k_scale_byte(at.p0 + l4) + 64 * at.which) = (uint16_t)(__builtin_bit_cast(uint32_t, s_mine) >> 16);
        __syncthreads();
        write_record(a.cache + (((int64_t)layer * a.n_kv + kh) * a.records + at.record) * kKv8Record, rec, at.from, at.to);
    }
}

template <int FORMAT, bool STREAM>
__global__ __launch_bounds__(kCopyThreads) void kv8_load_kernel(CopyArgs a) {
    __shared__ __attribute__((aligned(16))) char rec[kLdsScales + 128];
    const CopyPlace at = copy_place(a);
    const int kh = at.kh;
    uint16_t* dst = (at.which ? a.rows[1] : a.rows[0]) + (int64_t)at.record * 32 * a.row_stride + kh * a.head_stride + at.c0;
    for (int layer = blockIdx.y; layer < a.layers; layer += gridDim.y) {
        if (layer != (int)blockIdx.y) __syncthreads();
        const char* src = a.cache + (((int64_t)layer * a.n_kv + kh) * a.records + at.record) * kKv8Record;
        {
            // (all of a thread's loads before the first is waited for)
            const int i = (int)threadIdx.x;
            const u32x4* from = reinterpret_cast<const u32x4*>(src);
            const u32x4 x0 = load_chunk<STREAM>(from + i), x1 = load_chunk<STREAM>(from + i + 256);
            u32x4 x2{};
            if (i < 8) x2 = load_chunk<STREAM>(from + i + 512);
            *reinterpret_cast<u32x4*>(rec + in_lds(16 * i)) = x0;
            *reinterpret_cast<u32x4*>(rec + in_lds(16 * i + 4096)) = x1;
            if (i < 8) *reinterpret_cast<u32x4*>(rec + kLdsScales + 16 * i) = x2;
        }
        __syncthreads();
        uint32_t c[2][4];
        if (at.which == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(rec + in_lds(k_byte(at.p0 + i, at.c0)));
                c[0][i] = w[0];
                c[1][i] = w[1];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(rec + in_lds(v_byte(at.p0, at.c0 + 4 * e + j)));
                transpose_bytes(v, c[e]);
            }
        }
        const u32x2 scales = *reinterpret_cast<const u32x2*>(rec + kLdsScales - kScaleBytes + k_scale_byte(at.p0) + 64 * at.which);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t sw = scales[i >> 1];
            const float s = (i & 1) ? bf16_hi(sw) : bf16_lo(sw);
            u32x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t pair = (e & 1) ? kv8_pair<FORMAT, true>(c[e >> 1][i]) : kv8_pair<FORMAT, false>(c[e >> 1][i]);
                y[e] = pack_bf16(bf16_lo(pair) * s, bf16_hi(pair) * s);
            }
            const int p = at.p0 + i;
            if (p >= at.from && p < at.to) __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(dst + layer * a.layer_elems + (int64_t)p * a.row_stride));
        }
    }
}

// The rows of many tokens. The first workgroups, whose way is the longest, have a record of a KV head each as kv8_store has: wavefront w sixteen positions
// of K (w < 2) or V, a lane four of them; the others a token's queries each, sixteen lanes a row, the weights, sines and cosines in registers for all of a
// wavefront's.
template <int FORMAT>
__global__ __launch_bounds__(kCopyThreads) void kv8_append_many_kernel(RowsArgs a) {
    __shared__ __attribute__((aligned(16))) char rec[kLdsScales + 128];
    const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6), l16 = lane & 15, l4 = lane & 3;
    const int base = a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos;
    const u32x2* weight = reinterpret_cast<const u32x2*>(a.weight);
    if (blockIdx.x >= a.record_groups) {
        const int row = (int)(blockIdx.x - a.record_groups);
        const int64_t table = (int64_t)(base + row) * 64 + 4 * l16;
        const u32x2 wl = weight[l16], wh = weight[l16 + 16];
        const f32x4 sn = *reinterpret_cast<const f32x4*>(a.sin_cache + table), cs = *reinterpret_cast<const f32x4*>(a.cos_cache + table);
        const u32x2* src = reinterpret_cast<const u32x2*>(a.query_src + row * a.query_src_stride);
        u32x2* dst = reinterpret_cast<u32x2*>(a.query + row * a.query_stride);
        for (int h = (int)(threadIdx.x >> 4); h < a.head_num; h += kCopyThreads / 16) {
            u32x2 lo = src[h * 32 + l16], hi = src[h * 32 + 16 + l16];
            norm_rope_regs16(lo, hi, wl, wh, sn, cs, a.eps);
            dst[h * 32 + l16] = lo;
            dst[h * 32 + 16 + l16] = hi;
        }
        return;
    }
    const int b = (int)blockIdx.x, record = base / 32 + b / a.n_kv, kh = b % a.n_kv;
    const int from = max(base - record * 32, 0), to = min(base + a.rows - record * 32, 32);  // (max_seq_len bounds both sums)
    if (to <= 0) return;  // (a position read on the device needs a record less than the launch has room for, perhaps)
    const bool is_v = wave >> 1;
    const int p0 = 16 * (wave & 1) + 4 * (lane >> 4), c0 = 4 * l16;
    u32x2 lo[4], hi[4];
    int64_t row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        row[i] = record * 32 + max(from, min(p0 + i, to - 1)) - base;  // (rows that are not filed repeat one that is)
        const uint16_t* src = (is_v ? a.value_new + row[i] * a.value_new_stride : a.key_new + row[i] * a.key_new_stride) + kh * kHeadDim;
        lo[i] = reinterpret_cast<const u32x2*>(src)[l16];
        hi[i] = reinterpret_cast<const u32x2*>(src)[l16 + 16];
    }
    if (!is_v) {
        const u32x2 wl = weight[32 + l16], wh = weight[48 + l16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t table = (base + row[i]) * 64 + 4 * l16;
            norm_rope_regs16(lo[i], hi[i], wl, wh, *reinterpret_cast<const f32x4*>(a.sin_cache + table), *reinterpret_cast<const f32x4*>(a.cos_cache + table), a.eps);
        }
    }
    uint32_t top[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        top[i] = row16_max(max_u32(max_u32(pair_magnitude(lo[i][0]), pair_magnitude(lo[i][1])), max_u32(pair_magnitude(hi[i][0]), pair_magnitude(hi[i][1]))));
    const float s_mine = kv8_scale<FORMAT>(l4 < 2 ? (l4 == 0 ? top[0] : top[1]) : (l4 == 2 ? top[2] : top[3])), r_mine = 1.0f / s_mine;
    const float s[4] = {quad_lane<0>(s_mine), quad_lane<1>(s_mine), quad_lane<2>(s_mine), quad_lane<3>(s_mine)};
    const float r[4] = {quad_lane<0>(r_mine), quad_lane<1>(r_mine), quad_lane<2>(r_mine), quad_lane<3>(r_mine)};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w0 = e ? hi[i][0] : lo[i][0], w1 = e ? hi[i][1] : lo[i][1];
            c[i] = kv8_codes<FORMAT>(bf16_lo(w0), bf16_hi(w0), bf16_lo(w1), bf16_hi(w1), s[i], r[i]);
        }
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(rec + in_lds(k_byte(p0 + i, c0 + 64 * e))) = c[i];
        } else {
            uint32_t v[4];
            transpose_bytes(c, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(rec + in_lds(v_byte(p0, c0 + 64 * e + j))) = v[j];
        }
    }
    if ((lane & 12) == 0)
        *reinterpret_cast<uint16_t*>(rec + kLdsScales - kScaleBytes + k_scale_byte(p0 + l4) + 64 * is_v) = (uint16_t)(__builtin_bit_cast(uint32_t, s_mine) >> 16);
    __syncthreads();
    write_record(a.cache + (kh * a.records + record) * kKv8Record, rec, from, to);
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
    a.touched = (int32_t)(((int64_t)args.first_pos + args.num_pos - 1) / 32 - args.first_pos / 32 + 1);
    a.by_head = by_head;
    return a;
}

dim3 copy_grid(const CopyArgs& a) { return dim3((unsigned)a.touched * (unsigned)a.n_kv, (unsigned)(a.layers < 65535 ? a.layers : 65535)); }

// Whether what the call reads is more than the memory-side cache may still hold of what was written last (a prompt's prefill, the last step's rows): past
// the caches then. us, cached loads : past them: 57 MB stored 15.5 : 17.4, 557 MB 146.6 : 134.9; 12 MB read back 6.8 : 7.6, 283 MB 148.0 : 145.7.
// (What is written goes past them at every size: 57 MB stored 16.6 : 15.5, 12 MB read back 8.6 : 6.8 with cached stores : without, large ones 155.0 : 146.6, 157.6 : 148.0.)
constexpr int64_t kStreamFrom = 128 << 20;
bool streams(const llmi_kv8_copy_args& args, int64_t row_bytes) { return (int64_t)args.layer_num * args.num_pos * (args.kv_dim / kHeadDim) * row_bytes > kStreamFrom; }

using CopyKernel = void (*)(CopyArgs);
void launch_copy(const CopyArgs& a, hipStream_t stream, int format, bool past, CopyKernel e4m3, CopyKernel e4m3_past, CopyKernel whole, CopyKernel whole_past) {
    const CopyKernel kernel = format == LLMI_KV8_E4M3 ? (past ? e4m3_past : e4m3) : (past ? whole_past : whole);
    hipLaunchKernelGGL(kernel, copy_grid(a), dim3(kCopyThreads), 0, stream, a);
}

}  // namespace

int launch_kv8_store(const llmi_kv8_copy_args& args) {
    const CopyArgs a = copy_args(args);
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    launch_copy(a, stream, args.format, streams(args, 2 * 256), kv8_store_kernel<LLMI_KV8_E4M3, false>, kv8_store_kernel<LLMI_KV8_E4M3, true>, kv8_store_kernel<LLMI_KV8_INT8, false>,
                kv8_store_kernel<LLMI_KV8_INT8, true>);
    return check_launch();
}

int launch_kv8_load(const llmi_kv8_copy_args& args) {
    const CopyArgs a = copy_args(args);
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    launch_copy(a, stream, args.format, streams(args, 2 * 130), kv8_load_kernel<LLMI_KV8_E4M3, false>, kv8_load_kernel<LLMI_KV8_E4M3, true>, kv8_load_kernel<LLMI_KV8_INT8, false>,
                kv8_load_kernel<LLMI_KV8_INT8, true>);
    return check_launch();
}

// Tokens from which a record is put together by a workgroup: half a wavefront a row, which scatters V's bytes, has the shorter way. us, half a wavefront a row :
// records, 32 Q / 8 KV heads: 2.3 : 4.3 with 1 token, 3.2 : 4.7 with 40, 5.95 : 5.94 with 300, 12.3 : 8.6 with 1001; 64 Q heads 16.7 : 11.6, 16 Q 11.5 : 8.0.
// (E4M3; E4M3 : whole numbers 2.25 : 2.25 with 1, 2.99 : 2.96 with 40, 5.77 : 5.77 with 300, 8.62 : 8.78 with 1001.)
constexpr int kManyRows = 384;
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
    // (at a position on the device the rows may begin anywhere in a record)
    const int64_t records = args.pos_device ? ((int64_t)args.row_num + 30) / 32 + 1 : ((int64_t)args.pos + args.row_num - 1) / 32 - args.pos / 32 + 1;
    if (args.row_num >= kManyRows && args.row_num + records * a.n_kv <= kKv8MostGroups) {
        a.record_groups = (uint32_t)(records * a.n_kv);
        const dim3 grid((unsigned)args.row_num + a.record_groups);
        if (args.format == LLMI_KV8_E4M3) hipLaunchKernelGGL((kv8_append_many_kernel<LLMI_KV8_E4M3>), grid, dim3(kCopyThreads), 0, static_cast<hipStream_t>(args.stream), a);
        else hipLaunchKernelGGL((kv8_append_many_kernel<LLMI_KV8_INT8>), grid, dim3(kCopyThreads), 0, static_cast<hipStream_t>(args.stream), a);
        return check_launch();
    }
    const int per = kRowThreads / 32;
    const dim3 grid((unsigned)((args.head_num + 2 * a.n_kv + per - 1) / per), (unsigned)(args.row_num < 65535 ? args.row_num : 65535));
    const hipStream_t stream = static_cast<hipStream_t>(args.stream);
    if (args.format == LLMI_KV8_E4M3) hipLaunchKernelGGL((kv8_append_kernel<LLMI_KV8_E4M3>), grid, dim3(kRowThreads), 0, stream, a);
    else hipLaunchKernelGGL((kv8_append_kernel<LLMI_KV8_INT8>), grid, dim3(kRowThreads), 0, stream, a);
    return check_launch();
}

}  // namespace llmi
