// Attention of a tree of drafted tokens over a KV cache on gfx950 (no counterpart in the reference, which decodes one token per
// step): for node i and query head h, with g query heads per KV head,
//   out[i][h] = sum_j w_j V[j][h/g] / sum_j w_j,   w_j = exp(q[i][h].K[j][h/g] / sqrt(128) - max),
// over the cached positions 0..pos-1 and the nodes t (slots pos + t) that node i's 64-bit word names.
//
// A workgroup takes one node and one query head: sixteen rows of sixteen lanes, each a running softmax of its own over every
// sixteenth key, merged at the end.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "llmi_internal.h"
#include "mha_device_helpers.h"

namespace llmi {
namespace {

struct TreeArgs {
    const uint16_t* q;          // [nodes][n_q][128]
    const uint16_t* k;          // layer base
    const uint16_t* v;
    uint16_t* out;              // [nodes][n_q][128]
    float* out_f32;             // optional
    const uint64_t* mask;       // optional
    const int32_t* pos_dev;     // optional
    int64_t row_stride;         // elements between positions of one KV head
    int64_t head_stride;        // elements between KV heads
    int32_t pos, nodes, group, n_q;
    float scale_log2e;          // log2(e) / sqrt(128)
};

constexpr int kStreams = 16;

__global__ __launch_bounds__(256) void mha_tree_kernel(TreeArgs a) {
    __shared__ float part_o[kStreams][kHeadDim];
    __shared__ float part_m[kStreams], part_l[kStreams];
    const int hq = blockIdx.x, node = blockIdx.y;
    const int kvh = hq / a.group;
    const int stream = threadIdx.x >> 4, c = threadIdx.x & 15;
    const int pos = a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos;
    const uint64_t sees = a.mask ? a.mask[node] : ~0ull >> (63 - node);
    const u32x4 q = reinterpret_cast<const u32x4*>(a.q + ((int64_t)node * a.n_q + hq) * kHeadDim)[c];
    const uint16_t* kp = a.k + kvh * a.head_stride;
    const uint16_t* vp = a.v + kvh * a.head_stride;
    float m = -FLT_MAX, l = 0.0f, o[8] = {};  // (a finite maximum: scores of -inf get weight 0, not NaN)
    for (int j = stream; j < pos + a.nodes; j += kStreams) {
        if (j >= pos && !(sees >> (j - pos) & 1)) continue;
        const u32x4 kv = reinterpret_cast<const u32x4*>(kp + j * a.row_stride)[c];
        const u32x4 vv = reinterpret_cast<const u32x4*>(vp + j * a.row_stride)[c];
        float s = dot8_bf16(kv, q, 0.0f);
        s += dpp_partner<0xB1>(s);
        s += dpp_partner<0x4E>(s);
        s += dpp_partner<0x141>(s);
        s += dpp_partner<0x140>(s);
        s *= a.scale_log2e;
        const float m_new = fmaxf(m, s);
        const float alpha = fast_exp2(m - m_new), p = fast_exp2(s - m_new);
        m = m_new;
        l = l * alpha + p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = vv[e];
            o[2 * e] = o[2 * e] * alpha + p * bf16_lo(w);
            o[2 * e + 1] = o[2 * e + 1] * alpha + p * bf16_hi(w);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) part_o[stream][8 * c + e] = o[e];
    if (c == 0) {
        part_m[stream] = m;
        part_l[stream] = l;
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= kHeadDim) return;
    float top = part_m[0];
    for (int i = 1; i < kStreams; ++i) top = fmaxf(top, part_m[i]);
    float sum = 0.0f, num = 0.0f;
    for (int i = 0; i < kStreams; ++i) {
        const float w = fast_exp2(part_m[i] - top);
        sum += w * part_l[i];
        num += w * part_o[i][d];
    }
    const float r = sum == 0.0f ? 0.0f : num / sum;  // (no key: zeros)
    const int64_t at = ((int64_t)node * a.n_q + hq) * kHeadDim + d;
    a.out[at] = f32_to_bf16(r);
    if (a.out_f32) a.out_f32[at] = r;
}

}  // namespace

int launch_mha_tree(const llmi_mha_tree_args& args, const llmi_mha_plan&) {
    const llmi_mha_args& m = args.mha;
    TreeArgs a;
    const int64_t layer = (int64_t)m.layer_id * m.max_seq_len * m.kv_dim;
    a.q = static_cast<const uint16_t*>(m.query);
    a.k = static_cast<const uint16_t*>(m.key_cache) + layer;
    a.v = static_cast<const uint16_t*>(m.value_cache) + layer;
    a.out = static_cast<uint16_t*>(m.output);
    a.out_f32 = m.output_f32;
    a.mask = args.tree_mask;
    a.pos_dev = m.pos_device;
    const bool by_head = m.kv_layout == LLMI_KV_LAYOUT_HEAD_MAJOR;
    a.row_stride = by_head ? kHeadDim : m.kv_dim;
    a.head_stride = by_head ? (int64_t)m.max_seq_len * kHeadDim : kHeadDim;
    a.pos = m.pos;
    a.nodes = args.node_num;
    a.group = m.kv_mul;
    a.n_q = m.head_num;
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)kHeadDim);
    hipLaunchKernelGGL(mha_tree_kernel, dim3(m.head_num, args.node_num), dim3(256), 0, static_cast<hipStream_t>(m.stream), a);
    return check_launch();
}

}  // namespace llmi
