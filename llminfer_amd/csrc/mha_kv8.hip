// Decode attention of one token over an 8-bit KV cache on gfx950 (layout and codes: kv8.h): for query head h of KV head k
//   out[h] = sum_j w_j s'_j V_j / sum_j w_j,   w_j = exp(s_j q[h].K_j / sqrt(128) - max),
// over the positions 0..pos, K_j and V_j the codes, s_j and s'_j their scales; with the new token's rows normalised, rotated, quantised and
// filed first, in the same launch, where the caller asks for that.
//
// A wavefront takes a record of 32 positions at a time, ten loads of 1 KiB (the scales: 64 bytes) straight into registers, in the order in
// which the two products want them. Both run on the matrix cores in the transposed form, S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_16x16x32_bf16, the query
// heads of the KV head as the sixteen columns; columns behind the group repeat its last head): a lane has eight positions of one head,
//   S^T  lane L: head L%16, position 16 t + 4 (L/16) + r in register r of product t
//   P^T  lane L: those eight, place 8 (L/16) + 4 t + r          V^T  lane L: channel 16 b + L%16, the same positions: eight bytes of the record
//   O^T  lane L: head L%16, channel 16 b + 4 (L/16) + r in register r of accumulator b = 0..7
// so that the probabilities never leave their lane. Codes become bf16 on the way (exact); K's scale multiplies the score, V's the probability,
// which enters the product as the sum of two bf16 numbers (2^-16 of it lost at most). Maximum, sum and accumulators are fp32; the accumulators are
// rescaled only where a maximum has grown by more than 2^8.
//
// Records are dealt to the splits (workgroups of a KV head) and their wavefronts in turn. The workgroup of the last split joins the others inside the launch:
// every split leaves its partial outputs and, once they are acknowledged, a record {tag | maximum} {tag | sum} per head in the workspace, past the
// caches; the last one, which is dispatched behind the others, waits for those (bounded) and adds the parts up.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "kv8.h"
#include "llmi_internal.h"
#include "mha_device_helpers.h"

namespace llmi {
namespace {

constexpr int kHeads = 16;  // columns of the products

struct Kv8Args {
    const uint16_t* q;            // [n_q][128]; the raw rows where the new token's are filed too
    const char* cache;            // the layer's records
    float* ws;                    // partial outputs [n_q][splits][128]
    unsigned long long* arrivals; // [n_q][splits][2]
    uint16_t* out;
    float* out_f32;               // optional
    const int32_t* pos_dev;       // optional
    int64_t records;              // per KV head
    uint32_t tag;
    int32_t pos, group, n_q, splits, max_polls;
    float scale_log2e;            // log2(e) / sqrt(128)
    // the new token's
    const uint16_t* k_new;
    const uint16_t* v_new;
    const uint16_t* norm_w;
    const float* sin_cache;
    const float* cos_cache;
    float eps;
};

struct Record {
    u32x4 k[4], v[4], ks, vs;
};

// Streaming loads: nobody reads a record twice.
constexpr int kStream = 2;
__device__ __forceinline__ Record load_record(const char* at, uint32_t bytes, uint32_t lane) {
    // (a record that there is not: zeros, and nothing read)
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at), 0, bytes, 0x00020000);
    Record y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y.k[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16u, i * 1024, kStream));
    y.ks = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (lane >> 4) * 16u, kScaleBytes, kStream));
    y.vs = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (lane >> 4) * 16u, kScaleBytes + 64, kStream));
#pragma unroll
    for (int i = 0; i < 4; ++i) y.v[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane * 16u, kVBytes + i * 1024, kStream));
    return y;
}

template <int FORMAT, int NW, bool APPEND>
__global__ __launch_bounds__(NW * 64, 2) void mha_kv8_kernel(Kv8Args a) {
    constexpr int kAhead = 2;  // records in flight
    __shared__ __attribute__((aligned(16))) float parts[NW][kHeads][kHeadDim];
    __shared__ float part_m[kHeads][NW], part_l[kHeads][NW];
    __shared__ float weights[NW][kMaxSplits];
    __shared__ float fin[kHeads][2];
    __shared__ __attribute__((aligned(16))) uint16_t rows[APPEND ? kHeads : 1][kHeadDim];
    __shared__ __attribute__((aligned(16))) uint8_t new_codes[APPEND ? 2 : 1][kHeadDim];
    __shared__ float new_scale[2];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x, split = blockIdx.y;

    const int pos = __builtin_amdgcn_readfirstlane(a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos);
    const int64_t keys = (int64_t)pos + (APPEND ? 0 : 1);  // positions that come from the cache
    const int tiles = (int)((keys + 31) >> 5);
    const int active = max(1, min(a.splits, (tiles + NW - 1) / NW));
    if (split >= active) return;
    const bool last = split == active - 1;
    const char* head = a.cache + (int64_t)kvh * a.records * kKv8Record;
    const int step = active * NW, t0 = split * NW + wave;
    const int count = t0 < tiles ? (tiles - t0 + step - 1) / step : 0;
    auto fetch = [&](int i) __attribute__((always_inline)) {
        const int64_t t = t0 + (int64_t)i * step;
        return load_record(head + (i < count ? t : 0) * kKv8Record, i < count ? (uint32_t)kKv8Record : 0u, (uint32_t)lane);
    };

    // The new token's rows, half a wavefront each: the query heads, in the last split K and V behind them.
    const int half = threadIdx.x >> 5, p32 = lane & 31;
    const int work_rows = a.group + (last ? 2 : 0);
    if constexpr (APPEND) {
        for (int row = half; row < work_rows; row += 2 * NW) {
            const bool is_new = row >= a.group, is_v = row > a.group;
            const uint16_t* src = is_v ? a.v_new + kvh * kHeadDim : is_new ? a.k_new + kvh * kHeadDim : a.q + (int64_t)(kvh * a.group + row) * kHeadDim;
            const NewRow y = load_row32(src, a.norm_w + (is_new ? kHeadDim : 0), a.sin_cache + (int64_t)pos * 64, a.cos_cache + (int64_t)pos * 64, p32);
            uint32_t lo, hi;
            norm_rope_regs32(y, p32, a.eps, lo, hi);
            if (is_v) {
                lo = y.x[0];
                hi = y.x[1];
            }
            if (is_new) {
                float s;
                const uint32_t codes = quantise_row32<FORMAT>(lo, hi, s);
                file_row32(const_cast<char*>(head) + (int64_t)(pos >> 5) * kKv8Record, pos & 31, is_v, p32, codes, s);
                reinterpret_cast<uint16_t*>(new_codes[is_v])[p32] = (uint16_t)codes;
                reinterpret_cast<uint16_t*>(new_codes[is_v])[p32 + 32] = (uint16_t)(codes >> 16);
                if (p32 == 0) new_scale[is_v] = s;
            } else {
                reinterpret_cast<uint32_t*>(rows[row])[p32] = lo;
                reinterpret_cast<uint32_t*>(rows[row])[p32 + 32] = hi;
            }
        }
    }
    Record ring[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ring[i] = fetch(i);
    if constexpr (APPEND) __syncthreads();

    // The query heads: step s of the first product has channels 64 (s/2) + 16 g + 8 (s%2) .. + 7 in lane group g.
    u32x4 q[4];
    {
        const int hq = min(n, a.group - 1);
        const uint16_t* src = APPEND ? rows[hq] : a.q + (int64_t)(kvh * a.group + hq) * kHeadDim;
#pragma unroll
        for (int s = 0; s < 4; ++s) q[s] = *reinterpret_cast<const u32x4*>(src + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
    }
    float m_run = -FLT_MAX, l_run = 0.0f;  // (a finite maximum: scores of -inf get weight 0, not NaN)
    f32x4 o[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) o[b] = f32x4{};

    if constexpr (APPEND) {
        // The new token, as its codes stand for it, with weight 1.
        if (last && wave == 0) {
            const float ks = new_scale[0], vs = new_scale[1];
            f32x4 c{};
            // (all sixteen positions of the product are the new one)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(new_codes[0] + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand<FORMAT>(w[0], w[1]), __builtin_bit_cast(bf16x8, q[s]), c, 0, 0, 0);
            }
            const float s = c[0] * (ks * a.scale_log2e);
            m_run = fmaxf(m_run, s);
            const float w = fast_exp2(s - m_run);
            l_run = g == 0 ? w : 0.0f;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(new_codes[1] + 16 * b + 4 * g);
                const uint32_t v0 = kv8_pair<FORMAT, false>(v), v1 = kv8_pair<FORMAT, true>(v);
                const float ws = w * vs;
                o[b] = f32x4{bf16_lo(v0) * ws, bf16_hi(v0) * ws, bf16_lo(v1) * ws, bf16_hi(v1) * ws};
            }
        }
    }

    auto fold = [&](Record& r, int64_t t) __attribute__((always_inline)) {
        float c[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4 x{};
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const u32x4 w = r.k[2 * u + (s >> 1)];
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand<FORMAT>(w[2 * (s & 1)], w[2 * (s & 1) + 1]), __builtin_bit_cast(bf16x8, q[s]), x, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) c[4 * u + e] = x[e];
        }
        float vs[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t kw = r.ks[e >> 1], vw = r.vs[e >> 1];
            c[e] *= ((e & 1) ? bf16_hi(kw) : bf16_lo(kw)) * a.scale_log2e;
            vs[e] = (e & 1) ? bf16_hi(vw) : bf16_lo(vw);
        }
        if (t == tiles - 1 && (keys & 31)) {
            // The last record, not full: what lies behind the last position has no weight whatever it is.
            const int left = (int)(keys & 31) - 4 * g;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool there = 16 * (e >> 2) + (e & 3) < left;
                c[e] = there ? c[e] : -INFINITY;
                vs[e] = there ? vs[e] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int bytes = min(max(left - 16 * u, 0), 4);
                const uint32_t mask = bytes == 4 ? ~0u : (1u << (8 * bytes)) - 1u;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    r.v[i][u] &= mask;
                    r.v[i][2 + u] &= mask;
                }
            }
        }
        float top = c[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, c[e]);
        top = rows_max(top);
        if (__any(top > m_run + 8.0f)) {
            const float m_new = fmaxf(m_run, top);
            const float alpha = fast_exp2(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int b = 0; b < 8; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][e] *= alpha;
        }
        u32x4 ph, pl;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(c[2 * e] - m_run), p1 = fast_exp2(c[2 * e + 1] - m_run);
            l_run += p0 + p1;
            const float x0 = p0 * vs[2 * e], x1 = p1 * vs[2 * e + 1];
            const uint32_t w = pack_bf16(x0, x1);
            ph[e] = w;
            pl[e] = pack_bf16(x0 - bf16_lo(w), x1 - bf16_hi(w));
        }
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const bf16x8 v = kv8_operand<FORMAT>(r.v[b >> 1][2 * (b & 1)], r.v[b >> 1][2 * (b & 1) + 1]);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, ph), o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, pl), o[b], 0, 0, 0);
        }
    };
    for (int i = 0; i < count; i += kAhead) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            if (i + d >= count) break;
            fold(ring[d], t0 + (int64_t)(i + d) * step);
            ring[d] = fetch(i + d + kAhead);
        }
    }

    // The workgroup's wavefronts.
    l_run = rows_sum(l_run);
    if (n < a.group) {
#pragma unroll
        for (int b = 0; b < 8; ++b) *reinterpret_cast<f32x4*>(&parts[wave][n][16 * b + 4 * g]) = o[b];
        if (g == 0) {
            part_m[n][wave] = m_run;
            part_l[n][wave] = l_run;
        }
    }
    __syncthreads();
    const int S = a.splits;
    const int64_t part_bytes = (int64_t)a.n_q * S * kHeadDim * (int64_t)sizeof(float);
    const __amdgpu_buffer_rsrc_t part_rsrc = __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, (int)part_bytes, 0x00020000);
    auto write_out = [&](int hq, int c4, f32x4 x) __attribute__((always_inline)) {
        *reinterpret_cast<u32x2*>(a.out + (int64_t)hq * kHeadDim + 4 * c4) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
        if (a.out_f32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a.out_f32[(int64_t)hq * kHeadDim + 4 * c4 + e] = x[e];
        }
    };
    for (int u = threadIdx.x; u < a.group * 32; u += NW * 64) {
        const int h = u >> 5, c4 = u & 31, hq = kvh * a.group + h;
        float m = part_m[h][0];
#pragma unroll
        for (int w = 1; w < NW; ++w) m = fmaxf(m, part_m[h][w]);
        f32x4 x{};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = fast_exp2(part_m[h][w] - m);
            sum += f * part_l[h][w];
            const f32x4 y = *reinterpret_cast<const f32x4*>(&parts[w][h][4 * c4]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += f * y[e];
        }
        if (active == 1) {
            const float r = 1.0f / sum;
            write_out(hq, c4, f32x4{x[0] * r, x[1] * r, x[2] * r, x[3] * r});
            continue;
        }
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), part_rsrc, (uint32_t)(((hq * S + split) * kHeadDim + 4 * c4) * 4), 0, kCacheDevice);
        if (last) {
            if (c4 == 0) {
                fin[h][0] = m;
                fin[h][1] = sum;
            }
            continue;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a head's 32 columns are half a wavefront's)
        if (c4 == 0) {
            unsigned long long* to = a.arrivals + ((int64_t)hq * S + split) * 2;
            const unsigned long long tag = a.tag;
            __hip_atomic_store(to, tag | (unsigned long long)__builtin_bit_cast(uint32_t, m) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(to + 1, tag | (unsigned long long)__builtin_bit_cast(uint32_t, sum) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (active == 1 || !last) return;

    // The last split's workgroup: a wavefront a head.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int h = wave; h < a.group; h += NW) {
        const int hq = kvh * a.group + h;
        constexpr int kSlots = kMaxSplits / 64;
        float ms[kSlots], ls[kSlots];
        unsigned long long* from = a.arrivals + (int64_t)hq * S * 2;
        bool in = false;
        for (int spin = 0; spin < a.max_polls && !in; ++spin) {
            bool ok = true;
#pragma unroll
            for (int j = 0; j < kSlots; ++j) {
                const int s = lane + 64 * j;
                ms[j] = -FLT_MAX;
                ls[j] = 0.0f;
                if (s >= active) continue;
                if (s == split) {
                    ms[j] = fin[h][0];
                    ls[j] = fin[h][1];
                    continue;
                }
                const unsigned long long r0 = __hip_atomic_load(from + 2 * s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const unsigned long long r1 = __hip_atomic_load(from + 2 * s + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                ok = ok && (uint32_t)r0 == a.tag && (uint32_t)r1 == a.tag;
                ms[j] = __builtin_bit_cast(float, (uint32_t)(r0 >> 32));
                ls[j] = __builtin_bit_cast(float, (uint32_t)(r1 >> 32));
            }
            in = __all(ok);
        }
        if (!in && lane == 0) atomicAdd(&g_poll_timeouts, 1u);
        float m = -FLT_MAX;
        if (in) {
#pragma unroll
            for (int j = 0; j < kSlots; ++j) m = fmaxf(m, ms[j]);
        }
        m = wave_max(m);
        float sum = 0.0f;
        if (in) {
#pragma unroll
            for (int j = 0; j < kSlots; ++j) {
                const int s = lane + 64 * j;
                if (s >= active) continue;
                const float f = fast_exp2(ms[j] - m);
                weights[wave][s] = f;
                sum += f * ls[j];
                if (s == split) continue;
                // (a replay of a captured launch carries the same tag)
                __hip_atomic_store(from + 2 * s, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(from + 2 * s + 1, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        sum = wave_sum(sum);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        const int c4 = lane & 31, part = lane >> 5;
        f32x4 x{};
        constexpr int kBatch = 8;
        for (int s0 = part; s0 < active; s0 += 2 * kBatch) {
            f32x4 y[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int s = min(s0 + 2 * j, active - 1);
                y[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(part_rsrc, (uint32_t)(((hq * S + s) * kHeadDim + 4 * c4) * 4), 0, kCacheDevice));
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int s = s0 + 2 * j;
                const float f = weights[wave][min(s, active - 1)];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = s < active ? x[e] + f * y[j][e] : x[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = halves_sum(x[e]);
        const float r = in ? 1.0f / sum : __builtin_bit_cast(float, 0x7fc00000u);
        if (part == 0) write_out(hq, c4, f32x4{x[0] * r, x[1] * r, x[2] * r, x[3] * r});
    }
}

template <int FORMAT, bool APPEND>
void launch(const Kv8Args& a, int n_kv, hipStream_t stream) {
    hipLaunchKernelGGL((mha_kv8_kernel<FORMAT, kKv8Waves, APPEND>), dim3(n_kv, a.splits), dim3(kKv8Waves * 64), 0, stream, a);
}

}  // namespace

hipError_t poll_timeouts_kv8(unsigned int* n) { return hipMemcpyFromSymbol(n, HIP_SYMBOL(g_poll_timeouts), sizeof(*n)); }

int launch_mha_kv8(const llmi_mha_kv8_args& m, const llmi_mha_kv8_append_args* append, int splits) {
    Kv8Args a{};
    const int n_kv = m.kv_dim / kHeadDim;
    a.q = static_cast<const uint16_t*>(m.query);
    a.records = kv8_records(m.max_seq_len);
    a.cache = static_cast<const char*>(m.cache8) + (int64_t)m.layer_id * n_kv * a.records * kKv8Record;
    a.out = static_cast<uint16_t*>(m.output);
    a.out_f32 = m.output_f32;
    a.pos_dev = m.pos_device;
    a.pos = m.pos;
    a.group = m.kv_mul;
    a.n_q = m.head_num;
    a.splits = splits;
    a.max_polls = poll_limit();
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)kHeadDim);
    if (splits > 1) {
        a.ws = static_cast<float*>(m.workspace);
        a.arrivals = reinterpret_cast<unsigned long long*>(static_cast<char*>(m.workspace) + fused_workspace(m.head_num, kHeadDim, splits, false).partial_bytes);
        a.tag = record_tag(next_epoch());
    }
    if (append) {
        a.k_new = static_cast<const uint16_t*>(append->key_new);
        a.v_new = static_cast<const uint16_t*>(append->value_new);
        a.norm_w = static_cast<const uint16_t*>(append->norm_weight);
        a.sin_cache = append->sin_cache;
        a.cos_cache = append->cos_cache;
        a.eps = append->eps;
    }
    const hipStream_t stream = static_cast<hipStream_t>(m.stream);
    const bool e4m3 = m.format == LLMI_KV8_E4M3;
    if (append) e4m3 ? launch<LLMI_KV8_E4M3, true>(a, n_kv, stream) : launch<LLMI_KV8_INT8, true>(a, n_kv, stream);
    else e4m3 ? launch<LLMI_KV8_E4M3, false>(a, n_kv, stream) : launch<LLMI_KV8_INT8, false>(a, n_kv, stream);
    return check_launch();
}

}  // namespace llmi
