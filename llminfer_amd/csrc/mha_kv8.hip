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
// which enters the product as the sum of three bf16 numbers: all bits that it has in fp32. (Of two numbers 2^-17 of it is lost, and results are 2e-6 from 64 bits where these are 1 - 3e-7; us, two : three,
// 2.42 : 2.47 at 58 positions (16 Q), 4.67 : 4.73 at 1024, 5.60 : 5.70 at 4096, 14.4 : 14.6 at 32768, 44.4 : 44.7 at 131001, whole numbers 6.93 : 7.09 at 6008, with the new token 4.36 : 4.46 at 300.)
// Maximum, sum and accumulators are fp32; the accumulators are
// rescaled only where a maximum has grown by more than 2^8, so a weight is up to 2^8 and sums over V stay in range for values up to 10^36 / positions.
//
// Two forms (rules and measurements: kv8_api.cpp):
//   sliced  Short contexts of up to 64 KV heads: four workgroups a KV head, each with 32 of the columns and every position. K's codes are read (through the L2) and multiplied four
//           times, V's once; nothing is handed from workgroup to workgroup, which costs a call 1.8 us otherwise (a record a wavefront: 2.9 in one workgroup, 4.7 joined).
//   split   A KV head's records are dealt to up to 256 workgroups in contiguous runs, a workgroup's wavefronts take them in turn, one record of each on its way
//           (more in flight on a compute unit come back later, not faster). Every split leaves its partial outputs and, once they are acknowledged, a
//           record {tag | maximum} {tag | sum} per head in the workspace, past the caches; the last one (or the last ones, a head each), which are
//           dispatched behind the others, wait for those (bounded) and add the parts up.
// What bounds it: the launch and a trip to memory up to some hundred positions (32 Q / 8 KV heads, E4M3, captured: 2.6 us at 58, 4.6 at 512), the hand-over up to some
// thousand (4.9 at 1024, 5.8 at 4096), then memory: 14.8 us at 32768 (68 MB), 42 - 45 by card at 131001 with 64 Q heads (272 MB, 6.2 TB/s with everything, 6.9 beyond
// the 4.9). Over the bf16 cache the same calls took 7.0 at 4096, 23.6 and 87.2 beside them.
// Whole-number codes take three instructions for two values where E4M3's take one, E4M3 : whole numbers 6.9 : 7.3 at 6008 positions, 44.2 : 45.2 at 131001; with
// the new token 3.20 : 3.33 at 57 (16 Q), 5.20 : 5.41 at 1024, 6.56 : 6.96 at 4099, 14.8 : 15.5 at 32768.

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
    int32_t run, longer;          // records per split, and how many splits take one more (position known on the host)
    int32_t single, each;         // position read on the device: kv8_active_splits
    int32_t sliced;               // ... records up to which a workgroup has 32 columns and all of them, -1 where the launch is not for that
    int32_t spread_min;           // fewest splits at which a KV head's query heads are joined by different workgroups
    float scale_log2e;            // log2(e) / sqrt(128)
    // the new token's
    const uint16_t* k_new;
    const uint16_t* v_new;
    const uint16_t* norm_w;
    const float* sin_cache;
    const float* cos_cache;
    float eps;
};

// CHUNKS: the 1 KiB chunks of V's codes that a workgroup reads, all four or one.
template <int CHUNKS>
struct Record {
    u32x4 k[4], v[CHUNKS], ks, vs;  // codes, the lane's eight scales
};

// (a record that there is not: zeros, and nothing read). Whole records are streamed past the caches, nobody reads one twice: 14.45 us at 32768 positions, without the hint
// 16.0; 44.6 : 48.7 at 131001. Where four workgroups read the same K codes they are not.
template <int CHUNKS>
__device__ __forceinline__ Record<CHUNKS> load_record(const char* at, bool there, uint32_t lane, int chunk) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at), 0, there ? kKv8Record : 0, 0x00020000);
    auto load = [&](uint32_t lane_at, int offset) __attribute__((always_inline)) {
        constexpr int kStream = 2;
        return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_at, offset, CHUNKS == 4 ? kStream : 0));
    };
    Record<CHUNKS> y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y.k[i] = load(lane * 16u, i * 1024);
    y.ks = load((lane >> 4) * 16u, kScaleBytes);
    y.vs = load((lane >> 4) * 16u, kScaleBytes + 64);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) y.v[i] = load(lane * 16u, kVBytes + (chunk + i) * 1024);
    return y;
}

template <int NW, int COLUMNS>
struct Kv8Shared {
    __attribute__((aligned(16))) float parts[NW][kHeads][COLUMNS];
    __attribute__((aligned(16))) float weights[NW][2][32];
    __attribute__((aligned(16))) uint16_t rows[kHeads][kHeadDim];  // the new token's query heads
    __attribute__((aligned(16))) uint8_t new_codes[2][kHeadDim];
    float part_m[kHeads][NW], part_l[kHeads][NW], fin[kHeads][2];
    int rows_done;  // of the new token's query heads
    bool arrived[NW];
};

// The new token's row `at` of a KV head: its query heads, then K and V.
__device__ __forceinline__ void ask_row(const Kv8Args& a, NewRow& row, int kvh, int at, int p32) {
    const bool is_new = at >= a.group;
    const uint64_t new_row = reinterpret_cast<uint64_t>(at > a.group ? a.v_new : a.k_new) + (uint64_t)(uint32_t)(kvh * 256);
    const uint64_t q_row = reinterpret_cast<uint64_t>(a.q) + (uint64_t)(uint32_t)((kvh * a.group + at) * 256);
    load_row32(row, is_new ? new_row : q_row, reinterpret_cast<uint64_t>(a.norm_w) + (is_new ? 256u : 0u), p32);
}

// A lane's value, for all of them.
__device__ __forceinline__ float row_scalar(float x, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane)); }

// SLICED: the workgroup has 32 of the 128 columns and every position, split is which (nothing to join). Otherwise all columns and its split's run. `row`: what does
// not depend on the position of the half wavefront's first new row has been asked for.
template <int FORMAT, int NW, bool APPEND, bool SLICED, int COLUMNS>
__device__ __forceinline__ void kv8_attend(const Kv8Args& a, Kv8Shared<NW, COLUMNS>& sm, NewRow& row, int pos, int active, int run, int longer) {
    constexpr int kChunks = SLICED ? 1 : 4, kColumns = 32 * kChunks;
    auto& parts = sm.parts;
    auto& part_m = sm.part_m;
    auto& part_l = sm.part_l;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x, split = SLICED ? 0 : blockIdx.y, slice = SLICED ? blockIdx.y : 0;
    const int p32 = lane & 31;
    const int half = (int)(threadIdx.x >> 5);
    const int64_t keys = (int64_t)pos + (APPEND ? 0 : 1);  // positions that come from the cache
    const bool last = split == active - 1;
    // A split's records are a run of consecutive ones (runs differ by one at most), its wavefronts take them in turn.
    const int mine = run + (split < longer ? 1 : 0);
    const int first_tile = split * run + min(split, longer);
    const int last_tile = (int)((keys + 31) >> 5) - 1;
    const char* head = a.cache + (int64_t)kvh * a.records * kKv8Record;
    const char* from = head + (int64_t)(first_tile + wave) * kKv8Record;
    const int count = wave < mine ? (mine - wave + NW - 1) / NW : 0;
    auto fetch = [&](int i) __attribute__((always_inline)) {
        return load_record<kChunks>(from + (i < count ? (int64_t)i * (NW * kKv8Record) : 0), i < count, (uint32_t)lane, slice);
    };

    // The query heads: step s of the first product has channels 64 (s/2) + 16 g + 8 (s%2) .. + 7 in lane group g. (Columns behind the group repeat its
    // last head: nobody reads their outputs.)
    u32x4 q[4];
    const int hq = min(n, a.group - 1);
    if constexpr (!APPEND) {
        const uint16_t* src = a.q + (int64_t)(kvh * a.group + hq) * kHeadDim;
#pragma unroll
        for (int s = 0; s < 4; ++s) q[s] = *reinterpret_cast<const u32x4*>(src + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
    }
    auto ask_tables = [&]() __attribute__((always_inline)) { load_tables32(row, a.sin_cache + (int64_t)pos * 64, a.cos_cache + (int64_t)pos * 64, p32); };
    uint32_t new_lo = 0u, new_hi = 0u, codes = 0u;
    float scale = 0.0f;
    const bool takes_new = wave == NW - 1;
    if constexpr (APPEND) ask_tables();
    asm volatile("" ::: "memory");
    Record<kChunks> r = fetch(0);
    if constexpr (APPEND) {
        auto put_row = [&](int at) __attribute__((always_inline)) {
            reinterpret_cast<uint32_t*>(sm.rows[at])[p32] = new_lo;
            reinterpret_cast<uint32_t*>(sm.rows[at])[p32 + 32] = new_hi;
            // (a wavefront's LDS instructions are done in order)
            asm volatile("" ::: "memory");
            if (p32 == 0) __hip_atomic_fetch_add(&sm.rows_done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        };
        if (half < a.group || takes_new) norm_rope_regs32(row, p32, a.eps, new_lo, new_hi);
        if (!takes_new) {
            if (half < a.group) put_row(half);
            // (apart from the first one: a loop's wait would be for its newest loads, the record's too)
            for (int at = half + 2 * (NW - 1); at < a.group; at += 2 * (NW - 1)) {
                ask_row(a, row, kvh, at, p32);
                ask_tables();
                norm_rope_regs32(row, p32, a.eps, new_lo, new_hi);
                put_row(at);
            }
        } else if (last) {
            const bool is_v = lane >= 32;
            codes = quantise_row32<FORMAT>(is_v ? row.x[0] : new_lo, is_v ? row.x[1] : new_hi, scale);
            reinterpret_cast<uint16_t*>(sm.new_codes[is_v])[p32] = (uint16_t)codes;
            reinterpret_cast<uint16_t*>(sm.new_codes[is_v])[p32 + 32] = (uint16_t)(codes >> 16);
        }
        // The query heads are waited for by their number, not at a barrier: nobody waits for K and V but the wavefront that has them. (Those that finish
        // rows wait for nothing.)
        while (__builtin_amdgcn_readfirstlane(__hip_atomic_load(&sm.rows_done, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)) < a.group) {}
        asm volatile("" ::: "memory");
#pragma unroll
        for (int s = 0; s < 4; ++s) q[s] = *reinterpret_cast<const u32x4*>(sm.rows[hq] + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
    }
    float m_run = -FLT_MAX, l_run = 0.0f;  // (a finite maximum: scores of -inf get weight 0, not NaN)
    constexpr int kAccs = 2 * kChunks;  // b: columns 16 b .. + 15 of the workgroup's
    f32x4 o[kAccs];
#pragma unroll
    for (int b = 0; b < kAccs; ++b) o[b] = f32x4{};

    if constexpr (APPEND) {
        // The new token, as its codes stand for it, with weight 1: the wavefront that has the fewest records starts from it.
        if (last && takes_new) {
            const float ks = row_scalar(scale, 0), vs = row_scalar(scale, 32);
            f32x4 c{};
            // (all sixteen positions of the product are the new one)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(sm.new_codes[0] + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
                c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_operand<FORMAT>(w[0], w[1]), __builtin_bit_cast(bf16x8, q[s]), c, 0, 0, 0);
            }
            const float s = c[0] * (ks * a.scale_log2e);
            m_run = fmaxf(m_run, s);
            const float w = fast_exp2(s - m_run);
            l_run = g == 0 ? w : 0.0f;
#pragma unroll
            for (int b = 0; b < kAccs; ++b) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(sm.new_codes[1] + 32 * slice + 16 * b + 4 * g);
                const uint32_t v0 = kv8_pair<FORMAT, false>(v), v1 = kv8_pair<FORMAT, true>(v);
                const float ws = w * vs;
                o[b] = f32x4{bf16_lo(v0) * ws, bf16_hi(v0) * ws, bf16_lo(v1) * ws, bf16_hi(v1) * ws};
            }
        }
    }

    auto fold = [&](int t) __attribute__((always_inline)) {
        float c[8], vs[8];  // of position 16 (e / 4) + 4 g + e % 4: scores in the exp2 domain, V's scales
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
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t kw = r.ks[e >> 1], vw = r.vs[e >> 1];
            c[e] *= ((e & 1) ? bf16_hi(kw) : bf16_lo(kw)) * a.scale_log2e;
            vs[e] = (e & 1) ? bf16_hi(vw) : bf16_lo(vw);
        }
        if (t == last_tile && (keys & 31)) {
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
                for (int i = 0; i < kChunks; ++i) {
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
            // (a wavefront's first record finds zeros)
            if (__any(l_run != 0.0f)) {
                l_run *= alpha;
#pragma unroll
                for (int b = 0; b < kAccs; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[b][e] *= alpha;
            }
        }
        u32x4 ph, pm, pl;  // a weight's three numbers, all of its bits together
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(c[2 * e] - m_run), p1 = fast_exp2(c[2 * e + 1] - m_run);
            l_run += p0 + p1;
            const float x0 = p0 * vs[2 * e], x1 = p1 * vs[2 * e + 1];
            const uint32_t w = pack_bf16(x0, x1);
            ph[e] = w;
            const float y0 = x0 - bf16_lo(w), y1 = x1 - bf16_hi(w);
            const uint32_t z = pack_bf16(y0, y1);
            pm[e] = z;
            pl[e] = pack_bf16(y0 - bf16_lo(z), y1 - bf16_hi(z));
        }
#pragma unroll
        for (int b = 0; b < kAccs; ++b) {
            const bf16x8 x = kv8_operand<FORMAT>(r.v[b >> 1][2 * (b & 1)], r.v[b >> 1][2 * (b & 1) + 1]);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, ph), o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, pm), o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, __builtin_bit_cast(bf16x8, pl), o[b], 0, 0, 0);
        }
    };
    for (int i = 0; i < count; ++i) {
        fold(first_tile + wave + i * NW);
        r = fetch(i + 1);
    }

    // The workgroup's wavefronts.
    l_run = rows_sum(l_run);
    if (n < a.group) {
#pragma unroll
        for (int b = 0; b < kAccs; ++b) *reinterpret_cast<f32x4*>(&parts[wave][n][16 * b + 4 * g]) = o[b];
        if (g == 0) {
            part_m[n][wave] = m_run;
            part_l[n][wave] = l_run;
        }
    }
    __syncthreads();
    // (here, where nobody waits for this wavefront any more; ahead of the records their waits would be for these stores too)
    if (APPEND && last && takes_new && slice == 0)
        file_row32(const_cast<char*>(head) + (int64_t)(pos >> 5) * kKv8Record, pos & 31, lane >= 32, p32, codes, scale);
    const int S = a.splits;
    const int64_t part_bytes = (int64_t)a.n_q * S * kHeadDim * (int64_t)sizeof(float);
    const __amdgpu_buffer_rsrc_t part_rsrc = __builtin_amdgcn_make_buffer_rsrc(a.ws, 0, (int)part_bytes, 0x00020000);
    auto write_out = [&](int hq, int c4, f32x4 x) __attribute__((always_inline)) {
        c4 += 8 * slice;
        *reinterpret_cast<u32x2*>(a.out + (int64_t)hq * kHeadDim + 4 * c4) = u32x2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
        if (a.out_f32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) a.out_f32[(int64_t)hq * kHeadDim + 4 * c4 + e] = x[e];
        }
    };
    // Who joins a head's splits: the workgroup of the last one all of them, or, where there are enough, the last splits' workgroups a head each, so
    // that the parts are read back by several compute units.
    const bool spread = active >= a.spread_min && active >= a.group;
    const int my_head = spread && active - 1 - split < a.group ? active - 1 - split : -1;
    constexpr int kPerHead = kColumns / 4, kUnits = (kHeads * kPerHead + NW * 64 - 1) / (NW * 64);
    float unit_m[kUnits], unit_l[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = (int)threadIdx.x + i * NW * 64;
        if (u >= a.group * kPerHead) break;
        const int h = u / kPerHead, c4 = u % kPerHead, hq = kvh * a.group + h;
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
        unit_m[i] = m;
        unit_l[i] = sum;
        if (SLICED || active == 1) {
            const float r = 1.0f / sum;
            write_out(hq, c4, f32x4{x[0] * r, x[1] * r, x[2] * r, x[3] * r});
        } else {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), part_rsrc, (uint32_t)(((hq * S + split) * kHeadDim + 4 * c4) * 4), 0, kCacheDevice);
        }
    }
    if (SLICED || active == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a head's 32 columns are half a wavefront's: no barrier)
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = (int)threadIdx.x + i * NW * 64;
        if (u >= a.group * 32) break;
        const int h = u >> 5;
        if ((u & 31) != 0) continue;
        if (spread ? h == my_head : last) {
            sm.fin[h][0] = unit_m[i];
            sm.fin[h][1] = unit_l[i];
        } else {
            unsigned long long* to = a.arrivals + ((int64_t)(kvh * a.group + h) * S + split) * 2;
            const unsigned long long tag = a.tag;
            __hip_atomic_store(to, tag | (unsigned long long)__builtin_bit_cast(uint32_t, unit_m[i]) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(to + 1, tag | (unsigned long long)__builtin_bit_cast(uint32_t, unit_l[i]) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (spread ? my_head < 0 : !last) return;
    __syncthreads();

    // A wavefront's part of a head's join: splits s0 .. s0 + n - 1 (64 at most), a lane each for the records, a lane for four columns of every
    // second split for the parts.
    struct Part {
        float m, sum;
        f32x4 x;
        bool in;
    };
    const int c4 = lane & 31, part = lane >> 5;
    auto gather = [&](int h, int s0, int n) __attribute__((always_inline)) {
        constexpr int kBatch = 16;
        const int hq = kvh * a.group + h;
        unsigned long long* rec = a.arrivals + ((int64_t)hq * S + s0 + lane) * 2;
        Part y;
        float m = -FLT_MAX, l = 0.0f;
        const bool mine_is = lane < n && s0 + lane == split, polls = lane < n && !mine_is;
        if (mine_is) {
            m = sm.fin[h][0];
            l = sm.fin[h][1];
        }
        y.in = false;
        for (int spin = 0; spin < a.max_polls && !y.in; ++spin) {
            bool ok = true;
            if (polls) {
                const unsigned long long r0 = __hip_atomic_load(rec, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const unsigned long long r1 = __hip_atomic_load(rec + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                ok = (uint32_t)r0 == a.tag && (uint32_t)r1 == a.tag;
                m = __builtin_bit_cast(float, (uint32_t)(r0 >> 32));
                l = __builtin_bit_cast(float, (uint32_t)(r1 >> 32));
            }
            y.in = __all(ok);
        }
        // (rows behind the last split: zeros, and nothing read)
        const __amdgpu_buffer_rsrc_t rows_rsrc =
            __builtin_amdgcn_make_buffer_rsrc(a.ws + (int64_t)(hq * S + s0) * kHeadDim, 0, max(n, 0) * (kHeadDim * 4), 0x00020000);
        const uint32_t at = (uint32_t)(part * (kHeadDim * 4) + c4 * 16);
        f32x4 v[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) v[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc, at, j * 1024, kCacheDevice));
        if (polls && y.in) {
            // (a replay of a captured launch carries the same tag)
            __hip_atomic_store(rec, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(rec + 1, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        y.m = wave_max(m);
        const float f = lane < n ? fast_exp2(m - y.m) : 0.0f;
        sm.weights[wave][lane & 1][lane >> 1] = f;  // (a half wavefront's side by side)
        y.sum = wave_sum(f * l);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        f32x4 w[kBatch / 4];
        auto weigh = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < kBatch / 4; ++j) w[j] = *reinterpret_cast<const f32x4*>(&sm.weights[wave][part][j0 + 4 * j]);
        };
        auto add = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) y.x[e] = __builtin_fmaf(w[j >> 2][j & 3], v[j][e], y.x[e]);
        };
        y.x = f32x4{};
        weigh(0);
        add();
        if (n > 2 * kBatch) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) v[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc, at, (kBatch + j) * 1024, kCacheDevice));
            weigh(kBatch);
            add();
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y.x[e] = halves_sum(y.x[e]);
        return y;
    };
    if (active <= 64) {
        // a wavefront a head
        if (spread && wave != 0) return;
        for (int h = spread ? my_head : wave; h < a.group; h += NW) {
            const Part y = gather(h, 0, active);
            if (!y.in && lane == 0) atomicAdd(&g_poll_timeouts, 1u);
            const float r = y.in ? 1.0f / y.sum : __builtin_bit_cast(float, 0x7fc00000u);
            if (part == 0) write_out(kvh * a.group + h, c4, f32x4{y.x[0] * r, y.x[1] * r, y.x[2] * r, y.x[3] * r});
            if (spread) break;
        }
        return;
    }
    // All wavefronts a head: a share of the splits each.
    const int share = (active + NW - 1) / NW;
    for (int h = spread ? my_head : 0; h < a.group; ++h) {
        const Part y = gather(h, wave * share, min(share, active - wave * share));
        __syncthreads();  // (the parts' place is read for the last time in the turn before)
        if (part == 0) *reinterpret_cast<f32x4*>(&parts[wave][0][4 * c4]) = y.x;
        if (lane == 0) {
            part_m[0][wave] = y.m;
            part_l[0][wave] = y.sum;
            sm.arrived[wave] = y.in;
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            float m = part_m[0][0], sum = 0.0f;
            f32x4 x{};
#pragma unroll
            for (int w = 1; w < NW; ++w) m = fmaxf(m, part_m[0][w]);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = fast_exp2(part_m[0][w] - m);
                sum += f * part_l[0][w];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] += f * parts[w][0][4 * c4 + e];
            }
            bool in = true;
#pragma unroll
            for (int w = 0; w < NW; ++w) in = in && sm.arrived[w];
            if (!in && lane == 0) atomicAdd(&g_poll_timeouts, 1u);
            const float r = in ? 1.0f / sum : __builtin_bit_cast(float, 0x7fc00000u);
            write_out(kvh * a.group + h, c4, f32x4{x[0] * r, x[1] * r, x[2] * r, x[3] * r});
        }
        if (spread) break;
    }
}

enum class Kv8Kind { split, sliced, device };  // device: which of them the position read at run time decides

template <int FORMAT, int NW, bool APPEND, Kv8Kind KIND>
__global__ __launch_bounds__(NW * 64, 2) void mha_kv8_kernel(Kv8Args a) {
    __shared__ Kv8Shared<NW, KIND == Kv8Kind::sliced ? 32 : kHeadDim> sm;
    // The new token's rows, half a wavefront each: the query heads, in the last wavefront K and V (which the last split files). What does not depend on the
    // position is asked for in front of it, everything else in front of the records. (Half wavefronts without a row take a head again: a branch around
    // the loads would make their wait one for all of the records' too.) Only the wavefront that has K and V waits for their quantisation; one barrier for all rows,
    // K and V quantised by a third wavefront ahead of it : this, us: 3.32 : 3.17 at 57 positions (16 Q), 4.46 : 4.36 at 300, 5.00 : 5.13 at 511 (32 Q), 5.19 : 5.06 at
    // 1024, 6.08 : 5.83 at 4095, 14.87 : 14.64 at 32768; position on the device 5.97 : 5.83 at 1000, 6.97 : 6.90 at 4099.
    NewRow row;
    if constexpr (APPEND) {
        const int half = (int)(threadIdx.x >> 5), behind = half - 2 * (NW - 1);
        ask_row(a, row, blockIdx.x, behind >= 0 ? a.group + behind : min(half, a.group - 1), threadIdx.x & 31);
        if (threadIdx.x == 0) sm.rows_done = 0;
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    int pos = a.pos, active = a.splits, run = a.run, longer = a.longer;
    if constexpr (KIND == Kv8Kind::device) {
        // (constant address space: a scalar load; nothing in the launch writes the position)
        const auto word = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(a.pos_dev));
        pos = max(0, min(*word, a.pos));
        const int tiles = (int)(((int64_t)pos + (APPEND ? 0 : 1) + 31) >> 5), split = (int)blockIdx.y;
        // (only where the launch has workgroups for the slices: a chosen number of splits, or many KV heads, go the other way, a step without a record too)
        if (tiles <= a.sliced) {
            if (split < kKv8Slices) kv8_attend<FORMAT, NW, APPEND, true>(a, sm, row, pos, 1, tiles, 0);
            return;
        }
        active = kv8_active_splits(tiles, a.splits, a.single, a.each);
        if (split >= active) return;
        // (a quotient in two steps of 24 bits, then one up or down: shorter than the compiler's division, and on the way to the first load)
        const float inverse = 1.0f / (float)active;
        run = (int)((float)tiles * inverse);
        run += (int)((float)(tiles - run * active) * inverse);
        longer = tiles - run * active;
        if (longer < 0) {
            --run;
            longer += active;
        } else if (longer >= active) {
            ++run;
            longer -= active;
        }
    }
    kv8_attend<FORMAT, NW, APPEND, KIND == Kv8Kind::sliced>(a, sm, row, pos, active, run, longer);
}

template <int FORMAT, bool APPEND, Kv8Kind KIND>
void launch(const Kv8Args& a, int n_kv, const Kv8Form& form, hipStream_t stream) {
    const dim3 grid(n_kv, KIND == Kv8Kind::sliced ? kKv8Slices : KIND == Kv8Kind::device && form.sliced && a.splits < kKv8Slices ? kKv8Slices : a.splits);
    if (form.waves == 8) hipLaunchKernelGGL((mha_kv8_kernel<FORMAT, 8, APPEND, KIND>), grid, dim3(8 * 64), 0, stream, a);
    else hipLaunchKernelGGL((mha_kv8_kernel<FORMAT, 4, APPEND, KIND>), grid, dim3(4 * 64), 0, stream, a);
}

template <int FORMAT, bool APPEND>
void launch(const Kv8Args& a, int n_kv, const Kv8Form& form, hipStream_t stream) {
    if (a.pos_dev) launch<FORMAT, APPEND, Kv8Kind::device>(a, n_kv, form, stream);
    else if (form.sliced) launch<FORMAT, APPEND, Kv8Kind::sliced>(a, n_kv, form, stream);
    else launch<FORMAT, APPEND, Kv8Kind::split>(a, n_kv, form, stream);
}

}  // namespace

hipError_t poll_timeouts_kv8(unsigned int* n) { return hipMemcpyFromSymbol(n, HIP_SYMBOL(g_poll_timeouts), sizeof(*n)); }

int launch_mha_kv8(const llmi_mha_kv8_args& m, const llmi_mha_kv8_append_args* append, const Kv8Form& form) {
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
    a.splits = form.splits;
    a.max_polls = poll_limit();
    const int tiles = (int)(((int64_t)m.pos + (append ? 0 : 1) + 31) >> 5);
    a.run = tiles / form.splits;
    a.longer = tiles % form.splits;
    a.spread_min = form.spread_min;
    a.single = form.single;
    a.each = form.each;
    a.sliced = form.sliced ? form.single : -1;
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)kHeadDim);
    if (form.splits > 1) {
        a.ws = static_cast<float*>(m.workspace);
        a.arrivals = reinterpret_cast<unsigned long long*>(static_cast<char*>(m.workspace) + fused_workspace(m.head_num, kHeadDim, form.splits, false).partial_bytes);
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
    if (append) e4m3 ? launch<LLMI_KV8_E4M3, true>(a, n_kv, form, stream) : launch<LLMI_KV8_INT8, true>(a, n_kv, form, stream);
    else e4m3 ? launch<LLMI_KV8_E4M3, false>(a, n_kv, form, stream) : launch<LLMI_KV8_INT8, false>(a, n_kv, form, stream);
    return check_launch();
}

}  // namespace llmi
