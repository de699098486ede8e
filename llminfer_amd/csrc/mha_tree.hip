// Attention of a tree of drafted tokens over a KV cache on gfx950 (no counterpart in the reference, which decodes one token per
// step): for node i and query head h, with g query heads per KV head,
//   out[i][h] = sum_j w_j V[j][h/g] / sum_j w_j,   w_j = exp(q[i][h].K[j][h/g] / sqrt(128) - max),
// over the cached positions 0..pos-1 and the nodes t (slots pos + t) that node i's 64-bit word names.
//
// A KV head's nodes * g query rows are taken 32 to a wavefront, K and V read once per workgroup in tiles of 32 keys. Both products
// run on the matrix cores in the transposed form, S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_bf16): a lane then holds
// 16 keys of one query row, so that maximum and sum of a row are folds inside a lane and one swap of the wavefront's halves, and the
// probabilities are in the registers where the second product wants them:
//   S^T  lane L: query row L%32, keys 8*(r/4) + 4*(L/32) + r%4 in register r = 0..15
//   P^T  lane L: query row L%32; its eight values of step s (16 keys) are registers 8s..8s+7 of S^T, which fixes the order of the keys in
//        that product: place 8*(L/32) + j is key 16s + 8*(j/4) + 4*(L/32) + j%4
//   V^T  lane L: column 32*b + L%32 (b = 0..3), keys in that order: two transposing LDS reads (ds_read_b64_tr_b16), four keys each
//   O^T  lane L: query row L%32, columns 32*b + 8*(r/4) + 4*(L/32) + r%4
// Tiles lie in LDS as rows of 256 bytes, filled by LDS-DMA loads whose lanes fetch from where the swizzle wants it: K's 16-byte chunks are
// exchanged by the row's low four bits, V's 64-byte quarters rotated by the row's low two, which spreads either read over the banks.
//
// Keys are split over workgroups; a second launch joins the splits.

#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "llmi_internal.h"
#include "mha_device_helpers.h"

namespace llmi {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kKeys = kTreeKeys;       // keys per tile
constexpr int kTileBytes = 2 * kKeys * kHeadDim * 2;
constexpr int kWaves = 4;
constexpr int kSlots = 16;             // a lane's 64 accumulators of O^T as float4: slot 4*b + r/4

struct TreeArgs {
    const uint16_t* q;          // [nodes][n_q][128]
    const uint16_t* k;          // layer base
    const uint16_t* v;
    uint16_t* out;              // [nodes][n_q][128]
    float* out_f32;             // optional
    const uint64_t* mask;       // optional
    const int32_t* pos_dev;     // optional
    f32x4* part;                // [block][split][slot][lane]: a block is 32 query rows of a KV head
    float2* part_ml;            // [block][split][32]: maximum (exp2 domain), sum
    int64_t row_stride;         // elements between positions of one KV head
    int64_t head_stride;        // elements between KV heads
    int32_t pos, nodes, group, n_q, rows, blocks, splits;  // rows = nodes * group, blocks = per KV head
    float scale_log2e;          // log2(e) / sqrt(128)
};

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float halves_max(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned h0 = h[0], h1 = h[1];
    return fmaxf(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
}

// (scalar: everything that is the same for a workgroup's wavefronts derives from it)
__device__ __forceinline__ int position(const TreeArgs& a) {
    return __builtin_amdgcn_readfirstlane(a.pos_dev ? max(0, min(*a.pos_dev, a.pos)) : a.pos);
}

// A load's base in scalar registers, for long enough (see scalar_bases).
__device__ __forceinline__ void scalar_base(const char*& p) { asm volatile("s_nop 4" : "+s"(p)); }

// A finished row's four columns.
__device__ __forceinline__ void write_out(const TreeArgs& a, int kvh, int row, int col, f32x4 o, float sum) {
    if (row >= a.rows) return;
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;  // (no key: zeros)
    const int node = row / a.group;
    const int64_t at = ((int64_t)node * a.n_q + kvh * a.group + (row - node * a.group)) * kHeadDim + col;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = sum == 0.0f ? 0.0f : o[e] * r;
    *reinterpret_cast<u32x2*>(a.out + at) = u32x2{pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])};
    if (a.out_f32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) a.out_f32[at + e] = y[e];
    }
}

// WM wavefronts side by side on 32 query rows each, 4 / WM of them on a tile each of the same rows. EXACT: a probability enters the second
// product as the sum of two bf16 numbers (relative error 2^-17), otherwise as one (2^-8).
template <int WM, bool EXACT, int STAGES>
__global__ __launch_bounds__(kWaves * 64, 2) void mha_tree_kernel(TreeArgs a) {
    constexpr int WK = kWaves / WM;
    constexpr int kStageBytes = WK * kTileBytes;
    constexpr int kLoads = 16 / WM;  // 1 KiB blocks of a tile per wavefront: eight of K, eight of V
    __shared__ __attribute__((aligned(1024))) char smem[STAGES * kStageBytes];
    __shared__ float merge_m[kWaves][32], merge_l[kWaves][32];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wk = wave / WM;
    const int half = lane >> 5, n32 = lane & 31;
    const int kvh = blockIdx.x, split = blockIdx.y;
    const int block = blockIdx.z * WM + wm;  // of 32 query rows
    const int row = block * 32 + n32;
    const bool has_rows = block * 32 < a.rows;

    const int pos = position(a);
    const int keys = pos + a.nodes;
    const int tiles = (keys + kKeys - 1) / kKeys;
    const int run = __builtin_amdgcn_readfirstlane(tiles / a.splits), longer = tiles - run * a.splits;
    const int t0 = split * run + min(split, longer), t1 = t0 + run + (split < longer ? 1 : 0);
    const int iters = (t1 - t0 + WK - 1) / WK;

    // The query rows (those behind the last one repeat it) and the nodes they see.
    u32x4 q[8];
    const int row_in = min(row, a.rows - 1);
    const int node = row_in / a.group;
    {
        const u32x4* src = reinterpret_cast<const u32x4*>(a.q + ((int64_t)node * a.n_q + kvh * a.group + (row_in - node * a.group)) * kHeadDim);
#pragma unroll
        for (int s = 0; s < 8; ++s) q[s] = src[2 * s + half];
    }
    uint64_t sees = a.mask ? a.mask[node] : ~0ull >> (63 - node);
    sees &= ~0ull >> (64 - a.nodes);

    const uint32_t rs = (uint32_t)a.row_stride * 2u;
    const char* kb = reinterpret_cast<const char*>(a.k + (int64_t)kvh * a.head_stride);
    const char* vb = reinterpret_cast<const char*>(a.v + (int64_t)kvh * a.head_stride);
    const int rho = lane >> 4, c16 = lane & 15;
    const uint32_t v_col = (uint32_t)((((c16 >> 2) - rho) & 3) * 64 + (c16 & 3) * 16);
    const uint32_t smem0 = (uint32_t)(uintptr_t)smem;

    uint32_t k_off[4];  // (a block is four rows, and the low four bits of a row follow from the block's low two)
#pragma unroll
    for (int b = 0; b < 4; ++b) k_off[b] = (uint32_t)rho * rs + (uint32_t)((c16 ^ (4 * b + rho)) * 16);
    const uint32_t v_off = (uint32_t)rho * rs + v_col;

    auto issue = [&](int it, int stage) __attribute__((always_inline)) {
        const int t = t0 + it * WK + wk;
        if (t >= t1) return;
        const char* kt = kb + (int64_t)t * kKeys * rs;
        const char* vt = vb + (int64_t)t * kKeys * rs;
        const int last = keys - 1 - t * kKeys;  // rows past the keys repeat the last one: seen by nobody
        const uint32_t to = smem0 + (uint32_t)(stage * kStageBytes + wk * kTileBytes);
        const bool whole = last >= kKeys - 1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int b = wm * kLoads + i;  // (a wavefront of four has blocks of K or of V alone)
            const bool is_k = WM == 4 ? wm < 2 : WM == 2 ? wm < 1 : i < 8;
            const int b8 = b & 7;
            const uint32_t lane_off = is_k ? k_off[i & 3] : v_off;
            const char* base = is_k ? kt : vt;
            const uint32_t ragged = (uint32_t)min(4 * b8 + rho, last) * rs + (lane_off - (uint32_t)rho * rs);
            if (whole) base += (int64_t)(4 * b8) * rs;
            scalar_base(base);
            dma16(base, whole ? lane_off : ragged, to + (uint32_t)(b * 1024));
        }
    };

    const uint32_t k_x = (uint32_t)(half ^ (n32 & 15));  // chunk 2s + half of row n32 lies at chunk (2s) ^ k_x
    const uint32_t k_row = (uint32_t)n32 * 256u;
    const int i16 = lane & 15;
    const uint32_t v_row = (uint32_t)((4 * half + (i16 >> 2)) * 256 + ((lane >> 4) & 1) * 32 + (i16 & 3) * 8);
    float m_run = -FLT_MAX, l_run = 0.0f;  // (a finite maximum: scores of -inf get weight 0, not NaN)
    f32x16 o[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) o[b] = f32x16{};

    uint32_t broken = 0u;  // bits 15 and 31: a value that is not finite among the nodes' tiles
    auto compute = [&](int t, int stage) __attribute__((always_inline)) {
        const bool masked = (t + 1) * kKeys > pos;
        const char* kt = smem + stage * kStageBytes + wk * kTileBytes;
        const char* vt = kt + kTileBytes / 2;
        // (all of K's fragments are asked for before the first product waits for one; V's travel while the weights are formed)
        u32x4 kf[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) kf[s] = *reinterpret_cast<const u32x4*>(kt + k_row + (((uint32_t)(2 * s) ^ k_x) << 4));
        asm volatile("" : "+v"(kf[0]), "+v"(kf[1]), "+v"(kf[2]), "+v"(kf[3]), "+v"(kf[4]), "+v"(kf[5]), "+v"(kf[6]), "+v"(kf[7]));
        u32x2 vh[4][2][2];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    typedef __attribute__((address_space(3))) i16x4* lds4;
                    const char* at = vt + v_row + (uint32_t)(((b + (i16 >> 2)) & 3) * 64) + (s * 16 + x * 8) * 256;
                    vh[b][s][x] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(uintptr_t)(uint32_t)(uintptr_t)at));
                }
        f32x16 c{};
#pragma unroll
        for (int s = 0; s < 8; ++s) c = mfma(__builtin_bit_cast(bf16x8, kf[s]), __builtin_bit_cast(bf16x8, q[s]), c);
        // Tiles with nodes in them: what a row does not see has no weight.
        uint32_t vis = ~0u;  // bit o: the tile's key 4 * half + o
        if (masked) {
            const int at = t * kKeys + 4 * half - pos;
            vis = at <= -32 ? ~0u : at >= 64 ? 0u : at >= 0 ? (uint32_t)(sees >> at) : (uint32_t)(sees << -at) | ((1u << -at) - 1u);
#pragma unroll
            for (int r = 0; r < 16; ++r) c[r] = vis >> (8 * (r >> 2) + (r & 3)) & 1u ? c[r] : -INFINITY;
        }
        float top = c[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, c[r]);
        top = halves_max(top) * a.scale_log2e;
        // The accumulators are rescaled only where a row's maximum has grown by more than 2^8: up to that its weights are
        // just larger than 1.
        if (__any(top > m_run + 8.0f)) {
            const float m_new = fmaxf(m_run, top);
            const float alpha = fast_exp2(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
        }
        float p[16];
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            p[r] = fast_exp2(__builtin_fmaf(c[r], a.scale_log2e, -m_run));
            sum += p[r];
        }
        l_run += sum;
        u32x4 ph[2], pl[2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = p[8 * s + 2 * j], y = p[8 * s + 2 * j + 1];
                const uint32_t w = pack_bf16(x, y);
                ph[s][j] = w;
                if constexpr (EXACT) pl[s][j] = pack_bf16(x - bf16_lo(w), y - bf16_hi(w));
            }
        if (masked) {
            // A weight of 0 times an infinity or NaN would be NaN: those enter as 0 here and are added at the end, for the rows that
            // see them. (An exponent of all ones carries into the sign's place.)
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        typedef short i16x2 __attribute__((ext_vector_type(2)));
                        uint32_t w = vh[b][s][j >> 1][j & 1];
                        const uint32_t carry = (w & 0x7f807f80u) + 0x00800080u;
                        broken |= carry;
                        vh[b][s][j >> 1][j & 1] = w & ~__builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, carry) >> 15);
                    }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const u32x4 vf = {vh[b][s][0][0], vh[b][s][0][1], vh[b][s][1][0], vh[b][s][1][1]};
                o[b] = mfma(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, ph[s]), o[b]);
                if constexpr (EXACT) o[b] = mfma(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, pl[s]), o[b]);
            }
    };

#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s, s);
    // One stage after the other: the oldest has landed (newer ones stay in flight), for every wavefront, and all have read the one
    // that is refilled.
    int stage = 0;
#pragma unroll 1
    for (int it = 0; it < iters; ++it) {
        if (it + STAGES - 1 < iters) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (it + STAGES - 1 < iters) issue(it + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        const int t = t0 + it * WK + wk;
        if (has_rows && t < t1) compute(t, stage);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }

    // Infinities and NaN among the values of nodes, for the rows that see them.
    if (__builtin_expect(__any((broken & 0x80008000u) != 0u), 0)) {
#pragma unroll 1
        for (int n = 0; n < a.nodes; ++n) {
            const int t = (pos + n) / kKeys;
            if (t < t0 || t >= t1 || (t - t0) % WK != wk) continue;
            const char* at = vb + (int64_t)(pos + n) * rs + 8 * half;
            const bool seen = sees >> n & 1;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(at + 64 * b + 16 * r4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t we = w[e >> 1];
                        const float x = (e & 1) ? bf16_hi(we) : bf16_lo(we);
                        if (seen && !(fabsf(x) < INFINITY)) o[b][4 * r4 + e] += x;
                    }
                }
        }
    }

    // Join the wavefronts of the same rows, each a part of the columns; then out, or to the workspace.
    l_run = halves_sum(l_run);
    f32x4 mine[kSlots / WK];
    if constexpr (WK > 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        static_assert(kWaves * kSlots * 64 * 16 <= sizeof(smem), "the accumulators of all wavefronts fit the ring");
        f32x4* parts = reinterpret_cast<f32x4*>(smem);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                parts[(wave * kSlots + 4 * b + r4) * 64 + lane] = f32x4{o[b][4 * r4], o[b][4 * r4 + 1], o[b][4 * r4 + 2], o[b][4 * r4 + 3]};
        if (half == 0) {
            merge_m[wave][n32] = m_run;
            merge_l[wave][n32] = l_run;
        }
        __syncthreads();
        float m = -FLT_MAX, w[WK], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < WK; ++i) m = fmaxf(m, merge_m[i * WM + wm][n32]);
#pragma unroll
        for (int i = 0; i < WK; ++i) {
            w[i] = fast_exp2(merge_m[i * WM + wm][n32] - m);
            sum += w[i] * merge_l[i * WM + wm][n32];
        }
#pragma unroll
        for (int x = 0; x < kSlots / WK; ++x) {
            mine[x] = f32x4{};
#pragma unroll
            for (int i = 0; i < WK; ++i) {
                const f32x4 y = parts[((i * WM + wm) * kSlots + wk * (kSlots / WK) + x) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[x][e] += w[i] * y[e];
            }
        }
        m_run = m;
        l_run = sum;
    } else {
#pragma unroll
        for (int x = 0; x < kSlots; ++x) mine[x] = f32x4{o[x >> 2][4 * (x & 3)], o[x >> 2][4 * (x & 3) + 1], o[x >> 2][4 * (x & 3) + 2], o[x >> 2][4 * (x & 3) + 3]};
    }
    if (!has_rows) return;
    if (a.splits == 1) {
#pragma unroll
        for (int x = 0; x < kSlots / WK; ++x) {
            const int slot = wk * (kSlots / WK) + x;
            write_out(a, kvh, row, 32 * (slot >> 2) + 8 * (slot & 3) + 4 * half, mine[x], l_run);
        }
        return;
    }
    const int64_t at = (int64_t)(kvh * a.blocks + block) * a.splits + split;
    if (t1 > t0) {
#pragma unroll
        for (int x = 0; x < kSlots / WK; ++x) a.part[(at * kSlots + wk * (kSlots / WK) + x) * 64 + lane] = mine[x];
    }
    // (a split without keys leaves no part: a maximum of -inf says so)
    if (wk == 0 && half == 0) a.part_ml[at * 32 + n32] = t1 > t0 ? make_float2(m_run, l_run) : make_float2(-INFINITY, 0.0f);
}

// The splits of a block joined: a workgroup per slot, its wavefronts on every fourth split, eight of them asked for at once.
__global__ __launch_bounds__(kWaves * 64) void mha_tree_join_kernel(TreeArgs a) {
    constexpr int kAhead = 8;
    __shared__ f32x4 wave_o[kWaves][64];
    __shared__ float wave_m[kWaves][64], wave_l[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kvh = blockIdx.x, slot = blockIdx.y, block = blockIdx.z;
    const int half = lane >> 5, n32 = lane & 31;
    const int64_t first = (int64_t)(kvh * a.blocks + block) * a.splits;
    const float2* ml = a.part_ml + first * 32 + n32;
    const f32x4* part = a.part + (first * kSlots + slot) * 64 + lane;
    float m = -FLT_MAX, sum = 0.0f;
    f32x4 o{};
    for (int s0 = wave; s0 < a.splits; s0 += kWaves * kAhead) {
        float2 x[kAhead];
        f32x4 y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int s = min(s0 + kWaves * i, a.splits - 1);
            x[i] = ml[s * 32];
            y[i] = part[(int64_t)s * kSlots * 64];
            if (s0 + kWaves * i >= a.splits) x[i] = make_float2(-INFINITY, 0.0f);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) top = fmaxf(top, x[i].x);
        const float before = fast_exp2(m - top);
        m = top;
        sum *= before;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= before;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const float w = fast_exp2(x[i].x - m);
            sum += w * x[i].y;
            // (a split without keys has left no part)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = w == 0.0f ? o[e] : o[e] + w * y[i][e];
        }
    }
    wave_o[wave][lane] = o;
    wave_m[wave][lane] = m;
    wave_l[wave][lane] = sum;
    __syncthreads();
    if (wave != 0) return;
    float top = m;
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, wave_m[i][lane]);
    f32x4 all{};
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const float w = fast_exp2(wave_m[i][lane] - top);
        const f32x4 y = wave_o[i][lane];
        total += w * wave_l[i][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) all[e] += w * y[e];
    }
    write_out(a, kvh, block * 32 + n32, 32 * (slot >> 2) + 8 * (slot & 3) + 4 * half, all, total);
}

}  // namespace

int launch_mha_tree(const llmi_mha_tree_args& args, const llmi_mha_plan& plan) {
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
    a.rows = args.node_num * m.kv_mul;
    const int n_kv = m.kv_dim / kHeadDim, wm = plan.group_pad / 32;
    a.blocks = (a.rows + 31) / 32;
    a.splits = plan.num_splits;
    a.part = static_cast<f32x4*>(m.workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part + (size_t)n_kv * a.blocks * a.splits * kSlots * 64);
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)kHeadDim);
    const hipStream_t stream = static_cast<hipStream_t>(m.stream);
    const dim3 grid(n_kv, a.splits, (a.blocks + wm - 1) / wm);
    if (wm == 1) hipLaunchKernelGGL((mha_tree_kernel<1, true, 2>), grid, dim3(kWaves * 64), 0, stream, a);
    else if (wm == 2) hipLaunchKernelGGL((mha_tree_kernel<2, true, 2>), grid, dim3(kWaves * 64), 0, stream, a);
    else if (grid.z == 1) hipLaunchKernelGGL((mha_tree_kernel<4, true, 3>), grid, dim3(kWaves * 64), 0, stream, a);
    else hipLaunchKernelGGL((mha_tree_kernel<4, false, 3>), grid, dim3(kWaves * 64), 0, stream, a);
    if (a.splits > 1) hipLaunchKernelGGL(mha_tree_join_kernel, dim3(n_kv, kSlots, a.blocks), dim3(kWaves * 64), 0, stream, a);
    return check_launch();
}

}  // namespace llmi
