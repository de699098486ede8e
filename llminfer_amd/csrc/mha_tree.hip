// Attention of a tree of drafted tokens over a KV cache on gfx950 (no counterpart in the reference, which decodes one token per
// step): for node i and query head h, with g query heads per KV head,
//   out[i][h] = sum_j w_j V[j][h/g] / sum_j w_j,   w_j = exp(q[i][h].K[j][h/g] / sqrt(128) - max),
// over the cached positions 0..pos-1 and the nodes t (slots pos + t) that node i's 64-bit word names.
//
// A KV head's nodes * g query rows are taken 32 to a wavefront (16 where there are no more), K and V read once per workgroup in tiles
// of 32 keys. Both products run on the matrix cores in the transposed form, S^T = K Q^T and O^T = V^T P^T (v_mfma_f32_32x32x16_bf16,
// v_mfma_f32_16x16x32_bf16): a lane then holds 16 (8) keys of one query row, so that maximum and sum of a row are folds inside a lane and one
// swap of the wavefront's halves (two swaps), and the probabilities are in the registers where the second product wants them:
//   32 rows:  S^T  lane L: query row L%32, keys 8*(r/4) + 4*(L/32) + r%4 in register r = 0..15
//             P^T  lane L: query row L%32; its eight values of step s (16 keys) are registers 8s..8s+7 of S^T, which fixes the order of the
//                  keys in that product: place 8*(L/32) + j is key 16s + 8*(j/4) + 4*(L/32) + j%4
//             V^T  lane L: column 32*b + L%32 (b = 0..3), keys in that order: two transposing LDS reads (ds_read_b64_tr_b16), four keys each
//             O^T  lane L: query row L%32, columns 32*b + 8*(r/4) + 4*(L/32) + r%4
//   16 rows:  S^T  lane L: query row L%16, keys 16*u + 4*(L/16) + r in register r = 0..3 of product u = 0, 1
//             P^T  lane L: those eight: place 8*(L/16) + j is key 16*(j/4) + 4*(L/16) + j%4
//             V^T  lane L: column 16*b + L%16 (b = 0..7), keys in that order;  O^T  lane L: query row L%16, columns 16*b + 4*(L/16) + r
// Tiles lie in LDS as rows of 256 bytes, filled by LDS-DMA loads whose lanes fetch from where the swizzle wants it: K's 16-byte chunks are
// exchanged by the row's low four bits, V's 32-byte pieces rotated by the row's low three. K's reads are spread over the banks by that, and V's in
// the 16-row form. In the 32-row form half a wavefront of the transposing read takes two neighbouring pieces of four keys, at the places 0 1 2 3 and 1 2 3 4:
// two cycles a half in place of one (counters: 2.0 conflict cycles a read of V, a third of all LDS cycles).
//
// Keys are split over workgroups; a second launch joins the splits. What bounds it: the way to the first product and the join's launch up to a few
// thousand positions (8 nodes of 32 heads, 8 KV heads at 4099: 10.3 us, 17 MB), memory for few rows (8 nodes at 32768: 29.6 us, 4.5 TB/s), matrix cores and
// the exponentials between their products for many (64 nodes of 64 heads at 131000: 293 us, 0.94 PFLOP/s).

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
// A lane's accumulators of O^T as float4: slot 4*b + r/4 (32 rows), b (16 rows).
template <int ROWS>
constexpr int kSlots = ROWS / 2;

struct TreeArgs {
    const uint16_t* q;          // [nodes][n_q][128]
    const uint16_t* k;          // layer base
    const uint16_t* v;
    uint16_t* out;              // [nodes][n_q][128]
    float* out_f32;             // optional
    const uint64_t* mask;       // optional
    const int32_t* pos_dev;     // optional
    f32x4* part;                // [block][split][slot][lane]: a block is 32 (16) query rows of a KV head
    float2* part_ml;            // [block][split][row]: maximum (exp2 domain), sum
    int64_t row_stride;         // elements between positions of one KV head
    int64_t head_stride;        // elements between KV heads
    int32_t pos, nodes, group, n_q, rows, blocks, splits;  // rows = nodes * group, blocks = per KV head
    float scale_log2e;          // log2(e) / sqrt(128)
};

// The first of a slot's four columns.
template <int ROWS>
__device__ __forceinline__ int slot_column(int slot, int lane) {
    return ROWS == 32 ? 32 * (slot >> 2) + 8 * (slot & 3) + 4 * (lane >> 5) : 16 * slot + 4 * (lane >> 4);
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
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

// dma16 without the streaming hint: for the form of 32 rows whose tiles several workgroups read. Several blocks of 16 rows have the hint though they
// share tiles as well; us, with it : without, 8 KV heads: 8 nodes of 32 heads 7.3 : 7.3 at 250 positions, 8.5 : 8.7 at 2000, 10.2 : 10.2 at 4099, 26 nodes 8.5 : 8.3 at
// 500, 61 nodes 10.1 : 9.9 at 500, 5 nodes of 64 heads 10.3 : 10.1 at 3000; 16 nodes of 16 heads, 4 KV heads 13.2 : 11.7 at 8000. So two blocks lose a little without it and
// more of them gain.
__device__ __forceinline__ void dma16_kept(const char* base, uint32_t voff, uint32_t lds_off) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint32_t b_lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b), b_hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    const uint64_t sbase = ((uint64_t)b_hi << 32) | (uint64_t)b_lo;
    const uint32_t slds = (uint32_t)__builtin_amdgcn_readfirstlane(lds_off);
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(voff), "s"(sbase), "{m0}"(slds) : "memory");
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

// WM wavefronts side by side on ROWS query rows each, 4 / WM of them on a tile each of the same rows. EXACT: a probability enters the second
// product as the sum of two bf16 numbers (relative error 2^-16), otherwise as one (2^-8). KEPT: loads without the streaming hint.
template <int ROWS, int WM, bool EXACT, int STAGES, bool KEPT>
// (two workgroups on a compute unit where its LDS holds two rings: a hint without which the accumulators go to AGPRs and back)
__global__ __launch_bounds__(kWaves * 64, STAGES * (kWaves / WM) * kTileBytes <= 80 * 1024 ? 2 : 1) void mha_tree_kernel(TreeArgs a) {
    constexpr int WK = kWaves / WM;
    constexpr int kStageBytes = WK * kTileBytes;
    constexpr int kLoads = 16 / WM;      // 1 KiB blocks of a tile per wavefront: eight of K, eight of V
    constexpr int kScores = ROWS / 2;    // a lane's keys of a tile
    constexpr int kSteps = 128 * ROWS / 512;  // fragments of a query row per lane
    constexpr int kS = kSlots<ROWS>;
    __shared__ __attribute__((aligned(1024))) char smem[STAGES * kStageBytes];
    __shared__ float merge_m[kWaves][ROWS], merge_l[kWaves][ROWS];
    __shared__ uint64_t sees_s[WM][ROWS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wk = wave / WM;
    const int n = lane & (ROWS - 1), kg = lane / ROWS;  // query row; which of the lanes that share it
    const int i16 = lane & 15;
    const int kvh = blockIdx.x, split = blockIdx.y;
    const int block = blockIdx.z * WM + wm;  // of ROWS query rows
    const int row = block * ROWS + n;
    const bool has_rows = block * ROWS < a.rows;

    const int pos = position(a);
    const int keys = pos + a.nodes;
    const int tiles = (keys + kKeys - 1) / kKeys;
    const int run = __builtin_amdgcn_readfirstlane(tiles / a.splits), longer = tiles - run * a.splits;
    const int t0 = split * run + min(split, longer), t1 = t0 + run + (split < longer ? 1 : 0);
    const int iters = (t1 - t0 + WK - 1) / WK;

    // The query rows (those behind the last one repeat it) and the nodes they see.
    u32x4 q[kSteps];
    const int row_in = min(row, a.rows - 1);
    const int node = row_in / a.group;
    {
        const u32x4* src = reinterpret_cast<const u32x4*>(a.q + ((int64_t)node * a.n_q + kvh * a.group + (row_in - node * a.group)) * kHeadDim);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = src[(64 / ROWS) * s + kg];
    }
    uint64_t sees = a.mask ? a.mask[node] : ~0ull >> (63 - node);
    sees &= ~0ull >> (64 - a.nodes);

    const uint32_t rs = (uint32_t)a.row_stride * 2u;
    const char* kb = reinterpret_cast<const char*>(a.k + (int64_t)kvh * a.head_stride);
    const char* vb = reinterpret_cast<const char*>(a.v + (int64_t)kvh * a.head_stride);
    const uint32_t smem0 = (uint32_t)(uintptr_t)smem;

    // Where a lane of a load fetches from: row rho of a block of four, the chunk that the swizzle wants at place i16 (a row's low bits
    // follow from the block's).
    const int rho = lane >> 4;
    auto k_off = [&](int b) { return (uint32_t)rho * rs + (uint32_t)((i16 ^ (4 * (b & 3) + rho)) * 16); };
    auto v_off = [&](int b) { return (uint32_t)rho * rs + (uint32_t)((((i16 >> 1) - (4 * (b & 1) + rho)) & 7) * 32 + (i16 & 1) * 16); };
    // (several wavefronts share a tile's blocks: one has blocks of K or of V alone)
    uint32_t lane_off[WM == 1 ? 8 : 4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        if constexpr (WM == 1) {
            lane_off[b] = k_off(b);
            lane_off[4 + b] = v_off(b);
        } else {
            lane_off[b] = wm < WM / 2 ? k_off(b) : v_off(b);
        }
    }

    auto issue = [&](int it, int stage) __attribute__((always_inline)) {
        const int t = t0 + it * WK + wk;
        if (t >= t1) return;
        const char* kt = kb + (int64_t)t * kKeys * rs;
        const char* vt = vb + (int64_t)t * kKeys * rs;
        const int last = keys - 1 - t * kKeys;
        const uint32_t to = smem0 + (uint32_t)(stage * kStageBytes + wk * kTileBytes);
        auto load = [&](auto whole) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int b = wm * kLoads + i, b8 = b & 7;
                const bool is_k = WM == 1 ? i < 8 : wm < WM / 2;
                uint32_t off = lane_off[(i & 3) + (WM == 1 && i >= 8 ? 4 : 0)];
                const char* base = is_k ? kt : vt;
                if constexpr (decltype(whole)::value) base += (int64_t)(4 * b8) * rs;
                else off += (uint32_t)(min(4 * b8 + rho, last) - rho) * rs;  // rows past the keys repeat the last one: seen by nobody
                scalar_base(base);
                if constexpr (!KEPT) dma16(base, off, to + (uint32_t)(b * 1024));
                else dma16_kept(base, off, to + (uint32_t)(b * 1024));
            }
        };
        if (last >= kKeys - 1) load(std::true_type{});
        else load(std::false_type{});
    };

    const uint32_t k_x = (uint32_t)(kg ^ i16);  // chunk (64 / ROWS) * s + kg of row n lies at chunk ((64 / ROWS) * s) ^ k_x
    const uint32_t k_row = (uint32_t)n * 256u;
    const int v_key = 4 * kg + (i16 >> 2);      // a transposing read: sixteen lanes, four keys of a 32-byte piece
    const int v_piece = (ROWS == 32 ? (lane >> 4) & 1 : 0) + v_key;
    const uint32_t v_row = (uint32_t)(v_key * 256 + (i16 & 3) * 8);
    float m_run = -FLT_MAX, l_run = 0.0f;  // (a finite maximum: scores of -inf get weight 0, not NaN)
    using Acc = std::conditional_t<ROWS == 32, f32x16, f32x4>;
    constexpr int kAccs = ROWS == 32 ? 4 : 8, kAccSize = ROWS == 32 ? 16 : 4;
    Acc o[kAccs];
#pragma unroll
    for (int b = 0; b < kAccs; ++b) o[b] = Acc{};

    uint32_t broken = 0u;  // bits 15 and 31: a value that is not finite among the nodes' tiles
    constexpr int kV = kAccs * (ROWS == 32 ? 2 : 1);  // V fragments: step s of columns b
    typedef __attribute__((address_space(3))) char LdsChar;
    typedef __attribute__((address_space(3))) i16x4 LdsVec;
    const LdsChar* ring = (const LdsChar*)smem + wk * kTileBytes;
    struct VFrag {
        u32x2 half[2];
    };
    struct Scores {
        float c[kScores];
    };
    auto k_frag = [&](int stage, int x) __attribute__((always_inline)) {
        const int s = x % kSteps, u = x / kSteps;  // (16 rows: the tile's upper sixteen keys behind the lower)
        const LdsChar* at = ring + k_row + (((uint32_t)((64 / ROWS) * s) ^ k_x) << 4);
        return *(const __attribute__((address_space(3))) u32x4*)(at + (stage * kStageBytes + u * 4096));
    };
    auto v_frag = [&](int stage, int f) __attribute__((always_inline)) {
        const int b = ROWS == 32 ? f >> 1 : f;
        const LdsChar* at = ring + v_row + (uint32_t)(((b * (ROWS / 16) + v_piece) & 7) * 32);  // (the rest: a constant of the instruction)
        VFrag v;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int key = ROWS == 32 ? 16 * (f & 1) + 8 * x : 16 * x;
            v.half[x] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsVec*)(at + (stage * kStageBytes + kTileBytes / 2 + key * 256))));
        }
        return v;
    };
    auto scores = [&](int stage) __attribute__((always_inline)) {
        // (all of K's fragments are asked for before the first product waits for one)
        u32x4 k[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) k[x] = k_frag(stage, x);
        asm volatile("" : "+v"(k[0]), "+v"(k[1]), "+v"(k[2]), "+v"(k[3]), "+v"(k[4]), "+v"(k[5]), "+v"(k[6]), "+v"(k[7]));
        Scores y;
#pragma unroll
        for (int u = 0; u < 8 / kSteps; ++u) {
            Acc x{};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) x = mfma(__builtin_bit_cast(bf16x8, k[u * kSteps + s]), __builtin_bit_cast(bf16x8, q[s]), x);
#pragma unroll
            for (int r = 0; r < kAccSize; ++r) y.c[u * kAccSize + r] = x[r];
        }
        return y;
    };
    // A tile's scores and values (at `stage`) into the running softmax. NEXT: the next tile's keys are at `ahead`; its scores are formed
    // between the exponentials of this one's and returned. CACHED: the tile has no nodes.
    auto fold = [&](int t, Scores y, int stage, int ahead, auto next, auto cached) __attribute__((always_inline)) {
        constexpr bool NEXT = decltype(next)::value, CACHED = decltype(cached)::value;
        static_assert(!NEXT || ROWS == 32, "");
        auto& c = y.c;
        VFrag v[kV];
        u32x4 k[8];
        if constexpr (NEXT) {
#pragma unroll
            for (int x = 0; x < 4; ++x) k[x] = k_frag(ahead, x);
        } else {
#pragma unroll
            for (int f = 0; f < kV; ++f) v[f] = v_frag(stage, f);
        }
        // Tiles with nodes in them: what a row does not see has no weight. Bit of `vis`: the key less 4 * kg.
        const bool nodes = !CACHED && (t + 1) * kKeys > pos;
        if (nodes) {
            const int at = t * kKeys + 4 * kg - pos;
            const uint32_t vis = at <= -32 ? ~0u : at >= 64 ? 0u : at >= 0 ? (uint32_t)(sees >> at) : (uint32_t)(sees << -at) | ((1u << -at) - 1u);
#pragma unroll
            for (int r = 0; r < kScores; ++r) c[r] = vis >> ((ROWS == 32 ? 8 : 16) * (r >> 2) + (r & 3)) & 1u ? c[r] : -INFINITY;
        }
        float top = c[0];
#pragma unroll
        for (int r = 1; r < kScores; ++r) top = fmaxf(top, c[r]);
        top = (ROWS == 32 ? halves_max(top) : rows_max(top)) * a.scale_log2e;
        // The accumulators are rescaled only where a row's maximum has grown by more than 2^8: up to that its weights are
        // just larger than 1.
        if (__any(top > m_run + 8.0f)) {
            const float m_new = fmaxf(m_run, top);
            const float alpha = fast_exp2(m_run - m_new);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int b = 0; b < kAccs; ++b)
#pragma unroll
                for (int r = 0; r < kAccSize; ++r) o[b][r] *= alpha;
        }
        Scores y_next;
        Acc x_next{};
        float sum = 0.0f;
        u32x4 ph[kScores / 8], pl[kScores / 8];
#pragma unroll
        for (int s = 0; s < kScores / 2; ++s) {
            if constexpr (NEXT) {
                // (in this order: a product, the reads that later ones wait for, then the vector instructions of two scores, which wait for
                // neither)
                x_next = mfma(__builtin_bit_cast(bf16x8, k[s]), __builtin_bit_cast(bf16x8, q[s]), x_next);
                if (s < 4) k[s + 4] = k_frag(ahead, s + 4);
                v[s] = v_frag(stage, s);
            }
            const float p0 = fast_exp2(__builtin_fmaf(c[2 * s], a.scale_log2e, -m_run));
            const float p1 = fast_exp2(__builtin_fmaf(c[2 * s + 1], a.scale_log2e, -m_run));
            sum += p0 + p1;
            const uint32_t w = pack_bf16(p0, p1);
            ph[s >> 2][s & 3] = w;
            if constexpr (EXACT) pl[s >> 2][s & 3] = pack_bf16(p0 - bf16_lo(w), p1 - bf16_hi(w));
            if constexpr (NEXT) __builtin_amdgcn_sched_barrier(0);
        }
        l_run += sum;
        if constexpr (NEXT) {
#pragma unroll
            for (int r = 0; r < kAccSize; ++r) y_next.c[r] = x_next[r];
        }
        if (nodes) {
            // A weight of 0 times an infinity or NaN would be NaN: those enter as 0 here and are added at the end, for the rows that
            // see them. (An exponent of all ones carries into the sign's place.)
#pragma unroll
            for (int f = 0; f < kV; ++f)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    typedef short i16x2 __attribute__((ext_vector_type(2)));
                    const uint32_t w = v[f].half[j >> 1][j & 1];
                    const uint32_t carry = (w & 0x7f807f80u) + 0x00800080u;
                    broken |= carry;
                    v[f].half[j >> 1][j & 1] = w & ~__builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, carry) >> 15);
                }
        }
        // (the second product's wavefront goes first: its products keep the matrix cores busy while the other wavefront of the SIMD has its
        // vector instructions between them. 64 nodes of 64 heads at 131000 positions 322 : 290 us, 61 of 32 heads at 32768 55.8 : 52.2.)
        if constexpr (NEXT) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int f = 0; f < kV; ++f) {
            const int b = ROWS == 32 ? f >> 1 : f, s = ROWS == 32 ? f & 1 : 0;
            const u32x4 vf = {v[f].half[0][0], v[f].half[0][1], v[f].half[1][0], v[f].half[1][1]};
            o[b] = mfma(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, ph[s]), o[b]);
            if constexpr (EXACT) o[b] = mfma(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, pl[s]), o[b]);
        }
        if constexpr (NEXT) __builtin_amdgcn_s_setprio(0);
        return y_next;
    };
    const int my_tiles = t1 - t0 > wk ? (t1 - t0 - wk + WK - 1) / WK : 0;
    // This wavefront's tile `it` has landed, up to `newer` ones behind it stay in flight; then every wavefront's, and all have read what is
    // refilled next. (Needed where wavefronts share tiles; with WM == 1 each has its own, and they wait for one another all the same.)
    auto wait_for = [&](int it, int newer) __attribute__((always_inline)) {
        newer = min(newer, my_tiles - 1 - it);
        if (newer >= 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * kLoads) : "memory");
        else if (newer == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) issue(s, s);
    if constexpr (STAGES == 4) {
        // A tile's scores are formed an iteration ahead: matrix cores and vector ALU of one wavefront work side by side. In use are the next
        // tile's keys and this one's values; one tile is in flight, one is asked for in the place of the tile before.
        Scores y;
        if (iters > 0) {
            wait_for(0, 2);
            y = scores(0);
        }
        auto step = [&](int it, int stage, auto cached) __attribute__((always_inline)) {
            if (it + 1 < iters) wait_for(it + 1, 1);
            if (it + 3 < iters) issue(it + 3, (stage + 3) & 3);
            if (has_rows && it < my_tiles) {
                // (behind the last tile the scores are of whatever lies there, and not used)
                y = fold(t0 + it * WK + wk, y, stage, (stage + 1) & 3, std::true_type{}, cached);
            }
        };
        // Four at a time where no tile has nodes: the places in the ring are constants then, and the scores change registers by name.
        const int cached = min(max((pos / kKeys - t0) / WK, 0), iters);
        int it = 0;
        sees_s[wm][n] = sees;  // (not needed meanwhile, and the registers are)
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (; it + 4 <= cached; it += 4) static_for<0, 4>([&](auto s) __attribute__((always_inline)) { step(it + s.value, s.value, std::true_type{}); });
        sees = sees_s[wm][n];
#pragma unroll 1
        for (; it < iters; ++it) step(it, it & 3, std::false_type{});
    } else {
        int stage = 0;
#pragma unroll 1
        for (int it = 0; it < iters; ++it) {
            wait_for(it, 0);
            if (it + 1 < iters) issue(it + 1, stage ^ 1);
            if (has_rows && it < my_tiles) {
                const Scores y = scores(stage);
                fold(t0 + it * WK + wk, y, stage, 0, std::false_type{}, std::false_type{});
            }
            stage ^= 1;
        }
    }

    // Infinities and NaN among the values of the nodes' tiles, for the rows that see them: nodes, and (x < 0, seen by all) the cached positions
    // that share the first node's tile.
    if (__builtin_expect(__any((broken & 0x80008000u) != 0u), 0)) {
#pragma unroll 1
        for (int x = -(pos % kKeys); x < a.nodes; ++x) {
            const int t = (pos + x) / kKeys;
            if (t < t0 || t >= t1 || (t - t0) % WK != wk) continue;
            const char* at = vb + (int64_t)(pos + x) * rs;
            const bool seen = x < 0 || (sees >> x & 1);
#pragma unroll
            for (int slot = 0; slot < kS; ++slot) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(at + 2 * slot_column<ROWS>(slot, lane));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t we = w[e >> 1];
                    const float y = (e & 1) ? bf16_hi(we) : bf16_lo(we);
                    if (seen && !(fabsf(y) < INFINITY)) o[4 * slot / kAccSize][(4 * slot + e) % kAccSize] += y;
                }
            }
        }
    }

    // Join the wavefronts of the same rows, each a part of the columns; then out, or to the workspace.
    auto slot_of = [&](int x) __attribute__((always_inline)) {
        const int b = 4 * x / kAccSize, r = 4 * x % kAccSize;
        return f32x4{o[b][r], o[b][r + 1], o[b][r + 2], o[b][r + 3]};
    };
    l_run = ROWS == 32 ? halves_sum(l_run) : rows_sum(l_run);
    f32x4 mine[kS / WK];
    if constexpr (WK > 1) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        static_assert(kWaves * kS * 64 * 16 <= sizeof(smem), "the accumulators of all wavefronts fit the ring");
        f32x4* parts = reinterpret_cast<f32x4*>(smem);
#pragma unroll
        for (int x = 0; x < kS; ++x) parts[(wave * kS + x) * 64 + lane] = slot_of(x);
        if (kg == 0) {
            merge_m[wave][n] = m_run;
            merge_l[wave][n] = l_run;
        }
        __syncthreads();
        float m = -FLT_MAX, w[WK], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < WK; ++i) m = fmaxf(m, merge_m[i * WM + wm][n]);
#pragma unroll
        for (int i = 0; i < WK; ++i) {
            w[i] = fast_exp2(merge_m[i * WM + wm][n] - m);
            sum += w[i] * merge_l[i * WM + wm][n];
        }
#pragma unroll
        for (int x = 0; x < kS / WK; ++x) {
            mine[x] = f32x4{};
#pragma unroll
            for (int i = 0; i < WK; ++i) {
                const f32x4 y = parts[((i * WM + wm) * kS + wk * (kS / WK) + x) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[x][e] += w[i] * y[e];
            }
        }
        m_run = m;
        l_run = sum;
    } else {
#pragma unroll
        for (int x = 0; x < kS; ++x) mine[x] = slot_of(x);
    }
    if (!has_rows) return;
    if (a.splits == 1) {
#pragma unroll
        for (int x = 0; x < kS / WK; ++x) write_out(a, kvh, row, slot_column<ROWS>(wk * (kS / WK) + x, lane), mine[x], l_run);
        return;
    }
    const int64_t at = (int64_t)(kvh * a.blocks + block) * a.splits + split;
    if (t1 > t0) {
#pragma unroll
        for (int x = 0; x < kS / WK; ++x) a.part[(at * kS + wk * (kS / WK) + x) * 64 + lane] = mine[x];
    }
    // (a split without keys leaves no part: a maximum of -inf says so)
    if (wk == 0 && kg == 0) a.part_ml[at * ROWS + n] = t1 > t0 ? make_float2(m_run, l_run) : make_float2(-INFINITY, 0.0f);
}

// The splits of a block joined: a workgroup per slot, its W wavefronts on every W-th split, eight of them asked for at once.
template <int ROWS, int W>
__global__ __launch_bounds__(W * 64) void mha_tree_join_kernel(TreeArgs a) {
    constexpr int kAhead = 8;
    __shared__ f32x4 wave_o[W][64];
    __shared__ float wave_m[W][64], wave_l[W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kvh = blockIdx.x, slot = blockIdx.y, block = blockIdx.z;
    const int n = lane & (ROWS - 1);
    const int64_t first = (int64_t)(kvh * a.blocks + block) * a.splits;
    const float2* ml = a.part_ml + first * ROWS + n;
    const f32x4* part = a.part + (first * kSlots<ROWS> + slot) * 64 + lane;
    float m = -FLT_MAX, sum = 0.0f;
    f32x4 o{};
    for (int s0 = wave; s0 < a.splits; s0 += W * kAhead) {
        float2 x[kAhead];
        f32x4 y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int s = min(s0 + W * i, a.splits - 1);
            x[i] = ml[s * ROWS];
            y[i] = part[(int64_t)s * kSlots<ROWS> * 64];
            if (s0 + W * i >= a.splits) x[i] = make_float2(-INFINITY, 0.0f);
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
            // (a split without keys has left no part; a weight of 0 alone does not say that: an infinity or NaN counts with it too)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = x[i].x == -INFINITY ? o[e] : o[e] + w * y[i][e];
        }
    }
    wave_o[wave][lane] = o;
    wave_m[wave][lane] = m;
    wave_l[wave][lane] = sum;
    __syncthreads();
    if (wave != 0) return;
    float top = m;
#pragma unroll
    for (int i = 1; i < W; ++i) top = fmaxf(top, wave_m[i][lane]);
    f32x4 all{};
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float w = fast_exp2(wave_m[i][lane] - top);
        const f32x4 y = wave_o[i][lane];
        total += w * wave_l[i][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) all[e] += w * y[e];
    }
    write_out(a, kvh, block * ROWS + n, slot_column<ROWS>(slot, lane), all, total);
}

template <int ROWS, int WM, bool EXACT, int STAGES, bool KEPT>
void launch(const TreeArgs& a, int n_kv, hipStream_t stream) {
    const dim3 grid(n_kv, a.splits, (a.blocks + WM - 1) / WM), block(kWaves * 64);
    hipLaunchKernelGGL((mha_tree_kernel<ROWS, WM, EXACT, STAGES, KEPT>), grid, block, 0, stream, a);
    if (a.splits == 1) return;
    // (a trip to memory for all splits up to 128)
    const dim3 join(n_kv, kSlots<ROWS>, a.blocks);
    if (a.splits <= 32) hipLaunchKernelGGL((mha_tree_join_kernel<ROWS, 4>), join, dim3(4 * 64), 0, stream, a);
    else if (a.splits <= 64) hipLaunchKernelGGL((mha_tree_join_kernel<ROWS, 8>), join, dim3(8 * 64), 0, stream, a);
    else hipLaunchKernelGGL((mha_tree_join_kernel<ROWS, 16>), join, dim3(16 * 64), 0, stream, a);
}

}  // namespace

int launch_mha_tree(const llmi_mha_tree_args& args, const TreeForm& form) {
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
    const int n_kv = m.kv_dim / kHeadDim;
    a.blocks = form.blocks;
    a.splits = form.splits;
    a.part = static_cast<f32x4*>(m.workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part + (size_t)n_kv * a.blocks * a.splits * (form.rows / 2) * 64);
    a.scale_log2e = 1.4426950408889634f / sqrtf((float)kHeadDim);
    const hipStream_t stream = static_cast<hipStream_t>(m.stream);
    // Two wavefronts on each of two tiles: scores ahead from six pairs of tiles a split on, before that the longer way to the first product costs
    // more (two stages : four, us, 16 nodes of 32 heads, 8 KV heads: 13.2 : 14.3 at 6000 positions, 16.5 : 17.1 at 10000, 19.9 : 19.5 at 14000, 33.4 : 30.4
    // at 32768).
    constexpr int kPairsAhead = 6;
    const int pairs = (m.pos + args.node_num) / kKeys / (2 * a.splits);
    if (form.rows == 16) launch<16, 1, true, 2, false>(a, n_kv, stream);
    else if (form.row_waves == 1) launch<32, 1, true, 2, false>(a, n_kv, stream);
    else if (form.row_waves == 2 && pairs < kPairsAhead) launch<32, 2, true, 2, false>(a, n_kv, stream);
    else if (form.row_waves == 2) launch<32, 2, true, 4, false>(a, n_kv, stream);
    else if (form.blocks <= 4) launch<32, 4, true, 4, false>(a, n_kv, stream);
    // Beyond 128 query rows the matrix cores are the bound: with one bf16 number a probability, half as many of the second product's instructions; a
    // bf16 output rounds as much by itself. Whoever asks for the fp32 output gets both. us, one : two numbers: 64 nodes of 64 heads, 8 KV heads 35.5 : 41.1
    // at 8000 positions, 293 : 393 at 131000, 61 nodes of 32 heads 20.7 : 22.6 at 6000, 56.4 : 67.5 at 32768.
    else if (a.out_f32) launch<32, 4, true, 4, true>(a, n_kv, stream);
    else launch<32, 4, false, 4, true>(a, n_kv, stream);
    return check_launch();
}

}  // namespace llmi
