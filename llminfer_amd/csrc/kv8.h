// The 8-bit KV cache on the device: where a record keeps what, how a row becomes codes and a scale, and back.
//
// A row is 128 values of a KV head's K or V at a position, as the bf16 cache holds them. Its scale s is the smallest number of eight
// significant bits with s * top >= the largest magnitude (top = 448 for E4M3, 127 for whole numbers), 2^-64 at least; a code is x / s rounded to
// nearest even and stands for code * s. A row with an infinity or NaN has s = NaN and codes of 0: a row of NaN.
// Eight bits are what makes fp32 enough: x and s have 8-bit significands, a border between two codes has five (E4M3) or eight, so a quotient
// that is not on a border is at least 2^-17 of itself away from it, and the same holds for largest / top and the 8-bit numbers.
//
// The cache is [layer][KV head][record of 32 positions], a record 8320 bytes: 4096 of K codes, 4096 of V codes, 64 of K scales, 64 of V
// scales (bf16). Position 16 t + 4 g + i of a record (t < 2, g < 4, i < 4):
//   K codes  [position / 16][channel / 16][position % 16][channel % 16]: a 1 KiB load of 16 bytes a lane is an operand of S^T = K Q^T (lane L:
//            position L % 16, channels 16 (4 h + L / 16) .. + 15 of load h)
//   V codes  [channel / 32][g][channel % 16][channel / 16 % 2][t][i]: a 1 KiB load is two operands of O^T = V^T P^T (lane L: channel L % 16 of
//            two groups of sixteen, the positions that lane's P^T holds: g = L / 16)
//   scales   [g][t][i]: 16 bytes are a lane's eight
// so a record is ten loads of whole cache lines whose bytes are where the matrix instructions want them: no LDS, no transposition.
#ifndef LLMI_KV8_H
#define LLMI_KV8_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mha_device_helpers.h"

namespace llmi {
namespace {

constexpr int kVBytes = 4096, kScaleBytes = 8192;  // where a record's V codes and scales begin

// Bytes of a record that belong to position p and channel c; of the scales of position p (K; V's lie 64 behind).
__device__ __forceinline__ int k_byte(int p, int c) { return (p >> 4) * 2048 + (c >> 4) * 256 + (p & 15) * 16 + (c & 15); }
__device__ __forceinline__ int v_byte(int p, int c) {
    return kVBytes + (c >> 5) * 1024 + ((p >> 2) & 3) * 256 + (c & 15) * 16 + ((c >> 4) & 1) * 8 + (p >> 4) * 4 + (p & 3);
}
__device__ __forceinline__ int k_scale_byte(int p) { return kScaleBytes + ((p >> 2) & 3) * 16 + (p >> 4) * 8 + (p & 3) * 2; }

// A row's scale from its largest magnitude, the bits of a bf16 number (infinities and NaN: NaN).
template <int FORMAT>
__device__ __forceinline__ float kv8_scale(uint32_t top_bits) {
    if (top_bits >= 0x7f80u) return __builtin_bit_cast(float, 0x7fc00000u);
    const float least = __builtin_bit_cast(float, top_bits << 16) / (FORMAT == LLMI_KV8_E4M3 ? 448.0f : 127.0f);
    const uint32_t up = (__builtin_bit_cast(uint32_t, least) + 0xffffu) & 0xffff0000u;
    return __builtin_bit_cast(float, max(up, 0x1f800000u));
}

// x / s of finite x, rounded correctly where it matters: a quotient that fp32 holds (all that lie on a border between two codes) comes out as it
// is, others within two units of the last place. (The remainder is taken as y s - x: a zero keeps its sign.)
__device__ __forceinline__ float kv8_quotient(float x, float s, float r) {
    const float y = x * r;
    return __builtin_fmaf(-__builtin_fmaf(y, s, -x), r, y);
}

// Four values' codes, the first in the low byte; r = 1 / s. Of a scale of NaN: zeros.
template <int FORMAT>
__device__ __forceinline__ uint32_t kv8_codes(float x0, float x1, float x2, float x3, float s, float r) {
    const float y0 = kv8_quotient(x0, s, r), y1 = kv8_quotient(x1, s, r), y2 = kv8_quotient(x2, s, r), y3 = kv8_quotient(x3, s, r);
    uint32_t w;
    if constexpr (FORMAT == LLMI_KV8_E4M3) {
        w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false);
        w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y2, y3, (int)w, true);
    } else {
        const int i0 = (int)__builtin_rintf(y0), i1 = (int)__builtin_rintf(y1), i2 = (int)__builtin_rintf(y2), i3 = (int)__builtin_rintf(y3);
        w = ((uint32_t)i0 & 255u) | ((uint32_t)i1 & 255u) << 8 | ((uint32_t)i2 & 255u) << 16 | (uint32_t)i3 << 24;
    }
    return s == s ? w : 0u;
}

// What two codes of a word stand for, without the scale, as a pair of bf16 numbers (exact): bytes 0 and 1, or with UPPER 2 and 3.
template <int FORMAT, bool UPPER>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w) {
    if constexpr (FORMAT == LLMI_KV8_E4M3) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, UPPER));
    } else {
        return pack_bf16((float)(int8_t)(w >> (UPPER ? 16 : 0)), (float)(int8_t)(w >> (UPPER ? 24 : 8)));
    }
}
// Eight codes (two words) as a matrix instruction's operand.
template <int FORMAT>
__device__ __forceinline__ bf16x8 kv8_operand(uint32_t w0, uint32_t w1) {
    return __builtin_bit_cast(bf16x8, u32x4{kv8_pair<FORMAT, false>(w0), kv8_pair<FORMAT, true>(w0), kv8_pair<FORMAT, false>(w1), kv8_pair<FORMAT, true>(w1)});
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_partner_u32(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
}
// The largest over the sixteen lanes of a DPP row, in all of them.
__device__ __forceinline__ uint32_t row16_max(uint32_t x) {
    x = max_u32(x, dpp_partner_u32<0xB1>(x));
    x = max_u32(x, dpp_partner_u32<0x4E>(x));
    x = max_u32(x, dpp_partner_u32<0x141>(x));
    return max_u32(x, dpp_partner_u32<0x140>(x));
}
// ... over the 32 lanes of half a wavefront.
__device__ __forceinline__ uint32_t row32_max(uint32_t x) {
    x = row16_max(x);
    const auto q = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const uint32_t q0 = q[0], q1 = q[1];
    return max_u32(q0, q1);
}
// The larger magnitude of two bf16 numbers, as bits.
__device__ __forceinline__ uint32_t pair_magnitude(uint32_t w) { return max_u32(w & 0x7fffu, (w >> 16) & 0x7fffu); }

// Four words whose bytes are a 4 x 4 matrix, transposed: byte j of word i to byte i of word j.
__device__ __forceinline__ void transpose_bytes(const uint32_t (&a)[4], uint32_t (&b)[4]) {
    const uint32_t p = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), q = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u);  // rows 0, 1: columns 0 and 1, 2 and 3
    const uint32_t r = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u), s = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
    b[0] = __builtin_amdgcn_perm(r, p, 0x05040100u);
    b[1] = __builtin_amdgcn_perm(r, p, 0x07060302u);
    b[2] = __builtin_amdgcn_perm(s, q, 0x05040100u);
    b[3] = __builtin_amdgcn_perm(s, q, 0x07060302u);
}
// x of lane I of the caller's four neighbours.
template <int I>
__device__ __forceinline__ float quad_lane(float x) { return dpp_partner<I * 0x55>(x); }

// A row on 32 lanes: lane p has dwords p and p + 32 of it (channels 2p, 2p + 1, 64 + 2p, 64 + 2p + 1).
struct NewRow {
    uint32_t x[2], w[2];      // the row, its norm weights
    uint32_t neighbour[2];    // the dwords of the pair's other lane: what four_pairs_squared adds up
    u32x2 sn, cs;
};
// (addresses as numbers, so that they can be chosen by selects: global loads all the same, a flat one would wait for LDS too)
__device__ __forceinline__ void load_row32(NewRow& y, uint64_t row, uint64_t w, int p) {
    typedef const __attribute__((address_space(1))) uint32_t* Words;
    const Words r = reinterpret_cast<Words>(row), n = reinterpret_cast<Words>(w);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        y.x[h] = r[p + 32 * h];
        y.neighbour[h] = r[(p ^ 1) + 32 * h];
        y.w[h] = n[p + 32 * h];
    }
}
__device__ __forceinline__ void load_tables32(NewRow& y, const float* sin_row, const float* cos_row, int p) {
    y.sn = reinterpret_cast<const u32x2*>(sin_row)[p];
    y.cs = reinterpret_cast<const u32x2*>(cos_row)[p];
}
// RMS norm and rotation of such a row, rounded to bf16: the bits of norm_rope_row32.
__device__ __forceinline__ void norm_rope_regs32(const NewRow& y, int p, float eps, uint32_t& lo, uint32_t& hi) {
    uint32_t first[2], second[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        first[h] = (p & 1) ? y.neighbour[h] : y.x[h];
        second[h] = (p & 1) ? y.x[h] : y.neighbour[h];
    }
    const float a[4] = {bf16_lo(first[0]), bf16_hi(first[0]), bf16_lo(second[0]), bf16_hi(second[0])};
    const float b[4] = {bf16_lo(first[1]), bf16_hi(first[1]), bf16_lo(second[1]), bf16_hi(second[1])};
    float ss = four_pairs_squared(a, b);
    ss += dpp_partner<0x4E>(ss);
    ss += dpp_partner<0x141>(ss);
    ss += dpp_partner<0x140>(ss);
    {
        const unsigned u = __builtin_bit_cast(unsigned, ss);
        const auto q = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const unsigned q0 = q[0], q1 = q[1];
        ss = __builtin_bit_cast(float, q0) + __builtin_bit_cast(float, q1);
    }
    const float r = inverse_rms(ss, eps);
    const uint32_t sn0 = y.sn[0], sn1 = y.sn[1], cs0 = y.cs[0], cs1 = y.cs[1];
    float l0, l1, h0, h1;
    rotate_scaled(scaled(bf16_lo(y.x[0]), bf16_lo(y.w[0]), r), scaled(bf16_lo(y.x[1]), bf16_lo(y.w[1]), r), __builtin_bit_cast(float, sn0),
                  __builtin_bit_cast(float, cs0), l0, h0);
    rotate_scaled(scaled(bf16_hi(y.x[0]), bf16_hi(y.w[0]), r), scaled(bf16_hi(y.x[1]), bf16_hi(y.w[1]), r), __builtin_bit_cast(float, sn1),
                  __builtin_bit_cast(float, cs1), l1, h1);
    lo = pack_bf16(l0, l1);
    hi = pack_bf16(h0, h1);
}
// The same on 16 lanes, a DPP row: lane p has channels 4p .. 4p + 3 and the four 64 behind them. The bits of norm_rope_row32 (see four_pairs_squared).
__device__ __forceinline__ void norm_rope_regs16(u32x2& lo, u32x2& hi, u32x2 wl, u32x2 wh, f32x4 sn, f32x4 cs, float eps) {
    const uint32_t xl0 = lo[0], xl1 = lo[1], xh0 = hi[0], xh1 = hi[1], wl0 = wl[0], wl1 = wl[1], wh0 = wh[0], wh1 = wh[1];
    const float a[4] = {bf16_lo(xl0), bf16_hi(xl0), bf16_lo(xl1), bf16_hi(xl1)};
    const float b[4] = {bf16_lo(xh0), bf16_hi(xh0), bf16_lo(xh1), bf16_hi(xh1)};
    const float wa[4] = {bf16_lo(wl0), bf16_hi(wl0), bf16_lo(wl1), bf16_hi(wl1)};
    const float wb[4] = {bf16_lo(wh0), bf16_hi(wh0), bf16_lo(wh1), bf16_hi(wh1)};
    float ss = four_pairs_squared(a, b);
    ss += dpp_partner<0xB1>(ss);
    ss += dpp_partner<0x4E>(ss);
    ss += dpp_partner<0x141>(ss);
    ss += dpp_partner<0x140>(ss);
    const float r = inverse_rms(ss, eps);
    float ol[4], oh[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) rotate_pair(a[e], b[e], wa[e], wb[e], r, sn[e], cs[e], ol[e], oh[e]);
    lo = u32x2{pack_bf16(ol[0], ol[1]), pack_bf16(ol[2], ol[3])};
    hi = u32x2{pack_bf16(oh[0], oh[1]), pack_bf16(oh[2], oh[3])};
}
// Such a row quantised: its scale, and the codes of lo's and hi's channels in the word's bytes 0, 1 and 2, 3.
template <int FORMAT>
__device__ __forceinline__ uint32_t quantise_row32(uint32_t lo, uint32_t hi, float& s) {
    s = kv8_scale<FORMAT>(row32_max(max_u32(pair_magnitude(lo), pair_magnitude(hi))));
    return kv8_codes<FORMAT>(bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi), s, 1.0f / s);
}
// ... and filed in its record.
__device__ __forceinline__ void file_row32(char* record, int pos, bool is_v, int p, uint32_t codes, float s) {
    if (is_v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) record[v_byte(pos, 2 * p + (e & 1) + 64 * (e >> 1))] = (char)(codes >> (8 * e));
    } else {
        *reinterpret_cast<uint16_t*>(record + k_byte(pos, 2 * p)) = (uint16_t)codes;
        *reinterpret_cast<uint16_t*>(record + k_byte(pos, 2 * p + 64)) = (uint16_t)(codes >> 16);
    }
    if (p == 0) *reinterpret_cast<uint16_t*>(record + k_scale_byte(pos) + (is_v ? 64 : 0)) = (uint16_t)(__builtin_bit_cast(uint32_t, s) >> 16);
}

}  // namespace
}  // namespace llmi

#endif
