// vsl_attn_mods.h -- device helpers of attention with modified scores (vsl_attn_mods.hip, vsl_attn_mods_prefill.hip).
#pragma once
#include <cmath>

#include "vsl_device.h"

namespace attn_mods {

constexpr float kLog2e = 1.4426950408889634f;

// tanh(u) for |u| <= kTanhNear: u times a polynomial in u^2 (the weighted least squares fit whose largest relative error is
// smallest, found by reweighting: 1.4e-7). Scores of trained models lie here: a cap of 50 bends one of 10 by 0.13.
constexpr float kTanhNear = 0.64f;
constexpr int kTanhTerms = 5;
constexpr float kTanhPoly[kTanhTerms] = {0.999999866f, -0.33331689f, 0.133005777f, -0.0516386036f, 0.0147901969f};
__device__ __forceinline__ float tanh_near(float u) {
    const float z = u * u;
    float p = kTanhPoly[kTanhTerms - 1];
#pragma unroll
    for (int i = kTanhTerms - 2; i >= 0; --i) p = fmaf(p, z, kTanhPoly[i]);
    return u * p;
}
// The same anywhere: beyond, (1 - e) / (1 + e) with e = exp(-2 |u|) <= 0.28, which loses nothing to cancellation.
__device__ __forceinline__ float tanh_any(float u) {
    const float e = __builtin_amdgcn_exp2f(-2.f * kLog2e * fabsf(u)), n = 1.f - e, d = 1.f + e;
    const float r = __builtin_amdgcn_rcpf(d);
    float q = n * r;
    q = fmaf(fmaf(-q, d, n), r, q);
    q = copysignf(q, u);
    return fabsf(u) > kTanhNear ? q : tanh_near(u);  // NaN: the polynomial's
}

// Softmax against a reference per row (log2 units), raised to kRoom below the largest score seen and only when a score
// exceeds it by more than kRoom + kLazy: probabilities stay within binary16 (2^15), and what the planes drop of a small
// one is 2^-32 of the largest.
constexpr float kLazy = 8.f, kRoom = 7.f;

// Two values rounded to binary16 in one instruction, the pair through an empty register asm, so that what is used and
// what is subtracted from the values are the same rounding.
__device__ __forceinline__ half2v round2(float a, float b) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    half2v h = __builtin_convertvector((float2v{a, b}), half2v);
    asm volatile("" : "+v"(h));
    return h;
}

// LDS position (in halfs) of 16-byte chunk c of row r of a [rows][HD] tile: the chunks of a row exchanged (an xor by bits of
// the row) so that what a half wave reads at once lies in different banks: 16 bytes of one column of 16 rows (the operand
// K), and 64 bytes of four rows (a transpose read of V). The row's two low bits move whole 64-byte groups; with its bits in
// order (an xor by r & 15) four rows' 64 bytes fell onto the same 16 banks, 59 % of the LDS cycles of prompt attention.
template <int HD>
__device__ __forceinline__ constexpr int swizzle_bits(int r) {
    if constexpr (HD == 128) return (r & 3) << 2 | ((r >> 2) & 3);          // 256-byte rows
    else return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);                        // 128-byte rows: by pairs
}
template <int HD>
__device__ __forceinline__ int swizzle(int r, int c) {
    return r * HD + ((c ^ swizzle_bits<HD>(r)) * 8);
}

// Whether a word of two halfs holds an infinity or a NaN: the carry out of an exponent of ones, in bit 15 of either half.
__device__ __forceinline__ uint32_t odd_halfs(uint32_t w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// Whether a cap can be used with a scale: both factors of a score, scale / softcap and softcap * log2(e), normal numbers of 32 bits
// (below, they have fewer digits).
inline bool softcap_ok(float softcap, float scale) {
    return softcap == 0.f || (softcap > 0.f && std::isnormal(softcap * kLog2e) && (std::isnormal(scale / softcap) || scale == 0.f || !std::isfinite(scale)));
}

}  // namespace attn_mods
