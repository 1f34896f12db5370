// vsl_kv4.h -- layout of the 4-bit KV cache (VSL_DT_KV4, vsl_hip.h) and its expansion to binary16, shared by the
// kernels that write it and those that read it.
#pragma once
#include "vsl_device.h"

// Positions that a cache of `cap` holds room for (whole tiles of the kernels that read it), and the byte offset of its steps.
__device__ __host__ __forceinline__ constexpr uint64_t kv4_positions(uint32_t cap) { return ((uint64_t)cap + 127) & ~(uint64_t)127; }
__device__ __host__ __forceinline__ constexpr uint64_t kv4_steps_off(uint32_t n_kv, uint32_t cap, uint32_t hd) {
    return (n_kv * kv4_positions(cap) * hd / 2 + 255) & ~(uint64_t)255;
}
__device__ __host__ __forceinline__ constexpr uint64_t kv4_bytes(uint32_t n_kv, uint32_t cap, uint32_t hd) {
    return kv4_steps_off(n_kv, cap, hd) + n_kv * kv4_positions(cap) * (hd / 32) * 2;
}

constexpr uint32_t kKv4NaN = 0x7E00;  // the step of a block that reads back as NaN
// The largest other step that an append stores: d = 4352 (a range of 65280), z = 15. Past it (n - z) d may overflow, and
// so may what stands for a position that no append wrote, whose bits are anything.
constexpr uint32_t kKv4MaxStep = 0x6C4F;

// Shift of value e's nibble in a word of eight: values 2p and 2p + 1 lie 16 bits apart, so that one mask takes
// both into the halves of a register.
__device__ __host__ __forceinline__ constexpr uint32_t kv4_shift(uint32_t e) { return 4 * (e / 2 + 4 * (e & 1)); }

// The masks and exponents of the expansion, held in registers: as literals each mask-and-set would take two instructions
// (v_and_or_b32 takes no literal, and one scalar register).
struct Kv4Consts {
    uint32_t lo = 0x000F000Fu, hi = 0x00F000F0u, e1024 = 0x64006400u, e64 = 0x54005400u;
};
__device__ __forceinline__ Kv4Consts kv4_consts() {
    Kv4Consts c;
    asm volatile("" : "+s"(c.lo), "+s"(c.hi), "+v"(c.e1024), "+v"(c.e64));
    return c;
}

// Two steps as stored, apart: the step values d, and 1024 + z and 64 + z in binary16.
struct Kv4Step {
    half2v d, z1024, z64;
};
__device__ __forceinline__ Kv4Step kv4_step(uint32_t s2, const Kv4Consts& c) {
    return Kv4Step{__builtin_bit_cast(half2v, s2 & 0xFFF0FFF0u), __builtin_bit_cast(half2v, (s2 & c.lo) | c.e1024),
                   __builtin_bit_cast(half2v, ((s2 << 4) & c.hi) | c.e64)};
}

// Values 2p, 2p + 1 of a word. A nibble masked in place under the exponent of 1024 (bits 0-3, one unit each) or
// of 64 (bits 4-7, a sixteenth of a unit each) reads as 1024 + n or 64 + n, so the integer n - z is one packed
// subtraction, and its product with d is exact: 4 bits times 7 bits.
template <int p>
__device__ __forceinline__ half2v kv4_pair(uint32_t w, const Kv4Step& s, const Kv4Consts& c) {
    const uint32_t b = p >= 2 ? w >> 8 : w;
    if constexpr (p & 1) return (__builtin_bit_cast(half2v, (b & c.hi) | c.e64) - s.z64) * s.d;
    else return (__builtin_bit_cast(half2v, (b & c.lo) | c.e1024) - s.z1024) * s.d;
}
__device__ __forceinline__ half8 kv4_join(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The eight values of a word of K (one step for all) and of V (a step for each position: four pairs).
__device__ __forceinline__ half8 kv4_word(uint32_t w, const Kv4Step& s, const Kv4Consts& c) {
    return kv4_join(kv4_pair<0>(w, s, c), kv4_pair<1>(w, s, c), kv4_pair<2>(w, s, c), kv4_pair<3>(w, s, c));
}
__device__ __forceinline__ half8 kv4_word(uint32_t w, const Kv4Step (&s)[4], const Kv4Consts& c) {
    return kv4_join(kv4_pair<0>(w, s[0], c), kv4_pair<1>(w, s[1], c), kv4_pair<2>(w, s[2], c), kv4_pair<3>(w, s[3], c));
}

// Softmax against a reference m per row (log2 units) that is raised, to kKv4Room below the largest score seen, only when
// some score exceeds it by more than kKv4Room + kKv4Lazy: probabilities stay up to 2^15, within binary16, and what the pair
// of planes (or the one plane) drops of each, half a subnormal step 2^-25, is 2^-32 of the largest or less. (With m
// at the largest score it is 2^-25, and a tail of 16000 keys just below that share, 5e-4 of an output, is lost.) The
// excess is taken as the difference that the exponential gets, so the bound holds for scores that fp32 holds to whole
// powers of two, too.
constexpr float kKv4Lazy = 8.f, kKv4Room = 7.f;

// Two values rounded to binary16 in one instruction. The pair passes through an empty register asm, so that what is
// used and what is subtracted from the values are the same rounding.
__device__ __forceinline__ half2v pack_f16(float a, float b) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    half2v h = __builtin_convertvector((float2v{a, b}), half2v);
    asm volatile("" : "+v"(h));
    return h;
}
