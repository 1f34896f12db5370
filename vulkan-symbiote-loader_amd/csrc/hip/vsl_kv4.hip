// vsl_kv4.hip -- the 4-bit KV cache (VSL_DT_KV4): per-head norms of queries and keys with the rotation and the
// cache append in one pass, the cache read back as values, and decode attention over it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vsl_device.h"
#include "vsl_hip.h"
#include "vsl_internal.h"
#include "vsl_kv4.h"

namespace {

// ---------------------------------------------------------------------------------------------
// norms, rotation, append
// ---------------------------------------------------------------------------------------------
// A lane's double through a DPP move (two 32-bit moves).
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The same double of the lane 16 away (within 32 lanes), added.
__device__ __forceinline__ double add_lane16(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    return __builtin_bit_cast(double, (uint64_t)h[0] << 32 | l[0]) + __builtin_bit_cast(double, (uint64_t)h[1] << 32 | l[1]);
}
// Lane moves whose repeated use combines 2, 4, 8, 16 lanes: pairs, quads, half rows, rows.
constexpr int kDppPair = 0xB1, kDppQuad = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

template <int W>  // 16 or 32 lanes, every lane ending with the same sum
__device__ __forceinline__ double group_sum64(double v) {
    v += dpp64<kDppPair>(v);
    v += dpp64<kDppQuad>(v);
    v += dpp64<kDppHalfMirror>(v);
    v += dpp64<kDppMirror>(v);
    if constexpr (W == 32) v = add_lane16(v);
    return v;
}

// 1 / sqrt(x) to within an ulp or two: the hardware's estimate (26 bits or more) and two Newton steps, a third of the
// instructions of a 64-bit square root and division. 0 for infinite x.
__device__ __forceinline__ double rsqrt64(double x) {
    const double r0 = __builtin_amdgcn_rsq(x);
    double r = r0;
#pragma unroll
    for (int i = 0; i < 2; ++i) r = fma(0.5 * r, fma(-x * r, r, 1.0), r);
    return r0 == 0.0 ? 0.0 : r;
}

// Four consecutive dims of a head's row in one lane (HD / 4 lanes a row): the head's norm and rotation. T: float; or
// double for keys that become 4-bit codes, whose choice hangs on values next to a border: it is then the exact
// value's, and the same for every number of rows in a call. (In 64 bits throughout, 2048 rows of the 8B shape took 29.5
// us instead of 22.9, side by side: conversions and 64-bit operations, not memory, were the bound.)
struct RopeArgs {
    const float* q_gamma;
    const float* k_gamma;
    const float* rc;
    const float* rs;
    float eps;
    int halves;
};
// What a lane reads for its four dims: the row, and the rotation's angles (pairs: two; halves: four, of the dims' half).
struct RowIn {
    float4v x, co, si;
};
template <int HD>
__device__ __forceinline__ void load_angles(const RopeArgs& a, uint32_t pos, uint32_t c, RowIn& r) {
    const size_t row = (size_t)pos * (HD / 2);
    if (a.halves) {
        const uint32_t j = 4 * (c & (HD / 8 - 1));
        r.co = *reinterpret_cast<const float4v*>(a.rc + row + j);
        r.si = *reinterpret_cast<const float4v*>(a.rs + row + j);
    } else {
        const float2 co = *reinterpret_cast<const float2*>(a.rc + row + 2 * c);
        const float2 si = *reinterpret_cast<const float2*>(a.rs + row + 2 * c);
        r.co = float4v{co.x, co.y, 0.f, 0.f};
        r.si = float4v{si.x, si.y, 0.f, 0.f};
    }
}
// The gains of a lane's dims (ga; halves: of its dims of the first half ga, of the second gb).
struct Gains {
    float4v ga, gb;
};
template <int HD>
__device__ __forceinline__ Gains load_gains(const RopeArgs& a, const float* gamma, uint32_t c) {
    Gains g{{1.f, 1.f, 1.f, 1.f}, {1.f, 1.f, 1.f, 1.f}};
    if (!gamma) return g;
    const uint32_t j = a.halves ? 4 * (c & (HD / 8 - 1)) : 4 * c;
    g.ga = *reinterpret_cast<const float4v*>(gamma + j);
    if (a.halves) g.gb = *reinterpret_cast<const float4v*>(gamma + HD / 2 + j);
    return g;
}
template <int HD, typename T>
__device__ __forceinline__ void norm_rotate(const RowIn& r, bool norm, const Gains& g, const RopeArgs& a, uint32_t c, T (&y)[4]) {
    constexpr int L = HD / 4;
    T inv = 1;
    if (norm) {
        T ss = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fma((T)r.x[i], (T)r.x[i], ss);
        if constexpr (sizeof(T) == 8) {
            inv = rsqrt64(group_sum64<L>(ss) * (1.0 / HD) + (double)a.eps);
        } else {
            ss = group_sum_dpp<16>(ss);
            if constexpr (L == 32) {
                float s0, s1;
                lane_pair<16>(ss, s0, s1);
                ss = s0 + s1;
            }
            inv = 1.f / sqrtf(ss / HD + a.eps);
        }
    }
    if (!a.halves) {
        T v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (T)r.x[i] * inv * (T)g.ga[i];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const T co = (T)r.co[i / 2], si = (T)r.si[i / 2];
            y[i] = v[i] * co - v[i + 1] * si;
            y[i + 1] = v[i] * si + v[i + 1] * co;
        }
    } else {
        // the other half's four dims are L / 2 lanes away
        const bool first = c < (uint32_t)(L / 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float xa, xb;
            lane_pair<L / 2>(r.x[i], xa, xb);
            const T va = (T)xa * inv * (T)g.ga[i], vb = (T)xb * inv * (T)g.gb[i];
            const T co = (T)r.co[i], si = (T)r.si[i];
            y[i] = first ? va * co - vb * si : va * si + vb * co;
        }
    }
}

// rint(y / d), ties to even, from r near 1 / d (an ulp or two; |y / d| <= 15): the remainder of the nearest integer to
// y r is exact in either type (d has 7 significant bits), and tells on which side of a border y / d lies.
template <typename T>
__device__ __forceinline__ T rint_quotient(T y, T d, T r) {
    const T n = rint(y * r), rem = fma(-n, d, y), a = fabs(rem), h = (T)0.5 * d;
    const bool off = a > h || (a == h && ((int)n & 1));
    return off ? n + copysign((T)1, rem) : n;
}
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ double dpp_move(double v) {
    return dpp64<CTRL>(v);
}

// The 4-bit form of a block of 32 dims, four in each of 8 consecutive lanes: this lane's codes; returns the step
// as stored.
template <typename T>
__device__ __forceinline__ uint32_t kv4_quantize(const T (&y)[4], uint32_t (&n)[4]) {
    T lo = 0, hi = 0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo = fmin(lo, y[i]);
        hi = fmax(hi, y[i]);
        bad |= !(fabs(y[i]) < (T)INFINITY);
    }
    lo = fmin(lo, dpp_move<kDppPair>(lo));
    hi = fmax(hi, dpp_move<kDppPair>(hi));
    lo = fmin(lo, dpp_move<kDppQuad>(lo));
    hi = fmax(hi, dpp_move<kDppQuad>(hi));
    lo = fmin(lo, dpp_move<kDppHalfMirror>(lo));
    hi = fmax(hi, dpp_move<kDppHalfMirror>(hi));
    const uint64_t b = __builtin_amdgcn_ballot_w64(bad) >> (threadIdx.x & 56);
    const double range = (double)hi - (double)lo;
    if ((b & 0xFF) != 0 || range > 65280.0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) n[i] = 0;
        return kKv4NaN;
    }
    // d: the quotient by 15 cut to 7 significant bits, or the next such number where that is below it (15 times
    // either is exact)
    constexpr uint64_t one = 1ull << 46;
    const uint64_t u = __builtin_bit_cast(uint64_t, range * (1.0 / 15.0)) & ~(one - 1);
    const double cut = __builtin_bit_cast(double, u);
    const double dd = fmax(15.0 * cut >= range ? cut : __builtin_bit_cast(double, u + one), 0x1p-14);
    const T d = (T)dd;  // exact: 7 bits, 2^-14 .. 4352
    T r = (T)__builtin_amdgcn_rcpf((float)dd);  // 1 / d to 23 bits, in 64 bits two Newton steps
    if constexpr (sizeof(T) == 8) {
        r = fma(fma(-d, r, 1.0), r, r);
        r = fma(fma(-d, r, 1.0), r, r);
    }
    const T z = rint_quotient(-lo, d, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = (uint32_t)(int)fmin(fmax(rint_quotient(y[i], d, r) + z, (T)0), (T)15);
    const vsl_half dh = (vsl_half)(float)dd;
    return (uint32_t)__builtin_bit_cast(uint16_t, dh) | (uint32_t)(int)z;
}

struct AppendArgs {
    const float* qkv;
    uint32_t S, n_q, n_kv, pos0, cap;
    RopeArgs r;
    void* q_out;
    void* kc;
    void* vc;
};

enum { Q_F32 = 0, Q_F16 = 1, Q_F16X2 = 2 };
enum { KV_F32 = 0, KV_F16 = 1, KV_4 = 2 };

template <int QM>
__device__ __forceinline__ void store_q(void* q_out, size_t off, size_t plane, const float (&y)[4]) {
    if constexpr (QM == Q_F32) {
        *reinterpret_cast<float4v*>(static_cast<float*>(q_out) + off) =
            float4v{y[0], y[1], y[2], y[3]};
    } else {
        vsl_half* q = static_cast<vsl_half*>(q_out);
        half4 h, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            vsl_half hi, lo;
            split_f16(y[i], hi, lo);
            h[i] = hi;
            l[i] = lo;
        }
        *reinterpret_cast<half4*>(q + off) = h;
        if constexpr (QM == Q_F16X2) *reinterpret_cast<half4*>(q + plane + off) = l;
    }
}
template <int KVM>
__device__ __forceinline__ void store_kv(void* cache, size_t off, const float (&y)[4]) {
    if constexpr (KVM == KV_F32)
        *reinterpret_cast<float4v*>(static_cast<float*>(cache) + off) = float4v{y[0], y[1], y[2], y[3]};
    else
        *reinterpret_cast<half4*>(static_cast<vsl_half*>(cache) + off) =
            half4{(vsl_half)y[0], (vsl_half)y[1], (vsl_half)y[2], (vsl_half)y[3]};
}
// A row of K in 4 bits, `at` its place among the cache's rows; two lanes a word (dims 0-3 and 4-7 of eight).
template <int HD>
__device__ __forceinline__ void store_k4(void* cache, uint64_t soff, size_t at, uint32_t c, const double (&y)[4]) {
    uint32_t n[4];
    const uint32_t step = kv4_quantize(y, n);
    const uint32_t own = (n[0] | n[1] << 16 | n[2] << 4 | n[3] << 20) << (c & 1 ? 8 : 0);
    const uint32_t w = own | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own, kDppPair, 0xF, 0xF, false);
    if ((c & 1) == 0) static_cast<uint32_t*>(cache)[at * (HD / 8) + c / 2] = w;
    if ((c & 7) == 0) reinterpret_cast<uint16_t*>(static_cast<char*>(cache) + soff)[at * (HD / 32) + c / 8] = (uint16_t)step;
}

// Prompt rows, four dims a lane, everything that a lane reads requested before its first use. The first v_waves waves
// take one 32-dim block of a V head at the 8 positions of an octet each (8 lanes a position; the first and the last octet
// of a call may be partly outside it): the codes of a column are joined to its word over the lanes. The others take
// rows of q and k heads (of all heads with fp16 and fp32 caches), HD / 4 lanes a head, neighbouring heads in
// neighbouring lanes. Bound by memory in a large call: 2048 rows of the 8B shape with a split q (50 MB read, 36 MB
// written) 22.5 us (median of a trace; the least 19.8), 3.8 TB/s against the 5.3 of a large copy; 45 rows 3.5 us. Two
// and four rows a lane: 23.5 and 25.6, 4.3 and 6.3 us; an octet of rows of one head a lane: 38.4 and 12.0 us.
template <int HD, int QM, int KVM>
__global__ __launch_bounds__(256) void k_append_rows(AppendArgs a, uint32_t v_waves) {
    constexpr uint32_t L = HD / 4, NB = HD / 32;
    const uint32_t heads = a.n_q + 2 * a.n_kv, width = heads * HD, lane = threadIdx.x & 63;
    const uint64_t P = kv4_positions(a.cap), soff = kv4_steps_off(a.n_kv, a.cap, HD);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (KVM == KV_4 && wave < v_waves) {
        const uint32_t blk = wave % NB, kvh = wave / NB % a.n_kv, oct = a.pos0 / 8 + wave / NB / a.n_kv;
        const uint32_t e = lane >> 3, j = lane & 7, s = oct * 8 + e - a.pos0;  // wraps below pos0
        const bool in = s < a.S;
        const float4v x = *reinterpret_cast<const float4v*>(a.qkv + (size_t)(in ? s : 0) * width +
                                                            (size_t)(a.n_q + a.n_kv + kvh) * HD + 32 * blk + 4 * j);
        const float y[4] = {x[0], x[1], x[2], x[3]};
        uint32_t n[4];
        const uint32_t step = kv4_quantize(y, n);
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t v = in ? n[i] << kv4_shift(e) : 0u;
            v |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false);  // lane ^ 8
            const auto p16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);
            v = p16[0] | p16[1];
            const auto p32 = __builtin_amdgcn_permlane32_swap(v, v, false, false);
            w[i] = p32[0] | p32[1];
        }
        const size_t at = (size_t)kvh * (P / 8) + oct;
        if (lane < 8) {
            uint32_t mask = 0;  // of the octet's positions in this call; the others keep their codes
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) mask |= oct * 8 + i - a.pos0 < a.S ? 15u << kv4_shift(i) : 0u;
            u32x4* dst = reinterpret_cast<u32x4*>(static_cast<uint32_t*>(a.vc) + at * HD + 32 * blk + 4 * j);
            if (~mask) w |= *dst & ~mask;
            *dst = w;
        }
        if (j == 0 && in)
            reinterpret_cast<uint16_t*>(static_cast<char*>(a.vc) + soff)[(at * NB + blk) * 8 + e] = (uint16_t)step;
        return;
    }
    const uint32_t row_heads = KVM == KV_4 ? a.n_q + a.n_kv : heads, c = lane % L;
    const uint32_t item = (KVM == KV_4 ? wave - v_waves : wave) * (64 / L);  // the wave's first row of a head
    uint32_t s = item / row_heads, h = item % row_heads + lane / L;
    while (h >= row_heads) {
        h -= row_heads;
        ++s;
    }
    if (s >= a.S) return;
    const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + a.n_kv;
    const float* gamma = is_q ? a.r.q_gamma : is_k ? a.r.k_gamma : nullptr;
    const uint32_t pos = a.pos0 + s;
    RowIn in;
    in.x = *reinterpret_cast<const float4v*>(a.qkv + (size_t)s * width + (size_t)h * HD + 4 * c);
    const Gains g = load_gains<HD>(a.r, gamma, c);
    if (is_q || is_k) load_angles<HD>(a.r, pos, c, in);
    const uint32_t kvh = is_k ? h - a.n_q : h - a.n_q - a.n_kv;
    if constexpr (KVM == KV_4) {
        if (is_k) {
            double y[4];
            norm_rotate<HD>(in, gamma != nullptr, g, a.r, c, y);
            store_k4<HD>(a.kc, soff, (size_t)kvh * P + pos, c, y);
            return;
        }
    }
    float y[4] = {in.x[0], in.x[1], in.x[2], in.x[3]};
    if (is_q || is_k) norm_rotate<HD>(in, gamma != nullptr, g, a.r, c, y);
    if (is_q) store_q<QM>(a.q_out, ((size_t)s * a.n_q + h) * HD + 4 * c, (size_t)a.S * a.n_q * HD, y);
    else if constexpr (KVM != KV_4) store_kv<KVM>(is_k ? a.kc : a.vc, ((size_t)kvh * a.cap + pos) * HD + 4 * c, y);
}

// One row at ctrl->pos, an item a head. The row, and for V the octet's words, are requested at once.
template <int HD, int KVM>
__global__ __launch_bounds__(64) void k_append_decode(AppendArgs a, vsl_ctrl* ctrl) {
    constexpr uint32_t L = HD / 4, NB = HD / 32;
    const uint32_t heads = a.n_q + 2 * a.n_kv;
    const uint32_t t = blockIdx.x * 64 + threadIdx.x, h = t / L, c = t % L;
    const bool in = h < heads;
    const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + a.n_kv;
    const float* gamma = is_q ? a.r.q_gamma : is_k ? a.r.k_gamma : nullptr;
    const float4v x = *reinterpret_cast<const float4v*>(a.qkv + (in ? (size_t)h * HD + 4 * c : 0));
    const Gains g = load_gains<HD>(a.r, gamma, c);
    const uint32_t done = ctrl->done, pos = ctrl->pos;
    if (done) return;
    if (pos >= a.cap) {
        if (t == 0) {
            ctrl->error = 1u;
            ctrl->done = 1u;
        }
        return;
    }
    if (!in) return;
    const uint32_t kvh = is_q ? 0 : is_k ? h - a.n_q : h - a.n_q - a.n_kv;
    const uint64_t P = kv4_positions(a.cap), soff = kv4_steps_off(a.n_kv, a.cap, HD);
    RowIn in_row;
    in_row.x = x;
    if (is_q || is_k) load_angles<HD>(a.r, pos, c, in_row);
    if constexpr (KVM == KV_4) {
        if (is_k) {
            double y[4];
            norm_rotate<HD>(in_row, gamma != nullptr, g, a.r, c, y);
            store_k4<HD>(a.kc, soff, (size_t)kvh * P + pos, c, y);
            return;
        }
    }
    float y[4] = {x[0], x[1], x[2], x[3]};
    if (is_q || is_k) norm_rotate<HD>(in_row, gamma != nullptr, g, a.r, c, y);
    if (is_q) {
        store_q<Q_F32>(a.q_out, (size_t)h * HD + 4 * c, 0, y);
    } else if constexpr (KVM != KV_4) {
        store_kv<KVM>(is_k ? a.kc : a.vc, ((size_t)kvh * a.cap + pos) * HD + 4 * c, y);
    } else {
        const size_t oct = (size_t)kvh * (P / 8) + pos / 8;
        u32x4* dst = reinterpret_cast<u32x4*>(static_cast<uint32_t*>(a.vc) + oct * HD + 4 * c);
        const u32x4 old = *dst;
        const uint32_t sh = kv4_shift(pos & 7);
        uint32_t n[4];
        const uint32_t step = kv4_quantize(y, n);
        *dst = (old & ~(15u << sh)) | (u32x4{n[0], n[1], n[2], n[3]} << sh);
        if ((c & 7) == 0)
            reinterpret_cast<uint16_t*>(static_cast<char*>(a.vc) + soff)[(oct * NB + c / 8) * 8 + (pos & 7)] = (uint16_t)step;
    }
}

// ---------------------------------------------------------------------------------------------
// the cache as values
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void store8(vsl_half* p, half8 v) { *reinterpret_cast<half8*>(p) = v; }
__device__ __forceinline__ void store8(float* p, half8 v) {
    *reinterpret_cast<float4v*>(p) = float4v{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    *reinterpret_cast<float4v*>(p + 4) = float4v{(float)v[4], (float)v[5], (float)v[6], (float)v[7]};
}

// K: a thread for a word (8 dims of a position). V: a thread for 8 words (8 columns of an octet), turned in registers.
template <int HD, typename T>
__global__ __launch_bounds__(256) void k_kv4_read(const char* __restrict__ kc, const char* __restrict__ vc, uint32_t n_kv,
                                                  uint32_t cap, uint32_t pos0, uint32_t n, T* __restrict__ ko,
                                                  T* __restrict__ vo) {
    constexpr uint32_t WPR = HD / 8, NB = HD / 32;
    const uint64_t P = kv4_positions(cap), soff = kv4_steps_off(n_kv, cap, HD);
    const uint32_t o0 = pos0 / 8, n_oct = (pos0 + n - 1) / 8 - o0 + 1;
    const uint64_t nk = kc ? (uint64_t)n_kv * n * WPR : 0, nv = vc ? (uint64_t)n_kv * n_oct * WPR : 0;
    uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const Kv4Consts kc4 = kv4_consts();
    if (t < nk) {
        const uint32_t w = (uint32_t)(t % WPR);
        const uint64_t r = t / WPR, kvh = r / n, i = r % n, at = kvh * P + pos0 + i;
        const uint32_t word = reinterpret_cast<const uint32_t*>(kc)[at * WPR + w];
        const uint32_t s = reinterpret_cast<const uint16_t*>(kc + soff)[at * NB + w / 4];
        store8(ko + (kvh * n + i) * HD + 8 * w, kv4_word(word, kv4_step(s | s << 16, kc4), kc4));
        return;
    }
    t -= nk;
    if (t >= nv) return;
    const uint32_t w = (uint32_t)(t % WPR);
    const uint64_t r = t / WPR, kvh = r / n_oct, oct = o0 + r % n_oct, at = kvh * (P / 8) + oct;
    const u32x4* wp = reinterpret_cast<const u32x4*>(reinterpret_cast<const uint32_t*>(vc) + at * HD + 8 * w);
    const u32x4 wa = wp[0], wb = wp[1];
    const u32x4 sp = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(vc + soff) + (at * NB + w / 4) * 8);
    Kv4Step st[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) st[p] = kv4_step(sp[p], kc4);
    half8 col[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) col[j] = kv4_word(j < 4 ? wa[j & 3] : wb[j & 3], st, kc4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint64_t i = oct * 8 + e - pos0;
        if (i < n)
            store8(vo + (kvh * n + i) * HD + 8 * w,
                   half8{col[0][e], col[1][e], col[2][e], col[3][e], col[4][e], col[5][e], col[6][e], col[7][e]});
    }
}

// ---------------------------------------------------------------------------------------------
// decode attention
// ---------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
// Waves of a decode attention block, and tiles in flight a wave. With 8 waves, or 3 or 4 tiles, the 8B shape at 32 splits
// took 6.1, 5.6 or 5.9 us over 778 positions instead of 4.9, and 11.4, 13.4 or 14.0 us over 32001 instead of 11.9.
constexpr int kDecWaves = 4, kDecTiles = 2;

// LDS traffic alone (global loads stay in flight).
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// v of lane i ^ 8 of the 16-lane row, added
__device__ __forceinline__ float add_lane8(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
}

// Block (split s, KV head h) of WAVES waves; wave w of it owns the tiles of 32 positions (j nsplit + s) WAVES + w. Both
// products run on the matrix cores (v_mfma_f32_16x16x32_f16) over the expanded binary16 values, with no operand
// moved between lanes:
//  - S^T = K Q^T: the B columns 0-7 hold the group's query heads as the hi plane of q * scale * log2(e), the columns
//    8-15 the lo plane of the same heads, so that the sum of the two columns is the product of the fp32 q. Row r of
//    the tile's half t is position 8 (r / 4) + 4 t + r % 4, dims in the order of the cache's words;
//  - so lane l ends with the scores of head l % 8 (in both columns after one lane rotation by 8) at the 8 positions of
//    octet l / 16, which is the B operand P^T of O^T += V^T P^T when V's words are octets of positions: the lanes of
//    the columns 0-7 pass the probabilities' hi plane, the others the lo plane;
//  - lane l expands the V columns HD/16 (l % 16) .. + HD/16 - 1 of octet l / 16, whose steps are one 16-byte load.
// Softmax against a reference per head (kKv4Room), raised for the whole wave. Masked positions get probability 0 and
// their V steps are set to 0, so what the cache holds past the length never reaches a sum. Output as k_attn_decode's.
// Bound by latency at short lengths (8B shape, 32 splits, 778 positions 4.9 us: loads 1.0, one tile's chain 1.1, the waves'
// join and the partials 0.9, the launch), and by the expansion's vector instructions at long ones: 32001 positions 11.9 us,
// of which the loads alone, by the same pattern, take 8.6 (37 MB, 4.3 TB/s), against 22.4 for the fp16 cache's kernel
// (11.6 to 13 in a trace, where a launch starts on an idle card).
template <int HD, int G, bool WIN, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void k_attn_decode_kv4(const float* __restrict__ q, const char* __restrict__ kcache,
                                                                const char* __restrict__ vcache, uint32_t n_kv, uint32_t cap,
                                                                float scale, uint32_t nsplit, float* __restrict__ part_o,
                                                                float* __restrict__ part_ml, vsl_ctrl* ctrl, uint32_t win,
                                                                uint32_t n_glob, uint32_t thr) {
    constexpr int KS = HD / 32, NB = HD / 32, NC = HD / 16;  // k-steps; blocks a row; V columns a lane (and O^T tiles)
    constexpr uint32_t TP = 32;
    constexpr int NBUF = kDecTiles;
    static_assert(G >= 1 && G <= 8, "GQA group of 1..8 heads");
    __shared__ __attribute__((aligned(8))) float s_ml[WAVES][G][2];
    __shared__ __attribute__((aligned(16))) float s_acc[WAVES][G][HD];

    const uint32_t kvh = blockIdx.y, split = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15, rg = lane >> 4, head = col & 7;
    const uint32_t h0 = kvh * G;
    const Kv4Consts kc4 = kv4_consts();
    const uint64_t P = kv4_positions(cap), soff = kv4_steps_off(n_kv, cap, HD);
    const uint32_t all_tiles = (uint32_t)(P / TP);
    // this lane's part of tile 0
    const uint32_t krow = 8 * (col >> 2) + (col & 3);
    const char* Kc = kcache + ((uint64_t)kvh * P + krow) * (HD / 2) + rg * (HD / 8);
    const char* Ks = kcache + soff + (((uint64_t)kvh * P + krow) * NB + rg * NB / 4) * 2;
    const char* Vc = vcache + (((uint64_t)kvh * (P / 8) + rg) * HD + col * NC) * 4;
    const char* Vs = vcache + soff + ((((uint64_t)kvh * (P / 8) + rg) * NB + col * NC / 32) * 8) * 2;

    struct Tile {
        uint32_t k[2][KS], ks[2], v[NC];
        u32x4 vs;
    };
    auto issue = [&](Tile& b, uint32_t tile) {
        const uint64_t p0 = (uint64_t)tile * TP;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const char* kp = Kc + (p0 + 4 * t) * (HD / 2);
            if constexpr (KS == 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(kp);
#pragma unroll
                for (int i = 0; i < 4; ++i) b.k[t][i] = w[i];
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(kp);
                b.k[t][0] = w.x;
                b.k[t][1] = w.y;
            }
            b.ks[t] = *reinterpret_cast<const uint16_t*>(Ks + (p0 + 4 * t) * NB * 2);
        }
        const char* vp = Vc + p0 / 8 * HD * 4;
#pragma unroll
        for (int i = 0; i < NC; i += 4) {
            const u32x4 w = *reinterpret_cast<const u32x4*>(vp + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) b.v[i + j] = w[j];
        }
        b.vs = *reinterpret_cast<const u32x4*>(Vs + p0 / 8 * NB * 16);
    };
    auto vtile = [&](uint32_t j) { return (j * nsplit + split) * WAVES + wave; };

    // q (B operand: lane l holds head l % 8, dims HD/4 (l / 16) + 8 ks ..) and the first two tiles are requested before
    // the control block is read: without a window a tile's place does not depend on the length
    float4 qa[KS][2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const float* qp = q + (size_t)(h0 + (head < (uint32_t)G ? head : 0)) * HD + HD / 4 * rg + 8 * ks;
        qa[ks][0] = *reinterpret_cast<const float4*>(qp);
        qa[ks][1] = *reinterpret_cast<const float4*>(qp + 4);
    }
    Tile buf[NBUF];
    if constexpr (!WIN) {
#pragma unroll
        for (int i = 0; i < NBUF; ++i) issue(buf[i], vtile(i) < all_tiles ? vtile(i) : 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t done = ctrl->done;
    const uint32_t pos = ctrl->pos;
    const uint32_t p = pos < cap ? pos : cap - 1;  // pos >= cap only with done set
    // virtual tiles: with a window those of the n_glob first positions, then those from the window's start
    const uint32_t n_tiles = p / TP + 1;
    uint32_t n_gt = n_tiles, t_lo = n_tiles, lo = 0;
    if constexpr (WIN) {
        if (p + 1 > thr && p > win) {
            lo = p - win;
            t_lo = lo / TP;
            n_gt = min((n_glob + TP - 1) / TP, t_lo);
        }
    }
    const uint32_t n_vt = n_gt + (n_tiles - t_lo);
    auto phys = [&](uint32_t vt) {  // tiles past the last read tile 0
        if (vt >= n_vt) return 0u;
        return vt < n_gt ? vt : vt - n_gt + t_lo;
    };
    if constexpr (WIN) {
#pragma unroll
        for (int i = 0; i < NBUF; ++i) issue(buf[i], phys(vtile(i)));
    }

    half8 qf[KS];
    const float f = scale * kLog2e;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const float x[8] = {qa[ks][0].x, qa[ks][0].y, qa[ks][0].z, qa[ks][0].w,
                            qa[ks][1].x, qa[ks][1].y, qa[ks][1].z, qa[ks][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            vsl_half hi, lo16;
            split_f16(x[e] * f, hi, lo16);
            qf[ks][e] = head < (uint32_t)G ? (col < 8 ? hi : lo16) : (vsl_half)0.f;
        }
    }
    float m = -INFINITY, l = 0.f, minus_plane = col < 8 ? 0.f : -1.f;
    float4v o[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = float4v{0.f, 0.f, 0.f, 0.f};

    auto consume = [&](const Tile& b, uint32_t vt) {
        const uint32_t p0 = phys(vt) * TP;
        float s[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Kv4Step st = kv4_step(b.ks[t] | b.ks[t] << 16, kc4);
            float4v d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_word(b.k[t][ks], st, kc4), qf[ks], d, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * t + i] = add_lane8(d[i]);
        }
        u32x4 vs = b.vs;
        // wave-uniform: a tile that ends past the position or begins before the window
        const bool whole = p0 + TP - 1 <= p && (!WIN || p0 >= lo || p0 + TP <= n_glob);
        if (!whole) {
            asm volatile("");  // a branch, not selects in every tile
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t k = p0 + 8 * rg + e;
                const bool seen = k <= p && (!WIN || k >= lo || k < n_glob);
                s[e] = seen ? s[e] : -INFINITY;
                if (!seen) vs[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
            }
        }
        float bm = s[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) bm = fmaxf(bm, s[e]);
        if (__builtin_amdgcn_ballot_w64(bm - m > kKv4Lazy + kKv4Room)) {  // m = -inf: any finite score raises it
            float a0, a1;
            lane_pair<16>(bm, a0, a1);
            lane_pair<32>(fmaxf(a0, a1), a0, a1);
            const float mn = fmaxf(m, fmaxf(a0, a1) - kKv4Room);
            const float corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);  // m = -inf: 0
            l *= corr;
#pragma unroll
            for (int i = 0; i < NC; ++i) o[i] *= corr;
            m = mn;
        }
        // columns 0-7 take the hi plane, 8-15 what it leaves: fp16(p - plane * fp16(p)), plane 0 or 1
        half8 pf;
        const float ref = m == -INFINITY ? 0.f : m;  // no score seen yet: every s is -inf (or NaN)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p0 = fast_exp2(s[e] - ref), p1 = fast_exp2(s[e + 1] - ref);
            l += p0;
            l += p1;
            const half2v hi = pack_f16(p0, p1);
            const half2v w = pack_f16(fmaf((float)hi[0], minus_plane, p0), fmaf((float)hi[1], minus_plane, p1));
            pf[e] = w[0];
            pf[e + 1] = w[1];
        }
        Kv4Step st[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) st[i] = kv4_step(vs[i], kc4);
#pragma unroll
        for (int i = 0; i < NC; ++i) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_word(b.v[i], st, kc4), pf, o[i], 0, 0, 0);
    };

    // each buffer is refilled right after it is consumed (past the wave's last tile with the one just consumed)
    const uint32_t stride = nsplit * WAVES;
    uint32_t vt = vtile(0);
    bool more = vt < n_vt;
    while (more) {
#pragma unroll
        for (int i = 0; i < NBUF; ++i) {
            consume(buf[i], vt);
            const uint32_t ahead = vt + NBUF * stride;
            more = vt + stride < n_vt;
            if (!more) break;
            issue(buf[i], phys(ahead < n_vt ? ahead : vt));
            __builtin_amdgcn_sched_barrier(0);
            vt += stride;
        }
    }

    // the head's sums over the octets, the hi and lo columns joined; lane l holds head l % 8, dims
    // NC (4 (l / 16) + r) + i in o[i][r]
    float l0, l1;
    lane_pair<16>(l, l0, l1);
    lane_pair<32>(l0 + l1, l0, l1);
    l = l0 + l1;
    if (m == -INFINITY && l != 0.f) m = 0.f;  // only NaN scores: keep the sum in the merge
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] = add_lane8(o[i][r]);
    if (col < (uint32_t)G) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < NC; i += 4)
                *reinterpret_cast<float4v*>(&s_acc[wave][col][NC * (4 * rg + r) + i]) =
                    float4v{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
        if (rg == 0) {
            s_ml[wave][col][0] = m;
            s_ml[wave][col][1] = l;
        }
    }
    lds_barrier();
    // four dims a thread; the waves' statistics and sums are read at once
    static_assert(G * HD / 4 <= WAVES * 64, "one pass over the outputs");
    const uint32_t g = threadIdx.x / (HD / 4), dd = threadIdx.x % (HD / 4) * 4;
    if (g >= (uint32_t)G) return;
    float2 ml[WAVES];
    float4v acc[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        ml[w] = *reinterpret_cast<const float2*>(&s_ml[w][g][0]);
        acc[w] = *reinterpret_cast<const float4v*>(&s_acc[w][g][dd]);
    }
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, ml[w].x);
    float L = 0.f;
    float4v A = {0.f, 0.f, 0.f, 0.f};
    const float ref = M == -INFINITY ? 0.f : M;  // no tile at all: every weight and sum is 0
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float fw = fast_exp2(ml[w].x - ref);
        L = fmaf(ml[w].y, fw, L);
#pragma unroll
        for (int i = 0; i < 4; ++i) A[i] = fmaf(acc[w][i], fw, A[i]);
    }
    if (done) return;
    const size_t pidx = (size_t)(h0 + g) * nsplit + split;
    *reinterpret_cast<float4v*>(part_o + pidx * HD + dd) = A;
    if (dd == 0) *reinterpret_cast<float2*>(part_ml + pidx * 2) = make_float2(M, L);
}

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int check_kv4(const char* fn, const void* kcache, const void* vcache, uint32_t hd) {
    if (hd != 64 && hd != 128) return vsl_unsupported("%s: head_dim %u (64 or 128)", fn, hd);
    if (!aligned_to(kcache, 256) || !aligned_to(vcache, 256))
        return vsl_invalid("%s: a 4-bit cache must be 256-byte aligned", fn);
    return VSL_OK;
}

// Arguments that both append entries share; VSL_OK or the error code (nothing launched on error).
int check_append(const char* fn, const float* qkv, uint32_t n_q, uint32_t n_kv, uint32_t hd, const float* q_gamma,
                 const float* k_gamma, int rope, const float* rc, const float* rs, const void* q_out, const void* kcache,
                 const void* vcache, int kv_dtype, uint32_t cap) {
    if (!qkv || !rc || !rs || !q_out || !kcache || !vcache) return vsl_invalid("%s: null pointer", fn);
    if (hd != 64 && hd != 128) return vsl_unsupported("%s: head_dim %u (64 or 128)", fn, hd);
    if (n_q == 0 || n_kv == 0 || ((uint64_t)n_q + 2ull * n_kv) * hd > 0x7FFFFFFFull)
        return vsl_invalid("%s: n_q=%u n_kv=%u", fn, n_q, n_kv);
    if (rope != VSL_ROPE_PAIRS && rope != VSL_ROPE_HALVES) return vsl_invalid("%s: rotation %d", fn, rope);
    if (kv_dtype != VSL_DT_F16 && kv_dtype != VSL_DT_F32 && kv_dtype != VSL_DT_KV4)
        return vsl_unsupported("%s: kv dtype %d", fn, kv_dtype);
    if (cap == 0) return vsl_invalid("%s: capacity 0", fn);
    for (const void* p : {static_cast<const void*>(qkv), static_cast<const void*>(q_gamma), static_cast<const void*>(k_gamma),
                          static_cast<const void*>(rc), static_cast<const void*>(rs), q_out, kcache, vcache})
        if (!aligned_to(p, 16)) return vsl_invalid("%s: pointers must be 16-byte aligned", fn);
    if (kv_dtype == VSL_DT_KV4) return check_kv4(fn, kcache, vcache, hd);
    return VSL_OK;
}

template <int HD, int QM>
void launch_rows(hipStream_t s, const AppendArgs& a, int kv_dtype) {
    const bool kv4 = kv_dtype == VSL_DT_KV4;
    const uint64_t octets = ((uint64_t)a.pos0 + a.S - 1) / 8 - a.pos0 / 8 + 1;
    const uint64_t v_waves = kv4 ? octets * a.n_kv * (HD / 32) : 0;
    const uint64_t items = (uint64_t)a.S * (a.n_q + (kv4 ? 1 : 2) * (uint64_t)a.n_kv);
    const uint32_t grid = (uint32_t)((v_waves + (items + 256 / HD - 1) / (256 / HD) + 3) / 4);
    if (kv4) k_append_rows<HD, QM, KV_4><<<grid, 256, 0, s>>>(a, (uint32_t)v_waves);
    else if (kv_dtype == VSL_DT_F16) k_append_rows<HD, QM, KV_F16><<<grid, 256, 0, s>>>(a, 0);
    else k_append_rows<HD, QM, KV_F32><<<grid, 256, 0, s>>>(a, 0);
}
template <int HD>
void launch_decode(uint32_t grid, hipStream_t s, const AppendArgs& a, int kv_dtype, vsl_ctrl* ctrl) {
    if (kv_dtype == VSL_DT_KV4) k_append_decode<HD, KV_4><<<grid, 64, 0, s>>>(a, ctrl);
    else if (kv_dtype == VSL_DT_F16) k_append_decode<HD, KV_F16><<<grid, 64, 0, s>>>(a, ctrl);
    else k_append_decode<HD, KV_F32><<<grid, 64, 0, s>>>(a, ctrl);
}

}  // namespace

extern "C" uint64_t vsl_kv_cache_bytes(int kv_dtype, uint32_t n_kv, uint32_t cap, uint32_t hd) {
    if (kv_dtype == VSL_DT_F16) return 2ull * n_kv * cap * hd;
    if (kv_dtype == VSL_DT_F32) return 4ull * n_kv * cap * hd;
    if (kv_dtype == VSL_DT_KV4 && (hd == 64 || hd == 128)) return kv4_bytes(n_kv, cap, hd);
    return 0;
}

extern "C" int vsl_qk_norm_rope_append(const float* qkv, uint32_t S, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t pos0,
                                       const float* q_gamma, const float* k_gamma, float eps, int rope, const float* rope_cos,
                                       const float* rope_sin, void* q_out, int q_dtype, void* kcache, void* vcache,
                                       int kv_dtype, uint32_t cap, void* stream) {
    const char* fn = "vsl_qk_norm_rope_append";
    if (const int rc = check_append(fn, qkv, n_q, n_kv, hd, q_gamma, k_gamma, rope, rope_cos, rope_sin, q_out, kcache, vcache,
                                    kv_dtype, cap))
        return rc;
    if (q_dtype != VSL_DT_F32 && q_dtype != VSL_DT_F16 && q_dtype != VSL_DT_F16X2)
        return vsl_unsupported("%s: q dtype %d", fn, q_dtype);
    if ((uint64_t)pos0 + S > cap)
        return vsl_capacity("%s: %u positions from %u exceed capacity %u", fn, S, pos0, cap);
    if (S == 0) return VSL_OK;
    const AppendArgs a{qkv, S, n_q, n_kv, pos0, cap, RopeArgs{q_gamma, k_gamma, rope_cos, rope_sin, eps, rope},
                       q_out, kcache, vcache};
    if ((uint64_t)S * (n_q + 2 * n_kv) * hd > 1ull << 33) return vsl_unsupported("%s: %u rows in one call", fn, S);  // 2^31 lanes
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto hdc) {
        constexpr int HD = decltype(hdc)::value;
        if (q_dtype == VSL_DT_F32) launch_rows<HD, Q_F32>(s, a, kv_dtype);
        else if (q_dtype == VSL_DT_F16) launch_rows<HD, Q_F16>(s, a, kv_dtype);
        else launch_rows<HD, Q_F16X2>(s, a, kv_dtype);
    };
    if (hd == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 64>{});
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}

extern "C" int vsl_qk_norm_rope_append_decode(const float* qkv, uint32_t n_q, uint32_t n_kv, uint32_t hd,
                                              const float* q_gamma, const float* k_gamma, float eps, int rope,
                                              const float* rope_cos, const float* rope_sin, float* q_out, void* kcache,
                                              void* vcache, int kv_dtype, uint32_t cap, vsl_ctrl* ctrl, void* stream) {
    const char* fn = "vsl_qk_norm_rope_append_decode";
    if (const int rc = check_append(fn, qkv, n_q, n_kv, hd, q_gamma, k_gamma, rope, rope_cos, rope_sin, q_out, kcache, vcache,
                                    kv_dtype, cap))
        return rc;
    if (!ctrl) return vsl_invalid("%s: null pointer", fn);
    const AppendArgs a{qkv, 1, n_q, n_kv, 0, cap, RopeArgs{q_gamma, k_gamma, rope_cos, rope_sin, eps, rope},
                       q_out, kcache, vcache};
    const uint32_t grid = (uint32_t)(((uint64_t)(n_q + 2 * n_kv) * (hd / 4) + 63) / 64);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (hd == 128) launch_decode<128>(grid, s, a, kv_dtype, ctrl);
    else launch_decode<64>(grid, s, a, kv_dtype, ctrl);
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}

extern "C" int vsl_kv4_read(const void* kcache, const void* vcache, uint32_t n_kv, uint32_t cap, uint32_t hd, uint32_t pos0,
                            uint32_t n, void* k_out, void* v_out, int out_dtype, void* stream) {
    const char* fn = "vsl_kv4_read";
    if (!kcache != !k_out || !vcache != !v_out || (!kcache && !vcache)) return vsl_invalid("%s: null pointer", fn);
    if (n_kv == 0) return vsl_invalid("%s: n_kv=0", fn);
    if (const int rc = check_kv4(fn, kcache, vcache, hd)) return rc;
    if (out_dtype != VSL_DT_F16 && out_dtype != VSL_DT_F32) return vsl_unsupported("%s: dtype %d", fn, out_dtype);
    if (!aligned_to(k_out, 16) || !aligned_to(v_out, 16)) return vsl_invalid("%s: outputs must be 16-byte aligned", fn);
    if ((uint64_t)pos0 + n > cap) return vsl_capacity("%s: %u positions from %u exceed capacity %u", fn, n, pos0, cap);
    if (n == 0) return VSL_OK;
    const uint64_t n_oct = (pos0 + n - 1) / 8 - pos0 / 8 + 1;
    const uint64_t items = (uint64_t)n_kv * (hd / 8) * ((kcache ? n : 0) + (vcache ? n_oct : 0));
    if (items > 1ull << 31) return vsl_unsupported("%s: %u positions in one call", fn, n);
    const uint32_t blocks = (uint32_t)((items + 255) / 256);
    const char* kc = static_cast<const char*>(kcache);
    const char* vc = static_cast<const char*>(vcache);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto kernel, auto* ko, auto* vo) {
        kernel<<<blocks, 256, 0, s>>>(kc, vc, n_kv, cap, pos0, n, ko, vo);
    };
    if (out_dtype == VSL_DT_F16) {
        vsl_half *ko = static_cast<vsl_half*>(k_out), *vo = static_cast<vsl_half*>(v_out);
        if (hd == 128) go(k_kv4_read<128, vsl_half>, ko, vo);
        else go(k_kv4_read<64, vsl_half>, ko, vo);
    } else {
        float *ko = static_cast<float*>(k_out), *vo = static_cast<float*>(v_out);
        if (hd == 128) go(k_kv4_read<128, float>, ko, vo);
        else go(k_kv4_read<64, float>, ko, vo);
    }
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}

int vsl_kv4_attn_partials(const float* q, const void* kcache, const void* vcache, uint32_t n_q, uint32_t n_kv, uint32_t hd,
                          uint32_t cap, float scale, uint32_t nsplit, float* part_o, float* part_ml, vsl_ctrl* ctrl, bool window,
                          uint32_t win, uint32_t n_glob, uint32_t thr, void* stream) {
    if (const int rc = check_kv4("vsl_attn_decode", kcache, vcache, hd)) return rc;
    if (cap == 0) return vsl_invalid("vsl_attn_decode: capacity 0");
    if (!aligned_to(q, 16) || !aligned_to(part_o, 16) || !aligned_to(part_ml, 8))
        return vsl_invalid("vsl_attn_decode: a 4-bit cache needs q and part_o 16-byte, part_ml 8-byte aligned");
    const dim3 grid(nsplit, n_kv);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const char* kc = static_cast<const char*>(kcache);
    const char* vc = static_cast<const char*>(vcache);
    auto go = [&](auto hdc, auto gc) {
        constexpr int HD = decltype(hdc)::value, G = decltype(gc)::value;
        if (window)
            k_attn_decode_kv4<HD, G, true, kDecWaves><<<grid, kDecWaves * 64, 0, s>>>(q, kc, vc, n_kv, cap, scale, nsplit, part_o,
                                                                                      part_ml, ctrl, win, n_glob, thr);
        else
            k_attn_decode_kv4<HD, G, false, kDecWaves><<<grid, kDecWaves * 64, 0, s>>>(q, kc, vc, n_kv, cap, scale, nsplit, part_o,
                                                                                       part_ml, ctrl, 0, 0, 0);
    };
    auto by_group = [&](auto hdc) {
        switch (n_q / n_kv) {
            case 1: go(hdc, std::integral_constant<int, 1>{}); break;
            case 2: go(hdc, std::integral_constant<int, 2>{}); break;
            case 3: go(hdc, std::integral_constant<int, 3>{}); break;
            case 4: go(hdc, std::integral_constant<int, 4>{}); break;
            case 5: go(hdc, std::integral_constant<int, 5>{}); break;
            case 6: go(hdc, std::integral_constant<int, 6>{}); break;
            case 7: go(hdc, std::integral_constant<int, 7>{}); break;
            case 8: go(hdc, std::integral_constant<int, 8>{}); break;
            default: return vsl_unsupported("vsl_attn_decode: GQA ratio %u (supported 1..8)", n_q / n_kv);
        }
        return (int)VSL_OK;
    };
    const int rc = hd == 128 ? by_group(std::integral_constant<int, 128>{}) : by_group(std::integral_constant<int, 64>{});
    if (rc) return rc;
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}
