// vsl_rope.hip -- rotary tables with scaled frequencies, and rotation of part of each head with the cache append
// (vsl_rope_tables, vsl_rope_part_append, vsl_rope_part_append_decode). The reference rotates whole heads by unscaled
// angles that it computes in the shader (fused_matmul_rope.comp:48-81).
#include <cmath>

#include "vsl_device.h"
#include "vsl_internal.h"

namespace {

// ---------------------------------------------------------------------------------------------
// tables
// ---------------------------------------------------------------------------------------------
// Frequencies: theta^(-2j/rot) / ff_j, then a mix of f and f / factor (a of f, 1 - a of f / factor):
//   by pair index (yarn)    1 - a = (j - lo) / (hi - lo) within 0..1
//   by turns (llama3)       a = (turns - lo) / (hi - lo) within 0..1, turns = orig f / (2 pi)
struct FreqArgs {
    double log2_theta, inv_factor, turns;  // turns: orig / (2 pi)
    double lo, inv_span, mscale;
    int by_pair, by_turns;
};

// A thread takes a pair at kRun positions: the angles of the first and of one step in 64 bits, the others by rotation
// (each adds under 2^-52; 16 of them stay 2^24 below the results' rounding). Bound by the
// stores: 131072 positions of 32 pairs 8.1 us (4.1 TB/s); of fewer values a thread's two sincos show: 32768 positions of 64 pairs
// 6.0 us (2.8 TB/s). Runs of 8 / 32 / 64 positions 8.9 / 8.2 / 9.6 and 6.3 / 6.5 / 7.8, of 4 11.8 and 7.7.
constexpr uint32_t kRun = 16;
__global__ __launch_bounds__(256) void k_rope_tables(uint32_t half, uint32_t pos0, uint32_t rows, FreqArgs a, double rot,
                                                     const float* __restrict__ ff, float* __restrict__ cos_out,
                                                     float* __restrict__ sin_out) {
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t j = (uint32_t)(at % half);
    const uint64_t r0 = at / half * kRun;
    if (r0 >= rows) return;
    double f = exp2(-2.0 * (double)j / rot * a.log2_theta);
    if (ff) f /= (double)ff[j];
    if (a.by_pair) {
        const double mix = fmin(fmax(((double)j - a.lo) * a.inv_span, 0.0), 1.0);
        f = f * a.inv_factor * mix + f * (1.0 - mix);
    } else if (a.by_turns) {
        const double mix = fmin(fmax((f * a.turns - a.lo) * a.inv_span, 0.0), 1.0);
        f = f * a.inv_factor * (1.0 - mix) + f * mix;
    } else {
        f *= a.inv_factor;
    }
    double c, s, dc, ds;
    sincos((double)(pos0 + r0) * f, &s, &c);
    sincos(f, &ds, &dc);
    c *= a.mscale;
    s *= a.mscale;
    const uint32_t n = (uint32_t)min((uint64_t)kRun, rows - r0);
    float* co = cos_out + r0 * half + j;
    float* so = sin_out + r0 * half + j;
    for (uint32_t i = 0; i < n; ++i) {
        co[(size_t)i * half] = (float)c;
        so[(size_t)i * half] = (float)s;
        const double nc = c * dc - s * ds;
        s = s * dc + c * ds;
        c = nc;
    }
}

// ---------------------------------------------------------------------------------------------
// rotation of the first rot dims of each head, append
// ---------------------------------------------------------------------------------------------
enum { Q_F32 = 0, Q_F16 = 1, Q_F16X2 = 2 };

struct PartArgs {
    const float* qkv;
    uint32_t S, n_q, n_kv, hd, rot, pos0, cap, table_rows;
    int halves;
    const uint32_t* positions;
    const float* rc;
    const float* rs;
    void* q_out;
    void* kc;
    void* vc;
};

// Four dims a lane; bpr blocks a row. A rotated dim's partner is read again from the row (it is in the same lines).
// VEC: rot % 8 == 0, so that four dims are rotated or not as one and the partners and angles of a halves' rotation are
// aligned vectors; otherwise dim by dim (36 dims instead of 32: by halves 30.3 us instead of 19.2, by pairs 19.7). Bound by the projection read and the outputs written: 2048 rows of the 8B shape, 32
// dims of each head, split q: 92 MB in 16.4 us (5.6 TB/s; 19.2 with the launch; fp32 caches 21.8); a token 4.0.
template <bool VEC, int QM, typename KT, bool DEC>
__global__ __launch_bounds__(256) void k_rope_part(PartArgs a, uint32_t bpr, vsl_ctrl* ctrl) {
    const uint32_t s = blockIdx.x / bpr;
    const uint32_t c4 = (blockIdx.x - s * bpr) * 256 + threadIdx.x, per_head = a.hd / 4;
    const uint32_t h = c4 / per_head, d0 = (c4 - h * per_head) * 4;
    const uint32_t heads = a.n_q + 2 * a.n_kv;
    uint32_t pos = a.pos0 + s;
    if constexpr (DEC) {
        if (ctrl->done) return;
        pos = ctrl->pos;
        if (pos >= a.cap) {
            if (c4 == 0) {
                ctrl->error = 1u;
                ctrl->done = 1u;
            }
            return;
        }
    }
    if (h >= heads) return;
    const float* x = a.qkv + ((size_t)s * heads + h) * a.hd;
    float y[4];
    {
        const float4v v = *reinterpret_cast<const float4v*>(x + d0);
        y[0] = v[0]; y[1] = v[1]; y[2] = v[2]; y[3] = v[3];
    }
    if (h < a.n_q + a.n_kv && d0 < a.rot) {
        const uint32_t half = a.rot / 2, rpos = a.positions ? a.positions[s] : pos;
        const bool known = rpos < a.table_rows;  // a position that the tables lack gives NaN
        const float* rc = a.rc + (size_t)(known ? rpos : 0) * half;
        const float* rs = a.rs + (size_t)(known ? rpos : 0) * half;
        if (!a.halves) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t j = d0 / 2 + p;
                if (!VEC && j >= half) break;
                const float c = known ? rc[j] : NAN, sn = known ? rs[j] : NAN, u = y[2 * p], w = y[2 * p + 1];
                y[2 * p] = u * c - w * sn;
                y[2 * p + 1] = u * sn + w * c;
            }
        } else if constexpr (VEC) {
            const bool low = d0 < half;
            const uint32_t j = low ? d0 : d0 - half;
            const float4v o = *reinterpret_cast<const float4v*>(x + (low ? d0 + half : j));
            const float4v c = *reinterpret_cast<const float4v*>(rc + j), sn = *reinterpret_cast<const float4v*>(rs + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float r = low ? y[i] * c[i] - o[i] * sn[i] : o[i] * sn[i] + y[i] * c[i];
                y[i] = known ? r : NAN;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t d = d0 + i;
                if (d >= a.rot) break;
                const bool low = d < half;
                const uint32_t j = low ? d : d - half;
                const float o = x[low ? d + half : j];
                const float r = low ? y[i] * rc[j] - o * rs[j] : o * rs[j] + y[i] * rc[j];
                y[i] = known ? r : NAN;
            }
        }
    }
    if (h < a.n_q) {
        const size_t off = ((size_t)s * a.n_q + h) * a.hd + d0, plane = (size_t)a.S * a.n_q * a.hd;
        if constexpr (QM == Q_F32) {
            *reinterpret_cast<float4v*>(static_cast<float*>(a.q_out) + off) = float4v{y[0], y[1], y[2], y[3]};
        } else {
            vsl_half* q = static_cast<vsl_half*>(a.q_out);
            half4 hi4, lo4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vsl_half hi, lo;
                split_f16(y[i], hi, lo);
                hi4[i] = hi;
                lo4[i] = lo;
            }
            *reinterpret_cast<half4*>(q + off) = hi4;
            if constexpr (QM == Q_F16X2) *reinterpret_cast<half4*>(q + plane + off) = lo4;
        }
        return;
    }
    const bool is_k = h < a.n_q + a.n_kv;
    const uint32_t kvh = is_k ? h - a.n_q : h - a.n_q - a.n_kv;
    KT* dst = static_cast<KT*>(is_k ? a.kc : a.vc) + ((size_t)kvh * a.cap + pos) * a.hd + d0;
    if constexpr (sizeof(KT) == 4)
        *reinterpret_cast<float4v*>(dst) = float4v{y[0], y[1], y[2], y[3]};
    else
        *reinterpret_cast<half4*>(dst) = half4{(vsl_half)y[0], (vsl_half)y[1], (vsl_half)y[2], (vsl_half)y[3]};
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Arguments that both entries share; VSL_OK or the error code (nothing is launched on error).
int check_part(const char* fn, const PartArgs& a, int rope, int kv_dtype) {
    if (!a.qkv || !a.q_out || !a.kc || !a.vc || (a.rot && (!a.rc || !a.rs))) return vsl_invalid("%s: null pointer", fn);
    if (a.hd == 0 || a.hd % 8 || a.hd > 512) return vsl_unsupported("%s: head_dim %u (a multiple of 8 up to 512)", fn, a.hd);
    if (a.rot % 2 || a.rot > a.hd) return vsl_invalid("%s: %u rotated dims of %u (even, at most all)", fn, a.rot, a.hd);
    if (a.n_q == 0 || a.n_kv == 0 || ((uint64_t)a.n_q + 2ull * a.n_kv) * a.hd > 0x7FFFFFFFull)
        return vsl_invalid("%s: n_q=%u n_kv=%u", fn, a.n_q, a.n_kv);
    if (rope != VSL_ROPE_PAIRS && rope != VSL_ROPE_HALVES) return vsl_invalid("%s: rotation %d", fn, rope);
    if (kv_dtype != VSL_DT_F16 && kv_dtype != VSL_DT_F32) return vsl_unsupported("%s: kv dtype %d", fn, kv_dtype);
    if (a.cap == 0 || (a.rot && a.table_rows == 0)) return vsl_invalid("%s: capacity %u, %u table rows", fn, a.cap, a.table_rows);
    for (const void* p : {static_cast<const void*>(a.qkv), static_cast<const void*>(a.rc), static_cast<const void*>(a.rs),
                          static_cast<const void*>(a.q_out), static_cast<const void*>(a.kc), static_cast<const void*>(a.vc)})
        if (!aligned16(p)) return vsl_invalid("%s: pointers must be 16-byte aligned", fn);
    if (reinterpret_cast<uintptr_t>(a.positions) & 3) return vsl_invalid("%s: misaligned positions", fn);
    return VSL_OK;
}

template <bool VEC, int QM, bool DEC>
void launch_part(uint32_t grid, hipStream_t s, const PartArgs& a, uint32_t bpr, int kv_dtype, vsl_ctrl* ctrl) {
    if (kv_dtype == VSL_DT_F16) k_rope_part<VEC, QM, vsl_half, DEC><<<grid, 256, 0, s>>>(a, bpr, ctrl);
    else k_rope_part<VEC, QM, float, DEC><<<grid, 256, 0, s>>>(a, bpr, ctrl);
}

}  // namespace

extern "C" int vsl_rope_tables(uint32_t rot, uint32_t pos0, uint32_t rows, const vsl_rope_scaling* scaling,
                               const float* freq_factors, float* rope_cos, float* rope_sin, void* stream) {
    const char* fn = "vsl_rope_tables";
    if (!scaling || !rope_cos || !rope_sin) return vsl_invalid("%s: null pointer", fn);
    if (rot == 0 || rot % 2 || rot > 512) return vsl_unsupported("%s: %u rotated dims (even, 2..512)", fn, rot);
    if ((uint64_t)pos0 + rows > 1ull << 31) return vsl_unsupported("%s: %u positions from %u", fn, rows, pos0);
    if (rows == 0) return VSL_OK;
    const vsl_rope_scaling& p = *scaling;
    auto good = [](float v) { return v > 0.f && std::isfinite(v); };
    if (!good(p.theta)) return vsl_invalid("%s: theta %g", fn, (double)p.theta);
    if (!(p.mscale >= 0.f) || !std::isfinite(p.mscale)) return vsl_invalid("%s: scale of the tables %g", fn, (double)p.mscale);
    FreqArgs a{std::log2((double)p.theta), 1.0, 0.0, 0.0, 0.0, p.mscale > 0.f ? (double)p.mscale : 1.0, 0, 0};
    const double two_pi = 6.283185307179586;
    if (p.type != VSL_ROPE_SCALE_NONE) {
        if (!good(p.factor)) return vsl_invalid("%s: factor %g", fn, (double)p.factor);
        a.inv_factor = 1.0 / (double)p.factor;
    }
    if (p.type == VSL_ROPE_SCALE_TURNS || p.type == VSL_ROPE_SCALE_YARN) {
        if (!good(p.orig_ctx) || !good(p.low) || !good(p.high) || !(p.high > p.low))
            return vsl_invalid("%s: context %g, turns %g to %g", fn, (double)p.orig_ctx, (double)p.low, (double)p.high);
    }
    if (p.type == VSL_ROPE_SCALE_TURNS) {
        a.by_turns = 1;
        a.turns = (double)p.orig_ctx / two_pi;
        a.lo = p.low;
        a.inv_span = 1.0 / ((double)p.high - (double)p.low);
    } else if (p.type == VSL_ROPE_SCALE_YARN) {
        if (p.theta <= 1.f) return vsl_invalid("%s: theta %g", fn, (double)p.theta);
        auto pair = [&](double turns) {
            return (double)rot * std::log((double)p.orig_ctx / (two_pi * turns)) / (2.0 * std::log((double)p.theta));
        };
        auto within = [&](double d) { return std::fmin(std::fmax(d, 0.0), (double)rot - 1.0); };
        const double lo = within(std::floor(pair(p.high))), hi = within(std::ceil(pair(p.low)));
        a.by_pair = 1;
        a.lo = lo;
        a.inv_span = 1.0 / std::fmax(hi - lo, 0.001);
        if (!(p.mscale > 0.f)) a.mscale = p.factor > 1.f ? 0.1 * std::log((double)p.factor) + 1.0 : 1.0;
    } else if (p.type != VSL_ROPE_SCALE_NONE && p.type != VSL_ROPE_SCALE_LINEAR) {
        return vsl_unsupported("%s: scaling %d", fn, p.type);
    }
    if ((reinterpret_cast<uintptr_t>(rope_cos) | reinterpret_cast<uintptr_t>(rope_sin) |
         reinterpret_cast<uintptr_t>(freq_factors)) & 3)
        return vsl_invalid("%s: misaligned pointer", fn);
    const uint32_t half = rot / 2;
    const uint64_t threads = (uint64_t)half * ((rows + kRun - 1) / kRun);
    k_rope_tables<<<(uint32_t)((threads + 255) / 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
        half, pos0, rows, a, (double)rot, freq_factors, rope_cos, rope_sin);
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}

extern "C" int vsl_rope_part_append(const float* qkv, uint32_t S, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t rot,
                                    int rope, uint32_t pos0, const uint32_t* positions, const float* rope_cos,
                                    const float* rope_sin, uint32_t table_rows, void* q_out, int q_dtype, void* kcache,
                                    void* vcache, int kv_dtype, uint32_t cap, void* stream) {
    const char* fn = "vsl_rope_part_append";
    const PartArgs a{qkv, S, n_q, n_kv, hd, rot, pos0, cap, table_rows, rope == VSL_ROPE_HALVES, positions, rope_cos, rope_sin,
                     q_out, kcache, vcache};
    if (const int rc = check_part(fn, a, rope, kv_dtype)) return rc;
    if (q_dtype != VSL_DT_F32 && q_dtype != VSL_DT_F16 && q_dtype != VSL_DT_F16X2)
        return vsl_unsupported("%s: q dtype %d", fn, q_dtype);
    if ((uint64_t)pos0 + S > cap) return vsl_capacity("%s: %u positions from %u exceed capacity %u", fn, S, pos0, cap);
    if (S == 0) return VSL_OK;
    const uint32_t bpr = (uint32_t)((((uint64_t)n_q + 2ull * n_kv) * (hd / 4) + 255) / 256);
    if ((uint64_t)S * bpr > 1ull << 23) return vsl_unsupported("%s: %u rows in one call", fn, S);  // 2^31 lanes
    const uint32_t grid = S * bpr;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto vec) {
        constexpr bool VEC = decltype(vec)::value;
        if (q_dtype == VSL_DT_F32) launch_part<VEC, Q_F32, false>(grid, s, a, bpr, kv_dtype, nullptr);
        else if (q_dtype == VSL_DT_F16) launch_part<VEC, Q_F16, false>(grid, s, a, bpr, kv_dtype, nullptr);
        else launch_part<VEC, Q_F16X2, false>(grid, s, a, bpr, kv_dtype, nullptr);
    };
    if (rot % 8 == 0) go(std::true_type{});
    else go(std::false_type{});
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}

extern "C" int vsl_rope_part_append_decode(const float* qkv, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t rot, int rope,
                                           const uint32_t* position, const float* rope_cos, const float* rope_sin,
                                           uint32_t table_rows, float* q_out, void* kcache, void* vcache, int kv_dtype,
                                           uint32_t cap, vsl_ctrl* ctrl, void* stream) {
    const char* fn = "vsl_rope_part_append_decode";
    const PartArgs a{qkv, 1, n_q, n_kv, hd, rot, 0, cap, table_rows, rope == VSL_ROPE_HALVES, position, rope_cos, rope_sin,
                     q_out, kcache, vcache};
    if (const int rc = check_part(fn, a, rope, kv_dtype)) return rc;
    if (!ctrl) return vsl_invalid("%s: null pointer", fn);
    const uint32_t bpr = (uint32_t)((((uint64_t)n_q + 2ull * n_kv) * (hd / 4) + 255) / 256);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rot % 8 == 0) launch_part<true, Q_F32, true>(bpr, s, a, bpr, kv_dtype, ctrl);
    else launch_part<false, Q_F32, true>(bpr, s, a, bpr, kv_dtype, ctrl);
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}
