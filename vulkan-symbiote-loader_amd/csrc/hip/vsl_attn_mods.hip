// vsl_attn_mods.hip -- decode attention with capped scores, a distance bias and a range of keys (vsl_attn_decode_mods). No
// reference counterpart.
#include "vsl_attn_mods.h"
#include "vsl_internal.h"

using namespace attn_mods;

namespace {

constexpr uint32_t kMaxSplits = 1024;
constexpr int kWaves = 4, kTileKeys = 32;

struct DecodeArgs {
    const float* q;
    const void* kc;
    const void* vc;
    uint32_t G, cap, nsplit;
    float to_u;    // scale / softcap, or scale * log2(e) without a cap
    float from_u;  // softcap * log2(e)
    const float* slopes;
    const uint32_t* ranges;
    float* part_o;
    float* part_ml;
    vsl_ctrl* ctrl;
};

// keys [begin, end) of the row at position p
__device__ __forceinline__ void key_range(const uint32_t* ranges, uint32_t p, uint32_t& begin, uint32_t& end) {
    begin = ranges ? ranges[0] : 0;
    end = ranges ? min(ranges[1], p + 1) : p + 1;
    if (begin >= end) begin = end = 0;
}

// The waves' sums of a block joined, the split's partials written: part_ml = (m, l), part_o = sum of 2^(s - m) v.
template <int HD>
__device__ __forceinline__ void join_waves(const float (*s_ml)[8][2], const float (*s_acc)[8][HD], const DecodeArgs& a,
                                           uint32_t kvh, uint32_t split) {
    for (uint32_t e = threadIdx.x; e < a.G * (HD / 4); e += kWaves * 64) {
        const uint32_t g = e / (HD / 4), dd = e % (HD / 4) * 4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_ml[w][g][0]);
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4v A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = fast_exp2(s_ml[w][g][0] - ref);
            L = fmaf(s_ml[w][g][1], f, L);
#pragma unroll
            for (int i = 0; i < 4; ++i) A[i] = fmaf(s_acc[w][g][dd + i], f, A[i]);
        }
        const size_t at = (size_t)(kvh * a.G + g) * a.nsplit + split;
        *reinterpret_cast<float4v*>(a.part_o + at * HD + dd) = A;
        if (dd == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
    }
}

// fp16 caches. Block (split, KV head) of four waves; wave w takes the 32-key tiles (j nsplit + split) 4 + w from the range's
// start. Both products on the matrix cores (16 x 16 x 32):
//   S^T = K Q^T   columns 0-7 hold the group's heads as the hi plane of q (unscaled: times scale / softcap the lo plane would
//                 fall among binary16's subnormals), 8-15 as the lo plane, so that the sum of two columns is the product of
//                 the fp32 q. Row r of half t is key 8 (r / 4) + 4 t + r % 4, so lane l
//                 ends with the scores of head l % 8 at the 8 keys of octet l / 16,
//   O^T = V^T P^T which is this product's operand as it is; V goes through 8 KB of the wave's LDS, whose transpose reads give
//                 a lane 8 keys of a dim.
// Bound by reading the range once: 32001 keys, 8 KV heads of 128, cap 50, in 22.5 us, 5.8 TB/s (the join 4.6 more, 29.7 in all;
// 41 keys of a tiny model 6.9, two launches). For that two tiles' loads are in flight in each wave, in 128 registers.
template <int HD, bool CAP>
__global__ __launch_bounds__(kWaves * 64, 1) void k_decode_mods(DecodeArgs a) {
    constexpr int KS = HD / 32, NC = HD / 16, CPR = HD / 8, NV = kTileKeys * CPR / 64;
    __shared__ __attribute__((aligned(16))) vsl_half s_v[kWaves][kTileKeys * HD];
    __shared__ __attribute__((aligned(16))) float s_ml[kWaves][8][2];
    __shared__ __attribute__((aligned(16))) float s_acc[kWaves][8][HD];
    const uint32_t kvh = blockIdx.y, split = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15, rg = lane >> 4, head = col & 7;
    const bool in_group = head < a.G;
    const uint32_t h = kvh * a.G + (in_group ? head : 0);
    const vsl_half* Kb = static_cast<const vsl_half*>(a.kc) + (size_t)kvh * a.cap * HD;
    const vsl_half* Vb = static_cast<const vsl_half*>(a.vc) + (size_t)kvh * a.cap * HD;
    float4 qa[KS][2];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const float* qp = a.q + (size_t)h * HD + 32 * ks + 8 * rg;
        qa[ks][0] = *reinterpret_cast<const float4*>(qp);
        qa[ks][1] = *reinterpret_cast<const float4*>(qp + 4);
    }
    const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    if (a.ctrl->done) return;
    const uint32_t p = a.ctrl->pos < a.cap ? a.ctrl->pos : a.cap - 1;
    uint32_t begin, end;
    key_range(a.ranges, p, begin, end);

    struct Tile {
        u32x4 k[2][KS], v[NV];
    };
    const uint32_t krow = 8 * (col >> 2) + (col & 3);
    auto issue = [&](Tile& b, uint32_t k0) {  // keys past the range read its last one
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const vsl_half* kp = Kb + (size_t)min(k0 + krow + 4 * t, end - 1) * HD + 8 * rg;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) b.k[t][ks] = *reinterpret_cast<const u32x4*>(kp + 32 * ks);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = i * 64 + lane;
            b.v[i] = *reinterpret_cast<const u32x4*>(Vb + (size_t)min(k0 + c / CPR, end - 1) * HD + c % CPR * 8);
        }
    };
    half8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const float x[8] = {qa[ks][0].x, qa[ks][0].y, qa[ks][0].z, qa[ks][0].w,
                            qa[ks][1].x, qa[ks][1].y, qa[ks][1].z, qa[ks][1].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            vsl_half hi, lo;
            split_f16(x[e], hi, lo);
            qf[ks][e] = in_group ? (col < 8 ? hi : lo) : (vsl_half)0.f;
        }
    }
    float m = -INFINITY, l = 0.f;
    const float minus_plane = col < 8 ? 0.f : -1.f;
    float4v o[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = float4v{0.f, 0.f, 0.f, 0.f};

    auto consume = [&](const Tile& b, uint32_t k0) {
        float s[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float4v d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, b.k[t][ks]), qf[ks], d, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[4 * t + i] = a.to_u * (d[i] + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(d[i]), 0x128, 0xF, 0xF, false)));
        }
        if constexpr (CAP) {
            float um = fabsf(s[0]);
#pragma unroll
            for (int e = 1; e < 8; ++e) um = fmaxf(um, fabsf(s[e]));
            if (__builtin_amdgcn_ballot_w64(um > kTanhNear)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] = tanh_any(s[e]) * a.from_u;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] = tanh_near(s[e]) * a.from_u;
            }
        }
        const bool whole = k0 + kTileKeys <= end;  // wave-uniform
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t k = k0 + 8 * rg + e;
            s[e] = fmaf(slope, (float)((int)k - (int)p), s[e]);
            if (!whole) s[e] = k < end ? s[e] : -INFINITY;
        }
        // V to LDS; keys past the range as zeros, whatever the cache holds
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = i * 64 + lane, r = c / CPR;
            u32x4 w = b.v[i];
            if (!whole && k0 + r >= end) w = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(&s_v[wave][swizzle<HD>(r, c % CPR)]) = w;
        }
        float bm = s[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) bm = fmaxf(bm, s[e]);
        if (__builtin_amdgcn_ballot_w64(bm - m > kLazy + kRoom)) {  // m = -inf: any finite score raises it
            float a0, a1;
            lane_pair<16>(bm, a0, a1);
            lane_pair<32>(fmaxf(a0, a1), a0, a1);
            const float mn = fmaxf(m, fmaxf(a0, a1) - kRoom);
            const float corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
            l *= corr;
#pragma unroll
            for (int i = 0; i < NC; ++i) o[i] *= corr;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        half8 pf;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const float p0 = fast_exp2(s[e] - ref), p1 = fast_exp2(s[e + 1] - ref);
            l += p0;
            l += p1;
            const half2v hi = round2(p0, p1);
            const half2v w = round2(fmaf((float)hi[0], minus_plane, p0), fmaf((float)hi[1], minus_plane, p1));
            pf[e] = w[0];
            pf[e + 1] = w[1];
        }
        // lane i of 16 addresses V[8 rg + i / 4][16 c + 4 (i % 4) ..] and receives V[8 rg + j][16 c + i] as its value j
        const int gi = lane & 15, d4 = 4 * (gi & 3);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int d = 16 * i + d4, r = 8 * rg + (gi >> 2);
            const half4 x0 = lds_read_tr16(&s_v[wave][swizzle<HD>(r, d >> 3) + (d & 7)]);
            const half4 x1 = lds_read_tr16(&s_v[wave][swizzle<HD>(r + 4, d >> 3) + (d & 7)]);
            const half8 af = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af, pf, o[i], 0, 0, 0);
        }
    };

    const uint32_t step = a.nsplit * kWaves * kTileKeys;
    uint32_t k0 = begin + (split * kWaves + wave) * kTileKeys;
    if (k0 < end) {
        Tile b0, b1;
        issue(b0, k0);
        for (;;) {
            const bool more1 = end - k0 > step;  // another tile of this wave
            issue(b1, more1 ? k0 + step : k0);
            __builtin_amdgcn_sched_barrier(0);
            consume(b0, k0);
            if (!more1) break;
            k0 += step;
            const bool more0 = end - k0 > step;
            issue(b0, more0 ? k0 + step : k0);
            __builtin_amdgcn_sched_barrier(0);
            consume(b1, k0);
            if (!more0) break;
            k0 += step;
        }
    }
    // sums over the octets, the planes' columns joined; lane l holds head l % 8, dims 16 i + 4 (l / 16) + r in o[i][r]
    float l0, l1;
    lane_pair<16>(l, l0, l1);
    lane_pair<32>(l0 + l1, l0, l1);
    l = l0 + l1;
    if (m == -INFINITY && l != 0.f) m = 0.f;  // only NaN scores: keep the sum in the join
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            o[i][r] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(o[i][r]), 0x128, 0xF, 0xF, false));
    if (col < a.G) {
#pragma unroll
        for (int i = 0; i < NC; ++i) *reinterpret_cast<float4v*>(&s_acc[wave][col][16 * i + 4 * rg]) = o[i];
        if (rg == 0) {
            s_ml[wave][col][0] = m;
            s_ml[wave][col][1] = l;
        }
    }
    __syncthreads();
    join_waves<HD>(s_ml, s_acc, a, kvh, split);
}

// fp32 caches: a group of HD / 8 lanes a key, eight dims a lane, fp32 throughout. Bound by the latency of a key's loads, of which none
// is in flight ahead: 32001 keys, 8 KV heads of 128, 121 us, 2.2 TB/s (a tiny model's 41 keys 7.6). For caches of small models.
template <int HD, bool CAP>
__global__ __launch_bounds__(kWaves * 64, 1) void k_decode_mods_f32(DecodeArgs a) {
    constexpr int LPP = HD / 8, SLOTS = 64 / LPP;
    __shared__ __attribute__((aligned(16))) float s_ml[kWaves][8][2];
    __shared__ __attribute__((aligned(16))) float s_acc[kWaves][8][HD];
    const uint32_t kvh = blockIdx.y, split = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slot = lane / LPP, sub = lane % LPP;
    const float* Kb = static_cast<const float*>(a.kc) + (size_t)kvh * a.cap * HD + sub * 8;
    const float* Vb = static_cast<const float*>(a.vc) + (size_t)kvh * a.cap * HD + sub * 8;
    if (a.ctrl->done) return;
    const uint32_t p = a.ctrl->pos < a.cap ? a.ctrl->pos : a.cap - 1;
    uint32_t begin, end;
    key_range(a.ranges, p, begin, end);
    float q[8][8], slope[8], m[8], l[8], acc[8][8];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        const uint32_t h = kvh * a.G + (g < (int)a.G ? g : 0);
        slope[g] = a.slopes ? a.slopes[h] * kLog2e : 0.f;
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            q[g][i] = a.q[(size_t)h * HD + sub * 8 + i] * a.to_u;
            acc[g][i] = 0.f;
        }
    }
    const uint32_t step = a.nsplit * kWaves * SLOTS;
    for (uint32_t k0 = begin + (split * kWaves + wave) * SLOTS; k0 < end; k0 = end - k0 > step ? k0 + step : end) {
        const uint32_t k = k0 + slot;
        const bool in = k < end;
        const size_t at = (size_t)(in ? k : end - 1) * HD;
        float kf[8], vf[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            kf[i] = Kb[at + i];
            vf[i] = in ? Vb[at + i] : 0.f;
        }
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            if (g >= (int)a.G) break;
            float d = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) d = fmaf(q[g][i], kf[i], d);
            d = group_sum_dpp<LPP>(d);
            if constexpr (CAP) d = tanh_any(d) * a.from_u;
            d = fmaf(slope[g], (float)((int)k - (int)p), d);
            const float mn = in ? fmaxf(m[g], d) : m[g];
            const float corr = mn == -INFINITY ? 1.f : fast_exp2(m[g] - mn);
            const float w = in ? fast_exp2(d - (mn == -INFINITY ? 0.f : mn)) : 0.f;
            l[g] = fmaf(l[g], corr, w);
            m[g] = mn;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[g][i] = fmaf(acc[g][i], corr, w * vf[i]);
        }
    }
    // the wave's slots joined: lanes at distances LPP .. 32
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        if (g >= (int)a.G) break;
        if (m[g] == -INFINITY && l[g] != 0.f) m[g] = 0.f;  // only NaN scores
        auto join = [&](auto x) {
            constexpr int X = decltype(x)::value;
            float ma, mb, la, lb;
            lane_pair<X>(m[g], ma, mb);
            lane_pair<X>(l[g], la, lb);
            const float M = fmaxf(ma, mb);
            const float fa = ma == -INFINITY ? 0.f : fast_exp2(ma - M), fb = mb == -INFINITY ? 0.f : fast_exp2(mb - M);
            l[g] = la * fa + lb * fb;
            m[g] = M;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float aa, ab;
                lane_pair<X>(acc[g][i], aa, ab);
                acc[g][i] = aa * fa + ab * fb;
            }
        };
        if constexpr (LPP == 8) join(std::integral_constant<int, 8>());
        join(std::integral_constant<int, 16>());
        join(std::integral_constant<int, 32>());
        if (slot == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s_acc[wave][g][sub * 8 + i] = acc[g][i];
            if (sub == 0) {
                s_ml[wave][g][0] = m[g];
                s_ml[wave][g][1] = l[g];
            }
        }
    }
    __syncthreads();
    join_waves<HD>(s_ml, s_acc, a, kvh, split);
}

// out[head] = sum of the splits' sums / sum of their weights, zeros where no key was attended to. A block a head; the first
// 32 splits' sums are requested before their weights are known.
template <int HD>
__global__ __launch_bounds__(256) void k_join_decode(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                     uint32_t nsplit, float* __restrict__ out, const vsl_ctrl* ctrl) {
    constexpr int LPR = HD / 4, GRP = 256 / LPR, EARLY = 32 / GRP;
    __shared__ float s_w[kMaxSplits], s_red[4], s_l[4];
    __shared__ __attribute__((aligned(16))) float s_o[GRP][HD];
    const uint32_t h = blockIdx.x, t = threadIdx.x, grp = t / LPR, dd = t % LPR * 4;
    const float* po = part_o + (size_t)h * nsplit * HD + dd;
    float4v early[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
        const uint32_t s = grp + i * GRP;
        early[i] = *reinterpret_cast<const float4v*>(po + (size_t)(s < nsplit ? s : 0) * HD);
    }
    float mx = -INFINITY, mine[4], lsum = 0.f;
    float2 ml[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t s = t + 256 * i;
        ml[i] = s < nsplit ? *reinterpret_cast<const float2*>(part_ml + ((size_t)h * nsplit + s) * 2) : make_float2(-INFINITY, 0.f);
        mx = fmaxf(mx, ml[i].x);
    }
    const uint32_t done = ctrl->done;
    mx = wave_max_dpp(mx);
    if ((t & 63) == 0) s_red[t >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        mine[i] = fast_exp2(ml[i].x - ref);
        if (t + 256 * i < nsplit) s_w[t + 256 * i] = mine[i];
        lsum = fmaf(ml[i].y, mine[i], lsum);
    }
    lsum = wave_sum_dpp(lsum);
    if ((t & 63) == 0) s_l[t >> 6] = lsum;
    __syncthreads();
    float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
        const uint32_t s = grp + i * GRP;
        const float w = s < nsplit ? s_w[s] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = s < nsplit ? fmaf(early[i][j], w, acc[j]) : acc[j];
    }
    for (uint32_t s = grp + 32; s < nsplit; s += GRP) {
        const float4v v = *reinterpret_cast<const float4v*>(po + (size_t)s * HD);
        const float w = s_w[s];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(v[j], w, acc[j]);
    }
    *reinterpret_cast<float4v*>(&s_o[grp][dd]) = acc;
    __syncthreads();
    if (t >= (uint32_t)HD || done) return;
    float v = 0.f;
#pragma unroll
    for (int g = 0; g < GRP; ++g) v += s_o[g][t];
    const float L = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
    out[(size_t)h * HD + t] = L == 0.f ? 0.f : v / L;
}

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace

extern "C" int vsl_attn_decode_mods(const float* q, const void* kcache, const void* vcache, int kv_dtype, uint32_t n_q,
                                    uint32_t n_kv, uint32_t hd, uint32_t cap, float scale, uint32_t nsplit, float* part_o,
                                    float* part_ml, float* out, vsl_ctrl* ctrl, const vsl_attn_mods* mods, void* stream) {
    const char* fn = "vsl_attn_decode_mods";
    if (!q || !kcache || !vcache || !part_o || !part_ml || !out || !ctrl) return vsl_invalid("%s: null pointer", fn);
    if (n_kv == 0 || n_q == 0 || n_q % n_kv) return vsl_invalid("%s: n_q=%u not a multiple of n_kv=%u", fn, n_q, n_kv);
    if (cap == 0 || cap > 0x7FFFFFFFu) return vsl_invalid("%s: capacity %u", fn, cap);
    if (nsplit == 0 || nsplit > kMaxSplits) return vsl_invalid("%s: nsplit=%u (1..%u)", fn, nsplit, kMaxSplits);
    const uint32_t G = n_q / n_kv;
    if (G > 8 || n_kv > 65535) return vsl_unsupported("%s: GQA ratio %u (supported 1..8), %u KV heads", fn, G, n_kv);
    if ((hd != 64 && hd != 128) || (kv_dtype != VSL_DT_F16 && kv_dtype != VSL_DT_F32))
        return vsl_unsupported("%s: head_dim %u / kv dtype %d (supported 64,128 / f16,f32)", fn, hd, kv_dtype);
    for (const void* p : {static_cast<const void*>(q), kcache, vcache, static_cast<const void*>(part_o), static_cast<const void*>(out)})
        if (!aligned_to(p, 16)) return vsl_invalid("%s: pointers must be 16-byte aligned", fn);
    const vsl_attn_mods none{};
    const vsl_attn_mods& md = mods ? *mods : none;
    if (!aligned_to(part_ml, 8) || !aligned_to(md.slopes, 4) || !aligned_to(md.ranges, 8)) return vsl_invalid("%s: misaligned pointer", fn);
    if (!softcap_ok(md.softcap, scale)) return vsl_invalid("%s: softcap %g with scale %g", fn, (double)md.softcap, (double)scale);
    const bool capped = md.softcap > 0.f;
    const DecodeArgs a{q, kcache, vcache, G, cap, nsplit, capped ? scale / md.softcap : scale * kLog2e, md.softcap * kLog2e,
                       md.slopes, md.ranges, part_o, part_ml, ctrl};
    const dim3 grid(nsplit, n_kv);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto hdc, auto cc) {
        constexpr int HD = decltype(hdc)::value;
        constexpr bool CAP = decltype(cc)::value;
        if (kv_dtype == VSL_DT_F16) k_decode_mods<HD, CAP><<<grid, kWaves * 64, 0, s>>>(a);
        else k_decode_mods_f32<HD, CAP><<<grid, kWaves * 64, 0, s>>>(a);
        k_join_decode<HD><<<n_q, 256, 0, s>>>(part_o, part_ml, nsplit, out, ctrl);
    };
    if (hd == 128 && capped) go(std::integral_constant<int, 128>{}, std::true_type{});
    else if (hd == 128) go(std::integral_constant<int, 128>{}, std::false_type{});
    else if (capped) go(std::integral_constant<int, 64>{}, std::true_type{});
    else go(std::integral_constant<int, 64>{}, std::false_type{});
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}
