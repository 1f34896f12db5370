// vsl_kv4_prefill.hip -- causal flash attention of prompt rows over the 4-bit KV cache (VSL_DT_KV4).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vsl_device.h"
#include "vsl_hip.h"
#include "vsl_internal.h"
#include "vsl_kv4.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Half index of 16-byte chunk c of row r in an LDS tile of rows of N halfs (a power of two): the chunk xored with
// the row so that 16 lanes reading the same chunk of 16 rows hit all banks once.
template <int N>
__device__ __forceinline__ int sw(int r, int c) {
    if constexpr (N >= 128) return r * N + ((c ^ (r & 15)) * 8);  // 256-byte rows
    else return r * N + ((c ^ ((r >> 1) & 7)) * 8);               // 128-byte rows: row pairs
}

// S prompt rows at positions pos0.. (their keys and values already in the cache). Block = GB query heads of one KV head
// x 32 query rows, KSPLIT waves a head, each taking its share of every tile of TK keys, joined at the end. The codes of
// a tile are loaded by whole words, expanded to binary16 once for all the block's waves and left in LDS: K row-major,
// V by columns (a word of V is 8 positions of one column). Per tile each wave computes S^T = K Q^T by
// v_mfma_f32_32x32x16_f16, the online softmax of its 32 rows (a lane owns a row with lane ^ 32), and O^T += V^T P^T.
// MFMA row r of a 32-key fragment is the key with bits 2 and 3 of r exchanged, so that the scores a lane holds are
// octets of consecutive keys: the probabilities are the B operand as they are, and V^T's operand one 16-byte LDS read.
// The next tile's codes are in flight while a tile is computed.
template <int HD, int G, int GB, bool QX2, int KSPLIT, int TK>
__global__ __launch_bounds__(64 * GB * KSPLIT) void k_attn_prefill_kv4(
    const vsl_half* __restrict__ q, const char* __restrict__ kc, const char* __restrict__ vc, uint32_t S, uint32_t pos0,
    uint32_t n_q, uint32_t n_kv, uint32_t cap, float scale, vsl_half* __restrict__ out, int om, uint32_t win,
    uint32_t n_glob, uint32_t thr) {
    constexpr int NT = 64 * GB * KSPLIT, NB = HD / 32;
    constexpr int NKB = TK / 32 / KSPLIT;  // 32-key fragments of a tile per wave
    constexpr int NKW = TK * HD / 16 / NT; // pairs of words per thread and tile, of K and of V
    constexpr int QP = QX2 ? 2 : 1;        // q planes; with split q the probabilities are split too
    static_assert(G % GB == 0 && NKB >= 1 && NKB * KSPLIT * 32 == TK, "a tile's fragments divide over a head's waves");
    static_assert(NKW >= 1 && NKW * NT * 16 == TK * HD, "a tile's words divide over the block");
    __shared__ __attribute__((aligned(16))) vsl_half Ks[2][TK * HD];
    __shared__ __attribute__((aligned(16))) vsl_half Vs[2][TK * HD];
    __shared__ float s_stat[KSPLIT][GB][128];  // row statistics of the key shares, for their join
    __shared__ uint32_t s_nan;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t qb = gridDim.x - 1 - blockIdx.x;  // the longest (latest) query blocks start first
    const uint32_t kvh = blockIdx.y / (G / GB);
    const int ksp = wave / GB, kbase = ksp * NKB;
    const uint32_t h = kvh * G + (blockIdx.y % (G / GB)) * GB + wave % GB;
    const uint32_t s_base = qb * 32, my_s = s_base + (lane & 31), qw = n_q * HD;
    const size_t qplane = (size_t)S * qw;
    // scores are scaled within the exponential's argument, which the maximum then needs a positive factor for: a
    // negative scale negates q, a zero one is a factor that leaves no difference
    const float sl2 = fmaxf(fabsf(scale) * kLog2e, 1e-30f);
    const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;
    const uint32_t last_s = min(S, s_base + 32) - 1;
    const uint32_t kv_end = pos0 + last_s + 1, my_pos = pos0 + my_s;
    const uint32_t n_tiles = (kv_end + TK - 1) / TK;
    // windowed rows (position p with p + 1 > thr) see the keys below n_glob and from p - win on; where the first row is
    // windowed, the tiles between are skipped
    const uint32_t p_first = pos0 + s_base, p_last = pos0 + last_s;
    uint32_t n_gt = n_tiles, t_lo = n_tiles;
    if (p_first + 1 > thr && p_first > win) {
        t_lo = (p_first - win) / TK;
        n_gt = min((n_glob + TK - 1) / TK, t_lo);
    }
    const uint32_t n_vt = n_gt + (n_tiles - t_lo);
    auto phys = [&](uint32_t vt) { return vt < n_gt ? vt : vt - n_gt + t_lo; };
    const uint32_t my_lo = (my_pos + 1 > thr && my_pos > win) ? my_pos - win : 0;
    const uint32_t lo_max = (p_last + 1 > thr && p_last > win) ? p_last - win : 0;

    const uint64_t P = kv4_positions(cap), soff = kv4_steps_off(n_kv, cap, HD);
    const Kv4Consts kc4 = kv4_consts();
    const char* Kc = kc + (uint64_t)kvh * P * (HD / 2);
    const char* Kst = kc + soff + (uint64_t)kvh * P * NB * 2;
    const char* Vc = vc + (uint64_t)kvh * P * (HD / 2);
    const char* Vst = vc + soff + (uint64_t)kvh * P * NB * 2;

    // Pair i of a thread: K words 2w, 2w + 1 (16 dims) of a key row, V words of columns 2w, 2w + 1 of an octet.
    struct KWords {
        uint2 k[NKW];
        uint32_t s[NKW];
    };
    struct VWords {
        uint2 v[NKW];
        u32x4 s[NKW];
    };
    auto load_k = [&](KWords& b, uint32_t t) {
#pragma unroll
        for (int i = 0; i < NKW; ++i) {
            const int r = (i * NT + tid) / (HD / 16), w = (i * NT + tid) % (HD / 16);
            const uint64_t row = (uint64_t)t * TK + r;
            b.k[i] = *reinterpret_cast<const uint2*>(Kc + row * (HD / 2) + 8 * w);
            b.s[i] = *reinterpret_cast<const uint16_t*>(Kst + (row * NB + w / 2) * 2);
        }
    };
    auto load_v = [&](VWords& b, uint32_t t) {
#pragma unroll
        for (int i = 0; i < NKW; ++i) {
            const int r = (i * NT + tid) / (HD / 2), w = (i * NT + tid) % (HD / 2);
            const uint64_t oct = (uint64_t)t * (TK / 8) + r;
            b.v[i] = *reinterpret_cast<const uint2*>(Vc + (oct * HD + 2 * w) * 4);
            b.s[i] = *reinterpret_cast<const u32x4*>(Vst + (oct * NB + w / 16) * 16);
        }
    };
    // A tile's values into LDS. What lies past the block's last key is anything: its steps are taken as 0. So is a V
    // block that stands for NaN, as a NaN would reach rows that do not see it through a product with 0: the
    // block notes that there was one, and the rows that see it are found at the end.
    auto expand_k = [&](const KWords& b, int buf, uint32_t t) {
#pragma unroll
        for (int i = 0; i < NKW; ++i) {
            const int r = (i * NT + tid) / (HD / 16), w = (i * NT + tid) % (HD / 16);
            const uint32_t st = t * TK + r < kv_end ? b.s[i] : 0u;
            const Kv4Step s = kv4_step(st | st << 16, kc4);
            *reinterpret_cast<half8*>(&Ks[buf][sw<HD>(r, 2 * w)]) = kv4_word(b.k[i].x, s, kc4);
            *reinterpret_cast<half8*>(&Ks[buf][sw<HD>(r, 2 * w + 1)]) = kv4_word(b.k[i].y, s, kc4);
        }
    };
    auto expand_v = [&](const VWords& b, int buf, uint32_t t) {
#pragma unroll
        for (int i = 0; i < NKW; ++i) {
            const int r = (i * NT + tid) / (HD / 2), w = (i * NT + tid) % (HD / 2);
            u32x4 s = b.s[i];
            if ((t + 1) * TK > kv_end) {  // block-uniform
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const uint32_t key = t * TK + 8 * r + 2 * p;
                    s[p] = key >= kv_end ? 0u : key + 1 >= kv_end ? s[p] & 0xFFFFu : s[p];
                }
            }
            // an exponent of all ones carries into its half's top bit, which steps leave 0
            const u32x4 c = s + 0x04000400u;
            if (((c[0] | c[1] | c[2] | c[3]) & 0x80008000u) != 0) {
                s_nan = 1;
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    if ((s[p] & 0xFFFFu) == kKv4NaN) s[p] &= 0xFFFF0000u;
                    if (s[p] >> 16 == kKv4NaN) s[p] &= 0xFFFFu;
                }
            }
            Kv4Step vs[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) vs[p] = kv4_step(s[p], kc4);
            *reinterpret_cast<half8*>(&Vs[buf][sw<TK>(2 * w, r)]) = kv4_word(b.v[i].x, vs, kc4);
            *reinterpret_cast<half8*>(&Vs[buf][sw<TK>(2 * w + 1, r)]) = kv4_word(b.v[i].y, vs, kc4);
        }
    };

    // Q^T as the B operand of S^T = K Q^T: lane holds row l % 32, dims 16 c + 8 (l / 32) .. + 7
    half8 qf[QP][HD / 16];
#pragma unroll
    for (int p = 0; p < QP; ++p)
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
            const uint32_t row = my_s < S ? my_s : S - 1;  // rows past S are never stored
            const u32x4 x = *reinterpret_cast<const u32x4*>(q + p * qplane + (size_t)row * qw + (size_t)h * HD + c * 16 +
                                                            (lane >> 5) * 8);
            qf[p][c] = __builtin_bit_cast(half8, x ^ flip);
        }
    float16v o[HD / 32];
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] = 0.f;
    float m = -INFINITY, l = 0.f, minus_one = -1.f;
    asm volatile("" : "+v"(minus_one));  // a register, so that value - (float)half is one mixed-precision multiply-add
    constexpr float kLazy = 8.f;  // the reference maximum is raised only by more than this (log2 units)

    const int krow = (lane & 19) | (lane & 4) << 1 | (lane & 8) >> 1;  // bits 2 and 3 of l % 32 exchanged
    auto qk = [&](int buf, float16v (&st)[NKB]) {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
            for (int v = 0; v < 16; ++v) st[kb][v] = 0.f;
            half8 kf[HD / 16];
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
                kf[c] = *reinterpret_cast<const half8*>(&Ks[buf][sw<HD>((kbase + kb) * 32 + krow, 2 * c + (lane >> 5))]);
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
#pragma unroll
                for (int p = 0; p < QP; ++p) st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[c], qf[p][c], st[kb], 0, 0, 0);
        }
    };
    // the mask, where tile t reaches past the block's first row or begins before a row's window; returns the scaled
    // maximum of this lane's row. Element v of a fragment is key 16 (v / 8) + 8 (l / 32) + v % 8.
    auto mask_max = [&](float16v (&st)[NKB], uint32_t t) {
        if (!(t * TK + TK - 1 <= p_first && (t * TK >= lo_max || t * TK + TK <= n_glob))) {
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const uint32_t key = t * TK + (kbase + kb) * 32 + (v >> 3) * 16 + (lane >> 5) * 8 + (v & 7);
                    const bool seen = key <= my_pos && (key >= my_lo || key < n_glob);
                    st[kb][v] = seen ? st[kb][v] : -INFINITY;
                }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int v = 0; v < 16; ++v) bm = fmaxf(bm, st[kb][v]);
        float ba, bb;
        lane_pair<32>(bm, ba, bb);
        return fmaxf(ba, bb) * sl2;
    };
    auto rescale = [&](float bm) {
        const bool raise = bm > m + kLazy;  // m = -inf: any finite tile maximum raises it
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float mn = raise ? bm : m;
            const float corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);  // m = -inf: 0
            l *= corr;
            m = mn;
#pragma unroll
            for (int tt = 0; tt < HD / 32; ++tt)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[tt][v] *= corr;
        }
    };
    auto probs = [&](const float16v (&st)[NKB], half8 (&pf)[QP][NKB][2]) {
        float ps = 0.f;
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int v = 0; v < 16; v += 2) {
                const float p0 = fast_exp2(fmaf(st[kb][v], sl2, -ref)), p1 = fast_exp2(fmaf(st[kb][v + 1], sl2, -ref));
                ps += p0;
                ps += p1;
                const half2v hi = pack_f16(p0, p1);
                pf[0][kb][v >> 3][v & 7] = hi[0];
                pf[0][kb][v >> 3][(v & 7) + 1] = hi[1];
                if constexpr (QX2) {
                    const half2v lo = pack_f16(fmaf((float)hi[0], minus_one, p0), fmaf((float)hi[1], minus_one, p1));
                    pf[QP - 1][kb][v >> 3][v & 7] = lo[0];
                    pf[QP - 1][kb][v >> 3][(v & 7) + 1] = lo[1];
                }
            }
        float pa, pb;
        lane_pair<32>(ps, pa, pb);
        return pa + pb;
    };
    auto pv = [&](int buf, const half8 (&pf)[QP][NKB][2]) {
#pragma unroll
        for (int tt = 0; tt < HD / 32; ++tt)
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int hi = 0; hi < 2; ++hi) {
                    const half8 af = *reinterpret_cast<const half8*>(
                        &Vs[buf][sw<TK>(tt * 32 + (lane & 31), (kbase + kb) * 4 + 2 * hi + (lane >> 5))]);
#pragma unroll
                    for (int p = 0; p < QP; ++p)
                        o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af, pf[p][kb][hi], o[tt], 0, 0, 0);
                }
    };

    // Two buffers each for K and V, K one tile ahead. At the top of iteration t, K of t and t + 1 and V of t are in LDS
    // and the scores of t in registers: the codes of K of t + 2 and V of t + 1 are requested, the scores of t + 1 are
    // issued on the matrix cores while the vector pipe turns those of t into probabilities, then the products
    // of t with V; the codes go into the buffers that K of t and V of t - 1 have left (both last read before the
    // barrier that ended the previous iteration). Requests past the last tile repeat it.
    auto tile = [&](uint32_t t) { return phys(t < n_vt ? t : n_vt - 1); };
    if (tid == 0) s_nan = 0;
    __syncthreads();
    KWords kw;
    VWords vw;
    load_k(kw, tile(0));
    load_v(vw, tile(0));
    expand_k(kw, 0, tile(0));
    load_k(kw, tile(1));
    expand_v(vw, 0, tile(0));
    expand_k(kw, 1, tile(1));
    __syncthreads();
    float16v st[NKB];
    qk(0, st);
    for (uint32_t t = 0; t < n_vt; ++t) {
        load_k(kw, tile(t + 2));
        load_v(vw, tile(t + 1));
        rescale(mask_max(st, phys(t)));
        float16v sn[NKB];
        qk((int)((t + 1) & 1), sn);
        half8 pf[QP][NKB][2];
        l += probs(st, pf);
        pv((int)(t & 1), pf);
        // every wave has its scores of t (taken in the previous iteration)
        expand_k(kw, (int)(t & 1), tile(t + 2));
        expand_v(vw, (int)((t + 1) & 1), tile(t + 1));
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) st[kb] = sn[kb];
        __syncthreads();
    }
    const uint32_t any_nan = s_nan;

    if constexpr (KSPLIT > 1) {
        // the key shares of each head, joined in LDS (the tile buffers are done with): waves with ksp > 0 leave their
        // accumulators and row statistics, the ksp = 0 wave brings all to the largest maximum
        constexpr int SLOT = HD / 32 * 16 * 64;          // accumulator floats of a wave
        constexpr int PER = 2 * TK * HD * 2 / 4 / SLOT;  // slots in each of the two buffer sets
        static_assert(2 * PER >= (KSPLIT - 1) * GB, "the join does not fit in the tile buffers");
        const int hw = wave % GB;
        auto slot = [&](int j) {
            const int i = (j - 1) * GB + hw;
            return reinterpret_cast<float*>(i < PER ? &Ks[0][0] : &Vs[0][0]) + (i % PER) * SLOT;
        };
        if (ksp > 0) {
            float* xo = slot(ksp);
#pragma unroll
            for (int tt = 0; tt < HD / 32; ++tt)
#pragma unroll
                for (int v = 0; v < 16; ++v) xo[(tt * 16 + v) * 64 + lane] = o[tt][v];
            s_stat[ksp][hw][lane] = m;
            s_stat[ksp][hw][64 + lane] = l;
        }
        __syncthreads();
        if (ksp > 0) return;
        float mm = m;
#pragma unroll
        for (int j = 1; j < KSPLIT; ++j) mm = fmaxf(mm, s_stat[j][hw][lane]);
        if (mm == -INFINITY) mm = 0.f;  // only NaN scores: their sums are kept (below)
        // a share that saw no score has l = 0, or NaN from NaN scores: either way it joins with weight 1 or less
        auto weight = [&](float mj) { return mj == -INFINITY ? 1.f : fast_exp2(mj - mm); };
        const float c0 = weight(m);
        l *= c0;
#pragma unroll
        for (int tt = 0; tt < HD / 32; ++tt)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[tt][v] *= c0;
#pragma unroll
        for (int j = 1; j < KSPLIT; ++j) {
            const float* xo = slot(j);
            const float cj = weight(s_stat[j][hw][lane]);
            l += s_stat[j][hw][64 + lane] * cj;
#pragma unroll
            for (int tt = 0; tt < HD / 32; ++tt)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[tt][v] += xo[(tt * 16 + v) * 64 + lane] * cj;
        }
    }

    if (my_s >= S) return;
    uint32_t nan_blocks = 0;  // 32-dim blocks of V in which this row sees a NaN
    if (any_nan) {
        const uint16_t* vs = reinterpret_cast<const uint16_t*>(Vst);
        for (uint32_t key = 0; key <= my_pos; ++key) {
            if (key < my_lo && key >= n_glob) continue;
            for (int bl = 0; bl < NB; ++bl)
                if (vs[((size_t)(key / 8) * NB + bl) * 8 + key % 8] == kKv4NaN) nan_blocks |= 1u << bl;
        }
    }
    const float inv = 1.f / l;  // every row sees its own position
    vsl_half* orow = out + (size_t)my_s * qw + (size_t)h * HD;
    // element v of O^T fragment t is dim 32 t + 8 (v / 4) + 4 (l / 32) + v % 4: runs of four dims, one store a plane
#pragma unroll
    for (int t = 0; t < HD / 32; ++t) {
        const float f = nan_blocks >> t & 1 ? __builtin_nanf("") : inv;
#pragma unroll
        for (int v0 = 0; v0 < 16; v0 += 4) {
            const int dim = t * 32 + (v0 >> 2) * 8 + (lane >> 5) * 4;
            const float x[4] = {o[t][v0] * f, o[t][v0 + 1] * f, o[t][v0 + 2] * f, o[t][v0 + 3] * f};
            half4 hv, lv;
            if (om == 2) {
                uint32_t lo8;
                split4_f16_f8(x[0], x[1], x[2], x[3], hv, lo8);
                // the lo8 plane (bytes) follows the hi plane
                *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(out + qplane) + (size_t)my_s * qw +
                                             lo8_pos(h * HD + dim)) = lo8;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vsl_half hi, lo;
                    split_f16(x[i], hi, lo);
                    hv[i] = hi;
                    lv[i] = lo;
                }
                if (om == 1) *reinterpret_cast<half4*>(orow + qplane + dim) = lv;
            }
            *reinterpret_cast<half4*>(orow + dim) = hv;
        }
    }
}

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

struct Args {
    const vsl_half* q;
    const char* k;
    const char* v;
    uint32_t S, pos0, n_q, n_kv, cap;
    float scale;
    vsl_half* out;
    int om;
    uint32_t win, n_glob, thr;
};

template <int HD, int G, int GB, bool QX2, int KSPLIT, int TK>
void launch(hipStream_t s, const Args& a) {
    const dim3 grid((a.S + 31) / 32, a.n_kv * (G / GB));
    k_attn_prefill_kv4<HD, G, GB, QX2, KSPLIT, TK><<<grid, 64 * GB * KSPLIT, 0, s>>>(
        a.q, a.k, a.v, a.S, a.pos0, a.n_q, a.n_kv, a.cap, a.scale, a.out, a.om, a.win, a.n_glob, a.thr);
}

// Up to four heads share a block, two waves a head: groups of a power of two, or pairs or single heads of the others
// (a block's threads divide a tile's words).
template <int HD, int G, bool QX2>
void launch_group(hipStream_t s, const Args& a) {
    constexpr int GB = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
    launch<HD, G, GB, QX2, 2, 64 * 128 / HD>(s, a);
}

template <int HD, int G>
void launch_q(hipStream_t s, const Args& a, bool x2) {
    if (x2) launch_group<HD, G, true>(s, a);
    else launch_group<HD, G, false>(s, a);
}

int attn_prefill_kv4(const char* fn, const void* q, int q_dtype, const void* kcache, const void* vcache, uint32_t S,
                     uint32_t pos0, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t cap, float scale, void* out, int out_dtype,
                     uint32_t win, uint32_t n_glob, uint32_t thr, void* stream) {
    if (!q || !kcache || !vcache || !out) return vsl_invalid("%s: null pointer", fn);
    if (n_kv == 0 || n_q == 0 || n_q % n_kv) return vsl_invalid("%s: n_q=%u n_kv=%u", fn, n_q, n_kv);
    if (hd != 64 && hd != 128) return vsl_unsupported("%s: head_dim %u (64 or 128)", fn, hd);
    if (n_q / n_kv > 8) return vsl_unsupported("%s: GQA ratio %u (supported 1..8)", fn, n_q / n_kv);
    if ((q_dtype != VSL_DT_F16 && q_dtype != VSL_DT_F16X2) ||
        (out_dtype != VSL_DT_F16 && out_dtype != VSL_DT_F16X2 && out_dtype != VSL_DT_F16F8))
        return vsl_unsupported("%s: dtypes %d/%d", fn, q_dtype, out_dtype);
    if (!aligned_to(kcache, 256) || !aligned_to(vcache, 256)) return vsl_invalid("%s: a 4-bit cache must be 256-byte aligned", fn);
    if (!aligned_to(q, 16) || !aligned_to(out, 16)) return vsl_invalid("%s: q and out must be 16-byte aligned", fn);
    if ((uint64_t)pos0 + S > cap) return vsl_capacity("%s: %u positions from %u exceed capacity %u", fn, S, pos0, cap);
    if (!std::isfinite(scale)) return vsl_invalid("%s: scale is not finite", fn);
    if (cap > 0x80000000u) return vsl_unsupported("%s: capacity %u", fn, cap);
    if ((uint64_t)n_q * hd > 0x7FFFFFFFull || n_q > 65535u) return vsl_unsupported("%s: n_q=%u", fn, n_q);
    if (S == 0) return VSL_OK;
    const Args a{static_cast<const vsl_half*>(q), static_cast<const char*>(kcache), static_cast<const char*>(vcache), S, pos0,
                 n_q, n_kv, cap, scale, static_cast<vsl_half*>(out),
                 out_dtype == VSL_DT_F16X2 ? 1 : out_dtype == VSL_DT_F16F8 ? 2 : 0, win, n_glob, thr};
    const bool x2 = q_dtype == VSL_DT_F16X2;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto by_group = [&](auto hdc) {
        constexpr int HD = decltype(hdc)::value;
        switch (n_q / n_kv) {
            case 1: launch_q<HD, 1>(s, a, x2); break;
            case 2: launch_q<HD, 2>(s, a, x2); break;
            case 3: launch_q<HD, 3>(s, a, x2); break;
            case 4: launch_q<HD, 4>(s, a, x2); break;
            case 5: launch_q<HD, 5>(s, a, x2); break;
            case 6: launch_q<HD, 6>(s, a, x2); break;
            case 7: launch_q<HD, 7>(s, a, x2); break;
            default: launch_q<HD, 8>(s, a, x2); break;
        }
    };
    if (hd == 128) by_group(std::integral_constant<int, 128>{});
    else by_group(std::integral_constant<int, 64>{});
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}

}  // namespace

extern "C" int vsl_attn_prefill_kv4(const void* q, int q_dtype, const void* kcache, const void* vcache, uint32_t S,
                                    uint32_t pos0, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t cap, float scale,
                                    void* out, int out_dtype, void* stream) {
    // no window: every position is below the threshold
    return attn_prefill_kv4("vsl_attn_prefill_kv4", q, q_dtype, kcache, vcache, S, pos0, n_q, n_kv, hd, cap, scale, out,
                            out_dtype, 0, 0, 0xFFFFFFFFu, stream);
}

extern "C" int vsl_attn_prefill_kv4_window(const void* q, int q_dtype, const void* kcache, const void* vcache, uint32_t S,
                                           uint32_t pos0, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t cap, float scale,
                                           void* out, int out_dtype, uint32_t window, uint32_t n_global, uint32_t threshold,
                                           void* stream) {
    if ((uint64_t)window + n_global >= 0x80000000ull)
        return vsl_invalid("vsl_attn_prefill_kv4_window: window %u + global %u too large", window, n_global);
    return attn_prefill_kv4("vsl_attn_prefill_kv4_window", q, q_dtype, kcache, vcache, S, pos0, n_q, n_kv, hd, cap, scale, out,
                            out_dtype, window, n_global, threshold, stream);
}
