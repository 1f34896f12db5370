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
// The next tiles' codes are in flight while a tile is computed.
// Bound by power at large sizes, 2048 rows at 6144 of the 8B shape with a split q (0.48 TFLOP on the matrix cores): 427 us,
// 1.13 PFLOP/s, against 1.25 of a large fp16 library product on the same card. The clock is at 1.9 GHz then; with the two waves
// of a SIMD in opposite phases (one in its products, one in its probabilities and expansion, a barrier each) it falls to 1.75
// and the time stays (425 us; smaller calls lose 5-25 %). Before the order of blocks was what it is, 470 us fell to 412
// without the expansion in the loop and to 398 without the exponentials too.
template <int HD, int G, int GB, bool QX2, int KSPLIT, int TK>
__global__ __launch_bounds__(64 * GB * KSPLIT) void k_attn_prefill_kv4(
    const vsl_half* __restrict__ q, const char* __restrict__ kc, const char* __restrict__ vc, uint32_t S, uint32_t pos0,
    uint32_t n_q, uint32_t n_kv, uint32_t cap, float scale, vsl_half* __restrict__ out, int om, uint32_t win,
    uint32_t n_glob, uint32_t thr) {
    constexpr int NT = 64 * GB * KSPLIT, NB = HD / 32;
    constexpr int NKB = TK / 32 / KSPLIT;  // 32-key fragments of a tile per wave
    constexpr int NKW = TK * HD / 16 / NT; // pairs of words per thread and tile, of K and of V
    // q planes; with a split q the probabilities are split too. A caller who passes one plane has q in fp16 already: the
    // probabilities are then rounded to it as well, 2^-11 of each (512 rows of the 1B shape: 2.5e-4 from the exact values,
    // of which the fp16 output alone is 2.0e-4), for half the matrix work: 2048 rows at 6144 296 us, split 429.
    constexpr int QP = QX2 ? 2 : 1;
    static_assert(G % GB == 0 && NKB >= 1 && NKB * KSPLIT * 32 == TK, "a tile's fragments divide over a head's waves");
    static_assert(NKW >= 1 && NKW * NT * 16 == TK * HD, "a tile's words divide over the block");
    __shared__ __attribute__((aligned(16))) vsl_half smem[4 * TK * HD];  // two buffers of K, two of V
    auto Ks = [&](int buf) { return smem + buf * (TK * HD); };
    auto Vs = [&](int buf) { return smem + (2 + buf) * (TK * HD); };
    __shared__ float s_stat[KSPLIT][GB][128];  // row statistics of the key shares, for their join
    __shared__ uint32_t s_nan;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the longest (latest) query blocks of every head start first; neighbouring blocks, which go to different XCDs, take
    // different KV heads (with 8 of them each XCD's L2 holds one). Head by head instead, the last head's longest blocks start
    // in the second round: 2048 rows at 6144 458 us instead of 427, 1B shape 1500 rows at 500 55 instead of 44.
    const uint32_t hb = n_q / GB, qb = gridDim.x / hb - 1 - blockIdx.x / hb;
    const uint32_t kvh = blockIdx.x % hb % n_kv;
    const int ksp = wave / GB, kbase = ksp * NKB;
    const uint32_t h = kvh * G + (blockIdx.x % hb / n_kv) * GB + wave % GB;
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
    // A tile's values into LDS. A V block that stands for NaN would reach rows that do not see its key through a product
    // with 0, and so would an infinity from a step that no append stored (the bits past the block's last key, and of
    // positions that a window hides from all its rows, are anything). Tiles that some row sees in part (EDGE) take such
    // steps as 0; the block notes that there was a NaN, and the rows that see it are found at the end. (K needs none
    // of this: what a key's row of scores holds is replaced where it is masked.)
    auto expand_k = [&](const KWords& b, int buf) {
#pragma unroll
        for (int i = 0; i < NKW; ++i) {
            const int r = (i * NT + tid) / (HD / 16), w = (i * NT + tid) % (HD / 16);
            const Kv4Step s = kv4_step(b.s[i] | b.s[i] << 16, kc4);
            *reinterpret_cast<half8*>(Ks(buf) + sw<HD>(r, 2 * w)) = kv4_word(b.k[i].x, s, kc4);
            *reinterpret_cast<half8*>(Ks(buf) + sw<HD>(r, 2 * w + 1)) = kv4_word(b.k[i].y, s, kc4);
        }
    };
    auto expand_v = [&](const VWords& b, int buf, uint32_t t, auto edge) {
#pragma unroll
        for (int i = 0; i < NKW; ++i) {
            const int r = (i * NT + tid) / (HD / 2), w = (i * NT + tid) % (HD / 2);
            u32x4 s = b.s[i];
            if constexpr (decltype(edge)::value) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t x = s[e / 2] >> (16 * (e & 1)) & 0xFFFFu;
                    if (x <= kKv4MaxStep) continue;
                    s[e / 2] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                    if (t * TK + 8 * r + e < kv_end) s_nan = 1;
                }
            }
            Kv4Step vs[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) vs[p] = kv4_step(s[p], kc4);
            *reinterpret_cast<half8*>(Vs(buf) + sw<TK>(2 * w, r)) = kv4_word(b.v[i].x, vs, kc4);
            *reinterpret_cast<half8*>(Vs(buf) + sw<TK>(2 * w + 1, r)) = kv4_word(b.v[i].y, vs, kc4);
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

    const int krow = (lane & 19) | (lane & 4) << 1 | (lane & 8) >> 1;  // bits 2 and 3 of l % 32 exchanged
    auto read_k = [&](int buf, half8 (&kf)[NKB][HD / 16]) {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
                kf[kb][c] = *reinterpret_cast<const half8*>(Ks(buf) + sw<HD>((kbase + kb) * 32 + krow, 2 * c + (lane >> 5)));
    };
    auto qk = [&](const half8 (&kf)[NKB][HD / 16], float16v (&st)[NKB]) {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
#pragma unroll
            for (int v = 0; v < 16; ++v) st[kb][v] = 0.f;
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
#pragma unroll
                for (int p = 0; p < QP; ++p)
                    st[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kb][c], qf[p][c], st[kb], 0, 0, 0);
        }
    };
    // the mask of a tile that some row sees in part; returns the maximum of this lane's row. Element v of a
    // fragment is key 16 (v / 8) + 8 (l / 32) + v % 8.
    auto mask_max = [&](float16v (&st)[NKB], uint32_t t, auto edge) {
        if constexpr (decltype(edge)::value) {
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
        return fmaxf(ba, bb);
    };
    auto rescale = [&](float bm) {
        const bool raise = fmaf(bm, sl2, -m) > kKv4Lazy + kKv4Room;  // m = -inf: any finite tile maximum raises it
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float mn = raise ? fmaf(bm, sl2, -kKv4Room) : m;
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
                        Vs(buf) + sw<TK>(tt * 32 + (lane & 31), (kbase + kb) * 4 + 2 * hi + (lane >> 5)));
#pragma unroll
                    for (int p = 0; p < QP; ++p)
                        o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af, pf[p][kb][hi], o[tt], 0, 0, 0);
                }
    };

    // Two buffers each for K and V, K one tile ahead. At the top of iteration t, K of t and t + 1 and V of t are in LDS
    // and the scores of t in registers: the codes of K of t + 2 and V of t + 1 are requested, the scores of t + 1 are
    // issued on the matrix cores while the vector pipe turns those of t into probabilities, then the products
    // of t with V; the codes go into the buffers that K of t and V of t - 1 have left (both last read before the
    // barrier that ended the previous iteration; K of tile 0 before one of its own). Tiles that every row of the block
    // sees whole come first (without a window): they run without masks and checks, in one straight block of code past
    // the rescale.
    float16v st[NKB];
    KWords kw;
    VWords vw;
    auto body = [&](uint32_t t, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        const bool one = !EDGE || t + 1 < n_vt, two = t + 2 < n_vt;
        if (!EDGE || two) load_k(kw, phys(two ? t + 2 : t));
        if (one) load_v(vw, phys(t + 1));
        half8 kf[NKB][HD / 16];
        if (one) read_k((int)((t + 1) & 1), kf);
        if constexpr (!EDGE) __builtin_amdgcn_sched_barrier(0);
        rescale(mask_max(st, phys(t), edge));
        float16v sn[NKB];
        if (one) qk(kf, sn);
        half8 pf[QP][NKB][2];
        l += probs(st, pf);
        pv((int)(t & 1), pf);
        if (!EDGE || two) expand_k(kw, (int)(t & 1));  // every wave has its scores of t
        if (one) expand_v(vw, (int)((t + 1) & 1), phys(t + 1), edge);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) st[kb] = sn[kb];
        __syncthreads();
    };
    if (tid == 0) s_nan = 0;
    __syncthreads();
    load_k(kw, phys(0));
    load_v(vw, phys(0));
    expand_k(kw, 0);
    if (n_vt > 1) load_k(kw, phys(1));
    expand_v(vw, 0, phys(0), std::true_type{});
    if (n_vt > 1) expand_k(kw, 1);
    __syncthreads();
    {
        half8 kf[NKB][HD / 16];
        read_k(0, kf);
        __syncthreads();  // body(0) writes K of tile 2 where this read K of tile 0
        qk(kf, st);
    }
    const uint32_t n_whole = lo_max ? 0 : (p_first + 1) / TK;
    uint32_t t = 0;
    for (; t + 1 < n_whole; ++t) body(t, std::false_type{});
    for (; t < n_vt; ++t) body(t, std::true_type{});
    const uint32_t any_nan = s_nan;

    // The key shares of each head, joined in LDS (the tile buffers are done with): wave ksp of a head takes the 32-dim
    // fragments f with f % KSPLIT = ksp from all of them, brought to the largest maximum, and stores them.
    constexpr int NF = HD / 32;
    if constexpr (KSPLIT > 1) {
        constexpr int FS = 16 * 64;  // floats of a fragment
        static_assert(GB * NF * (KSPLIT - 1) * FS * 4 <= 4 * TK * HD * 2, "the join does not fit in the tile buffers");
        const int hw = wave % GB;
        // fragment f as share j leaves it to its taker (j is not the taker)
        auto slot = [&](int f, int j) {
            return reinterpret_cast<float*>(smem) + ((hw * NF + f) * (KSPLIT - 1) + (j < f % KSPLIT ? j : j - 1)) * FS + lane;
        };
#pragma unroll
        for (int f = 0; f < NF; ++f)
            if (f % KSPLIT != ksp) {
#pragma unroll
                for (int v = 0; v < 16; ++v) slot(f, ksp)[v * 64] = o[f][v];
            }
        s_stat[ksp][hw][lane] = m;
        s_stat[ksp][hw][64 + lane] = l;
        __syncthreads();
        float mj[KSPLIT], wj[KSPLIT], mm = -INFINITY;
#pragma unroll
        for (int j = 0; j < KSPLIT; ++j) mm = fmaxf(mm, mj[j] = s_stat[j][hw][lane]);
        if (mm == -INFINITY) mm = 0.f;  // only NaN scores
        l = 0.f;
#pragma unroll
        for (int j = 0; j < KSPLIT; ++j) {
            // a share that saw no score has sums of 0, or of NaN from NaN scores, which are kept
            wj[j] = mj[j] == -INFINITY ? 1.f : fast_exp2(mj[j] - mm);
            l = fmaf(s_stat[j][hw][64 + lane], wj[j], l);
        }
        const float own = m == -INFINITY ? 1.f : fast_exp2(m - mm);
#pragma unroll
        for (int f = 0; f < NF; ++f)
            if (f % KSPLIT == ksp) {
#pragma unroll
                for (int v = 0; v < 16; ++v) o[f][v] *= own;
#pragma unroll
                for (int j = 0; j < KSPLIT; ++j)
                    if (j != ksp) {
#pragma unroll
                        for (int v = 0; v < 16; ++v) o[f][v] = fmaf(slot(f, j)[v * 64], wj[j], o[f][v]);
                    }
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
    for (int t = 0; t < NF; ++t) {
        if (KSPLIT > 1 && t % KSPLIT != ksp) continue;
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

// The same for few rows, where a block for a head and 32 rows leaves CUs idle and no tile is shared: block (row block,
// head) of WAVES waves that go through the keys by themselves, wave w the tiles of 32 keys w, w + WAVES, ..., straight from
// the cache into registers (two tiles in flight, no barrier before the join). As above but for the orders of dims, which
// follow the cache's words so that a lane reads its codes by 16 bytes: lane group g = l / 32 takes the dims HD/2 g + 8 c ..
// of the scores' step c, and row r of the product's fragment f is dim NF r + f. Join: every wave leaves its sums in LDS,
// and takes two of their 16 registers from all of them.
template <int HD, bool QX2, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void k_attn_prefill_kv4_few(
    const vsl_half* __restrict__ q, const char* __restrict__ kc, const char* __restrict__ vc, uint32_t S, uint32_t pos0,
    uint32_t n_q, uint32_t n_kv, uint32_t cap, float scale, vsl_half* __restrict__ out, int om, uint32_t win,
    uint32_t n_glob, uint32_t thr) {
    constexpr int NB = HD / 32, NF = HD / 32, NS = HD / 16, QP = QX2 ? 2 : 1, VPW = 16 / WAVES;
    constexpr uint32_t TK = 32;
    typedef float fragv __attribute__((ext_vector_type(NF)));
    __shared__ __attribute__((aligned(16))) fragv s_o[WAVES][16][64];
    __shared__ float s_stat[WAVES][2][64];
    __shared__ uint32_t s_nan;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5;
    const uint32_t kvh = blockIdx.x % n_q % n_kv, h = kvh * (n_q / n_kv) + blockIdx.x % n_q / n_kv;  // order: see above
    const uint32_t s_base = blockIdx.x / n_q * 32, my_s = s_base + (lane & 31), qw = n_q * HD;
    const size_t qplane = (size_t)S * qw;
    const float sl2 = fmaxf(fabsf(scale) * kLog2e, 1e-30f);  // see above
    const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;
    const uint32_t last_s = min(S, s_base + 32) - 1;
    const uint32_t p_first = pos0 + s_base, p_last = pos0 + last_s, my_pos = pos0 + my_s, kv_end = p_last + 1;
    const uint32_t n_tiles = (kv_end + TK - 1) / TK;
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
    const uint32_t krow = (lane & 19) | (lane & 4) << 1 | (lane & 8) >> 1;  // bits 2 and 3 of l % 32 exchanged
    const char* Kc = kc + ((uint64_t)kvh * P + krow) * (HD / 2) + g * (HD / 4);
    const char* Kst = kc + soff + (((uint64_t)kvh * P + krow) * NB + g * NB / 2) * 2;
    const char* Vc = vc + (((uint64_t)kvh * (P / 8) + g) * HD + NF * (lane & 31)) * 4;
    const char* Vst0 = vc + soff + (uint64_t)kvh * P * NB * 2;
    const char* Vst = Vst0 + ((uint64_t)g * NB + NF * (lane & 31) / 32) * 16;

    struct Tile {
        uint32_t k[NS], ks, v[2][NF];
        u32x4 vs[2];
    };
    auto issue = [&](Tile& b, uint32_t t) {
        const uint64_t p0 = (uint64_t)t * TK;
        const u32x4* kp = reinterpret_cast<const u32x4*>(Kc + p0 * (HD / 2));
#pragma unroll
        for (int i = 0; i < NS / 4; ++i) {
            const u32x4 w = kp[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) b.k[4 * i + j] = w[j];
        }
        if constexpr (NB == 4) b.ks = *reinterpret_cast<const uint32_t*>(Kst + p0 * NB * 2);
        else b.ks = *reinterpret_cast<const uint16_t*>(Kst + p0 * NB * 2);
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
            const uint64_t oct = p0 / 8 + 2 * hi;
            if constexpr (NF == 4) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(Vc + oct * HD * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) b.v[hi][j] = w[j];
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(Vc + oct * HD * 4);
                b.v[hi][0] = w.x;
                b.v[hi][1] = w.y;
            }
            b.vs[hi] = *reinterpret_cast<const u32x4*>(Vst + oct * NB * 16);
        }
    };

    half8 qf[QP][NS];
#pragma unroll
    for (int p = 0; p < QP; ++p)
#pragma unroll
        for (int c = 0; c < NS; ++c) {
            const uint32_t row = my_s < S ? my_s : S - 1;  // rows past S are never stored
            const u32x4 x = *reinterpret_cast<const u32x4*>(q + p * qplane + (size_t)row * qw + (size_t)h * HD + g * (HD / 2) + 8 * c);
            qf[p][c] = __builtin_bit_cast(half8, x ^ flip);
        }
    float16v o[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[f][v] = 0.f;
    float m = -INFINITY, l = 0.f, minus_one = -1.f;
    asm volatile("" : "+v"(minus_one));
    if (threadIdx.x == 0) s_nan = 0;
    __syncthreads();

    auto consume = [&](Tile& b, uint32_t vt) {
        const uint32_t p0 = phys(vt) * TK;
        float16v st;
#pragma unroll
        for (int v = 0; v < 16; ++v) st[v] = 0.f;
#pragma unroll
        for (int c = 0; c < NS; ++c) {
            // a lane group's dims: one or two blocks
            const uint32_t x = c < 4 ? b.ks & 0xFFFFu : b.ks >> 16;
            const half8 kf = kv4_word(b.k[c], kv4_step(x | x << 16, kc4), kc4);
#pragma unroll
            for (int p = 0; p < QP; ++p) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[p][c], st, 0, 0, 0);
        }
        if (!(p0 + TK - 1 <= p_first && (p0 >= lo_max || p0 + TK <= n_glob))) {  // some row sees the tile in part
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const uint32_t key = p0 + (v >> 3) * 16 + g * 8 + (v & 7);
                st[v] = key <= my_pos && (key >= my_lo || key < n_glob) ? st[v] : -INFINITY;
            }
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t x = b.vs[hi][e / 2] >> (16 * (e & 1)) & 0xFFFFu;
                    if (x <= kKv4MaxStep) continue;
                    b.vs[hi][e / 2] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                    if (p0 + 16 * hi + 8 * g + e < kv_end) s_nan = 1;
                }
        }
        float bm = st[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) bm = fmaxf(bm, st[v]);
        float ba, bb;
        lane_pair<32>(bm, ba, bb);
        bm = fmaxf(ba, bb);
        const bool raise = fmaf(bm, sl2, -m) > kKv4Lazy + kKv4Room;  // m = -inf: any finite tile maximum raises it
        if (__builtin_amdgcn_ballot_w64(raise)) {
            const float mn = raise ? fmaf(bm, sl2, -kKv4Room) : m;
            const float corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);  // m = -inf: 0
            l *= corr;
            m = mn;
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[f][v] *= corr;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        half8 pf[QP][2];
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
            const float p_0 = fast_exp2(fmaf(st[v], sl2, -ref)), p_1 = fast_exp2(fmaf(st[v + 1], sl2, -ref));
            l += p_0;
            l += p_1;
            const half2v hi = pack_f16(p_0, p_1);
            pf[0][v >> 3][v & 7] = hi[0];
            pf[0][v >> 3][(v & 7) + 1] = hi[1];
            if constexpr (QX2) {
                const half2v lo = pack_f16(fmaf((float)hi[0], minus_one, p_0), fmaf((float)hi[1], minus_one, p_1));
                pf[QP - 1][v >> 3][v & 7] = lo[0];
                pf[QP - 1][v >> 3][(v & 7) + 1] = lo[1];
            }
        }
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
            Kv4Step vs[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) vs[p] = kv4_step(b.vs[hi][p], kc4);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const half8 vf = kv4_word(b.v[hi][f], vs, kc4);
#pragma unroll
                for (int p = 0; p < QP; ++p) o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[p][hi], o[f], 0, 0, 0);
            }
        }
    };
    Tile ta, tb;
    uint32_t vt = wave;
    if (vt < n_vt) issue(ta, phys(vt));
    if (vt + WAVES < n_vt) issue(tb, phys(vt + WAVES));
    while (vt < n_vt) {
        consume(ta, vt);
        vt += WAVES;
        if (vt >= n_vt) break;
        issue(ta, phys(vt + WAVES < n_vt ? vt + WAVES : vt));  // past the wave's last tile the one just read
        __builtin_amdgcn_sched_barrier(0);
        consume(tb, vt);
        vt += WAVES;
        if (vt >= n_vt) break;
        issue(tb, phys(vt + WAVES < n_vt ? vt + WAVES : vt));
        __builtin_amdgcn_sched_barrier(0);
    }
    float l0, l1;
    lane_pair<32>(l, l0, l1);
    l = l0 + l1;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
        fragv x;
#pragma unroll
        for (int f = 0; f < NF; ++f) x[f] = o[f][v];
        s_o[wave][v][lane] = x;
    }
    s_stat[wave][0][lane] = m;
    s_stat[wave][1][lane] = l;
    __syncthreads();
    if (my_s >= S) return;
    float w[WAVES], mm = -INFINITY;
#pragma unroll
    for (int j = 0; j < WAVES; ++j) mm = fmaxf(mm, w[j] = s_stat[j][0][lane]);
    if (mm == -INFINITY) mm = 0.f;  // only NaN scores
    l = 0.f;
#pragma unroll
    for (int j = 0; j < WAVES; ++j) {
        // a wave that saw no score has sums of 0, or of NaN from NaN scores, which are kept
        w[j] = w[j] == -INFINITY ? 1.f : fast_exp2(w[j] - mm);
        l = fmaf(s_stat[j][1][lane], w[j], l);
    }
    uint32_t nan_blocks = 0;  // 32-dim blocks of V in which this row sees a NaN
    if (s_nan) {
        const uint16_t* vs = reinterpret_cast<const uint16_t*>(Vst0);
        for (uint32_t key = 0; key <= my_pos; ++key) {
            if (key < my_lo && key >= n_glob) continue;
            for (int bl = 0; bl < NB; ++bl)
                if (vs[((size_t)(key / 8) * NB + bl) * 8 + key % 8] == kKv4NaN) nan_blocks |= 1u << bl;
        }
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < VPW; ++i) {
        const int v = VPW * wave + i;
        fragv x;
#pragma unroll
        for (int f = 0; f < NF; ++f) x[f] = 0.f;
#pragma unroll
        for (int j = 0; j < WAVES; ++j) {
            const fragv y = s_o[j][v][lane];
#pragma unroll
            for (int f = 0; f < NF; ++f) x[f] = fmaf(y[f], w[j], x[f]);
        }
        const uint32_t dim = NF * ((v >> 2) * 8 + g * 4 + (v & 3));  // dims dim .. dim + NF - 1
        x *= nan_blocks >> (dim / 32) & 1 ? __builtin_nanf("") : inv;
        const size_t at = (size_t)my_s * qw + (size_t)h * HD + dim;
        typedef vsl_half halfn __attribute__((ext_vector_type(NF)));
        halfn hv, lv;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            vsl_half hi, lo;
            split_f16(x[f], hi, lo);
            hv[f] = hi;
            lv[f] = lo;
        }
        *reinterpret_cast<halfn*>(out + at) = hv;
        if (om == 1) *reinterpret_cast<halfn*>(out + qplane + at) = lv;
        if (om == 2) {
            uint8_t* lo8 = reinterpret_cast<uint8_t*>(out + qplane) + (size_t)my_s * qw + lo8_pos(h * HD + dim);
            if constexpr (NF == 4) {
                *reinterpret_cast<uint32_t*>(lo8) = lo8_code4(x[0] - (float)hv[0], x[1] - (float)hv[1], x[2] - (float)hv[2],
                                                              x[3] - (float)hv[3]);
            } else {
                *reinterpret_cast<uint16_t*>(lo8) =
                    (uint16_t)lo8_code4(x[0] - (float)hv[0], x[1] - (float)hv[1], 0.f, 0.f);
            }
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
    const uint32_t grid = (a.S + 31) / 32 * (a.n_q / GB);
    k_attn_prefill_kv4<HD, G, GB, QX2, KSPLIT, TK><<<grid, 64 * GB * KSPLIT, 0, s>>>(
        a.q, a.k, a.v, a.S, a.pos0, a.n_q, a.n_kv, a.cap, a.scale, a.out, a.om, a.win, a.n_glob, a.thr);
}

// As long as a CU holds every block of one head and 32 rows, those (k_attn_prefill_kv4_few). Past that up to four heads
// share a block and its expanded tiles, two waves a head (groups of a power of two; pairs or single heads of the others: a
// block's threads divide a tile's words), or, while that leaves CUs idle, two heads with four waves each on tiles of 128 keys:
// twice the blocks, half the tiles in a chain. Measured, split q unless said: blocks of several heads / of one, 8B shape
// (head_dim 128, 4 heads a group) 128 rows 9.8 / 9.1 us, 45 rows at 3000 51.5 / 30.4, 250 rows at 500 23.2 / 15.2, 300 rows at
// 1000 36.8 / 34.6, behind longer caches (traced) 45 rows at 12000 206 / 92, 128 at 30000 503 / 226, 250 at 30000
// 506 / 271; 400 rows 18.2 / 20.6, one plane 700 rows 23.0 / 29.2, 1B shape (64), one plane, 512 rows 10.8 / 13.3; four
// heads a block / two: 1B shape, one plane, 512 rows 12.7 / 10.8.
template <int HD, int G, bool QX2>
void launch_group(hipStream_t s, const Args& a) {
    constexpr int GB = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
    constexpr uint64_t kCUs = 256;  // MI355X compute units
    const uint64_t groups = (uint64_t)((a.S + 31) / 32) * a.n_kv;
    if (groups * G <= kCUs) {
        constexpr int W = 8;
        k_attn_prefill_kv4_few<HD, QX2, W><<<(a.S + 31) / 32 * a.n_q, W * 64, 0, s>>>(
            a.q, a.k, a.v, a.S, a.pos0, a.n_q, a.n_kv, a.cap, a.scale, a.out, a.om, a.win, a.n_glob, a.thr);
        return;
    }
    if constexpr (GB == 4) {
        if (groups * (G / 2) <= kCUs) {
            launch<HD, G, 2, QX2, 4, 128>(s, a);
            return;
        }
    }
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
    if ((uint64_t)n_q * hd > 0x7FFFFFFFull) return vsl_unsupported("%s: n_q=%u", fn, n_q);
    if (((uint64_t)S + 31) / 32 * n_q >= 1ull << 22) return vsl_unsupported("%s: %u rows in one call", fn, S);  // 2^30 lanes
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
