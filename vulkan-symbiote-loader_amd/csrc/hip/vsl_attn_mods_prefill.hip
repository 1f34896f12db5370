// vsl_attn_mods_prefill.hip -- prompt attention with capped scores, a distance bias and a range of keys for each row
// (vsl_attn_prefill_mods). No reference counterpart.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vsl_attn_mods.h"
#include "vsl_internal.h"

using namespace attn_mods;

namespace {

constexpr int kTiles = 4;   // query tiles of a block: 32 rows of one head each
constexpr int kShares = 2;  // waves of a query tile, each with one 32-key half of every key tile
constexpr int kTK = 64, kBufs = 2, kThreads = 64 * kTiles * kShares;

struct PrefillArgs {
    const vsl_half* q;
    const vsl_half* kc;
    const vsl_half* vc;
    uint32_t S, pos0, n_q, n_kv, cap, G, n_chunk;
    float to_u;    // scale / softcap, or scale * log2(e) without a cap
    float from_u;  // softcap * log2(e)
    float near;    // |q.k| up to which the polynomial is tanh (below 0: never)
    float poly[kTanhTerms];  // its coefficients, in q.k and times softcap * log2(e)
    int out_mode;  // 0 fp16, 1 hi / lo fp16 planes, 2 fp16 + fp8 planes
    const float* slopes;
    const uint32_t* ranges;
    vsl_half* out;
    float* part_o;   // where the keys are split over blocks: a query tile's sums as its wave holds them (part_tile)
    float* part_ml;  // its rows' references and weights
};

// row of D of a 32 x 32 product in register v
__device__ __forceinline__ int d_row(int v, int lane) { return (v >> 2) * 8 + (lane >> 5) * 4 + (v & 3); }

// o * inv (four consecutive dims of a head's row) as the output's type
template <int HD>
__device__ __forceinline__ void store4(const PrefillArgs& a, uint32_t s, uint32_t h, int dim, const float (&y)[4]) {
    const size_t qw = (size_t)a.n_q * HD, plane = (size_t)a.S * qw, at = (size_t)s * qw + (size_t)h * HD + dim;
    half4 hv, lv;
    if (a.out_mode == 2) {
        uint32_t lo8;
        split4_f16_f8(y[0], y[1], y[2], y[3], hv, lo8);
        *reinterpret_cast<half4*>(a.out + at) = hv;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(a.out + plane) + (size_t)s * qw + lo8_pos(h * HD + dim)) = lo8;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        vsl_half hi, lo;
        split_f16(y[i], hi, lo);
        hv[i] = hi;
        lv[i] = lo;
    }
    *reinterpret_cast<half4*>(a.out + at) = hv;
    if (a.out_mode == 1) *reinterpret_cast<half4*>(a.out + plane + at) = lv;
}

// A query tile's place in the partial sums, [n_chunk][row blocks][n_q]: 32 rows of references and weights, and of sums as
// [HD / 4 groups of four dims in pairs][64 lanes][4], so that a wave stores and loads whole lines. (By rows, every store of a
// wave went to 64 of them: 45 rows at 3001 23.3 us.)
__device__ __forceinline__ size_t part_tile(const PrefillArgs& a, uint32_t chunk, uint32_t rb, uint32_t h) {
    return ((size_t)chunk * ((a.S + 31) / 32) + rb) * a.n_q + h;
}

// keys [lo, hi) of row s
__device__ __forceinline__ void row_range(const PrefillArgs& a, uint32_t s, uint32_t& lo, uint32_t& hi) {
    lo = 0;
    hi = a.pos0 + s + 1;
    if (a.ranges) {
        const uint2 r = reinterpret_cast<const uint2*>(a.ranges)[s];
        lo = r.x;
        hi = min(r.y, a.pos0 + a.S);
        if (lo >= hi) lo = hi = 0;
    }
}

// The rows of a query tile over the keys k0 .. k1 - 1 without matrix products: a wave takes one row after the other, a lane a
// key for the scores and HD / 64 dims for the sums, and multiplies no masked key's V. (A call: within the kernel it would cost
// the tiles' loop 50 registers spilled.)
template <int HD, bool QX2, bool CAP>
__device__ __noinline__ void rows_one_by_one(const PrefillArgs& a, uint32_t rb, uint32_t h, uint32_t chunk, uint32_t k0, uint32_t k1) {
    constexpr int D = HD / 64;
    const uint32_t lane = threadIdx.x & 63, qw = a.n_q * HD, kvh = h / a.G;
    const vsl_half* Kb = a.kc + (size_t)kvh * a.cap * HD;
    const vsl_half* Vb = a.vc + (size_t)kvh * a.cap * HD;
    const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    for (uint32_t s = rb * 32; s < min(rb * 32 + 32, a.S); ++s) {
        uint32_t lo, hi;
        row_range(a, s, lo, hi);
        lo = max(lo, k0);
        hi = min(hi, k1);
        const vsl_half* q = a.q + (size_t)s * qw + (size_t)h * HD;
        float m = -INFINITY, l = 0.f, acc[D];
#pragma unroll
        for (int i = 0; i < D; ++i) acc[i] = 0.f;
        for (uint32_t kb = lo; kb < hi; kb += 64) {
            const uint32_t k = kb + lane;
            float sc = 0.f;
            if (k < hi) {
                for (int d = 0; d < HD; ++d) {
                    float x = (float)q[d];
                    if constexpr (QX2) x += (float)q[(size_t)a.S * qw + d];
                    sc = fmaf(x, (float)Kb[(size_t)k * HD + d], sc);
                }
            }
            sc *= a.to_u;
            if constexpr (CAP) sc = tanh_any(sc) * a.from_u;
            sc = fmaf(-slope, fabsf((float)((int)k - (int)(a.pos0 + s))), sc);
            if (k >= hi) sc = -INFINITY;
            const float mn = fmaxf(m, wave_max_dpp(sc)), ref = mn == -INFINITY ? 0.f : mn, corr = fast_exp2(m - ref);
            const float w = fast_exp2(sc - ref);
            l = fmaf(l, corr, wave_sum_dpp(w));
            m = mn;
#pragma unroll
            for (int i = 0; i < D; ++i) acc[i] *= corr;
            for (uint32_t j = 0; j < min(64u, hi - kb); ++j) {
                const float wj = __shfl(w, (int)j, 64);
#pragma unroll
                for (int i = 0; i < D; ++i) acc[i] = fmaf(wj, (float)Vb[(size_t)(kb + j) * HD + 64 * i + lane], acc[i]);
            }
        }
        if (m == -INFINITY && l != 0.f) m = 0.f;
        if (a.n_chunk > 1) {
            const size_t tile = part_tile(a, chunk, rb, h);
#pragma unroll
            for (int i = 0; i < D; ++i) {
                const uint32_t dim = 64 * i + lane;
                a.part_o[tile * 32 * HD + (dim / 8 * 64 + (dim & 4) * 8 + s % 32) * 4 + dim % 4] = acc[i];
            }
            if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + (tile * 32 + s % 32) * 2) = make_float2(m, l);
            continue;
        }
        // four consecutive dims in every fourth lane, for the output's types
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < D; ++i) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __shfl(acc[i], (int)((lane & ~3u) + j), 64) * inv;
            if ((lane & 3) == 0) store4<HD>(a, s, h, 64 * i + (int)lane, y);
        }
    }
}

// Planes: a split q has split probabilities (2^-22 of each is lost), as in attention without modifications. A caller who passes one
// plane has q in fp16 already: the probabilities are then one plane too, 2^-11 of each, for half the matrix work.
//
// Block: four query tiles (32 rows of one head) of one KV head, numbered row block by row block with the group's heads
// within; two waves each, a wave the one 32-key half of every 64-key tile. Key tiles go from the cache straight into LDS
// (two buffers of K and two of V), shared by the four query tiles. Per tile a wave takes S^T = K Q^T (its D: a lane has 16
// keys of one row) and turns the scores into probabilities, which are the operand of O^T += V^T P^T as they lie. The halves
// are joined through LDS at the end.
// Bound: the two products (4 head_dim flops a row and key, twice as many for a split q) and, for every score, a dozen vector
// instructions of cap, exponential and rounding; LDS, which each query tile reads anew, is as busy as the matrix cores. 2048 rows
// at 6144 of the 8B shape, split q, cap 30: 506 us whatever the output's type, 951 TFLOP/s in products where a large plain fp16
// product reaches 1084 on this card. Under the counters the clock is 2.05 GHz, the matrix cores are busy 44 % of the cycles and
// vector instructions are issued in 50 %; LDS has no bank conflicts. Single-plane q 350; without a cap 479; scores past 0.64 of the
// cap (tanh by its exponential) 630; a distance bias, whose tiles take the general way, 528, with the cap 595. With the
// probabilities in one plane, 424 there, slower were: the next tile's K in registers ahead of its product 451 to 470, products and
// vector code mixed by scheduling barriers 485.
// A row's keys are a range [lo, hi); tiles that lie within the ranges of all of a wave's rows take no masks, and tiles
// outside all of them are skipped. In the others a masked probability is 0; where V then holds an infinity or a NaN, whose
// product with 0 would reach the sums, the query tile's rows are computed again, one by one (rows_one_by_one).
template <int HD, bool QX2, bool CAP>
__global__ __launch_bounds__(kThreads, 2) void k_prefill_mods(PrefillArgs a) {
    constexpr int CPR = HD / 8, NCH = kTK * CPR / kThreads, QP = QX2 ? 2 : 1, ND = HD / 32;
    static_assert(NCH >= 1 && kTK * CPR % kThreads == 0, "a tile divides over the block");
    __shared__ __attribute__((aligned(256))) vsl_half s_tiles[2 * kBufs][kTK * HD];  // K's buffers, then V's
    vsl_half(*Ks)[kTK * HD] = s_tiles;
    vsl_half(*Vs)[kTK * HD] = s_tiles + kBufs;
    __shared__ __attribute__((aligned(16))) vsl_half s_q[kTiles][QP * 32 * HD];
    __shared__ uint32_t s_lo[kTiles * kShares], s_hi[kTiles * kShares];
    // (not in s_lo's place: where a chunk has no tiles, no barrier lies between the reads of s_lo and these flags)
    __shared__ uint32_t s_odd[kTiles * kShares];
    __shared__ float s_m[kTiles * kShares][64], s_l[kTiles * kShares][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // blocks in the order of their rows, the last (longest under the causal mask) first, KV heads next to each other
    const uint32_t n_rb = (a.S + 31) / 32, n_qt = n_rb * a.G, n_grp = (n_qt + kTiles - 1) / kTiles;
    const uint32_t kvh = blockIdx.x % a.n_kv, grp = n_grp - 1 - blockIdx.x / a.n_kv, chunk = blockIdx.y;
    const uint32_t qt = grp * kTiles + wave / kShares;
    const bool active = qt < n_qt;
    const int share = wave % kShares;
    const uint32_t rb = active ? qt / a.G : 0, h = kvh * a.G + (active ? qt % a.G : 0);
    const uint32_t my_s = rb * 32 + (lane & 31), row = min(my_s, a.S - 1);  // rows past S are those of row S - 1, not stored
    const uint32_t qw = a.n_q * HD;
    const size_t qplane = (size_t)a.S * qw;
    const uint32_t my_pos = a.pos0 + row;

    // this row's keys, the wave's (within some row's and within all rows') and the block's
    uint32_t lo, hi, some_lo, some_hi, all_lo, all_hi, blk_lo, blk_hi;
    row_range(a, row, lo, hi);
    if (!a.ranges) {
        some_lo = all_lo = blk_lo = 0;
        some_hi = active ? a.pos0 + min(a.S, rb * 32 + 32) : 0;
        all_hi = a.pos0 + rb * 32 + 1;
        blk_hi = a.pos0 + min(a.S, (min(grp * kTiles + kTiles, n_qt) - 1) / a.G * 32 + 32);
    } else {
        some_lo = all_lo = hi > lo ? lo : 0xFFFFFFFFu;
        some_hi = all_hi = hi;
#pragma unroll
        for (int o = 16; o; o >>= 1) {  // the two half waves hold the same rows
            some_lo = min(some_lo, (uint32_t)__shfl_xor((int)some_lo, o, 64));
            some_hi = max(some_hi, (uint32_t)__shfl_xor((int)some_hi, o, 64));
            all_lo = max(all_lo, (uint32_t)__shfl_xor((int)all_lo, o, 64));
            all_hi = min(all_hi, (uint32_t)__shfl_xor((int)all_hi, o, 64));
        }
        if (!active) {
            some_lo = 0xFFFFFFFFu;
            some_hi = 0;
        }
        some_lo = __builtin_amdgcn_readfirstlane(some_lo);
        some_hi = __builtin_amdgcn_readfirstlane(some_hi);
        all_lo = __builtin_amdgcn_readfirstlane(all_lo);
        all_hi = __builtin_amdgcn_readfirstlane(all_hi);
        if (lane == 0) {
            s_lo[wave] = some_lo;
            s_hi[wave] = some_hi;
        }
        __syncthreads();
        blk_lo = 0xFFFFFFFFu;
        blk_hi = 0;
#pragma unroll
        for (int w = 0; w < kTiles * kShares; ++w) {
            blk_lo = min(blk_lo, s_lo[w]);
            blk_hi = max(blk_hi, s_hi[w]);
        }
        blk_lo = __builtin_amdgcn_readfirstlane(blk_lo);
        blk_hi = __builtin_amdgcn_readfirstlane(blk_hi);
    }
    // the block's key tiles, or its chunk of them
    uint32_t t0 = 0, t1 = 0;
    if (blk_hi > blk_lo) {
        t0 = blk_lo / kTK;
        t1 = (blk_hi + kTK - 1) / kTK;
        const uint32_t n = t1 - t0, per = n / a.n_chunk, rest = n % a.n_chunk;
        t0 += chunk * per + min(chunk, rest);
        t1 = t0 + per + (chunk < rest ? 1 : 0);
    }

    const vsl_half* Kb = a.kc + (size_t)kvh * a.cap * HD;
    const vsl_half* Vb = a.vc + (size_t)kvh * a.cap * HD;
    // Tile copy: LDS chunk i * kThreads + tid holds row r, and of it the chunk whose swizzled place that is. Positions past
    // the block's keys read the last of them.
    uint32_t coff[NCH];
    int crow[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int P = i * kThreads + tid, r = P / CPR;
        crow[i] = r;
        coff[i] = (uint32_t)(swizzle<HD>(r, P % CPR) - r * HD);
    }
    auto issue = [&](const vsl_half* src, vsl_half* buf, uint32_t t) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            lds_load16(src + (size_t)min(t * kTK + crow[i], blk_hi - 1) * HD + coff[i], 0, buf + (i * kThreads + wave * 64) * 8);
    };

    // q's rows by way of LDS too, each wave half of its query tile's: a lane needs 16 bytes of its row at a time, and 32 rows'
    // lines for each such load kept a block for 4000 cycles (45 rows at 3001 21.6 -> 19.2 us). The first tiles' copies follow.
    constexpr int NQ = QP * CPR / 4;
    if (t1 > t0) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int at = (share * NQ + i) * 64, P = at + lane, r = P / CPR % 32;
            lds_load16(a.q + P / (32 * CPR) * qplane + (size_t)min(rb * 32 + r, a.S - 1) * qw + (size_t)h * HD + (swizzle<HD>(r, P % CPR) - r * HD), 0,
                       &s_q[wave / kShares][at * 8]);
        }
        issue(Kb, Ks[0], t0);
        issue(Kb, Ks[1], min(t0 + 1, t1 - 1));
        issue(Vb, Vs[0], t0);
    }
    half8 qf[QP][HD / 16];
    const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.f;
    float16v o[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] = 0.f;
    float m = -INFINITY, l = 0.f;

    // LDS byte addresses: the swizzle is an xor of the chunk, so all chunks that a lane reads of a row are its first one's
    // address xor a constant. (The address passes through an empty asm, or the compiler keeps all of them in registers.)
    typedef __attribute__((address_space(3))) const char* lds_ptr;
    constexpr int kTile = kTK * HD * 2;  // bytes
    static_assert(__alignof__(s_tiles) >= HD * 2, "an xor of the address is one of the chunk where rows start at multiples of their size");
    const uint32_t k_at = (uint32_t)(uintptr_t)(lds_ptr)&Ks[0][swizzle<HD>(share * 32 + (lane & 31), lane >> 5)];
    auto qk = [&](int buf, float16v& st) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < 16; ++v) st[v] = 0.f;
        half8 kf[HD / 16];
        uint32_t at = k_at + buf * kTile;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
            kf[c] = *reinterpret_cast<const __attribute__((address_space(3))) half8*>((lds_ptr)(uintptr_t)(at ^ (c * 32)));
#pragma unroll
        for (int c = 0; c < HD / 16; ++c)
#pragma unroll
            for (int p = 0; p < QP; ++p) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[c], qf[p][c], st, 0, 0, 0);
    };
    // the reference raised to scores of up to bm (log2 units), where that is far above it in some row
    auto raise = [&](float bm) __attribute__((always_inline)) {
        if (__builtin_amdgcn_ballot_w64(bm - m > kLazy + kRoom)) {  // m = -inf: any finite score raises it
            float a0, a1;
            lane_pair<32>(bm, a0, a1);
            const float mn = fmaxf(m, fmaxf(a0, a1) - kRoom);
            const float corr = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
            l *= corr;
#pragma unroll
            for (int t = 0; t < ND; ++t)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[t][v] *= corr;
            m = mn;
        }
    };
    auto largest = [&](const float16v& st) {
        float bm = st[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) bm = fmaxf(bm, st[v]);
        return bm;
    };
    auto largest_size = [&](const float16v& st) __attribute__((always_inline)) {
        float most = 0.f;
#pragma unroll
        for (int v = 0; v < 16; ++v) most = fmaxf(most, fabsf(st[v]));
        return most;
    };
    // two probabilities 2^x into their place in P^T; the row's sum takes them as they are multiplied
    auto put_probs = [&](int v, float x0, float x1, half8 (&pf)[QP][2]) __attribute__((always_inline)) {
        const half2v one = {(vsl_half)1.f, (vsl_half)1.f};
        const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
        const half2v hi2 = round2(p0, p1);
        pf[0][v >> 3][v & 7] = hi2[0];
        pf[0][v >> 3][(v & 7) + 1] = hi2[1];
        l = __builtin_amdgcn_fdot2(hi2, one, l, false);
        if constexpr (QX2) {
            const half2v lo2 = round2(p0 - (float)hi2[0], p1 - (float)hi2[1]);
            pf[QP - 1][v >> 3][v & 7] = lo2[0];
            pf[QP - 1][v >> 3][(v & 7) + 1] = lo2[1];
            l = __builtin_amdgcn_fdot2(lo2, one, l, false);
        }
    };
    // V^T operand of dims 32 tt .., keys 16 half ..: slots of P^T are the keys (v / 4) 8 + (lane / 32) 4 + v % 4, which the
    // transpose reads match: lane i of 16 addresses V[r0 + i / 4][d0 + 4 (i % 4) ..] and receives V[r0 + j][d0 + i] as value j
    const int gi = lane & 15, gdim = ((lane >> 4) & 1) * 16 + 4 * (gi & 3), grow = share * 32 + (lane >> 5) * 4 + (gi >> 2);
    const uint32_t v_at = (uint32_t)(uintptr_t)(lds_ptr)&Vs[0][swizzle<HD>(grow, gdim >> 3) + (gdim & 7)];
    auto v_frag = [&](uint32_t at, int tt, int half) {
        const int off = half * 16 * HD * 2;
        const auto* p0 = (const vsl_half*)((lds_ptr)(uintptr_t)(at ^ (tt * 64)) + off);
        const auto* p1 = (const vsl_half*)((lds_ptr)(uintptr_t)(at ^ (tt * 64) ^ (swizzle_bits<HD>(8) * 16)) + off + 8 * HD * 2);
        const half4 x0 = lds_read_tr16(p0), x1 = lds_read_tr16(p1);
        return half8{x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    };
    auto pv = [&](int buf, const half8 (&pf)[QP][2]) __attribute__((always_inline)) {
        uint32_t at = v_at + buf * kTile;
        asm volatile("" : "+v"(at));
#pragma unroll
        for (int tt = 0; tt < ND; ++tt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const half8 af = v_frag(at, tt, half);
#pragma unroll
                for (int p = 0; p < QP; ++p) o[tt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af, pf[p][half], o[tt], 0, 0, 0);
            }
    };
    // infinities and NaN in this wave's half of the tile's V
    uint32_t odd = 0;
    auto note_odd = [&](int buf) __attribute__((always_inline)) {
#pragma unroll 1
        for (int tt = 0; tt < ND; ++tt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const u32x4 w = __builtin_bit_cast(u32x4, v_frag(v_at + buf * kTile, tt, half));
                odd |= odd_halfs(w[0]) | odd_halfs(w[1]) | odd_halfs(w[2]) | odd_halfs(w[3]);
            }
        asm volatile("" ::: "memory");  // the products read V again: nothing of it is kept in registers here
    };
    const float to_u = a.to_u, from_u = a.from_u, near = a.near;
    auto poly = [&](float x) {  // x polynomial(x^2) = the capped score
        const float z = x * x;
        float p = a.poly[kTanhTerms - 1];
#pragma unroll
        for (int i = kTanhTerms - 2; i >= 0; --i) p = fmaf(p, z, a.poly[i]);
        return p;
    };

    // probabilities of tile t from its products: the short way where no mask or bias applies, the polynomial serves all its
    // scores and none, of either sign, raises the reference
    float16v st;
    half8 pf[QP][2];
    auto whole_of = [&](uint32_t t) { return t * kTK + share * 32 >= all_lo && t * kTK + share * 32 + 32 <= all_hi; };
    auto softmax = [&](uint32_t t) __attribute__((always_inline)) {
        const uint32_t k0 = t * kTK + share * 32;
        const bool whole = whole_of(t);
        bool plain = whole && !a.slopes;
        if (plain) {
            const float most = largest_size(st);
            plain = !__builtin_amdgcn_ballot_w64((CAP && !(most <= near)) || !(fabsf(most * (CAP ? poly(most) : to_u)) - m <= kLazy + kRoom));
        }
        if (plain) {
#pragma unroll
            for (int v = 0; v < 16; v += 2) {
                if constexpr (CAP) put_probs(v, fmaf(st[v], poly(st[v]), -m), fmaf(st[v + 1], poly(st[v + 1]), -m), pf);
                else put_probs(v, fmaf(st[v], to_u, -m), fmaf(st[v + 1], to_u, -m), pf);
            }
            return;
        }
        auto masked = [&](int v, float x) {
            x = fmaf(-slope, fabsf((float)((int)(k0 + d_row(v, lane)) - (int)my_pos)), x);
            return whole || k0 + d_row(v, lane) - lo < hi - lo ? x : -INFINITY;
        };
        if constexpr (!CAP) {
#pragma unroll
            for (int v = 0; v < 16; ++v) st[v] = masked(v, st[v] * to_u);
        } else {  // a wave's first tile comes here, its code fetched for the first time: what does not apply is branched over (45
                  // rows at 3001 25.8 -> 23.3 us; without a cap, where less is to skip, 512 packed rows 12.4 -> 13.2)
            if (__builtin_amdgcn_ballot_w64(!(largest_size(st) <= near))) {
#pragma unroll
                for (int v = 0; v < 16; ++v) st[v] = tanh_any(st[v] * to_u) * from_u;
            } else {
#pragma unroll
                for (int v = 0; v < 16; ++v) st[v] *= poly(st[v]);
            }
            if (!whole || a.slopes) {
#pragma unroll
                for (int v = 0; v < 16; ++v) st[v] = masked(v, st[v]);
            }
        }
        raise(largest(st));
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int v = 0; v < 16; v += 2) put_probs(v, st[v] - ref, st[v + 1] - ref, pf);
    };
    auto any_of = [&](uint32_t t) { return t * kTK + share * 32 < some_hi && t * kTK + share * 32 + 32 > some_lo; };

    // A wave turns by turns forms probabilities (of t) and multiplies (V of t, K of t + 1), with the block meeting after each.
    // The second wave of every SIMD (of the eight, the last four) runs one turn behind the first, so that one multiplies while
    // the other is on the vector unit: side by side they were on the same unit at the same time, 462 us instead of 442 for
    // 2048 rows at 6144. In the turn in which the first waves multiply for t, K of t + 2 and V of t + 1 are requested, by all
    // waves: their buffers were last read a turn before, by the late waves for t - 1. They are waited for at the end of the
    // next turn, and read in the one after that.
    const bool late = wave >= kTiles * kShares / 2;
    auto request = [&](uint32_t t, int buf) __attribute__((always_inline)) {
        issue(Kb, Ks[buf], min(t + 2, t1 - 1));
        issue(Vb, Vs[buf ^ 1], min(t + 1, t1 - 1));
    };
    auto step = [&](uint32_t t, int buf) __attribute__((always_inline)) {  // buf: of t
        const bool any = any_of(t);
        if (late) request(t, buf);
        if (any) softmax(t);
        if (!late) VSL_VMCNT_WAIT(0);
        __syncthreads();
        if (!late) request(t, buf);
        if (any) {
            if (!whole_of(t)) note_odd(buf);
            pv(buf, pf);
        }
        if (t + 1 < t1 && any_of(t + 1)) qk(buf ^ 1, st);
        if (late) VSL_VMCNT_WAIT(0);
        __syncthreads();
    };
    if (t1 > t0) {
        VSL_VMCNT_WAIT(0);
        __syncthreads();
        // Q^T as the B operand: lane holds row lane % 32, dims 16 c + 8 (lane / 32) ..
#pragma unroll
        for (int p = 0; p < QP; ++p)
#pragma unroll
            for (int c = 0; c < HD / 16; ++c)
                qf[p][c] = *reinterpret_cast<const half8*>(&s_q[wave / kShares][p * 32 * HD + swizzle<HD>(lane & 31, 2 * c + (lane >> 5))]);
        if (any_of(t0)) qk(0, st);
        __syncthreads();  // (K of t0 is overwritten in the first turn but one)
        if (late) __syncthreads();
        int buf = 0;
        for (uint32_t t = t0; t < t1; ++t, buf ^= 1) step(t, buf);
        if (!late) __syncthreads();
        VSL_VMCNT_WAIT(0);
        __syncthreads();  // the buffers are free
    }
    // a row's weights lie in two lanes
    {
        float a0, a1;
        lane_pair<32>(l, a0, a1);
        l = a0 + a1;
        if (m == -INFINITY && l != 0.f) m = 0.f;  // only NaN scores: keep the sum in the join
    }
    // the halves of each query tile joined: each wave takes half of the dims, and leaves the other half of its sums in the tile
    // buffers (every read and copy is over)
    const bool any_odd = __builtin_amdgcn_ballot_w64(odd != 0) != 0;
    constexpr int NJ = ND / 2, OSZ = NJ * 16 * 64;
    static_assert(kTiles * kShares * OSZ * 4 <= 2 * kBufs * kTK * HD * 2, "every query tile's sums in the tile buffers");
    const int w = wave / kShares;
    float* sums = reinterpret_cast<float*>(&s_tiles[0][0]) + (w * kShares) * OSZ;
    auto leave = [&](auto first) __attribute__((always_inline)) {  // tiles of dims first .. for the other wave
        float* x = sums + (share ^ 1) * OSZ;
#pragma unroll
        for (int t = 0; t < NJ; ++t)
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const float16v& from = o[decltype(first)::value + t];
                *reinterpret_cast<float4v*>(x + ((t * 4 + v / 4) * 64 + lane) * 4) = float4v{from[v], from[v + 1], from[v + 2], from[v + 3]};
            }
    };
    using std::integral_constant;
    if (share) leave(integral_constant<int, 0>());
    else leave(integral_constant<int, NJ>());
    s_m[wave][lane] = m;
    s_l[wave][lane] = l;
    if (lane == 0) s_odd[wave] = any_odd;
    __syncthreads();
    if (!active) return;
    if (s_odd[w * kShares] || s_odd[w * kShares + 1]) {
        if (share) return;
        // the arguments where the launch put them: the address of `a` would move them all to scratch memory
        const auto* args = reinterpret_cast<const PrefillArgs*>((const void*)__builtin_amdgcn_kernarg_segment_ptr());
        rows_one_by_one<HD, QX2, CAP>(*args, rb, h, chunk, t0 * kTK, t1 * kTK);
        return;
    }
    const float mb = s_m[wave ^ 1][lane], mm = fmaxf(m, mb), ref = mm == -INFINITY ? 0.f : mm;
    const float ca = fast_exp2(m - ref), cb = fast_exp2(mb - ref);
    l = l * ca + s_l[wave ^ 1][lane] * cb;
    m = mm;
    if (my_s >= a.S) return;
    auto finish = [&](auto first) __attribute__((always_inline)) {
        constexpr int F = decltype(first)::value;
        const float* x = sums + share * OSZ;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t tile = part_tile(a, chunk, rb, h);
#pragma unroll
        for (int t = 0; t < NJ; ++t)
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const float4v b = *reinterpret_cast<const float4v*>(x + ((t * 4 + v / 4) * 64 + lane) * 4);
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = o[F + t][v + i] * ca + b[i] * cb;
                if (a.n_chunk > 1) {  // dims 32 t + 2 v + 4 (lane / 32) ..
                    *reinterpret_cast<float4v*>(a.part_o + tile * 32 * HD + (((F + t) * 4 + v / 4) * 64 + lane) * 4) = float4v{y[0], y[1], y[2], y[3]};
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] *= inv;
                    store4<HD>(a, my_s, h, (F + t) * 32 + d_row(v, lane), y);
                }
            }
        if (a.n_chunk > 1 && F == 0 && lane < 32) *reinterpret_cast<float2*>(a.part_ml + (tile * 32 + lane) * 2) = make_float2(m, l);
    };
    if (share) finish(integral_constant<int, NJ>());
    else finish(integral_constant<int, 0>());
}

// The chunks' sums joined: a block 32 dims of a query tile, a wave 8 of them, its lanes as those that stored them.
template <int HD>
__global__ __launch_bounds__(256) void k_join_prefill(PrefillArgs a) {
    constexpr uint32_t ND = HD / 32;
    const uint32_t lane = threadIdx.x & 63, group = blockIdx.x % ND * 4 + threadIdx.x / 64;
    const uint32_t in_chunk = blockIdx.x / ND, h = in_chunk % a.n_q, s = in_chunk / a.n_q * 32 + (lane & 31);
    if (s >= a.S) return;
    const size_t n = (size_t)((a.S + 31) / 32) * a.n_q;
    float M = -INFINITY, L = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t c0 = 0; c0 < a.n_chunk; c0 += 8) {  // eight chunks' sums are requested at once
        float2 ml[8];
        float4v v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const size_t tile = min(c0 + j, a.n_chunk - 1) * n + in_chunk;
            ml[j] = *reinterpret_cast<const float2*>(a.part_ml + (tile * 32 + (lane & 31)) * 2);
            v[j] = *reinterpret_cast<const float4v*>(a.part_o + tile * 32 * HD + (group * 64 + lane) * 4);
        }
        float top = M;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, ml[j].x);
        const float ref = top == -INFINITY ? 0.f : top, old = fast_exp2(M - ref);
        M = top;
        L *= old;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] *= old;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = c0 + j < a.n_chunk ? fast_exp2(ml[j].x - ref) : 0.f;
            if (c0 + j < a.n_chunk) {
                L = fmaf(ml[j].y, f, L);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = fmaf(v[j][i], f, y[i]);
            }
        }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] *= inv;
    store4<HD>(a, s, h, (int)(group * 8 + lane / 32 * 4), y);
}

uint64_t blocks_of(uint32_t S, uint32_t n_q, uint32_t n_kv) {
    const uint64_t n_qt = ((uint64_t)S + 31) / 32 * (n_q / n_kv);
    return (n_qt + kTiles - 1) / kTiles * n_kv;
}

// Key chunks: as many as fill the CUs (45 rows at 3001 of the 8B shape 19.4 us, half as many 23.1; at 20000 59.6, half as many 98.7, up
// to two blocks a CU 66.8), none shorter than three tiles of the longest rows (45 rows at 3001 two tiles 19.4, four 20.7, six 23.1; 5
// rows at 2500 16.3, 19.0 and 22.7 against 18.2). Calls of less than 12 tiles run unsplit: 512 packed rows of the 1B shape 11.4,
// in two chunks 15.4; the rule goes by pos0 + S, not by what rows see, and 45 rows at 600 of the 8B shape would take 17.2 split
// instead of 28.
uint32_t chunks_of(uint32_t S, uint32_t pos0, uint32_t n_q, uint32_t n_kv) {
    const uint64_t blocks = blocks_of(S, n_q, n_kv), tiles = ((uint64_t)pos0 + S + kTK - 1) / kTK;
    if (blocks >= 256 || tiles < 12) return 1;
    return (uint32_t)std::min<uint64_t>({256 / blocks, tiles / 3, 32});
}

// A chunk's partial sums: whole query tiles. With at most 256 / blocks chunks, and a block for four query tiles at most, all of them
// together are VSL_ATTN_MODS_WS_MAX(hd) = 256 * 4 * 32 * (hd + 2) * 4 bytes or less, whatever the call.
uint64_t part_bytes(uint32_t S, uint32_t n_q, uint32_t hd) { return ((uint64_t)S + 31) / 32 * 32 * n_q * (hd + 2) * 4; }

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace

extern "C" uint64_t vsl_attn_prefill_mods_ws_bytes(uint32_t S, uint32_t pos0, uint32_t n_q, uint32_t n_kv, uint32_t hd) {
    if (S == 0 || n_kv == 0 || n_q == 0 || n_q % n_kv || (hd != 64 && hd != 128)) return 0;
    const uint64_t c = chunks_of(S, pos0, n_q, n_kv);
    return c > 1 ? c * part_bytes(S, n_q, hd) : 0;
}

extern "C" int vsl_attn_prefill_mods(const void* q, int q_dtype, const void* kcache, const void* vcache, uint32_t S,
                                     uint32_t pos0, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t cap, float scale,
                                     void* out, int out_dtype, const vsl_attn_mods* mods, void* workspace, uint64_t ws_bytes,
                                     void* stream) {
    const char* fn = "vsl_attn_prefill_mods";
    if (!q || !kcache || !vcache || !out) return vsl_invalid("%s: null pointer", fn);
    if (n_kv == 0 || n_q == 0 || n_q % n_kv) return vsl_invalid("%s: n_q=%u not a multiple of n_kv=%u", fn, n_q, n_kv);
    if ((q_dtype != VSL_DT_F16 && q_dtype != VSL_DT_F16X2) ||
        (out_dtype != VSL_DT_F16 && out_dtype != VSL_DT_F16X2 && out_dtype != VSL_DT_F16F8))
        return vsl_unsupported("%s: dtypes %d/%d", fn, q_dtype, out_dtype);
    if (hd != 64 && hd != 128) return vsl_unsupported("%s: head_dim %u (64 or 128)", fn, hd);
    const uint32_t G = n_q / n_kv;
    if (G > 8 || n_q > 65535) return vsl_unsupported("%s: GQA ratio %u (supported 1..8), %u heads", fn, G, n_q);
    if (cap > 0x7FFFFFFFu) return vsl_invalid("%s: capacity %u", fn, cap);
    if ((uint64_t)pos0 + S > cap) return vsl_capacity("%s: %u positions from %u exceed capacity %u", fn, S, pos0, cap);
    for (const void* p : {q, kcache, vcache, static_cast<const void*>(out), static_cast<const void*>(workspace)})
        if (!aligned_to(p, 16)) return vsl_invalid("%s: pointers must be 16-byte aligned", fn);
    const vsl_attn_mods none{};
    const vsl_attn_mods& md = mods ? *mods : none;
    if (!aligned_to(md.slopes, 4) || !aligned_to(md.ranges, 8)) return vsl_invalid("%s: misaligned pointer", fn);
    if (!softcap_ok(md.softcap, scale)) return vsl_invalid("%s: softcap %g with scale %g", fn, (double)md.softcap, (double)scale);
    if (S == 0) return VSL_OK;
    const uint64_t blocks = blocks_of(S, n_q, n_kv);
    if (blocks > 1u << 23 || (uint64_t)S * n_q > 1u << 26) return vsl_unsupported("%s: %u rows in one call", fn, S);
    const bool capped = md.softcap > 0.f;
    const uint32_t n_rb = (S + 31) / 32;
    uint32_t chunks = workspace ? chunks_of(S, pos0, n_q, n_kv) : 1;
    if (chunks > 1 && ws_bytes < chunks * part_bytes(S, n_q, hd)) chunks = 1;
    PrefillArgs a{};
    a.q = static_cast<const vsl_half*>(q);
    a.kc = static_cast<const vsl_half*>(kcache);
    a.vc = static_cast<const vsl_half*>(vcache);
    a.S = S;
    a.pos0 = pos0;
    a.n_q = n_q;
    a.n_kv = n_kv;
    a.cap = cap;
    a.G = G;
    a.n_chunk = chunks;
    a.to_u = capped ? scale / md.softcap : scale * kLog2e;
    a.from_u = md.softcap * kLog2e;
    // the polynomial in q.k itself, where its coefficients are normal numbers (at head_dim 128 caps of 4e-5 to 2200)
    if (capped) {
        bool normal = true;
        double f = (double)a.from_u * a.to_u;
        for (int i = 0; i < kTanhTerms; ++i, f *= (double)a.to_u * a.to_u) {
            a.poly[i] = (float)(kTanhPoly[i] * f);
            normal = normal && std::isnormal(a.poly[i]);
        }
        a.near = normal ? kTanhNear / std::fabs(a.to_u) : -1.f;
    }
    a.out_mode = out_dtype == VSL_DT_F16X2 ? 1 : out_dtype == VSL_DT_F16F8 ? 2 : 0;
    a.slopes = md.slopes;
    a.ranges = md.ranges;
    a.out = static_cast<vsl_half*>(out);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)chunks * n_rb * 32 * n_q * hd;
    const dim3 grid((uint32_t)blocks, chunks);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto hdc, auto x2, auto cc) {
        constexpr int HD = decltype(hdc)::value;
        k_prefill_mods<HD, decltype(x2)::value, decltype(cc)::value><<<grid, kThreads, 0, s>>>(a);
        if (chunks > 1) k_join_prefill<HD><<<n_rb * n_q * (HD / 32), 256, 0, s>>>(a);
    };
    using T = std::true_type;
    using F = std::false_type;
    auto pick = [&](auto hdc) {
        if (q_dtype == VSL_DT_F16) capped ? go(hdc, F{}, T{}) : go(hdc, F{}, F{});
        else capped ? go(hdc, T{}, T{}) : go(hdc, T{}, F{});
    };
    if (hd == 128) pick(std::integral_constant<int, 128>{});
    else pick(std::integral_constant<int, 64>{});
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}
