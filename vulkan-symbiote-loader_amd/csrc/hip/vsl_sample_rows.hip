// vsl_sample_rows.hip -- one token for each row of a batch of logits, by temperature, top-k, top-p and min-p, from given
// uniform numbers (vsl_sample_rows). No reference counterpart: the reference samples one vector by its host code
// (Utils.cpp:140-172) and reads no top_p (Common.h:59).
//
// With w_i = exp((l_i - max) / T), the kept tokens are a run of the order (logit descending, index ascending): every one
// of the three filters cuts that order somewhere, and the shortest run counts. So nothing is sorted: a cut is one 64-bit
// rank key (the float's order, then the inverted index), found by narrowing down, and the draw walks the kept tokens by
// index. Weights are summed in 64 bits (fixed point where atomics add them, so that no order of arrival matters): the
// token is that of exact sums but where u falls within about 1e-10 of a border.
//
// Three launches. k_rows_scan reads the row's slices (a block each) once and leaves, by what the row asks for,
//   GREEDY  the slice's maximum
//   TOPK    (k <= kLeanK) the slice's tokens that can be among the k largest: at least k of them lie at or above the k-th
//           largest of the block's per-thread maxima
//   SUM     (no cut but min-p) the maximum
//   HIST    (top-p, or a larger k) counts and weights by bins of 1/8 in l / T, whose grid is the same for every slice, so
//           that no slice has to know the row's maximum
// k_rows_cut ends GREEDY and TOPK rows in one block; for SUM its blocks sum the kept weights of the slices, for HIST each
// joins the slices' bins, which tells in which bins a cut falls, and collects its tokens of those. k_rows_draw, a block a
// row, finds the cuts among the collected tokens, the slice in which u falls and the token there. (The last
// block of the second kernel to arrive took the draw at first: its fences write the L2 caches back, and a pass over one row of
// 131072 took 66 us.) Where ties or ranges make a list too long, it narrows the cuts down over the whole row instead, which is
// slow, one block and several passes: more than 32768 tokens in the cut's bin (a flat row of 131072 by top-p 1.7 ms, 64 of them
// 1.8), |max l / T| above 16384 (1.0 ms), a top-k list of more than 256 tokens of a slice within 1/510 of its range (flat, k = 40:
// 32000 .24 ms, 131072 .9).
//
// What bounds it: for few rows the three launches and, within each, a chain of loads, sums over the block and code run for the
// first time: 1 x 32000 with k = 40 14.8 us, 1 x 131072 with top-p 32.5 (7 + 12 + 14). For many the two passes over the logits
// with 64-bit arithmetic per token, and a block a row in the draw: 64 x 131072 of mixed parameters 59 us (20.9 + 19.6 + 20.5;
// one read of the 33.6 MB takes about 7).
#include <float.h>

#include <cmath>

#include "vsl_device.h"
#include "vsl_internal.h"

namespace {

constexpr int kThreads = 256, kDrawThreads = 512;
constexpr uint32_t kMaxSlices = 128, kMaxEpt = 32;
constexpr uint32_t kMaxRowsV = kMaxSlices * kMaxEpt * kThreads;  // 2^20 tokens
// TOPK up to this k, HIST above. us, TOPK / HIST: k = 40 of 32000 15 / 22, of 131072 19 / 27, 64 rows of it 30 / 58; k = 128 25 / 23,
// 39 / 30, 47 / 59.
constexpr uint32_t kLeanK = 128;
constexpr uint32_t kLeanCap = 256;   // TOPK: tokens a slice's list holds
constexpr int kLeanRegs = 4, kDrawRegs = 4;  // tokens of a list that a thread holds
constexpr uint32_t kLeanList = kLeanRegs * kThreads, kListCap = 32768;  // tokens of a row's list: TOPK (in LDS), HIST
constexpr uint32_t kFinish = 256;    // keys that are left to a key a thread
constexpr uint32_t kBins = 512;     // of 1/8 in l / T; the last one takes all below e^-63.9 of the largest, never drawn
constexpr int kBinFrac = 36;        // weights in a bin: what they lie below its upper edge (up to .1175), in units of 2^-36
constexpr int kCountShift = 46;     // 8192 of them stay below 2^46; the count above
// Sums over bins are off by up to 2^-37 of their weights, and a little of the grid's rounding. Cuts and draws that meet a
// border exactly (equal logits: whole numbers of equal weights) are decided as exact sums are: a share is reached a little
// below it, a draw has passed a border a little above it.
constexpr double kBinNoise = 4e-11;
constexpr double kMaxTop = 16384.0;  // l / T up to which the grid's rounding (2^-39) is far below a weight's
// Fixed point of weights: so many units for a weight of 1 that the sum of those that take part stays below 2^62. For lists of a
// known length from that (k_rows_cut), else from their sum (unit_of): units for a row of 2^20 weights of 1 would leave 2^-42, and
// as many weights of that size 2^-22 of the sum.
constexpr double kFewOne = 0x1p54, kLeanOne = 0x1p52;

enum { MODE_GREEDY = 0, MODE_TOPK = 1, MODE_SUM = 2, MODE_HIST = 3 };

struct RowParams {
    int mode;
    uint32_t k;  // 1 .. V
    double inv_t, p, m;
    bool cut_p;
};

__device__ __forceinline__ RowParams row_params(const vsl_row_sampler& s, uint32_t V) {
    RowParams r;
    r.k = s.top_k == 0 || s.top_k > V ? V : s.top_k;
    r.cut_p = s.top_p < 1.f;  // NaN: no cut
    r.p = (double)s.top_p;
    r.m = s.min_p > 0.f ? (double)s.min_p : 0.0;
    r.inv_t = 1.0 / (double)s.temperature;
    if (!(s.temperature > 0.f) || r.k == 1 || s.top_p <= 0.f || s.min_p > 1.f) r.mode = MODE_GREEDY;
    else if (r.k <= kLeanK) r.mode = MODE_TOPK;
    else if (r.k == V && !r.cut_p) r.mode = MODE_SUM;
    else r.mode = MODE_HIST;
    return r;
}

struct SliceRec {
    uint64_t top;     // the largest rank key (0: nothing above -inf)
    uint32_t count;   // TOPK: tokens found (kLeanCap of them stored); HIST: bins up to the last one that holds a token
    float floor_v;    // TOPK: all tokens of the slice at or above this value are in its list, and there are k of them (-inf: all that can be drawn)
    double sum;       // weights kept for sure
};

struct RowRec {
    uint32_t kb, plo, phi, sure;  // HIST: the bin of the k-th token, those in which the top-p cut can fall, those kept whole
    uint32_t cut_k, k_left;       // whether k ends within its bin, and how many of that bin's tokens count
    double lo_total, hi_total;    // the first k tokens' weights, without and with the k-th's bin
    uint32_t whole;               // TOPK: the lists do not hold the tokens, or too many of the same size
    double cum_w[kBins];          // HIST: weights up to and with each bin
};

constexpr uint32_t kCounter = 64;
struct Work {
    SliceRec* rec;       // [rows][nsl]
    RowRec* row;         // [rows]
    uint32_t* counters;  // [rows][kCounter]: the row list's length, in lines of their own (side by side 1024 blocks' atomics
                         // met in two lines)
    uint64_t* lists;     // [rows][list_stride]
    uint64_t* hist;      // [rows][nsl][kBins]
    uint32_t list_stride;
};

// Logits as the samplers take them: NaN counts as -inf, +inf as the largest finite number.
__device__ __forceinline__ float clean(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
__device__ __forceinline__ float load_logit(const float* p, uint32_t i) { return clean(p[i]); }
__device__ __forceinline__ float load_logit(const vsl_half* p, uint32_t i) { return clean((float)p[i]); }

// Rank key: larger = earlier in the order (logit descending, index ascending); 0 for -inf.
__device__ __forceinline__ uint64_t rank_of(float v, uint32_t i) {
    if (v == -INFINITY) return 0;
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 as +0
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float value_of(uint64_t rank) {
    const uint32_t k = (uint32_t)(rank >> 32);
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ uint32_t index_of(uint64_t rank) { return ~(uint32_t)rank; }

// Waves: scans and reductions of 64-bit values by DPP lane moves (rows of 16 by shifts, then row 0 into 1, 2 into 3, and both
// into the upper half); lanes that a move does not reach read 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_move64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}
template <class T, class Op>
__device__ __forceinline__ T wave_steps(T v, Op op) {
    auto step = [&](auto ctrl, auto rows) {
        v = op(v, __builtin_bit_cast(T, dpp_move64<decltype(ctrl)::value, decltype(rows)::value>(__builtin_bit_cast(uint64_t, v))));
    };
    using std::integral_constant;
    step(integral_constant<int, 0x111>(), integral_constant<int, 0xF>());  // row_shr:1
    step(integral_constant<int, 0x112>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());
    step(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());  // row_bcast:15 into rows 1 and 3
    step(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());  // row_bcast:31 into rows 2 and 3
    return v;
}
template <class T>
__device__ __forceinline__ T last_lane(T v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {  // inclusive
    return wave_steps(v, [](T a, T b) { return a + b; });
}
template <class T>
__device__ __forceinline__ T wave_add(T v) { return last_lane(wave_scan(v)); }
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    return last_lane(wave_steps(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; }));
}
__device__ __forceinline__ uint64_t wave_or64(uint64_t v) {
    return last_lane(wave_steps(v, [](uint64_t a, uint64_t b) { return a | b; }));
}

struct Keyed {
    uint64_t key, weight;
};
struct Shared {
    uint64_t red[2 * kDrawThreads / 64];
    uint64_t digits[256];
    uint32_t counts[256];
    __attribute__((aligned(16))) Keyed keyed[kFinish];
    uint64_t sel_key, sel_left;
    uint32_t sel_count, n;
};

// Block-wide sums, maxima and scans of 64-bit values, every thread ending with the result. All threads call.
template <int NT, class T>
__device__ __forceinline__ T block_add(Shared& sh, T v) {
    v = wave_add(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = __builtin_bit_cast(uint64_t, v);
    __syncthreads();
    T s = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += __builtin_bit_cast(T, sh.red[w]);
    return s;
}
// Two maxima at once.
template <int NT>
__device__ __forceinline__ void block_max2(Shared& sh, uint64_t& a, uint64_t& b) {
    a = wave_max64(a);
    b = wave_max64(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        sh.red[threadIdx.x >> 6] = a;
        sh.red[NT / 64 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        a = sh.red[w] > a ? sh.red[w] : a;
        b = sh.red[NT / 64 + w] > b ? sh.red[NT / 64 + w] : b;
    }
}
// Inclusive scan; `total`: the sum over the block.
template <int NT, class T>
__device__ __forceinline__ T block_scan(Shared& sh, T v, T& total) {
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.red[threadIdx.x >> 6] = __builtin_bit_cast(uint64_t, v);
    __syncthreads();
    const int wave = threadIdx.x >> 6;
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const T x = __builtin_bit_cast(T, sh.red[w]);
        if (w < wave) before += x;
        total += x;
    }
    return before + v;
}

// The last key of the shortest run of keys, in descending order, whose measures reach `target` (the smallest key of all if
// they do not). visit(f) calls f(rank, weight) for each of the thread's elements, weight() being its weight;
// map(rank, weight, key, measure) is false where one takes no part; measures are integers, keys differ and are not 0. `n` bounds the elements that take part. Narrowed down by
// digits of 8 bits, from the highest bit in which keys differ, until kFinish keys are left, whose threads sum up the
// measures before their own. All threads call; 0 without elements.
template <int NT, class Visit, class Map>
__device__ __forceinline__ uint64_t select_key(Shared& sh, uint32_t n, uint64_t target, Visit visit, Map map) {
    const uint32_t t = threadIdx.x;
    uint64_t prefix = 0, mask = 0;
    if (n > kFinish) {
        uint64_t all_or = 0, none_or = 0;  // bits that some key has, that some key lacks
        visit([&](uint64_t rank, auto weight) {
            uint64_t key, w;
            if (map(rank, weight, key, w)) {
                all_or |= key;
                none_or |= ~key;
            }
        });
        all_or = wave_or64(all_or);
        none_or = wave_or64(none_or);
        __syncthreads();
        if ((t & 63) == 0) {
            sh.red[t >> 6] = all_or;
            sh.red[NT / 64 + (t >> 6)] = none_or;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            all_or |= sh.red[w];
            none_or |= sh.red[NT / 64 + w];
        }
        const uint64_t diff = all_or & none_or;
        if (diff == 0) return all_or;              // one key, or none
        const int top = 64 - __builtin_clzll(diff);  // bits 0 .. top - 1 differ
        int shift = top > 8 ? top - 8 : 0;
        if (top < 64) {
            mask = ~0ull << top;
            prefix = all_or & mask;
        }
        for (;;) {
            __syncthreads();
            if (t < 256) {
                sh.digits[t] = 0;
                sh.counts[t] = 0;
            }
            __syncthreads();
            visit([&](uint64_t rank, auto weight) {
                uint64_t key, w;
                if (map(rank, weight, key, w) && (key & mask) == prefix) {
                    const uint32_t d = (uint32_t)(key >> shift) & 255u;
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits[d]), (unsigned long long)w);
                    atomicAdd(&sh.counts[d], 1u);
                }
            });
            __syncthreads();
            if (t < 64) {  // lane t: digits 255 - 4 t .. 252 - 4 t, descending
                uint64_t d4[4], s = 0;
                uint32_t c4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    d4[j] = sh.digits[255 - 4 * t - j];
                    c4[j] = sh.counts[255 - 4 * t - j];
                    s += d4[j];
                }
                uint64_t run = wave_scan(s) - s, left = 0, last_left = 0;
                uint32_t hit = 0, last = 0, hit_n = 0, last_n = 0;  // digit + 1
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (c4[j]) {
                        last = 256 - 4 * t - j;
                        last_n = c4[j];
                        last_left = target > run ? target - run : 0;
                        if (!hit && run + d4[j] >= target) {
                            hit = last;
                            hit_n = last_n;
                            left = last_left;
                        }
                    }
                    run += d4[j];
                }
                const uint64_t reach = __builtin_amdgcn_ballot_w64(hit != 0), some = __builtin_amdgcn_ballot_w64(last != 0);
                // the first digit that reaches the target; where none does, the smallest
                const int who = reach ? __builtin_ctzll(reach) : 63 - __builtin_clzll(some | 1);
                if ((int)t == who) {
                    sh.sel_key = (reach ? hit : last) - 1;
                    sh.sel_left = reach ? left : last_left;
                    sh.sel_count = reach ? hit_n : last_n;
                }
            }
            __syncthreads();
            prefix |= sh.sel_key << shift;
            mask |= 255ull << shift;
            target = sh.sel_left;
            if (sh.sel_count <= kFinish || shift == 0) break;
            shift = shift > 8 ? shift - 8 : 0;
        }
    }
    __syncthreads();
    if (t < kFinish) sh.keyed[t] = Keyed{0, 0};
    if (t == 0) {
        sh.n = 0;
        sh.sel_key = 0;
        sh.sel_left = 0;
    }
    __syncthreads();
    visit([&](uint64_t rank, auto weight) {
        uint64_t key, w;
        if (map(rank, weight, key, w) && (key & mask) == prefix) {
            const uint32_t at = atomicAdd(&sh.n, 1u);
            if (at < kFinish) sh.keyed[at] = Keyed{key, w};
        }
    });
    __syncthreads();
    const uint32_t m = min(sh.n, kFinish);
    if (t < m) {
        const Keyed mine = sh.keyed[t];
        uint64_t before = 0;
        bool least = true;
        for (uint32_t j0 = 0; j0 < m; j0 += 8) {
            Keyed x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = sh.keyed[j0 + j];  // zeros behind the last
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                before += x[j].key > mine.key ? x[j].weight : 0;
                least &= x[j].key == 0 || x[j].key >= mine.key;
            }
        }
        if (before < target && before + mine.weight >= target) sh.sel_key = mine.key;
        if (least) sh.sel_left = mine.key;
    }
    __syncthreads();
    return sh.sel_key ? sh.sel_key : sh.sel_left;
}

struct RowOut {
    uint32_t* token;
    float* prob;
};
__device__ __forceinline__ void put(const RowOut& o, uint32_t token, double prob) {
    *o.token = token;
    if (o.prob) *o.prob = (float)prob;
}

__device__ __forceinline__ double weight_of(float v, double vmax, double inv_t) { return exp(((double)v - vmax) * inv_t); }

// A weight in units: none above 0 counts as 0, so that u = 0 gives the first kept token however small its weight.
__device__ __forceinline__ uint64_t units(double w, double one) {
    const uint64_t n = (uint64_t)(w * one + 0.5);
    return n || !(w > 0.0) ? n : 1;
}
// Units for weights whose sum is `sum`, about 1 or above: the power of two that makes it 2^61 to 2^62. 2^20 roundings are 2^-41 of it,
// and as much of the sum of any first ones in descending order, each of which is no smaller than the others.
__device__ __forceinline__ double unit_of(double sum) {
    const uint64_t e = __builtin_bit_cast(uint64_t, sum) >> 52;  // 1023 + its exponent
    return __builtin_bit_cast(double, (2 * 1023 + 61 - e) << 52);
}

// The draw over elements (visit and n as for select_key) that hold every token of the first k: the three cuts, then the index
// at which the running sum passes u. one: units of a weight of 1.
template <int NT, class Visit>
__device__ __forceinline__ void draw_exact(Shared& sh, uint32_t n, const RowParams& rp, double vmax, double u, const RowOut& out,
                                           bool cut_k, double one, Visit visit) {
    uint64_t low = 1;  // the smallest kept rank key
    if (cut_k) low = select_key<NT>(sh, n, rp.k, visit, [&](uint64_t rank, auto, uint64_t& key, uint64_t& w) {
        key = rank;
        w = 1;
        return true;
    });
    if (rp.cut_p) {
        uint64_t s = 0;
        visit([&](uint64_t rank, auto weight) { s += rank >= low ? units(weight(), one) : 0; });
        const uint64_t target = (uint64_t)ceil((double)block_add<NT>(sh, s) * rp.p);
        low = select_key<NT>(sh, n, target, visit, [&](uint64_t rank, auto weight, uint64_t& key, uint64_t& w) {
            key = rank;
            w = rank >= low ? units(weight(), one) : 0;
            return rank >= low;
        });
    }
    // min-p: the weight itself decides
    auto heavy = [&](uint64_t rank) { return weight_of(value_of(rank), vmax, rp.inv_t) >= rp.m; };
    uint64_t s = 0;
    visit([&](uint64_t rank, auto weight) { s += rank >= low && heavy(rank) ? units(weight(), one) : 0; });
    const uint64_t total = block_add<NT>(sh, s);
    uint64_t target = (uint64_t)((double)total * u) + 1;
    if (target > total) target = total;
    const uint64_t at = select_key<NT>(sh, n, target, visit, [&](uint64_t rank, auto weight, uint64_t& key, uint64_t& w) {
        if (rank < low || !heavy(rank)) return false;
        w = units(weight(), one);
        key = (rank & 0xFFFFFFFFull) + 1;  // the inverted index: ascending indices are descending keys (+ 1: not 0)
        return w != 0;
    });
    const uint32_t idx = ~(uint32_t)(at - 1);
    visit([&](uint64_t rank, auto weight) {
        if (index_of(rank) == idx) put(out, idx, weight() * one / (double)total);
    });
}

// The same for at most a token a thread of k_rows_cut, list[0 .. n - 1]: put into their order by counting, so that each cut
// is a number of tokens and the kept ones are the smallest of the three. 45 tokens (k = 40 of 32000) 14.8 us by draw_exact.
__device__ __forceinline__ void draw_few(Shared& sh, uint64_t* list, uint32_t n, const RowParams& rp, double vmax, double u,
                                         const RowOut& out) {
    const uint32_t t = threadIdx.x;
    const uint64_t mine = t < n ? list[t] : 0;
    if (t >= n && t < ((n + 15) & ~15u)) list[t] = 0;  // up to a whole batch
    const double w = weight_of(mine ? value_of(mine) : (float)vmax, vmax, rp.inv_t);
    const bool heavy = w >= rp.m;
    const uint64_t fixed = units(w, kFewOne);
    __syncthreads();
    uint32_t rank = 0;
    for (uint32_t j0 = 0; j0 < n; j0 += 16) {
        uint64_t x[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = list[j0 + j];
#pragma unroll
        for (int j = 0; j < 16; ++j) rank += x[j] > mine;
    }
    // by rank: inverted index + 1 and weight; whether the weight is below min-p in the key's top bit
    if (t < n) sh.keyed[rank] = Keyed{((mine & 0xFFFFFFFFull) + 1) | (heavy ? 0 : 1ull << 63), fixed};
    __syncthreads();
    const Keyed k = t < n ? sh.keyed[t] : Keyed{0, 0};
    const bool first = t < min(n, rp.k);
    uint64_t total;
    const uint64_t incl = block_scan<kThreads>(sh, first ? k.weight : 0, total), before = incl - k.weight;
    const uint64_t target_p = rp.cut_p ? (uint64_t)ceil((double)total * rp.p) : ~0ull;
    const bool keep = first && (t == 0 || (before < target_p && !(k.key >> 63)));
    // the kept ones are the ranks below the first that is not
    const uint64_t m64 = __builtin_amdgcn_ballot_w64(keep);
    if ((t & 63) == 0) sh.counts[t >> 6] = (uint32_t)__builtin_popcountll(m64);
    __syncthreads();
    uint32_t kept = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) kept += sh.counts[i];
    if (t == kept - 1) sh.sel_left = incl;
    if (t >= kept && t < ((kept + 7) & ~7u) && t < kFinish) sh.keyed[t] = Keyed{0, 0};
    __syncthreads();
    const uint64_t sum = sh.sel_left;
    if (t < kept) {
        uint64_t target = (uint64_t)((double)sum * u);
        if (target >= sum) target = sum - 1;
        const uint64_t key = k.key & ~(1ull << 63);
        uint64_t below = 0;  // weights of lower indices
        for (uint32_t j0 = 0; j0 < kept; j0 += 8) {
            Keyed x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = sh.keyed[j0 + j];
#pragma unroll
            for (int j = 0; j < 8; ++j) below += (x[j].key & ~(1ull << 63)) > key ? x[j].weight : 0;
        }
        if (below <= target && below + k.weight > target) sh.sel_key = key;
    }
    __syncthreads();
    if (t < n && (mine & 0xFFFFFFFFull) + 1 == sh.sel_key) put(out, index_of(mine), w * kFewOne / (double)sum);
}

// The smallest value that can be drawn beside one of vmax: 64 temperatures below it weights are 2^-92. Top-k lists leave out what
// lies further down, or a mask of finite values (-1e9, the type's lowest) would count among the k largest where fewer are allowed,
// fill the lists and send the row to the draw over the whole row: 1 x 32000 with 20 allowed 567 us,
// 30 now (slices of masked tokens alone still list theirs), 11 with -infinity; with 1000 allowed 15 either way.
__device__ __forceinline__ float least_drawn(float vmax, float temperature) {
    return (float)((double)vmax - 64.0 * (double)temperature);
}

// Bin of a value on the grid that all slices share: floor(8 l / T), as a double (exact to 2^53, and monotone above).
__device__ __forceinline__ double bin_of(float v, double inv_t) { return floor((double)v * inv_t * 8.0); }
__device__ __forceinline__ uint32_t bin_below(double top_bin, double bin) { return (uint32_t)fmin(top_bin - bin, (double)(kBins - 1)); }
// 1 - exp(y) for -1/8 <= y <= 0, to 2^-45 (the series' first eight terms).
__device__ __forceinline__ double one_less_exp(double y) {
    double p = 1.0 / 40320.0;
    p = fma(p, y, 1.0 / 5040.0);
    p = fma(p, y, 1.0 / 720.0);
    p = fma(p, y, 1.0 / 120.0);
    p = fma(p, y, 1.0 / 24.0);
    p = fma(p, y, 1.0 / 6.0);
    p = fma(p, y, 0.5);
    p = fma(p, y, 1.0);
    return -p * y;
}

// Values between vmax and vmin in kBins - 1 bins (NaN, of an infinite range, and what lies below: the last one).
struct ValueBins {
    float vmax, step;
    __device__ ValueBins(float hi, float lo) : vmax(hi), step(hi - lo > 0.f ? (float)(kBins - 2) / (hi - lo) : 0.f) {}
    __device__ uint32_t operator()(float x) const {
        const float b = (vmax - x) * step;
        return b < (float)(kBins - 1) ? (uint32_t)b : kBins - 1;
    }
};
// The bin of counts that holds the k-th value, to *cut (unchanged where there are fewer); the first wave calls.
__device__ __forceinline__ void find_kth(const uint32_t* count, uint32_t k, uint32_t* cut) {
    constexpr int N = kBins / 64;
    const uint32_t t = threadIdx.x;
    uint32_t c[N];
    uint64_t s = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        c[j] = count[t * N + j];
        s += c[j];
    }
    uint64_t run = wave_scan(s) - s;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (run < k && run + c[j] >= k) *cut = t * N + j;
        run += c[j];
    }
}

template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void k_rows_scan(const T* __restrict__ logits, uint32_t V, uint64_t stride,
                                                        const vsl_row_sampler* __restrict__ params, Work ws) {
    __shared__ Shared sh;
    __shared__ uint64_t s_hist[kBins];
    __shared__ uint32_t s_n, s_low;
    const uint32_t row = blockIdx.y, slice = blockIdx.x, nsl = gridDim.x, t = threadIdx.x;
    const T* l = logits + (size_t)row * stride;
    const uint32_t first = slice * (EPT * kThreads);
    float v[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const uint32_t e = first + i * kThreads + t;
        v[i] = e < V ? load_logit(l, e) : -INFINITY;
    }
    const vsl_row_sampler ps = params[row];
    const RowParams rp = row_params(ps, V);
    if (slice == 0 && t == 0) ws.counters[row * kCounter] = 0;
#pragma unroll
    for (uint32_t b = 0; b < kBins; b += kThreads) s_hist[b + t] = 0;
    if (t == 0) {
        s_n = 0;
        s_low = 0xFFFFFFFFu;
        sh.sel_count = kBins - 1;
    }
    float mx = v[0];
    int arg = 0;
#pragma unroll
    for (int i = 1; i < EPT; ++i)
        if (v[i] > mx) {
            mx = v[i];
            arg = i;
        }
    const uint64_t best = rank_of(mx, first + arg * kThreads + t);
    uint64_t top = best, low_key = best ? ~(best | 0xFFFFFFFFull) : 0;  // the smallest of the threads' maxima, inverted
    block_max2<kThreads>(sh, top, low_key);
    SliceRec* rec = ws.rec + (size_t)row * nsl + slice;
    if (t == 0) rec->top = top;
    if (rp.mode == MODE_GREEDY || rp.mode == MODE_SUM) return;
    if (rp.mode == MODE_TOPK) {
        // threads' maxima in bins between their largest and their smallest: the bin of the k-th bounds the k-th token
        const float hi = top ? value_of(top) : 0.f, least = least_drawn(hi, ps.temperature);
        const ValueBins bin(hi, top ? fmaxf(value_of(~low_key), least) : 0.f);
        uint32_t* count = reinterpret_cast<uint32_t*>(s_hist);
        if (best && mx >= least) atomicAdd(&count[bin(mx)], 1u);
        __syncthreads();
        if (t < 64) find_kth(count, rp.k, &sh.sel_count);
        __syncthreads();
        const uint32_t cut = sh.sel_count;  // the last bin: fewer than k threads hold a token
        uint64_t* list = ws.lists + (size_t)row * ws.list_stride + (size_t)slice * kLeanCap;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            if (v[i] == -INFINITY || v[i] < least || bin(v[i]) > cut) continue;
            const uint32_t at = atomicAdd(&s_n, 1u);
            const uint64_t r = rank_of(v[i], first + i * kThreads + t);
            if (at < kLeanCap) list[at] = r;
            atomicMin(&s_low, (uint32_t)(r >> 32));
        }
        __syncthreads();
        // the list's smallest value: with k tokens in it, no token below that value is among the row's k largest
        if (t == 0) {
            rec->count = s_n;
            rec->floor_v = s_n >= rp.k ? value_of((uint64_t)s_low << 32) : -INFINITY;
        }
        return;
    }
    const double top_bin = top ? bin_of(value_of(top), rp.inv_t) : 0.0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        if (v[i] == -INFINITY) continue;
        const double x = (double)v[i] * rp.inv_t, b = floor(x * 8.0);
        const uint32_t r = bin_below(top_bin, b);
        // what the weight lies below its bin's upper edge, 0 .. 1 - exp(-1/8), in units of 2^-36: the mantissa behind 2^16
        const double d = one_less_exp(x - (b + 1.0) * 0.125) + 0x1p16;
        if (r < kBins - 1)
            atomicAdd(reinterpret_cast<unsigned long long*>(&s_hist[r]),
                      __builtin_bit_cast(unsigned long long, d) + ((1ull << kCountShift) - __builtin_bit_cast(unsigned long long, 0x1p16)));
    }
    __syncthreads();
    uint64_t* h = ws.hist + ((size_t)row * nsl + slice) * kBins;
    uint64_t used = 0, unused = 0;
#pragma unroll
    for (uint32_t b = 0; b < kBins; b += kThreads) {
        const uint64_t x = s_hist[b + t];
        h[b + t] = x;  // the last one is 0: what lies outside the bins is read from there
        if (x) used = b + t + 1;
    }
    block_max2<kThreads>(sh, used, unused);
    if (t == 0) rec->count = (uint32_t)used;
}

template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void k_rows_cut(const T* __restrict__ logits, uint32_t V, uint64_t stride,
                                                       const vsl_row_sampler* __restrict__ params, const float* __restrict__ us,
                                                       Work ws, uint32_t* __restrict__ tokens, float* __restrict__ probs) {
    constexpr int NT = kThreads;
    __shared__ Shared sh;
    __shared__ uint64_t s_list[kLeanList];
    __shared__ double s_cum_w[kBins], s_edge[kBins];
    __shared__ uint32_t s_cum_n[kBins];
    __shared__ uint32_t s_count[kMaxSlices], s_off[kMaxSlices], s_n, s_plo, s_phi, s_kb, s_base;
    const uint32_t row = blockIdx.y, slice = blockIdx.x, nsl = gridDim.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    SliceRec* rec = ws.rec + (size_t)row * nsl;
    // requested together: parameters, u and the slices' records
    const vsl_row_sampler ps = params[row];
    const float uf = us[row];
    uint64_t my_top = 0, top, bound = 0;
    uint32_t my_count = 0;
    float my_floor = -INFINITY;
    if (t < nsl) {
        my_top = rec[t].top;
        my_count = rec[t].count;
        my_floor = rec[t].floor_v;
    }
    const RowParams rp = row_params(ps, V);
    const double u = uf > 0.f ? fmin((double)uf, 1.0 - 0x1p-24) : 0.0;  // NaN and below 0: 0; 1 and above: the float below 1
    if (rp.mode <= MODE_TOPK && slice != 0) return;
    const T* l = logits + (size_t)row * stride;
    const uint32_t first = slice * (EPT * kThreads);
    float v[EPT];
    if (rp.mode >= MODE_SUM) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const uint32_t e = first + i * kThreads + t;
            v[i] = e < V ? load_logit(l, e) : -INFINITY;
        }
    }
    const RowOut out{tokens + row, probs ? probs + row : nullptr};
    // (count and floor_v are this call's in the modes that use them)
    if (rp.mode == MODE_TOPK) bound = rank_of(my_floor, 0xFFFFFFFFu);  // the smallest rank of that value
    if (t < kMaxSlices) s_count[t] = my_count;
    if (t == 0) {
        s_n = 0;
        s_kb = s_plo = s_phi = kBins - 1;
    }
    top = my_top;
    block_max2<NT>(sh, top, bound);
    if (top == 0) {  // nothing above -inf
        if (slice == 0 && t == 0) put(out, 0, 0.0);
        return;
    }
    if (rp.mode == MODE_GREEDY) {
        if (t == 0) put(out, index_of(top), 1.0);
        return;
    }
    const double vmax = (double)value_of(top);

    if (rp.mode == MODE_TOPK) {
        // the slices' tokens at or above the highest of their bounds, and of what can be drawn
        const uint64_t drawn = rank_of(least_drawn((float)vmax, ps.temperature), 0xFFFFFFFFu);
        bound = drawn > bound ? drawn : bound;
        const uint64_t* lists = ws.lists + (size_t)row * ws.list_stride;
        auto each = [&](auto f) {
            auto take = [&](uint64_t r) {
                if (r >= bound && r != 0) f(r);
            };
            for (uint32_t s0 = wave; s0 < nsl; s0 += 4 * (NT / 64)) {  // four slices' first 64 entries at a time
                uint64_t r[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t s = s0 + j * (NT / 64);
                    r[j] = s < nsl && lane < s_count[s] ? lists[(size_t)s * kLeanCap + lane] : 0;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t s = s0 + j * (NT / 64);
                    take(r[j]);
                    if (s < nsl)
                        for (uint32_t i = 64 + lane; i < min(s_count[s], kLeanCap); i += 64) take(lists[(size_t)s * kLeanCap + i]);
                }
            }
        };
        each([&](uint64_t r) {
            const uint32_t at = atomicAdd(&s_n, 1u);
            if (at < kLeanList) s_list[at] = r;
        });
        const bool over = __syncthreads_or(my_count > kLeanCap && my_top >= bound);
        const uint32_t n = s_n;
        // each slice's k-th bounds them: of k = 40 from 16 slices 490 are left, from 32 slices 1000, so they are binned once more; what
        // s_list does not hold is read again for that (16 x 131072 with k = 40 took 741 us when it sent a row to the draw over the
        // whole row, 1 x 32000 with k = 100 211)
        auto listed = [&](auto f) {
            if (n > kLeanList) return each(f);
            for (uint32_t i = t; i < n; i += NT) f(s_list[i]);
        };
        uint32_t m = n;
        uint64_t* few = s_list;
        if (n > rp.k && n > 64 && !over) {
            const ValueBins bin((float)vmax, bound ? value_of(bound) : (float)vmax);
            few = reinterpret_cast<uint64_t*>(s_cum_w);
#pragma unroll
            for (uint32_t b = 0; b < kBins; b += NT) s_cum_n[b + t] = 0;
            if (t == 0) {
                sh.sel_count = kBins - 1;
                sh.n = 0;
            }
            __syncthreads();
            listed([&](uint64_t x) { atomicAdd(&s_cum_n[bin(value_of(x))], 1u); });
            __syncthreads();
            if (t < 64) find_kth(s_cum_n, rp.k, &sh.sel_count);
            __syncthreads();
            const uint32_t cut = sh.sel_count;
            listed([&](uint64_t x) {
                if (bin(value_of(x)) > cut) return;
                const uint32_t at = atomicAdd(&sh.n, 1u);
                if (at < kThreads) few[at] = x;
            });
            __syncthreads();
            m = sh.n;
        }
        const bool whole = over || (m > kThreads && n > kLeanList);
        if (t == 0) ws.row[row].whole = whole;
        if (whole) return;
        if (m <= kThreads) {
            draw_few(sh, few, m, rp, vmax, u, out);
            return;
        }
        uint64_t r[kLeanRegs];
#pragma unroll
        for (int i = 0; i < kLeanRegs; ++i) r[i] = i * NT + t < n ? s_list[i * NT + t] : 0;
        draw_exact<NT>(sh, n, rp, vmax, u, out, n > rp.k, kLeanOne, [&](auto f) {
#pragma unroll
            for (int i = 0; i < kLeanRegs; ++i)
                if (r[i]) f(r[i], [&] { return weight_of(value_of(r[i]), vmax, rp.inv_t); });
        });
        return;
    }

    if (rp.mode == MODE_SUM) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const double w = v[i] == -INFINITY ? 0.0 : weight_of(v[i], vmax, rp.inv_t);
            if (w >= rp.m) sum += w;
        }
        sum = block_add<NT>(sh, sum);
        if (t == 0) rec[slice].sum = sum;
        return;
    }

    if (fabs(vmax * rp.inv_t) > kMaxTop) return;  // drawn from the whole row
    // HIST: the slices' bins on the row's grid, thread t the bins 2 t and 2 t + 1 below the row's top bin
    const double top_bin = bin_of(value_of(top), rp.inv_t);
    const uint64_t* hist = ws.hist + (size_t)row * nsl * kBins;
    constexpr uint64_t kLess = (1ull << kCountShift) - 1;
    constexpr double kUnit = 1.0 / (double)(1ull << kBinFrac);
    // bins between the row's top and the slice's, and those that hold something
    uint64_t used = 0, unused = 0;
    if (t < nsl) {
        const uint32_t o = my_top ? bin_below(top_bin, bin_of(value_of(my_top), rp.inv_t)) : kBins - 1;
        s_off[t] = o;
        used = min(o + my_count, kBins - 1);
    }
    // weights of the bins' upper edges relative to the largest token
    const double top_edge = (top_bin + 1.0) * 0.125 - vmax * rp.inv_t;
#pragma unroll
    for (uint32_t b = 0; b < kBins; b += kThreads) s_edge[b + t] = exp(top_edge - 0.125 * (double)(b + t));
    block_max2<NT>(sh, used, unused);
    uint32_t n2[2] = {0, 0};
    uint64_t less[2] = {0, 0};
    if (2 * t < (uint32_t)used) {
        for (uint32_t s0 = 0; s0 < nsl; s0 += 16) {
            uint64_t h[16][2];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t s = min(s0 + j, nsl - 1), at = 2 * t - s_off[s];  // wraps below the slice's top
                const bool in = s0 + j < nsl;
                const uint64_t* hs = hist + (size_t)s * kBins;
                h[j][0] = hs[in && at < kBins ? at : kBins - 1];
                h[j][1] = hs[in && at + 1 < kBins ? at + 1 : kBins - 1];
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    n2[i] += (uint32_t)(h[j][i] >> kCountShift);
                    less[i] += h[j][i] & kLess;
                }
        }
    }
    if (2 * t + 1 == kBins - 1) n2[1] = 0, less[1] = 0;  // below all bins that count
    double w2[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) w2[i] = ((double)n2[i] - (double)less[i] * kUnit) * s_edge[2 * t + i];
    uint64_t all_n;
    double all_w;
    const uint64_t cn1 = block_scan<NT>(sh, (uint64_t)n2[0] + n2[1], all_n), cn0 = cn1 - n2[1];
    const double cw1 = block_scan<NT>(sh, w2[0] + w2[1], all_w), cw0 = cw1 - w2[1];
    s_cum_n[2 * t] = (uint32_t)cn0;
    s_cum_n[2 * t + 1] = (uint32_t)cn1;
    s_cum_w[2 * t] = cw0;
    s_cum_w[2 * t + 1] = cw1;
    // the bin of the k-th token (kBins - 1: below all bins that count) and the bins in which the top-p cut can fall
    if (n2[0] && cn0 >= rp.k && cn0 - n2[0] < rp.k) s_kb = 2 * t;
    if (n2[1] && cn1 >= rp.k && cn0 < rp.k) s_kb = 2 * t + 1;
    __syncthreads();
    const uint32_t kb = s_kb;
    const bool cut_k = kb < kBins - 1 && s_cum_n[kb] != rp.k;
    const double hi_total = s_cum_w[kb], lo_total = cut_k ? (kb ? s_cum_w[kb - 1] : 0.0) : hi_total;
    if (rp.cut_p) {
        // the first bin with a token whose running sum reaches the share, a lane of each wave (one address for all lanes
        // that reach it took 4 us)
        auto first_of = [&](double share, uint32_t* at) {
            const bool r0 = n2[0] && cw0 >= share, r1 = n2[1] && cw1 >= share;
            const uint64_t some = __builtin_amdgcn_ballot_w64(r0 || r1);
            if (some && lane == (uint32_t)__builtin_ctzll(some)) atomicMin(at, 2 * t + (r0 ? 0 : 1));
        };
        first_of(lo_total * rp.p * (1.0 - kBinNoise), &s_plo);
        first_of(hi_total * rp.p * (1.0 - kBinNoise), &s_phi);
    }
    __syncthreads();
    const uint32_t plo = s_plo, phi = s_phi;
    const uint32_t mb = rp.m > 0.0 ? bin_below(top_bin, fmin(floor((vmax * rp.inv_t + log(rp.m)) * 8.0), top_bin)) : kBins - 1;
    // Bins that are kept whole whatever the cuts turn out to be: those before the first in which one can fall (from there
    // on to the last one kept, a cut can fall in every bin, or they lie below min-p). This slice's weight in them, and its tokens in the others.
    const uint32_t sure = min(min(rp.cut_p ? plo : kBins - 1, mb), kb < kBins - 1 ? (cut_k ? kb : kb + 1) : kBins - 1);
    if (slice == 0) {
        RowRec& r = ws.row[row];
        r.cum_w[2 * t] = cw0;
        r.cum_w[2 * t + 1] = cw1;
        if (t == 0) {
            r.kb = kb;
            r.plo = plo;
            r.phi = phi;
            r.sure = sure;
            r.cut_k = cut_k;
            r.k_left = rp.k - (cut_k && kb ? s_cum_n[kb - 1] : 0);
            r.lo_total = lo_total;
            r.hi_total = hi_total;
        }
    }
    {
        const uint64_t* hs = hist + (size_t)slice * kBins;
        const uint32_t o = s_off[slice];
        double sum = 0.0;
#pragma unroll
        for (uint32_t b0 = 0; b0 < kBins; b0 += kThreads) {
            const uint32_t b = b0 + t;
            if (b < o || b >= sure) continue;
            const uint64_t h = hs[b - o];
            sum += ((double)(h >> kCountShift) - (double)(h & kLess) * kUnit) * s_edge[b];
        }
        sum = block_add<NT>(sh, sum);
        if (t == 0) rec[slice].sum = sum;
    }
    uint64_t* list = ws.lists + (size_t)row * ws.list_stride;
    // The tokens of bins b1 .. b2, by value: within some 2^-21 of an edge also the next bins' (the draw takes no token by its
    // being listed). In 64 bits, bin by bin, this took 9000 cycles of 32 tokens a thread.
    uint32_t mine = 0;
    auto collect = [&](uint32_t b1, uint32_t b2) {
        b2 = min(b2, kBins - 2);
        if (b1 > b2) return;
        const double eighth = 0.125 * (double)ps.temperature, most = (double)FLT_MAX;
        const double lo = fmax((top_bin - (double)b2) * eighth, -most), hi = fmin((top_bin - (double)b1 + 1.0) * eighth, most);
        const float mid = (float)(0.5 * (lo + hi));
        const float reach = (float)fmin((hi - lo) * 0.5 + (hi - lo + fabs(lo + hi)) * 0x1p-22 + 0x1p-140, most);
#pragma unroll
        for (int i = 0; i < EPT; ++i) mine |= fabsf(v[i] - mid) <= reach ? 1u << i : 0u;
    };
    if (rp.cut_p) collect(plo, phi);
    if (cut_k) collect(kb, kb);
    if (mb <= min(rp.cut_p ? phi : kBins, kb)) collect(mb, mb);
    uint64_t total;
    const uint64_t c = __builtin_popcount(mine);
    uint32_t at = (uint32_t)(block_scan<NT>(sh, c, total) - c);
    if (total == 0) return;
    if (t == 0) s_base = atomicAdd(&ws.counters[row * kCounter], (uint32_t)total);
    __syncthreads();
    at += s_base;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
        if (mine >> i & 1) {
            if (at < kListCap) list[at] = rank_of(v[i], first + i * kThreads + t);
            ++at;
        }
}

// A block a row of mode SUM or HIST, or of one whose lists overflowed. SL: tokens a slice.
template <class T, int SL>
__global__ __launch_bounds__(kDrawThreads) void k_rows_draw(const T* __restrict__ logits, uint32_t V, uint64_t stride,
                                                            const vsl_row_sampler* __restrict__ params, const float* __restrict__ us,
                                                            uint32_t nsl, Work ws, uint32_t* __restrict__ tokens,
                                                            float* __restrict__ probs) {
    constexpr int NT = kDrawThreads, E = SL / NT;
    __shared__ Shared sh;
    __shared__ uint64_t s_slice[kMaxSlices];
    const uint32_t row = blockIdx.x, t = threadIdx.x;
    const vsl_row_sampler ps = params[row];
    const RowRec& rr = ws.row[row];
    // requested together with the parameters; each is this call's in the modes that use it
    const uint32_t kb = rr.kb, plo = rr.plo, phi = rr.phi, rec_sure = rr.sure, rec_cut_k = rr.cut_k, k_left = rr.k_left, whole = rr.whole;
    const double lo_total = rr.lo_total, hi_total = rr.hi_total;
    const float uf = us[row];
    const uint32_t listed = ws.counters[row * kCounter];
    const RowParams rp = row_params(ps, V);
    if (rp.mode == MODE_GREEDY || (rp.mode == MODE_TOPK && !whole)) return;
    const T* l = logits + (size_t)row * stride;
    const RowOut out{tokens + row, probs ? probs + row : nullptr};
    const double u = uf > 0.f ? fmin((double)uf, 1.0 - 0x1p-24) : 0.0;
    const uint32_t n_list = rp.mode == MODE_HIST ? listed : 0;
    const SliceRec* rec = ws.rec + (size_t)row * nsl;
    uint64_t top = 0, none = 0;
    double slice_sum = 0.0;
    if (t < nsl) {
        top = rec[t].top;
        slice_sum = rec[t].sum;
    }
    const uint64_t* list = ws.lists + (size_t)row * ws.list_stride;
    uint64_t r[kDrawRegs];
#pragma unroll
    for (int i = 0; i < kDrawRegs; ++i) r[i] = i * NT + t < min(n_list, kListCap) ? list[i * NT + t] : 0;
    block_max2<NT>(sh, top, none);
    if (top == 0) return;
    const double vmax = (double)value_of(top);
    // batches of eight elements, requested together
    auto in_batches = [&](uint32_t from, uint32_t n, auto load, auto f) {
        for (uint32_t i0 = from + t; i0 < n; i0 += 8 * NT) {
            uint64_t x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = i0 + j * NT < n ? load(i0 + j * NT) : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (x[j]) f(x[j], [&] { return weight_of(value_of(x[j]), vmax, rp.inv_t); });
        }
    };
    if (rp.mode == MODE_TOPK || (rp.mode == MODE_HIST && (n_list > kListCap || fabs(vmax * rp.inv_t) > kMaxTop))) {
        auto visit = [&](auto f) { in_batches(0, V, [&](uint32_t i) { return rank_of(load_logit(l, i), i); }, f); };
        double one = kFewOne;  // TOPK: only the first k count
        if (rp.mode == MODE_HIST) {
            double sum = 0.0;
            visit([&](uint64_t, auto weight) { sum += weight(); });
            one = unit_of(block_add<NT>(sh, sum));
        }
        draw_exact<NT>(sh, V, rp, vmax, u, out, rp.k < V, one, visit);
        return;
    }
    // the list's tokens: the first ones from registers, their weights taken once, the others from memory
    double wts[kDrawRegs];
#pragma unroll
    for (int i = 0; i < kDrawRegs; ++i) wts[i] = (uint32_t)i * NT < n_list ? weight_of(r[i] ? value_of(r[i]) : (float)vmax, vmax, rp.inv_t) : 0.0;
    auto visit = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kDrawRegs; ++i)
            if (r[i]) f(r[i], [&] { return wts[i]; });
        in_batches(kDrawRegs * NT, n_list, [&](uint32_t i) { return list[i]; }, f);
    };
    const double top_bin = bin_of(value_of(top), rp.inv_t);
    auto row_bin = [&](float x) { return bin_below(top_bin, bin_of(x, rp.inv_t)); };
    uint64_t low = 1;  // the smallest kept rank key
    uint32_t cb = kBins - 2, sure = 0;  // the last bin that keeps a token; the bins kept whole are in the slices' sums
    const bool hist = rp.mode == MODE_HIST;
    const double one = unit_of(hist ? hi_total : block_add<NT>(sh, slice_sum));  // kept weights add up to no more
    if (hist) {
        sure = rec_sure;
        double total = hi_total;
        if (rec_cut_k) {
            low = select_key<NT>(sh, n_list, k_left, visit, [&](uint64_t rank, auto, uint64_t& key, uint64_t& w) {
                key = rank;
                w = 1;
                return row_bin(value_of(rank)) == kb;
            });
            if (rp.cut_p) {
                uint64_t part = 0;
                visit([&](uint64_t rank, auto weight) { part += rank >= low && row_bin(value_of(rank)) == kb ? units(weight(), one) : 0; });
                total = lo_total + (double)block_add<NT>(sh, part) / one;
            }
        }
        if (rp.cut_p) {
            const double target = total * rp.p * (1.0 - kBinNoise);
            uint32_t pb = plo;
            while (pb < phi && rr.cum_w[pb] < target) ++pb;
            const double base = pb ? rr.cum_w[pb - 1] : 0.0;
            const uint64_t left = target > base ? (uint64_t)ceil((target - base) * one) : 1;
            const uint64_t cut = select_key<NT>(sh, n_list, left, visit, [&](uint64_t rank, auto weight, uint64_t& key, uint64_t& w) {
                if (rank < low || row_bin(value_of(rank)) != pb) return false;
                key = rank;
                w = units(weight(), one);
                return true;
            });
            if (cut > low) low = cut;
        }
        cb = low > 1 ? row_bin(value_of(low)) : kb < kBins - 1 ? kb : kBins - 2;
    }
    auto kept = [&](uint64_t rank, double w) { return rank >= low && w >= rp.m && (!hist || row_bin(value_of(rank)) <= cb); };
    // the slices' kept weights, in fixed point; of the bins that a cut divides, the list's tokens
    if (t < kMaxSlices) s_slice[t] = units(slice_sum, one);
    __syncthreads();
    visit([&](uint64_t rank, auto weight) {
        if (rank < low) return;
        const uint32_t b = row_bin(value_of(rank));
        if (b < sure || b > cb || (rp.m > 0.0 && weight_of(value_of(rank), vmax, rp.inv_t) < rp.m)) return;
        atomicAdd(reinterpret_cast<unsigned long long*>(&s_slice[index_of(rank) / SL]), (unsigned long long)units(weight(), one));
    });
    __syncthreads();
    // the slice in which their running sum passes u
    if (t < 64) {
        const uint64_t a = s_slice[2 * t], b = s_slice[2 * t + 1];
        const uint64_t incl = wave_scan(a + b), sum = last_lane(incl), before = incl - a - b;
        const double target = (double)sum * (hist ? u * (1.0 + kBinNoise) : u);
        const bool in_a = a && (double)(before + a) > target, in_b = b && (double)incl > target;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(in_a || in_b), some = __builtin_amdgcn_ballot_w64(a || b);
        const int who = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some | 1);
        if ((int)t == who) {
            const bool second = hit ? !in_a : b != 0;
            sh.sel_count = 2 * t + (second ? 1 : 0);
            sh.sel_key = second ? before + a : before;
            sh.sel_left = sum;
        }
    }
    __syncthreads();
    // the token in it: thread t takes E neighbours
    const double total = (double)sh.sel_left / one;
    const double target = total * (hist ? u * (1.0 + kBinNoise) : u) - (double)sh.sel_key / one;
    const uint32_t first = sh.sel_count * SL, from = first + t * E;
    double w[E], mine = 0.0, all;
    uint64_t last = 0;  // the last kept index + 1
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float x = from + i < V ? load_logit(l, from + i) : -INFINITY;
        const double wx = weight_of(x, vmax, rp.inv_t);
        w[i] = x != -INFINITY && kept(rank_of(x, from + i), wx) ? wx : 0.0;
        mine += w[i];
        if (w[i] > 0.0) last = from + i + 1;
    }
    const double incl = block_scan<NT>(sh, mine, all);
    // the first thread whose sum passes the target (rounding may leave none: the last kept token)
    uint64_t hit = incl > target && mine > 0.0 ? ~(uint64_t)t : 0, end = last;
    block_max2<NT>(sh, hit, end);
    const uint32_t who = hit ? (uint32_t)~hit : (uint32_t)(end - 1 - first) / E;
    if (end == 0 || t != who) return;
    double run = incl - mine, share = 0.0;
    uint32_t token = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        run += w[i];
        if (w[i] > 0.0 && !found) {
            token = from + i;
            share = w[i];
            found = hit && run > target;
        }
    }
    put(out, token, share / total);
}

uint64_t up256(uint64_t b) { return (b + 255) & ~255ull; }

// Elements a thread: enough slices to fill the CUs with the rows there are, at most kMaxSlices of them. us for 8 / 16 / 32, k = 40 and
// top-p: 1 x 32000 15 / 17 / 19 and 23 / 29 / 39, 1 x 131072 24 / 19 / 20 and 29 / 32 / 42, 64 x 131072 59 / 42 / 30 and
// 88 / 64 / 62. Between, rows of 32000 would do better with 8: 16 rows 16 / 17 / 20 and 24 / 30 / 41.
uint32_t elements_per_thread(uint32_t rows, uint32_t V) {
    for (uint32_t e : {8u, 16u})
        if ((uint64_t)rows * ((V + e * kThreads - 1) / (e * kThreads)) <= (e == 8 ? 32 : 1024) && (V + e * kThreads - 1) / (e * kThreads) <= kMaxSlices)
            return e;
    return kMaxEpt;
}

struct Layout {
    uint32_t ept, nsl, list_stride;
    uint64_t row, counters, lists, hist, bytes;
};
Layout layout(uint32_t rows, uint32_t V) {
    Layout y;
    y.ept = elements_per_thread(rows, V);
    y.nsl = (V + y.ept * kThreads - 1) / (y.ept * kThreads);
    const uint32_t wide = V < kListCap ? V : kListCap;
    y.list_stride = y.nsl * kLeanCap > wide ? y.nsl * kLeanCap : wide;
    y.row = up256((uint64_t)rows * y.nsl * sizeof(SliceRec));
    y.counters = y.row + up256((uint64_t)rows * sizeof(RowRec));
    y.lists = y.counters + up256((uint64_t)rows * kCounter * 4);
    y.hist = y.lists + up256((uint64_t)rows * y.list_stride * 8);
    y.bytes = y.hist + up256((uint64_t)rows * y.nsl * kBins * 8);
    return y;
}

template <class T, int EPT>
void launch(hipStream_t s, const Layout& y, const T* logits, uint32_t rows, uint32_t V, uint64_t stride,
            const vsl_row_sampler* params, const float* u, const Work& w, uint32_t* tokens, float* probs) {
    const dim3 grid(y.nsl, rows);
    k_rows_scan<T, EPT><<<grid, kThreads, 0, s>>>(logits, V, stride, params, w);
    k_rows_cut<T, EPT><<<grid, kThreads, 0, s>>>(logits, V, stride, params, u, w, tokens, probs);
    k_rows_draw<T, EPT * kThreads><<<rows, kDrawThreads, 0, s>>>(logits, V, stride, params, u, y.nsl, w, tokens, probs);
}

}  // namespace

extern "C" uint64_t vsl_sample_rows_ws_bytes(uint32_t rows, uint32_t V) {
    if (rows == 0 || rows > 65535 || V == 0 || V > kMaxRowsV) return 0;
    return layout(rows, V).bytes;
}

extern "C" int vsl_sample_rows(const void* logits, int dtype, uint32_t rows, uint32_t V, uint64_t stride,
                               const vsl_row_sampler* params, const float* u, uint32_t* tokens, float* probs, void* workspace,
                               uint64_t ws_bytes, void* stream) {
    const char* fn = "vsl_sample_rows";
    if (rows == 0) return VSL_OK;
    if (!logits || !params || !u || !tokens || !workspace) return vsl_invalid("%s: null pointer", fn);
    if (dtype != VSL_DT_F32 && dtype != VSL_DT_F16) return vsl_unsupported("%s: dtype %d", fn, dtype);
    if (V == 0 || V > kMaxRowsV || rows > 65535)
        return vsl_unsupported("%s: %u rows of %u logits (up to 65535 of 1..%u)", fn, rows, V, kMaxRowsV);
    if (stride < V) return vsl_invalid("%s: row stride %llu below %u logits", fn, (unsigned long long)stride, V);
    if (reinterpret_cast<uintptr_t>(workspace) & 15 || reinterpret_cast<uintptr_t>(params) & 3 ||
        reinterpret_cast<uintptr_t>(logits) & (dtype == VSL_DT_F32 ? 3 : 1) || reinterpret_cast<uintptr_t>(u) & 3 ||
        reinterpret_cast<uintptr_t>(tokens) & 3 || reinterpret_cast<uintptr_t>(probs) & 3)
        return vsl_invalid("%s: misaligned pointer", fn);
    const Layout y = layout(rows, V);
    if (ws_bytes < y.bytes)
        return vsl_capacity("%s: workspace of %llu bytes, %llu needed", fn, (unsigned long long)ws_bytes,
                            (unsigned long long)y.bytes);
    char* base = static_cast<char*>(workspace);
    const Work w{reinterpret_cast<SliceRec*>(base), reinterpret_cast<RowRec*>(base + y.row), reinterpret_cast<uint32_t*>(base + y.counters),
                 reinterpret_cast<uint64_t*>(base + y.lists), reinterpret_cast<uint64_t*>(base + y.hist), y.list_stride};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto* l) {
        if (y.ept == 8) launch<std::remove_const_t<std::remove_pointer_t<decltype(l)>>, 8>(s, y, l, rows, V, stride, params, u, w, tokens, probs);
        else if (y.ept == 16) launch<std::remove_const_t<std::remove_pointer_t<decltype(l)>>, 16>(s, y, l, rows, V, stride, params, u, w, tokens, probs);
        else launch<std::remove_const_t<std::remove_pointer_t<decltype(l)>>, 32>(s, y, l, rows, V, stride, params, u, w, tokens, probs);
    };
    if (dtype == VSL_DT_F32) go(static_cast<const float*>(logits));
    else go(static_cast<const vsl_half*>(logits));
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}
