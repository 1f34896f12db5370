// vsl_sample_rows.hip -- one token for each row of a batch of logits, by temperature, top-k, top-p and min-p, from given
// uniform numbers (vsl_sample_rows). No reference counterpart: the reference samples one vector by its host code
// (Utils.cpp:140-172) and reads no top_p (Common.h:59).
//
// With w_i = exp((l_i - max) / T), the kept tokens are a run of the order (logit descending, index ascending): every one
// of the three filters cuts that order somewhere, and the shortest run counts. So nothing is sorted: a cut is one 64-bit
// rank key (the float's order, then the inverted index), found by narrowing down, and the draw walks the kept tokens by
// index. Weights are summed in 64 bits (fixed point where atomics add them, so that no order of arrival matters): the
// token is that of exact sums but where u falls within about 1e-12 of a border.
//
// Two launches. k_rows_scan reads the row's slices (a block each) once and leaves, by what the row asks for,
//   GREEDY  the slice's maximum
//   TOPK    (k <= kLeanK) the slice's tokens that can be among the k largest: at least k of them lie at or above the k-th
//           largest of the block's per-thread maxima
//   SUM     (no cut but min-p) the maximum
//   HIST    (top-p, or a larger k) counts and weights by bins of 1/8 in l / T, whose grid is the same for every slice, so
//           that no slice has to know the row's maximum
// k_rows_pick ends GREEDY and TOPK rows in one block; for SUM its blocks sum the kept weights of the slices, for HIST they
// collect the tokens of the bins in which a cut falls, and the last block to arrive draws. Where ties or ranges make a
// list too long, that block narrows the cuts down over the whole row instead.
#include <float.h>

#include <cmath>

#include "vsl_device.h"
#include "vsl_internal.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr uint32_t kMaxSlices = 128, kMaxEpt = 8;
constexpr uint32_t kMaxRowsV = kMaxSlices * kMaxEpt * kThreads;  // 2^20 tokens
constexpr uint32_t kLeanK = 256;   // TOPK up to this k
constexpr uint32_t kLeanCap = 512;  // tokens a slice's list holds
constexpr uint32_t kListCap = 4096;  // tokens a row's list holds, in LDS too
constexpr uint32_t kBins = 512;     // of 1/8 in l / T; the last one takes all below e^-63.9 of the largest, never drawn
constexpr double kBinSpan = 0.11751;  // above 1 - exp(-1/8), the most that a weight lies below its bin's upper edge
constexpr int kBinFrac = 36;        // weights in a bin: what they lie below it, in units of 2^-36
constexpr int kCountShift = 46;     // 8192 of them stay below 2^46; the count above
// Sums over bins are off by up to 2^-37 of their weights, and a little of the grid's rounding. Cuts and draws that meet a
// border exactly (equal logits: whole numbers of equal weights) are decided as exact sums are: a share is reached a little
// below it, a draw has passed a border a little above it.
constexpr double kBinNoise = 4e-11;
constexpr double kMaxTop = 16384.0;  // l / T up to which the grid's rounding (2^-39) is far below a weight's
constexpr double kListOne = 0x1p50, kRowOne = 0x1p42;  // fixed point of weights in lists (<= 2^13 tokens) and rows (<= 2^20)

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
    uint32_t count;   // TOPK: tokens found (kLeanCap of them stored)
    float floor_v;    // TOPK: all tokens of the slice at or above this value are in its list, and there are k of them (-inf: all)
    double sum;       // SUM: kept weights
    uint64_t pad;
};

struct Work {
    SliceRec* rec;       // [rows][nsl]
    uint32_t* counters;  // [rows][2]: the row list's length, blocks that have arrived
    uint64_t* lists;     // [rows][max(nsl * kLeanCap, kListCap)]
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

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
    return (uint64_t)__shfl_xor((uint32_t)(v >> 32), m, 64) << 32 | __shfl_xor((uint32_t)v, m, 64);
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const uint64_t x = shfl_xor64(v, o);
        v = x > v ? x : v;
    }
    return v;
}
template <class T>
__device__ __forceinline__ T wave_add(T v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __builtin_bit_cast(T, shfl_xor64(__builtin_bit_cast(uint64_t, v), o));
    return v;
}
// Inclusive sum over the wave's lanes below and at this one.
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint64_t x = (uint64_t)__shfl_up((uint32_t)(b >> 32), o, 64) << 32 | __shfl_up((uint32_t)b, o, 64);
        if (lane >= o) v += __builtin_bit_cast(T, x);
    }
    return v;
}

struct Shared {
    uint64_t red[kWaves + 1];
    uint64_t digits[256];
    uint32_t counts[256];
    uint64_t sel_key, sel_left;
    uint32_t sel_count, sel_done;
};

// Block-wide sums, maxima and scans of 64-bit values, every thread ending with the result. All threads call.
template <class T>
__device__ T block_add(Shared& sh, T v) {
    v = wave_add(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = __builtin_bit_cast(uint64_t, v);
    __syncthreads();
    T s = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s += __builtin_bit_cast(T, sh.red[w]);
    return s;
}
__device__ uint64_t block_max64(Shared& sh, uint64_t v) {
    v = wave_max64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) s = sh.red[w] > s ? sh.red[w] : s;
    return s;
}
template <class T>
__device__ T block_scan(Shared& sh, T v) {
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.red[threadIdx.x >> 6] = __builtin_bit_cast(uint64_t, v);
    __syncthreads();
    const int wave = threadIdx.x >> 6;
    T before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        if (w < wave) before += __builtin_bit_cast(T, sh.red[w]);
    return before + v;
}

// The last key of the shortest run of keys, in descending order, whose measures reach `target` (the smallest key of all if
// they do not). src(i, key, measure) for i < n: false where the element takes no part; measure is an integer, keys differ.
// Digits of 8 bits from the highest bit in which keys differ; ends early when a digit holds one key. All threads call;
// 0 without elements.
template <class Src>
__device__ uint64_t select_key(Shared& sh, uint32_t n, uint64_t target, Src src) {
    const uint32_t t = threadIdx.x;
    uint64_t all_or = 0, all_and = ~0ull;
    for (uint32_t i = t; i < n; i += kThreads) {
        uint64_t key, w;
        if (src(i, key, w)) {
            all_or |= key;
            all_and &= key;
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        all_or |= shfl_xor64(all_or, o);
        all_and &= shfl_xor64(all_and, o);
    }
    __syncthreads();
    if ((t & 63) == 0) {
        sh.digits[t >> 6] = all_or;
        sh.digits[kWaves + (t >> 6)] = all_and;
    }
    __syncthreads();
    all_or = 0;
    all_and = ~0ull;
    for (int w = 0; w < kWaves; ++w) {
        all_or |= sh.digits[w];
        all_and &= sh.digits[kWaves + w];
    }
    __syncthreads();
    if (all_or == 0) return 0;
    const uint64_t diff = all_or ^ all_and;  // keys that differ somewhere (one key: none)
    if (diff == 0) return all_or;
    const int top = 64 - __builtin_clzll(diff);  // bits 0 .. top - 1 differ
    int shift = top > 8 ? top - 8 : 0;
    uint64_t prefix = top >= 64 ? 0 : all_and >> top << top, mask = top >= 64 ? 0 : ~0ull << top;
    for (;;) {
        for (uint32_t i = t; i < 256; i += kThreads) {
            sh.digits[i] = 0;
            sh.counts[i] = 0;
        }
        __syncthreads();
        for (uint32_t i = t; i < n; i += kThreads) {
            uint64_t key, w;
            if (src(i, key, w) && (key & mask) == prefix) {
                const uint32_t d = (uint32_t)(key >> shift) & 255u;
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits[d]), (unsigned long long)w);
                atomicAdd(&sh.counts[d], 1u);
            }
        }
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
            const uint64_t incl = wave_scan(s);
            uint64_t run = incl - s;
            int hit = -1, last = -1;
            uint64_t left = target, last_run = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (c4[j]) {
                    last = j;
                    last_run = run;
                }
                if (hit < 0 && c4[j] && run + d4[j] >= target) {
                    hit = j;
                    left = target - run;
                }
                run += d4[j];
            }
            const uint64_t reach = __builtin_amdgcn_ballot_w64(hit >= 0), some = __builtin_amdgcn_ballot_w64(last >= 0);
            const bool none = reach == 0;  // the sums fall short of the target: the smallest key
            const int who = none ? 63 - __builtin_clzll(some) : __builtin_ctzll(reach);
            if ((int)t == who) {
                const int j = none ? last : hit;
                sh.sel_left = none ? (target > last_run ? target - last_run : 0) : left;
                sh.sel_key = 255 - 4 * t - j;
                sh.sel_count = c4[j == 0 ? 0 : j == 1 ? 1 : j == 2 ? 2 : 3];
            }
        }
        __syncthreads();
        prefix |= sh.sel_key << shift;
        mask |= 255ull << shift;
        target = sh.sel_left;
        const uint32_t count = sh.sel_count;
        __syncthreads();
        if (count == 1 || shift == 0) break;
        shift = shift > 8 ? shift - 8 : 0;
    }
    // the one key with that prefix
    for (uint32_t i = t; i < n; i += kThreads) {
        uint64_t key, w;
        if (src(i, key, w) && (key & mask) == prefix) sh.sel_key = key;
    }
    __syncthreads();
    const uint64_t key = sh.sel_key;
    __syncthreads();
    return key;
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

// The draw over elements elem(i) -> rank key (0: none), i < n, that hold every token of the first k: the three cuts, then
// the index at which the running sum passes u. `one`: the fixed point of weights.
template <class Elem>
__device__ void draw_exact(Shared& sh, uint32_t n, const RowParams& rp, double vmax, double u, double one, const RowOut& out,
                           bool cut_k, Elem elem) {
    auto fixed = [&](uint64_t rank) { return (uint64_t)(weight_of(value_of(rank), vmax, rp.inv_t) * one + 0.5); };
    uint64_t low = 1;  // the smallest kept rank key
    if (cut_k) low = select_key(sh, n, rp.k, [&](uint32_t i, uint64_t& key, uint64_t& w) {
        key = elem(i);
        w = 1;
        return key != 0;
    });
    auto total_of = [&](auto kept) {
        uint64_t s = 0;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const uint64_t key = elem(i);
            if (key >= low && kept(key)) s += fixed(key);
        }
        return block_add(sh, s);
    };
    if (rp.cut_p) {
        const uint64_t total = total_of([](uint64_t) { return true; });
        const uint64_t target = (uint64_t)ceil((double)total * rp.p);
        low = select_key(sh, n, target, [&](uint32_t i, uint64_t& key, uint64_t& w) {
            key = elem(i);
            w = key >= low ? fixed(key) : 0;
            return key >= low;
        });
    }
    // min-p: the weight itself decides
    auto heavy = [&](uint64_t key) { return weight_of(value_of(key), vmax, rp.inv_t) >= rp.m; };
    const uint64_t total = total_of(heavy);
    uint64_t target = (uint64_t)((double)total * u) + 1;
    if (target > total) target = total;
    const uint64_t at = select_key(sh, n, target, [&](uint32_t i, uint64_t& key, uint64_t& w) {
        const uint64_t rank = elem(i);
        if (rank < low || !heavy(rank)) return false;
        w = fixed(rank);
        key = (rank & 0xFFFFFFFFull) + 1;  // the inverted index: ascending indices are descending keys (+ 1: not 0)
        return w != 0;
    });
    const uint32_t idx = ~(uint32_t)(at - 1);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t rank = elem(i);
        if (rank && index_of(rank) == idx) put(out, idx, (double)fixed(rank) / (double)total);
    }
}

// Bin of a value on the grid that all slices share: floor(8 l / T), as a double (exact to 2^53, and monotone above).
__device__ __forceinline__ double bin_of(float v, double inv_t) { return floor((double)v * inv_t * 8.0); }
__device__ __forceinline__ uint32_t bin_below(double top_bin, double bin) { return (uint32_t)fmin(top_bin - bin, (double)(kBins - 1)); }

template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void k_rows_scan(const T* __restrict__ logits, uint32_t V, uint64_t stride,
                                                        const vsl_row_sampler* __restrict__ params, Work ws) {
    __shared__ Shared sh;
    __shared__ uint64_t s_hist[kBins];
    __shared__ uint32_t s_n;
    const uint32_t row = blockIdx.y, slice = blockIdx.x, nsl = gridDim.x, t = threadIdx.x;
    const T* l = logits + (size_t)row * stride;
    const uint32_t first = slice * (EPT * kThreads);
    float v[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const uint32_t e = first + i * kThreads + t;
        v[i] = e < V ? load_logit(l, e) : -INFINITY;
    }
    const RowParams rp = row_params(params[row], V);
    if (slice == 0 && t < 2) ws.counters[2 * row + t] = 0;
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const uint64_t r = rank_of(v[i], first + i * kThreads + t);
        best = r > best ? r : best;
    }
    const uint64_t top = block_max64(sh, best);
    SliceRec* rec = ws.rec + (size_t)row * nsl + slice;
    if (t == 0) rec->top = top;
    if (rp.mode == MODE_GREEDY || rp.mode == MODE_SUM) return;
    for (uint32_t b = t; b < kBins; b += kThreads) s_hist[b] = 0;
    if (t == 0) s_n = 0;
    if (rp.mode == MODE_TOPK) {
        // threads' maxima in 512 bins between their largest and their smallest: the bin of the k-th bounds the k-th token
        const float vmax = top ? value_of(top) : 0.f, mine = best ? value_of(best) : INFINITY;
        const uint64_t low_key = block_max64(sh, best ? ~(best | 0xFFFFFFFFull) : 0);
        const float vmin = top ? value_of(~low_key) : 0.f, range = vmax - vmin;
        const float step = range > 0.f ? (float)(kBins - 2) / range : 0.f;
        auto bin = [&](float x) {
            const float b = (vmax - x) * step;
            return b < (float)(kBins - 1) ? (uint32_t)b : kBins - 1;  // NaN (an infinite range): the last
        };
        if (best) atomicAdd(reinterpret_cast<unsigned long long*>(&s_hist[bin(mine)]), 1ull);
        __syncthreads();
        uint64_t c = t < kBins ? s_hist[t] : 0;
        const uint64_t incl = block_scan(sh, c);
        if (t == 0) sh.sel_count = kBins - 1;
        __syncthreads();
        if (t < kBins && incl >= rp.k && incl - c < rp.k) sh.sel_count = t;
        __syncthreads();
        const uint32_t cut = sh.sel_count;
        float lowest = INFINITY;
        uint64_t* list = ws.lists + (size_t)row * ws.list_stride + (size_t)slice * kLeanCap;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            if (v[i] == -INFINITY || bin(v[i]) > cut) continue;
            const uint32_t at = atomicAdd(&s_n, 1u);
            if (at < kLeanCap) list[at] = rank_of(v[i], first + i * kThreads + t);
            lowest = fminf(lowest, v[i]);
        }
        // the list's smallest value: with k tokens in it, no token below that value is among the row's k largest
        const uint64_t lk = block_max64(sh, lowest < INFINITY ? ~(rank_of(lowest, 0) | 0xFFFFFFFFull) : 0);
        if (t == 0) {
            rec->count = s_n;
            rec->floor_v = s_n >= rp.k ? value_of(~lk) : -INFINITY;
        }
        return;
    }
    __syncthreads();
    const double top_bin = top ? bin_of(value_of(top), rp.inv_t) : 0.0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        if (v[i] == -INFINITY) continue;
        const double x = (double)v[i] * rp.inv_t, b = floor(x * 8.0);
        const uint32_t r = bin_below(top_bin, b);
        const double d = 1.0 - exp(x - (b + 1.0) * 0.125);
        const uint64_t add = (1ull << kCountShift) + (r < kBins - 1 ? (uint64_t)(fmin(fmax(d, 0.0), kBinSpan) * (double)(1ull << kBinFrac) + 0.5) : 0);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s_hist[r]), (unsigned long long)add);
    }
    __syncthreads();
    uint64_t* h = ws.hist + ((size_t)row * nsl + slice) * kBins;
    for (uint32_t b = t; b < kBins; b += kThreads) h[b] = s_hist[b];
}

// Draws from one slice: the token at which the kept weights' running sum, by index, passes `target`.
template <class T, int EPT, class Kept>
__device__ void walk_slice(Shared& sh, const T* l, uint32_t V, uint32_t first, double target, double total, double vmax,
                           double inv_t, const RowOut& out, Kept kept) {
    const uint32_t t = threadIdx.x, from = first + t * EPT;
    double w[EPT], mine = 0.0;
    uint64_t last = 0;  // the last kept index + 1
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        w[i] = 0.0;
        if (from + i >= V) continue;
        const float v = load_logit(l, from + i);
        const double x = v == -INFINITY ? 0.0 : weight_of(v, vmax, inv_t);
        if (v == -INFINITY || !kept(rank_of(v, from + i), x)) continue;
        w[i] = x;
        mine += x;
        if (x > 0.0) last = from + i + 1;
    }
    const double incl = block_scan(sh, mine), before = incl - mine;
    // the first thread whose sum passes the target (rounding may leave none: the last kept token)
    const uint64_t hit = block_max64(sh, incl > target && mine > 0.0 ? ~(uint64_t)t : 0);
    const uint64_t end = block_max64(sh, last);
    const uint32_t who = hit ? (uint32_t)~hit : (uint32_t)(end - 1 - first) / EPT;
    if (end == 0 || t != who) return;
    double run = before;
    uint32_t token = 0;
    double weight = 0.0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        run += w[i];
        if (w[i] > 0.0 && !found) {
            token = from + i;
            weight = w[i];
            found = hit && run > target;
        }
    }
    put(out, token, weight / total);
}

template <class T, int EPT>
__global__ __launch_bounds__(kThreads) void k_rows_pick(const T* __restrict__ logits, uint32_t V, uint64_t stride,
                                                        const vsl_row_sampler* __restrict__ params, const float* __restrict__ us,
                                                        Work ws, uint32_t* __restrict__ tokens, float* __restrict__ probs) {
    __shared__ Shared sh;
    __shared__ uint64_t s_list[kListCap];
    __shared__ double s_cum_w[kBins];
    __shared__ uint32_t s_cum_n[kBins];
    __shared__ uint64_t s_slice[kMaxSlices];
    __shared__ uint32_t s_n, s_plo, s_phi, s_kb;
    __shared__ bool s_last;
    const uint32_t row = blockIdx.y, slice = blockIdx.x, nsl = gridDim.x, t = threadIdx.x;
    const RowParams rp = row_params(params[row], V);
    if (rp.mode <= MODE_TOPK && slice != 0) return;
    const SliceRec* rec = ws.rec + (size_t)row * nsl;
    const T* l = logits + (size_t)row * stride;
    const RowOut out{tokens + row, probs ? probs + row : nullptr};
    const float uf = us[row];
    const double u = uf > 0.f ? fmin((double)uf, 1.0 - 0x1p-24) : 0.0;  // NaN and below 0: 0; 1 and above: the float below 1
    const uint64_t top = block_max64(sh, t < nsl ? rec[t].top : 0);
    if (top == 0) {  // nothing above -inf
        if (slice == 0 && t == 0) put(out, 0, 0.0);
        return;
    }
    if (rp.mode == MODE_GREEDY) {
        if (t == 0) put(out, index_of(top), 1.0);
        return;
    }
    const double vmax = (double)value_of(top);
    auto whole_row = [&] {
        draw_exact(sh, V, rp, vmax, u, kRowOne, out, rp.k < V, [&](uint32_t i) { return rank_of(load_logit(l, i), i); });
    };

    if (rp.mode == MODE_TOPK) {
        // tokens at or above the highest of the slices' bounds
        float bound = -INFINITY;
        for (uint32_t s = 0; s < nsl; ++s) bound = fmaxf(bound, rec[s].floor_v);
        if (t == 0) s_n = 0;
        __syncthreads();
        const uint64_t* lists = ws.lists + (size_t)row * ws.list_stride;
        bool whole = false;
        for (uint32_t i = t; i < nsl * kLeanCap; i += kThreads) {
            const uint32_t s = i / kLeanCap, c = rec[s].count;
            whole |= c > kLeanCap;
            if (i % kLeanCap >= min(c, kLeanCap)) continue;
            const uint64_t r = lists[i];
            if (value_of(r) < bound) continue;
            const uint32_t at = atomicAdd(&s_n, 1u);
            if (at < kListCap) s_list[at] = r;
        }
        if (__syncthreads_or(whole) || s_n > kListCap) {
            whole_row();
            return;
        }
        draw_exact(sh, s_n, rp, vmax, u, kListOne, out, s_n > rp.k, [&](uint32_t i) { return s_list[i]; });
        return;
    }

    const uint32_t first = slice * (EPT * kThreads);
    uint32_t* counters = ws.counters + 2 * row;
    auto last_block = [&] {
        __threadfence();
        __syncthreads();
        if (t == 0) s_last = atomicAdd(&counters[1], 1u) == nsl - 1;
        __syncthreads();
        __threadfence();
        return s_last;
    };
    // the slice in which the running sum of s_slice (fixed point kRowOne) passes u; then the walk
    auto draw_slice = [&](double u, auto kept) {
        __syncthreads();
        if (t < 64) {
            const uint64_t a = 2 * t < nsl ? s_slice[2 * t] : 0, b = 2 * t + 1 < nsl ? s_slice[2 * t + 1] : 0;
            const uint64_t incl = wave_scan(a + b);
            if (t == 63) sh.sel_left = incl;
            const uint64_t sum = (uint64_t)__shfl((uint32_t)(incl >> 32), 63, 64) << 32 | __shfl((uint32_t)incl, 63, 64);
            const double target = (double)sum * u;
            const uint64_t before = incl - a - b;
            const bool in_a = a && (double)(before + a) > target, in_b = b && (double)incl > target;
            const uint64_t hit = __builtin_amdgcn_ballot_w64(in_a || in_b);
            const uint64_t some = __builtin_amdgcn_ballot_w64(a || b);
            const int who = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some | 1);
            if ((int)t == who) {
                const bool second = hit ? !in_a : b != 0;
                sh.sel_count = 2 * t + (second ? 1 : 0);
                sh.sel_key = second ? before + a : before;
            }
        }
        __syncthreads();
        const double total = (double)sh.sel_left / kRowOne, before = (double)sh.sel_key / kRowOne;
        const uint32_t s = sh.sel_count;
        __syncthreads();
        walk_slice<T, EPT>(sh, l, V, s * (EPT * kThreads), total * u - before, total, vmax, rp.inv_t, out, kept);
    };

    if (rp.mode == MODE_SUM) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const uint32_t e = first + i * kThreads + t;
            const float v = e < V ? load_logit(l, e) : -INFINITY;
            const double w = v == -INFINITY ? 0.0 : weight_of(v, vmax, rp.inv_t);
            if (w >= rp.m) sum += w;
        }
        sum = block_add(sh, sum);
        if (t == 0) ws.rec[(size_t)row * nsl + slice].sum = sum;
        if (!last_block()) return;
        if (t < nsl) s_slice[t] = (uint64_t)(rec[t].sum * kRowOne + 0.5);
        draw_slice(u, [&](uint64_t, double w) { return w >= rp.m; });
        return;
    }

    if (fabs(vmax * rp.inv_t) > kMaxTop) {
        if (slice == 0) whole_row();
        return;
    }
    // HIST: the slices' bins on the row's grid, thread b bin b below the row's top bin
    const double top_bin = bin_of(value_of(top), rp.inv_t);
    const uint64_t* hist = ws.hist + (size_t)row * nsl * kBins;
    // weight of bin b's upper edge relative to the largest token
    auto edge = [&](uint32_t b) { return exp((top_bin + 1.0 - (double)b) * 0.125 - vmax * rp.inv_t); };
    auto bin_weight = [](uint64_t h) {  // of a bin's tokens, relative to its upper edge
        return (double)(h >> kCountShift) - (double)(h & ((1ull << kCountShift) - 1)) * (1.0 / (double)(1ull << kBinFrac));
    };
    auto offset_of = [&](uint32_t s) {  // bins between the row's top and the slice's
        return rec[s].top ? bin_below(top_bin, bin_of(value_of(rec[s].top), rp.inv_t)) : kBins - 1;
    };
    uint64_t n = 0;
    double w = 0.0;
    if (t < kBins - 1) {
        for (uint32_t s = 0; s < nsl; ++s) {
            const uint32_t o = offset_of(s);
            if (t < o) continue;
            const uint64_t h = hist[(size_t)s * kBins + t - o];
            n += h >> kCountShift;
            w += bin_weight(h);
        }
        w *= edge(t);
    }
    const uint64_t cum_n = block_scan(sh, n);
    const double cum_w = block_scan(sh, w);
    if (t < kBins) {
        s_cum_n[t] = (uint32_t)cum_n;
        s_cum_w[t] = cum_w;
    }
    if (t == 0) {
        s_kb = kBins - 1;
        s_plo = s_phi = kBins - 1;
    }
    __syncthreads();
    // the bin of the k-th token (kBins - 1: below all bins that count) and the bins in which the top-p cut can fall
    if (t < kBins - 1 && n && cum_n >= rp.k && cum_n - n < rp.k) s_kb = t;
    __syncthreads();
    const uint32_t kb = s_kb;
    const bool cut_k = kb < kBins - 1 && s_cum_n[kb] != rp.k;
    const double hi_total = s_cum_w[min(kb, kBins - 2)], lo_total = cut_k ? (kb ? s_cum_w[kb - 1] : 0.0) : hi_total;
    if (rp.cut_p && t < kBins - 1 && n) {
        if (cum_w >= lo_total * rp.p * (1.0 - kBinNoise)) atomicMin(&s_plo, t);
        if (cum_w >= hi_total * rp.p * (1.0 - kBinNoise)) atomicMin(&s_phi, t);
    }
    __syncthreads();
    const uint32_t plo = s_plo, phi = s_phi;
    const uint32_t mb = rp.m > 0.0 ? bin_below(top_bin, fmin(floor((vmax * rp.inv_t + log(rp.m)) * 8.0), top_bin)) : kBins - 1;
    auto row_bin = [&](float v) { return bin_below(top_bin, bin_of(v, rp.inv_t)); };
    auto wanted = [&](uint32_t b) {
        return b < kBins - 1 && ((cut_k && b == kb) || (rp.cut_p && b >= plo && b <= phi) || b == mb);
    };
    // this slice's tokens in those bins
    uint64_t* list = ws.lists + (size_t)row * ws.list_stride;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const uint32_t e = first + i * kThreads + t;
        const float v = e < V ? load_logit(l, e) : -INFINITY;
        if (v == -INFINITY || !wanted(row_bin(v))) continue;
        const uint32_t at = atomicAdd(&counters[0], 1u);
        if (at < kListCap) list[at] = rank_of(v, e);
    }
    if (!last_block()) return;
    const uint32_t n_list = __hip_atomic_load(&counters[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (n_list > kListCap) {
        whole_row();
        return;
    }
    for (uint32_t i = t; i < n_list; i += kThreads) s_list[i] = list[i];
    __syncthreads();
    auto fixed = [&](uint64_t rank) { return (uint64_t)(weight_of(value_of(rank), vmax, rp.inv_t) * kListOne + 0.5); };
    uint64_t low = 1;
    double total = hi_total;
    if (cut_k) {
        low = select_key(sh, n_list, rp.k - (kb ? s_cum_n[kb - 1] : 0), [&](uint32_t i, uint64_t& key, uint64_t& w1) {
            key = s_list[i];
            w1 = 1;
            return row_bin(value_of(key)) == kb;
        });
        uint64_t part = 0;
        for (uint32_t i = t; i < n_list; i += kThreads)
            if (s_list[i] >= low && row_bin(value_of(s_list[i])) == kb) part += fixed(s_list[i]);
        total = lo_total + (double)block_add(sh, part) / kListOne;
    }
    if (rp.cut_p) {
        const double target = total * rp.p * (1.0 - kBinNoise);
        uint32_t pb = plo;
        while (pb < phi && s_cum_w[pb] < target) ++pb;
        const double base = pb ? s_cum_w[pb - 1] : 0.0;
        const uint64_t left = target > base ? (uint64_t)ceil((target - base) * kListOne) : 1;
        const uint64_t cut = select_key(sh, n_list, left, [&](uint32_t i, uint64_t& key, uint64_t& w1) {
            key = s_list[i];
            if (key < low || row_bin(value_of(key)) != pb) return false;
            w1 = fixed(key);
            return true;
        });
        if (cut > low) low = cut;
    }
    // whole bins above the cut's, and of its own bin the list's tokens
    uint32_t cb = low > 1 ? row_bin(value_of(low)) : kBins - 1;
    if (low <= 1 && kb < kBins - 1) cb = kb + 1;  // k ends with a whole bin
    const uint32_t whole_bins = min(cb, mb);
    auto kept = [&](uint64_t rank, double wt) {
        return rank >= low && wt >= rp.m && row_bin(value_of(rank)) <= cb - (low > 1 ? 0 : 1);
    };
    const uint32_t lane = t & 63;
    for (uint32_t s = t >> 6; s < nsl; s += kWaves) {
        const uint32_t o = offset_of(s);
        double sum = 0.0;
        for (uint32_t b = o + lane; b < whole_bins; b += 64) sum += bin_weight(hist[(size_t)s * kBins + b - o]) * edge(b);
        sum = wave_add(sum);
        if (lane == 0) s_slice[s] = (uint64_t)(sum * kRowOne + 0.5);
    }
    __syncthreads();
    for (uint32_t i = t; i < n_list; i += kThreads) {
        const uint64_t r = s_list[i];
        const double wt = weight_of(value_of(r), vmax, rp.inv_t);
        const uint32_t b = row_bin(value_of(r));
        if (b < whole_bins || !kept(r, wt)) continue;
        atomicAdd(reinterpret_cast<unsigned long long*>(&s_slice[index_of(r) / (EPT * kThreads)]), (unsigned long long)(wt * kRowOne + 0.5));
    }
    draw_slice(u * (1.0 + kBinNoise), kept);
}

uint64_t up256(uint64_t b) { return (b + 255) & ~255ull; }

// Elements a thread: enough slices to fill the CUs with the rows there are, at most kMaxSlices of them.
uint32_t elements_per_thread(uint32_t rows, uint32_t V) {
    for (uint32_t e : {2u, 4u})
        if ((uint64_t)rows * ((V + e * kThreads - 1) / (e * kThreads)) <= 256 && (V + e * kThreads - 1) / (e * kThreads) <= kMaxSlices)
            return e;
    return kMaxEpt;
}

struct Layout {
    uint32_t ept, nsl, list_stride;
    uint64_t counters, lists, hist, bytes;
};
Layout layout(uint32_t rows, uint32_t V) {
    Layout y;
    y.ept = elements_per_thread(rows, V);
    y.nsl = (V + y.ept * kThreads - 1) / (y.ept * kThreads);
    y.list_stride = y.nsl * kLeanCap > kListCap ? y.nsl * kLeanCap : kListCap;
    y.counters = up256((uint64_t)rows * y.nsl * sizeof(SliceRec));
    y.lists = y.counters + up256((uint64_t)rows * 8);
    y.hist = y.lists + up256((uint64_t)rows * y.list_stride * 8);
    y.bytes = y.hist + up256((uint64_t)rows * y.nsl * kBins * 8);
    return y;
}

template <class T, int EPT>
void launch(hipStream_t s, const Layout& y, const T* logits, uint32_t rows, uint32_t V, uint64_t stride,
            const vsl_row_sampler* params, const float* u, const Work& w, uint32_t* tokens, float* probs) {
    const dim3 grid(y.nsl, rows);
    k_rows_scan<T, EPT><<<grid, kThreads, 0, s>>>(logits, V, stride, params, w);
    k_rows_pick<T, EPT><<<grid, kThreads, 0, s>>>(logits, V, stride, params, u, w, tokens, probs);
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
    const Work w{reinterpret_cast<SliceRec*>(base), reinterpret_cast<uint32_t*>(base + y.counters),
                 reinterpret_cast<uint64_t*>(base + y.lists), reinterpret_cast<uint64_t*>(base + y.hist), y.list_stride};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto go = [&](auto* l) {
        if (y.ept == 2) launch<std::remove_const_t<std::remove_pointer_t<decltype(l)>>, 2>(s, y, l, rows, V, stride, params, u, w, tokens, probs);
        else if (y.ept == 4) launch<std::remove_const_t<std::remove_pointer_t<decltype(l)>>, 4>(s, y, l, rows, V, stride, params, u, w, tokens, probs);
        else launch<std::remove_const_t<std::remove_pointer_t<decltype(l)>>, 8>(s, y, l, rows, V, stride, params, u, w, tokens, probs);
    };
    if (dtype == VSL_DT_F32) go(static_cast<const float*>(logits));
    else go(static_cast<const vsl_half*>(logits));
    HIP_TRY(hipGetLastError());
    return VSL_OK;
}
