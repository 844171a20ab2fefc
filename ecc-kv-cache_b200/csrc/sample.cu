// sample.cu -- the next token of every sequence from its logits and a given
// uniform number (sm_100a): temperature, top-k, top-p, min-p.
//
// Per row, x the logits as fp32 (NaN counts as -inf), M = max x, T the
// temperature:
//   w_i = exp((x_i - M) / T)                       (w = 1 where x_i = M)
//   top-k: the k largest x; top-p: of those, in descending order, every token
//   before which less than p of the mass lies; min-p: w_i >= min_p;
//   equal logits rank by ascending index
//   token = first index, ascending, with cumulative kept mass > u * total
//   logprob = log(w_token / total).  T = 0: the first maximum, logprob 0.
//   A row without a logit above -inf: token -1, logprob -inf.
//
// No sort of the row: one cluster of CTAs per row keeps it in shared memory.
// A pass bins the tokens by their distance from the maximum:
//   top-k: counts alone.  When everything down to the bin of the k-th fits the
//     list (4096), one CTA sorts that and finishes, top-p and min-p included.
//   top-p alone: counts and places inside the bins, from which each bin's mass
//     is estimated; a second pass adds up the exact masses above the bins around
//     the estimated end and lists theirs, and the draw takes its sums over.
//   otherwise (a long top-k list with top-p; an end that the estimate missed):
//     counts and exact masses, and the bin in which the set ends is sorted on its
//     own.  A bin of too many (nearly) equal logits is descended by key bits
//     (cluster_select.cuh).
// Then a pass draws.  Masses are sums of fixed-point numbers w * 2^S, so they do
// not depend on the order of the additions, and atomics give the same bits every
// time.  S leaves room for the row's own sum (62 - ceil(log2) of a bound of it:
// of top-p from its counts, of a long top-k list from its entries, without a
// filter from a pass of fp32 exponentials, 2 us for one row and 4 for 64): 41 to
// 61 bits behind the point, and a running sum of V tokens is off by at most V
// 2^-61 + 2^-45 of the whole, however long and flat the tail.  (With room for V
// maxima in every row, 2^20 - 1 equal logits 14 below one peak were known to
// 2^-23, and one draw in a hundred fell on a neighbour.)
// A drawn token hangs on which side of a sum u * total falls: fp32 exponentials
// would move one draw in a few thousand, so w is computed in fp64 to 2^-45
// relative, by table and polynomial:
//   2^y = 2^n 2^(i / 512) 2^f,  2^f = 1 + c1 f + c2 f^2 + c3 f^3,  ck = ln(2)^k / k!,
// |f| <= 2^-10: the polynomial is off by 2^-46.7 (Tang, Table-driven implementation
// of the exponential function, 1989).
//
// Measured per call at 128256 bf16 logits: top-k 50 + top-p 0.9 17 us for one
// row and 27 us for 64; top-p 0.9 alone 31 and 55 us; no filter 12 and 25 us;
// greedy 4 and 7 us.  A row alone is bound by the latency of its phases (about
// a microsecond per cluster barrier with the sums around it); 64 rows by the
// issue of their passes, two CTAs a row: weights 10 us (45 instructions a token,
// 8 of them fp64), counts by distance 12 us (two shared-memory atomics), weights
// with the list of the last bin 16 us.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "cluster_select.cuh"

namespace ecc {

int launch_status();
int sm_count();

namespace samp {

using namespace sel;

constexpr int kTab = 512;

struct Args {
    const void *logits;
    int64_t row_stride;
    int B, V;
    const float *u;
    const float *temperature, *top_p, *min_p;  // per row, or null: the value below
    const int *top_k;
    float temperature0, top_p0, min_p0;
    int top_k0;
    int64_t *token;
    float *logprob;
    int slice;  // elements of a row per CTA
};

template <class T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// A value's key (cluster_select.cuh).  fp16 values have 10 bits of mantissa
// behind fp32's exponent, bf16 values 7: the bits below `key_low` say nothing
// and are cleared, which saves a pass or two of a descent.
template <class T>
__host__ __device__ constexpr int key_low() {
    return std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 13 : 16;
}
template <class T>
__device__ __forceinline__ uint32_t value_key(float x) { return key_of(x) & (0xffffffffu << key_low<T>()); }
template <class T>
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~(k | ~(0xffffffffu << key_low<T>())));
}

struct Settings {  // of a row
    float temp, top_p, min_p, u;
    int top_k;
};
struct Work {
    Shared sel;
    Settings first, set;  // as this CTA read them; the cluster's: the first CTA's
    unsigned long long tot_mass[kBins];  // the cluster's masses and counts, this CTA's share of the bins
    uint32_t tot_count[kBins];
    double tab[kTab];
    float best;
    uint32_t best_at;
    float cta_best;       // of this CTA, read by the cluster
    uint32_t cta_best_at;
    uint64_t bound[kMaxCluster];  // of the CTAs' masses, written by each of them
    uint32_t listed;      // entries of this CTA's list
    uint32_t kth, cut;    // written by rank 0
    uint64_t bin_mass;
    unsigned long long part[kWarps];
    int lo, hi;           // the part that holds the drawn token, and the mass before it
    uint64_t before;
};
// In the place of the count descent's bins: this CTA's counts and masses of
// the first pass, later the list of one bin's tokens.
struct Bins {
    uint32_t count[kBins];
    union {
        unsigned long long mass[kBins];
        uint32_t place[kBins];
    };
};
static_assert(sizeof(Bins) <= sizeof(Shared::hist), "room for the bins");

// w * 2^S as an integer.  With y = (x - M) log2(e) / T, -63 < y <= 0, one product adds y to 192 + 2^-10, whose last
// bit is 2^-45: the sum's bits are, from the top, floor(y') + 64 (y' = y + 2^-10), the first 9 bits behind the point
// and the rest, from which 2^-10 is taken off again: |f| <= 2^-10.
struct Mass {
    const double *tab;        // 2^(i / 512) 2^(S - 64)
    double best, scale;
    float cut;                // what lies below has w < 2^-62.8: nothing of it is left by the rounding to 2^-S, S <= 61
    __device__ __forceinline__ Mass(const double *tab_, float best_, float temp) : tab(tab_), best(best_) {
        const double t = temp < INFINITY ? (double)temp : 1e300;
        scale = 1.442695040888963407 / t;
        cut = __double2float_ru(best - 43.6 * t);  // finite: x = -inf lies below
    }
    __device__ __forceinline__ uint64_t operator()(float x) const {  // the maximum itself: exactly 2^S
        const double d = (double)x - best, at = fma(d, scale, 192.0 + 1.0 / 1024.0);
        const double y = x >= cut ? at : 129.0;  // (2^-63)
        const int hi = __double2hiint(y);
        const double f = __hiloint2double((hi & 0xf) | 0x40600000, __double2loint(y)) - (128.0 + 1.0 / 1024.0);
        constexpr double c1 = 0.693147180559945309, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;  // 2^f = e^(f ln 2)
        const double p = fma(f, fma(f, fma(f, c3, c2), c1), 1.0);
        const double t = tab[(hi >> 4) & (kTab - 1)];
        const double w = __hiloint2double(__double2hiint(t) + ((hi & 0xfe000) << 7), __double2loint(t));  // its exponent by addition
        return __double2ull_rn(p * w);
    }
};

// A bound of a row's mass, as a sum of integers, whatever the order: w in units of 2^-kBoundBits, to the nearest, in
// the low bits of a float of exponent 23.  x - M, the scale and their product are off by 2^-24 of themselves, ex2 by
// 2^-22: by less than 2^-16 of w where w reaches half a unit, and smaller ones are covered by a unit a token.
constexpr int kBoundBits = 22;
struct Bound {
    float best, scale;
    bool most;  // taken for n maxima: every weight is whole (T infinite), or the differences leave fp32's range
    __device__ __forceinline__ Bound(float best_, float temp)
        : best(best_), scale(fminf(1.44269504f / temp, 3e38f)), most(!(temp < INFINITY) || best > 1e31f) {}
    __device__ __forceinline__ uint32_t operator()(float x) const {
        float e;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(x - best, scale, (float)kBoundBits)));
        return __float_as_uint(e + 8388608.0f) - 0x4b000000u;
    }
    // The fixed-point position S, 41 to 61, of n <= 2^20 tokens whose bounds add up to `sum`: their masses together stay
    // below 2^62 (and half a unit each); unless `most`, 2^-S is less than 2^-61 of their sum and n 2^-21.
    __device__ __forceinline__ int bits(uint64_t sum, int n) const {
        const uint64_t all = most ? (uint64_t)n << kBoundBits : sum + (sum >> 15) + (uint64_t)n;
        return min(61, 62 + kBoundBits - (64 - __clzll((long long)(all - 1))));  // 62 - ceil(log2(all 2^-22))
    }
};

// floor(f * total) and whether something was cut off, without rounding: f in
// (0, 1) is an integer of 24 bits times a power of two.  Sums that lie on a
// border exactly (equal logits, a number of 1/2) fall to the right side.
__device__ __forceinline__ uint64_t share_of(float f, uint64_t total, bool *cut_off) {
    const uint32_t bits = __float_as_uint(f), e = bits >> 23;
    const int s = 150 - (int)e;  // f = m * 2^-s, s >= 24
    const uint64_t m = (bits & 0x7fffffu) | 0x800000u;
    *cut_off = true;
    if (e == 0 || s >= 128) return 0;
    const uint64_t hi = __umul64hi(m, total), lo = m * total;
    if (s < 64) {
        *cut_off = (lo & ((1ull << s) - 1)) != 0;
        return (hi << (64 - s)) | (lo >> s);
    }
    *cut_off = lo != 0 || (hi & ((1ull << (s - 64)) - 1)) != 0;
    return hi >> (s - 64);
}

// Sum of v over the cluster's threads.
__device__ __forceinline__ uint64_t cluster_sum(Shared &sh, const Cluster &cl, uint64_t v) {
    uint64_t all;
    block_exclusive(v, sh.warp64, &all);
    if (threadIdx.x == 0) sh.cta64 = all;
    cl.sync();
    all = 0;
    for (unsigned r = 0; r < cl.num_blocks(); ++r) all += *of_rank(cl, &sh.cta64, r);
    cl.sync();
    return all;
}

// Two sums at once: a pair per CTA in the first CTAs' entries of `share`.
__device__ __forceinline__ ulonglong2 cluster_sum2(Shared &sh, const Cluster &cl, uint64_t x, uint64_t y) {
    static_assert(kMaxCluster >= 16, "two entries for each of 8 CTAs");
    const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    uint64_t ax, ay;
    block_exclusive(x, sh.warp64, &ax);
    block_exclusive(y, sh.warp64, &ay);
    if (threadIdx.x < ranks) {
        uint64_t *to = of_rank(cl, sh.cross.share, threadIdx.x);
        to[2 * rank] = ax;
        to[2 * rank + 1] = ay;
    }
    cl.sync();
    ulonglong2 s = make_ulonglong2(0, 0);
    for (int r = 0; r < ranks; ++r) s.x += sh.cross.share[2 * r], s.y += sh.cross.share[2 * r + 1];
    cl.sync();  // share may be written again
    return s;
}

// The top-p threshold inside a bin of many (nearly) equal logits, by the bits
// of their keys: a descent like kth_largest's whose digits are found by mass.
// Returns the new threshold key and cut.
template <class T, class Load, class Keep, class BinOf>
__device__ __noinline__ uint2 mass_descent(Shared &sh, Load load, Keep keep, BinOf bin_of, Mass mass, int n, int base,
                                           int bin, uint64_t above, uint64_t want, uint32_t kth, uint32_t cut) {
    const Cluster cl;
    unsigned long long *from = reinterpret_cast<unsigned long long *>(sh.hist), *to = from + kBins;
    const int tid = threadIdx.x, low = key_low<T>();
    uint32_t prefix = 0, mask = 0;
    uint64_t at = 0;
    for (int top = 32; top > low;) {
        const int bits = min(11, top - low), shift = top - bits;
        for (int i = tid; i < kBins; i += kThreads) from[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const float x = load(i);
            const uint32_t kx = value_key<T>(x);
            if ((kx & mask) != prefix || !keep(kx, i) || bin_of(x) != bin) continue;
            const uint64_t w = mass(x);
            if (w) atomicAdd(&from[kBins - 1 - ((kx >> shift) & ((1u << bits) - 1))], (unsigned long long)w);
        }
        cl.sync();
        cluster_share(cl, from, to);
        share_sums(sh.cross, cl, to, sh.warp64);
        const Crossing f = crossing(sh.cross, cl, to, want - above, sh.warp64);
        above += f.before;
        at = f.here;
        prefix |= (kBins - 1 - f.slot) << shift;
        mask |= ((1u << bits) - 1) << shift;
        top = shift;
    }
    // every kept token with this key has the same mass: the smallest m with above + m w >= want > above
    const uint64_t w = max((uint64_t)1, mass(key_value<T>(prefix)));
    const uint64_t m = (want - above + w - 1) / w, count = at / w;
    uint32_t new_cut = prefix == kth ? cut : 0xffffffffu;
    if (m < count)
        new_cut = tie_cut(sh, cl, n, base, (uint32_t)m, [&](int i) {
            const uint32_t kx = value_key<T>(load(i));
            return kx == prefix && keep(kx, i);
        });
    return make_uint2(prefix, new_cut);
}

template <class T, bool kCached>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    Work &wk = *reinterpret_cast<Work *>(dyn);
    Shared &sh = wk.sel;
    T *x_s = reinterpret_cast<T *>(dyn + (sizeof(Work) + 15) / 16 * 16);
    const Cluster cl;
    const int C = cl.num_blocks(), rank = cl.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C;
    for (int i = tid; i < kTab; i += kThreads) wk.tab[i] = exp2((double)i / kTab - 64.0);
    if (tid == 0) wk.listed = 0;
    pdl_trigger();
    pdl_wait();
    // one thread reads the row's settings for the whole cluster, which branches on them together
    if (tid == 0) {
        wk.first.temp = a.temperature ? __ldg(a.temperature + row) : a.temperature0;
        wk.first.top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p0;
        wk.first.min_p = a.min_p ? __ldg(a.min_p + row) : a.min_p0;
        wk.first.u = __ldg(a.u + row);
        wk.first.top_k = a.top_k ? __ldg(a.top_k + row) : a.top_k0;
    }

    const int base = min(a.V, rank * a.slice), n = min(a.V, base + a.slice) - base;
    const T *x_g = reinterpret_cast<const T *>(a.logits) + (int64_t)row * a.row_stride + base;
    // Element i: NaN counts as -inf; with an infinite maximum, the maximum as 0 and all else as -inf (`infinite`).
    // A slice in shared memory is put that way once.
    bool infinite = false;
    auto load = [x_s, x_g, &infinite](int i) {
        if (kCached) return to_float<T>(x_s[i]);
        const float x = to_float<T>(x_g[i]);
        if (infinite) return x == INFINITY ? 0.0f : -INFINITY;
        return x != x ? -INFINITY : x;
    };

    // ---- the row, its maximum and the maximum's first place
    float best = -INFINITY;
    uint32_t best_at = 0xffffffffu;
    if (kCached) {
        constexpr int kVec = 16 / sizeof(T);
        const int n_wide = ((uintptr_t)x_g & 15) == 0 ? n / kVec : 0;
#pragma unroll 4
        for (int i = tid; i < n_wide; i += kThreads)
            reinterpret_cast<uint4 *>(x_s)[i] = __ldg(reinterpret_cast<const uint4 *>(x_g) + i);
        for (int i = n_wide * kVec + tid; i < n; i += kThreads) x_s[i] = x_g[i];
        __syncthreads();
    }
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads) {
        const float x = load(i);
        if (kCached && x != x) x_s[i] = from_float<T>(-INFINITY);
        if (x > best) best = x, best_at = base + i;  // ascending i: the first of equals; not a NaN
    }
    auto better = [](float x, uint32_t i, float &bx, uint32_t &bi) {
        if (x > bx || (x == bx && i < bi)) bx = x, bi = i;
    };
    auto warp_best = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_at, o), best, best_at);
    };
    warp_best();
    if (lane == 0) sh.warp_a[warp] = __float_as_uint(best), sh.warp_b[warp] = best_at;
    __syncthreads();
    if (warp == 0) {
        best = __uint_as_float(sh.warp_a[lane]), best_at = sh.warp_b[lane];
        warp_best();
        if (lane == 0) wk.cta_best = best, wk.cta_best_at = best_at;
    }
    cl.sync();
    if (warp == 0) {
        best = -INFINITY, best_at = 0xffffffffu;
        if (lane < C) best = *of_rank(cl, &wk.cta_best, lane), best_at = *of_rank(cl, &wk.cta_best_at, lane);
        warp_best();
        if (lane == 0) wk.best = best, wk.best_at = best_at, wk.set = *of_rank(cl, &wk.first, 0);
    }
    cl.sync();  // also: nobody reads a CTA's shared memory after it may have left
    best = wk.best;
    best_at = wk.best_at;
    const float temp = wk.set.temp;
    if (best == -INFINITY || !(temp > 0.0f)) {  // cluster-uniform
        if (rank == 0 && tid == 0) {
            a.token[row] = best == -INFINITY ? -1 : (int64_t)best_at;
            if (a.logprob) a.logprob[row] = best == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    if (best == INFINITY) {  // cluster-uniform
        if (kCached) {
            for (int i = tid; i < n; i += kThreads) {  // each thread the elements that it alone has read so far
                const bool top = to_float<T>(x_s[i]) == INFINITY;
                x_s[i] = from_float<T>(top ? 0.0f : -INFINITY);
            }
        }
        infinite = true;
        best = 0.0f;
    }
    if (kCached) __syncthreads();  // the slice as the other threads read it from here on

    // ---- masses: not before it is known how many bits S behind the point the sums leave room for
    const Mass mass(wk.tab, best, temp);
    const Bound bound(best, temp);
    const float mp = wk.set.min_p;
    double unit = 0.0;   // 2^S
    uint64_t least = 0;  // the smallest mass that min-p leaves
    auto set_bits = [&](int S) {  // by the whole block
        unit = __hiloint2double((1023 + S) << 20, 0);
        for (int i = tid; i < kTab; i += kThreads) wk.tab[i] *= unit;
        // w >= min_p as whole masses; the most likely token stays in any case
        least = mp > 0.0f ? (uint64_t)ceil(fmin((double)mp, 1.0) * unit) : 0;
        __syncthreads();
    };
    auto set_bits_by_a_pass = [&]() {
        uint32_t sum = 0;   // of at most 128 tokens (V <= 2^20): 2^29
        if (!bound.most) {  // cluster-uniform
#pragma unroll 8
            for (int i = tid; i < n; i += kThreads) sum += bound(load(i));
        }
        uint64_t all;
        block_exclusive((uint64_t)sum, sh.warp64, &all);
        if (tid < C) of_rank(cl, wk.bound, tid)[rank] = all;
        cl.sync();
        all = 0;
        for (int r = 0; r < C; ++r) all += wk.bound[r];
        set_bits(bound.bits(all, a.V));
    };

    // What is kept so far: keys above `kth`, equal ones below the row position `cut`.
    uint32_t kth = 0, cut = 0xffffffffu;
    auto key = [&](int i) { return value_key<T>(load(i)); };
    auto keep = [&](uint32_t x, int i) { return x > kth || (x == kth && (uint32_t)(base + i) < cut); };

    const int k = wk.set.top_k;
    const float p = wk.set.top_p;
    const bool by_count = k > 0 && k < a.V, by_mass = p < 1.0f;
    const float u = wk.set.u;
    // cumulative mass > u * total, of whole masses: > floor(u * total); a number of 1 or more takes the last
    // kept token, one that is not above 0 the first
    auto need_of = [u](uint64_t total) -> uint64_t {
        bool ignored;
        return !(u > 0.0f) ? 0 : u < 1.0f ? share_of(u, total, &ignored) : total - 1;
    };
    // ceil(p * total): whole sums below it are below p * total.  p <= 0: the first token alone.
    auto want_of = [p](uint64_t total) {
        bool more = true;
        const uint64_t want = p > 0.0f ? share_of(p, total, &more) : 0;
        return want + (more ? 1 : 0);
    };

    bool parts_known = false;  // wk.part holds the kept masses of the warps' parts
    if (by_count || by_mass) {
        // ---- counts and masses by the distance from the maximum, in bins of 1/64 of an e-fold: monotone in
        // x, and spread however the logits lie
        Bins &bins = *reinterpret_cast<Bins *>(sh.hist);
        unsigned long long *list = reinterpret_cast<unsigned long long *>(sh.hist);
        // (above 0 for an infinite temperature too: a logit of -inf is infinitely far, never NaN bins, which would
        // pass every test for a bin; finite logits are at most 8 bins off then, in their order)
        const float inv_bin = fmaxf(fminf(64.0f / temp, 3e38f), 1.2e-38f);
        auto distance = [best, inv_bin](float x) { return (best - x) * inv_bin; };  // in bins; -inf: infinity
        auto bin_of = [distance](float x) {
            const float d = distance(x);
            return d < (float)(kBins - 1) ? (int)d : kBins - 1;
        };
        // What a pass adds up per bin: counts, and with them nothing, the places inside the bin (a sum of
        // kPlaces-ths of its width), or the masses.
        constexpr int kCount = 0, kPlace = 1, kMassToo = 2;
        constexpr float kPlaces = 1024.0f;
        auto count_bins = [&](auto what) {
            constexpr bool kMass = decltype(what)::value == kMassToo, kPlaced = decltype(what)::value == kPlace;
            for (int i = tid; i < kBins; i += kThreads) {
                bins.count[i] = 0;
                if (kMass) bins.mass[i] = 0;
                if (kPlaced) bins.place[i] = 0;
            }
            __syncthreads();
            // everything far below goes to the last bin: added up per thread first
            uint32_t far_count = 0;
            uint64_t far_mass = 0;
#pragma unroll 4
            for (int i = tid; i < n; i += kThreads) {
                const float x = load(i), d = distance(x);
                const uint64_t w = kMass ? mass(x) : 0;
                if (!(d < (float)(kBins - 1))) {
                    ++far_count;
                    far_mass += w;
                } else {
                    const int b = (int)d;
                    atomicAdd(&bins.count[b], 1u);
                    if (kMass) atomicAdd(&bins.mass[b], (unsigned long long)w);
                    // at most 2^20 tokens, fewer than 2^10 places each
                    if (kPlaced) {
                        const float fb = __int_as_float(0x4b000000 | b) - 8388608.0f;  // (float)b
                        atomicAdd(&bins.place[b], (uint32_t)((d - fb) * kPlaces));
                    }
                }
            }
            far_count = __reduce_add_sync(0xffffffffu, far_count);
            if (kMass) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) far_mass += __shfl_xor_sync(0xffffffffu, far_mass, o);
            }
            if (lane == 0 && far_count) {
                atomicAdd(&bins.count[kBins - 1], far_count);
                if (kMass) atomicAdd(&bins.mass[kBins - 1], (unsigned long long)far_mass);
            }
            cl.sync();
            cluster_share(cl, bins.count, wk.tot_count);
            if (kMass) cluster_share(cl, bins.mass, wk.tot_mass);
            if (kPlaced) cluster_share(cl, bins.place, wk.tot_mass);
            share_sums(sh.cross, cl, wk.tot_count, sh.warp64);  // its barrier: the bins' place is free
        };
        // Puts the kept ones of a warp's elements as (key, ~row position) into the CTA's list (room for kList) or,
        // when few are expected, into rank 0's, which saves join_lists' barrier.
        unsigned long long *list_to = list;
        uint32_t *listed_to = &wk.listed;
        auto straight_to_rank0 = [&](uint32_t expected) {  // at most `expected` entries in all; cluster-uniform
            const bool yes = expected <= 512;
            list_to = yes ? of_rank(cl, list, 0) : list;
            listed_to = yes ? of_rank(cl, &wk.listed, 0) : &wk.listed;
            return yes;
        };
        // A lane's elements come as bits: bit j for element first + j step.
        auto append = [&](uint32_t mask, int first, int step) {
            if (kth != 0) {  // cluster-uniform
                for (uint32_t m = mask; m; m &= m - 1) {
                    const int i = first + (__ffs(m) - 1) * step;
                    if (!keep(value_key<T>(load(i)), i)) mask &= ~(m & -m);
                }
            }
            if (!__any_sync(0xffffffffu, mask)) return;
            const uint32_t c = __popc(mask);
            uint32_t upto = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            uint32_t at = 0;
            if (lane == 31) at = atomicAdd(listed_to, upto);
            at = __shfl_sync(0xffffffffu, at, 31) + upto - c;
            for (; mask; mask &= mask - 1, ++at) {
                const int i = first + (__ffs(mask) - 1) * step;
                if (at < kList) list_to[at] = ((unsigned long long)value_key<T>(load(i)) << 32) | (uint32_t)~(uint32_t)(base + i);
            }
        };
        // After a cluster barrier: brings the lists to rank 0 and sorts them there, descending.  Returns how
        // many entries there are; more than kList: no list.
        auto sorted = [&](bool at_rank0) {
            const int m = at_rank0 ? (int)wk.listed : (int)join_lists(cl, list, &wk.listed);
            if (rank == 0 && m <= kList) sort_descending(list, m);
            return m;  // at_rank0: known there
        };
        // The kept tokens of bins b0 .. b1, at most `expected`, in rank 0's list, sorted.  Returns their number there.
        auto gather = [&](int b0, int b1, uint32_t expected) {
            const bool at_rank0 = straight_to_rank0(expected);
            const float d0 = (float)b0, d1 = b1 < kBins - 1 ? (float)(b1 + 1) : __int_as_float(0x7fc00000);
            for (int i0 = warp * 32; i0 < n; i0 += kThreads * 32) {
                uint32_t mask = 0;
                for (int j = 0; j < 32 && i0 + j * kThreads < n; j += 2) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int i = i0 + (j + q) * kThreads + lane;
                        const float d = i < n ? distance(load(i)) : -1.0f;
                        const bool hit = !(d < d0) & !(d >= d1);
                        mask |= (uint32_t)hit << (j + q);
                    }
                }
                append(mask, i0 + lane, kThreads);
            }
            cl.sync();
            return min(sorted(at_rank0), kList);
        };
        auto listed_mass = [&](int i) { return mass(key_value<T>((uint32_t)(list[i] >> 32))); };
        // Rank 0's finding reaches the cluster; the list is free again.
        auto publish = [&](unsigned long long entry) {
            for (int r = 0; r < C; ++r)
                *of_rank(cl, &wk.kth, r) = (uint32_t)(entry >> 32), *of_rank(cl, &wk.cut, r) = ~(uint32_t)entry + 1;
        };
        auto take = [&]() {
            cl.sync();
            kth = wk.kth;
            cut = wk.cut;
            if (tid == 0) wk.listed = 0;
            cl.sync();
        };

        Crossing at_k{};
        if (by_count) {
            count_bins(std::integral_constant<int, kCount>());
            at_k = crossing(sh.cross, cl, wk.tot_count, (uint64_t)k, sh.warp64);
            if (at_k.before + at_k.here <= kList) {
                // everything that may be kept fits the list: rank 0 finishes alone
                gather(0, (int)at_k.slot, (uint32_t)(at_k.before + at_k.here));
                if (rank != 0) return;  // nobody reads the other CTAs' shared memory any more
                int kept = k;
                if (k <= 256) {  // room for k maxima leaves S >= 54: k roundings are at most 2^-47 of the sum
                    set_bits(min(61, 62 - (32 - __clz(k - 1))));
                } else {
                    uint32_t sum = 0;
                    for (int i = tid; i < k; i += kThreads) sum += bound(key_value<T>((uint32_t)(list[i] >> 32)));
                    uint64_t all;
                    block_exclusive((uint64_t)sum, sh.warp64, &all);
                    set_bits(bound.bits(all, k));
                }
                if (by_mass || least > 0) {
                    uint64_t sum = 0, want = 0, total;
                    if (by_mass) {
                        for (int i = tid; i < kept; i += kThreads) sum += listed_mass(i);
                        block_exclusive(sum, sh.warp64, &total);
                        want = want_of(total);
                    }
                    uint64_t before = 0;
                    uint32_t stay = 0;
                    for (int i0 = 0; i0 < kept; i0 += kThreads) {  // block-uniform
                        const int i = i0 + tid;
                        const uint64_t w = i < kept ? listed_mass(i) : 0;
                        uint64_t all;
                        const uint64_t mine = before + block_exclusive(w, sh.warp64, &all);
                        // both conditions hold for a first part of the list
                        stay += i < kept && (i == 0 || ((!by_mass || mine < want) && w >= least)) ? 1 : 0;
                        before += all;
                    }
                    uint32_t all;
                    block_exclusive(stay, sh.warp_a, &all);
                    kept = (int)all;
                }
                // by row position, and the draw
                for (int i = tid; i < kept; i += kThreads) list[i] = (list[i] << 32) | (list[i] >> 32);
                __syncthreads();
                sort_descending(list, kept);
                auto drawn_mass = [&](int i) { return mass(key_value<T>((uint32_t)list[i])); };
                uint64_t sum = 0, total;
                for (int i = tid; i < kept; i += kThreads) sum += drawn_mass(i);
                block_exclusive(sum, sh.warp64, &total);
                const uint64_t need = need_of(total);
                uint64_t before = 0;
                for (int i0 = 0; i0 < kept; i0 += kThreads) {
                    const int i = i0 + tid;
                    const uint64_t w = i < kept ? drawn_mass(i) : 0;
                    uint64_t all;
                    const uint64_t mine = before + block_exclusive(w, sh.warp64, &all);
                    if (mine <= need && need < mine + w) {
                        a.token[row] = (uint32_t)~(uint32_t)(list[i] >> 32);
                        if (a.logprob) a.logprob[row] = (float)log((double)w / (double)total);
                    }
                    before += all;
                }
                return;
            }
            set_bits_by_a_pass();
        }
        if (by_mass && !by_count) {
            // ---- top-p alone: the bins' masses from counts and places tell where it ends, to 10^-4 of the mass;
            // one pass over exact masses then adds up what surely stays and lists what lies near the end.
            count_bins(std::integral_constant<int, kPlace>());
            const int W = kBins / C;
            for (int i = tid; i < W; i += kThreads) {
                // e^(-f/64), 0 <= f < 1, as its chord less half its sag: off by 1.6e-5.  A place is off by half
                // of 1/1024 of a bin: 8e-6.  fp32 here: 2e-7.  Everything in the last bin weighs at most e^-32.
                const float n_b = (float)wk.tot_count[i];
                const float f = ((float)(uint32_t)wk.tot_mass[i] + 0.5f * n_b) * (1.0f / kPlaces);
                constexpr float kChord = 0.015503561f;  // 1 - e^(-1/64)
                const float m = expf(-(float)(rank * W + i) * (1.0f / 64.0f)) * (n_b * (1.0f - 1.52e-5f) - kChord * f);
                wk.tot_mass[i] = (unsigned long long)(fmaxf(m, 0.0f) * 1099511627776.0f);  // 2^40
            }
            __syncthreads();
            const uint64_t about = share_sums(sh.cross, cl, wk.tot_mass, sh.warp64);
            // with 1/8192 for its error, a bound of the row's mass too (the last bin counts at its near edge)
            set_bits(bound.bits((about >> (40 - kBoundBits)) + (about >> (53 - kBoundBits)), a.V));
            const uint64_t slack = about / 8192, aim = want_of(about);
            const uint64_t ends[2] = {aim > slack ? aim - slack : 1, min(aim + slack, about)};
            Crossing at[2];
            crossings(sh.cross, cl, wk.tot_mass, ends, at, sh.warp64);
            const int b0 = (int)at[0].slot, b1 = ends[1] < about ? (int)at[1].slot : kBins - 1;
            {
                const float d0 = (float)b0, d1 = b1 < kBins - 1 ? (float)(b1 + 1) : 3e38f;
                // (mass beyond d1, at a vast temperature: the list misses the end, and the exact search below finds it)
                int lo, hi;
                warp_part(n, lo, hi);
                uint64_t all = 0, above = 0, part = 0;
                auto add_up = [&](auto by_min) {  // with min-p the kept masses are not all of those above
                    for (int i0 = lo; i0 < hi; i0 += 32 * 32) {
                        uint32_t mask = 0;
                        for (int j = 0; j < 32 && i0 + 32 * j < hi; j += 4) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const int i = i0 + 32 * (j + q) + lane;
                                const float x = i < hi ? load(i) : -INFINITY, d = distance(x);
                                const uint64_t w = mass(x);
                                all += w;
                                const bool stays = d < d0;
                                const uint64_t kept = stays ? w : 0;
                                above += kept;
                                if (decltype(by_min)::value) part += kept >= least ? kept : 0;
                                const bool hit = !stays & (d < d1);
                                mask |= (uint32_t)hit << (j + q);
                            }
                        }
                        append(mask, i0 + lane, 32);
                    }
                };
                if (least > 0) {
                    add_up(std::true_type());
                } else {
                    add_up(std::false_type());
                    part = above;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
                if (lane == 0) wk.part[warp] = part;
                const ulonglong2 sums = cluster_sum2(sh, cl, all, above);
                const uint64_t want = want_of(sums.x);
                above = sums.y;
                const int m = sorted(false);  // (cluster_sum2 ended with a barrier)
                if (rank == 0) {
                    if (tid == 0) for (int r = 0; r < C; ++r) *of_rank(cl, &wk.kth, r) = 0;
                    __syncthreads();
                    // the part of a row position: its CTA's slice, its warp's share of the slice
                    uint64_t before = above;
                    for (int i0 = 0; i0 < m && m <= kList; i0 += kThreads) {  // block-uniform
                        const int i = i0 + tid;
                        const uint64_t w = i < m ? listed_mass(i) : 0;
                        uint64_t sum;
                        const uint64_t mine = before + block_exclusive(w, sh.warp64, &sum);
                        if (i < m && mine < want) {
                            if (want <= mine + w) publish(list[i]);
                            if (w >= least) {
                                const int at = (int)~(uint32_t)list[i], r = at / a.slice;
                                atomicAdd(of_rank(cl, wk.part, r) + part_of(min(a.slice, a.V - r * a.slice), at - r * a.slice),
                                          (unsigned long long)w);
                            }
                        }
                        before += sum;
                    }
                }
                take();
                parts_known = kth != 0;  // no key is 0
                if (!parts_known) cut = 0xffffffffu;  // the list was too short: the exact search below
            }
        }
        if (by_mass && !parts_known) count_bins(std::integral_constant<int, kMassToo>());
        if (by_count) {
            const int b = (int)at_k.slot;
            const uint32_t rest = (uint32_t)k - (uint32_t)at_k.before;
            uint64_t dropped = 0;
            if (at_k.here <= kList) {
                const int m = gather(b, b, (uint32_t)at_k.here);
                if (rank == 0) {
                    if (tid == 0) publish(list[(rest - 1) & (kList - 1)]);
                    uint64_t mine = 0;
                    if (by_mass)
                        for (int i = rest + tid; i < m; i += kThreads) mine += listed_mass(i);
                    block_exclusive(mine, sh.warp64, &dropped);
                    if (tid < C) *of_rank(cl, &wk.bin_mass, tid) = dropped;
                }
                take();
                dropped = wk.bin_mass;
            } else {
                // a bin with more equal or nearly equal logits than the list holds
                uint32_t ties, equal;
                const uint32_t x = kth_largest(sh, cl, key, n, (uint32_t)k, key_low<T>(), &ties, &equal);
                if (ties < equal) cut = tie_cut(sh, cl, n, base, ties, [&](int i) { return key(i) == x; });
                kth = x;
                if (by_mass) {
                    uint64_t mine = 0;
                    for (int i = tid; i < n; i += kThreads)
                        if (bin_of(load(i)) == b && !keep(key(i), i)) mine += mass(load(i));
                    dropped = cluster_sum(sh, cl, mine);
                }
            }
            if (by_mass) {
                // the masses of what is left: the bins below are empty, this one has lost `dropped`
                const int W = kBins / C;
                for (int i = tid; i < W; i += kThreads) {
                    if (rank * W + i > b) wk.tot_mass[i] = 0;
                    if (rank * W + i == b) wk.tot_mass[i] -= dropped;
                }
                __syncthreads();
            }
        }
        if (by_mass && !parts_known) {
            const uint64_t want = want_of(share_sums(sh.cross, cl, wk.tot_mass, sh.warp64));
            const Crossing at = crossing(sh.cross, cl, wk.tot_mass, want, sh.warp64);
            const int b = (int)at.slot, W = kBins / C;
            const uint32_t count = *of_rank(cl, wk.tot_count + b % W, b / W);
            if (count <= kList) {
                const int m = gather(b, b, count);
                if (rank == 0) {
                    uint64_t before = at.before;
                    for (int i0 = 0; i0 < m; i0 += kThreads) {  // block-uniform
                        const int i = i0 + tid;
                        const uint64_t w = i < m ? listed_mass(i) : 0;
                        uint64_t all;
                        const uint64_t mine = before + block_exclusive(w, sh.warp64, &all);
                        if (mine < want && want <= mine + w) publish(list[i]);
                        before += all;
                    }
                }
                take();
            } else {
                const auto kept = [kth, cut, base](uint32_t x, int i) {
                    return x > kth || (x == kth && (uint32_t)(base + i) < cut);
                };
                const uint2 found = mass_descent<T>(sh, load, kept, bin_of, mass, n, base, b, at.before, want, kth, cut);
                kth = found.x;
                cut = found.y;
            }
        }
    }

    // ---- the draw: masses of the warps' parts, then the part that holds the number
    if (!by_count && !by_mass) set_bits_by_a_pass();
    auto kept_mass = [&](int i) -> uint64_t {
        const float x = load(i);
        if (!keep(value_key<T>(x), i)) return 0;
        const uint64_t w = mass(x);
        return w >= least ? w : 0;
    };
    int lo, hi;
    warp_part(n, lo, hi);
    uint64_t part = 0;
    if (parts_known) {
        part = wk.part[warp];
    } else {
        if (kth == 0 && least == 0) {  // everything is kept
#pragma unroll 4
            for (int i = lo + lane; i < hi; i += 32) part += mass(load(i));
        } else {
#pragma unroll 4
            for (int i = lo + lane; i < hi; i += 32) part += kept_mass(i);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    }
    uint64_t cta_all;
    uint64_t before = block_exclusive(lane == 0 ? part : 0, sh.warp64, &cta_all);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (tid < C) of_rank(cl, sh.cross.share, tid)[rank] = cta_all;
    cl.sync();  // nobody reads or writes another CTA's shared memory after this
    uint64_t total = 0, cta_before = 0;
    for (int r = 0; r < C; ++r) {
        cta_before += r < rank ? sh.cross.share[r] : 0;
        total += sh.cross.share[r];
    }
    const uint64_t need = need_of(total);
    if (need < cta_before || need >= cta_before + cta_all) return;  // block-uniform
    before += cta_before;
    if (lane == 0 && before <= need && need < before + part) wk.lo = lo, wk.hi = hi, wk.before = before;
    __syncthreads();
    // the part's elements over the block, a run of neighbours per thread
    lo = wk.lo;
    hi = wk.hi;
    const int run = (hi - lo + kThreads - 1) / kThreads;
    const int i0 = lo + tid * run, i1 = min(hi, i0 + run);
    uint64_t mine = 0;
    for (int i = i0; i < i1; ++i) mine += kept_mass(i);
    uint64_t ignored;
    before = wk.before + block_exclusive(mine, sh.warp64, &ignored);
    if (need < before || need >= before + mine) return;
    for (int i = i0; i < i1; ++i) {
        const uint64_t w = kept_mass(i);
        if (need < before + w) {
            a.token[row] = base + i;
            if (a.logprob) a.logprob[row] = (float)log((double)w / (double)total);
            break;
        }
        before += w;
    }
}

template <class T>
static int launch(Args &a, cudaStream_t s) {
    constexpr size_t kHead = (sizeof(Work) + 15) / 16 * 16, kRoom = 227 * 1024 - kHead;
    int C = cluster_size(sample_kernel<T, true>, a.B, a.V, 2048);
    while (C < 8 && (size_t)(a.V + C - 1) / C * sizeof(T) > kRoom - 64) C *= 2;
    a.slice = ((a.V + C - 1) / C + 15) / 16 * 16;  // slices start 16-byte aligned when the row does
    const size_t bytes = (size_t)a.slice * sizeof(T);
    const cudaError_t e = bytes <= kRoom ? launch_cluster(sample_kernel<T, true>, C, a.B, kHead + bytes, s, a)
                                         : launch_cluster(sample_kernel<T, false>, C, a.B, kHead, s, a);
    if (e != cudaSuccess) return ECC_ERR_LAUNCH;
    return launch_status();
}

}  // namespace samp
}  // namespace ecc

using namespace ecc;

extern "C" int ecc_sample(const void *logits, int64_t row_stride, int dtype, int B, int64_t V, const float *uniform,
                          const float *temperature, float temperature_all, const int *top_k, int top_k_all,
                          const float *top_p, float top_p_all, const float *min_p, float min_p_all, int64_t *token,
                          float *logprob, ecc_stream_t stream) {
    if (B == 0) return ECC_OK;
    if (!logits || !uniform || !token) return ECC_ERR_NULL;
    if (B < 0 || B > (1 << 24) || V < 1 || V > (1 << 20) || row_stride < 0) return ECC_ERR_SHAPE;
    if (dtype < ECC_SAMPLE_F16 || dtype > ECC_SAMPLE_F32) return ECC_ERR_SHAPE;
    if ((!temperature && !(temperature_all >= 0.0f)) || (!top_p && !(top_p_all > 0.0f)) ||
        (!min_p && !(min_p_all >= 0.0f && min_p_all <= 1.0f)) || (!top_k && top_k_all < 0))
        return ECC_ERR_PARAM;
    if ((uintptr_t)logits % (dtype == ECC_SAMPLE_F32 ? 4 : 2) || (uintptr_t)uniform % 4 || (uintptr_t)token % 8 ||
        (uintptr_t)logprob % 4 || (uintptr_t)temperature % 4 || (uintptr_t)top_k % 4 || (uintptr_t)top_p % 4 ||
        (uintptr_t)min_p % 4)
        return ECC_ERR_ALIGN;
    samp::Args a{};
    a.logits = logits;
    a.row_stride = row_stride;
    a.B = B;
    a.V = (int)V;
    a.u = uniform;
    a.temperature = temperature;
    a.temperature0 = temperature_all;
    a.top_k = top_k;
    a.top_k0 = top_k_all;
    a.top_p = top_p;
    a.top_p0 = top_p_all;
    a.min_p = min_p;
    a.min_p0 = min_p_all;
    a.token = token;
    a.logprob = logprob;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ECC_SAMPLE_F16: return samp::launch<__half>(a, s);
        case ECC_SAMPLE_BF16: return samp::launch<__nv_bfloat16>(a, s);
        default: return samp::launch<float>(a, s);
    }
}
