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
// No sort: one cluster of CTAs per row keeps the row in shared memory and
// finds the thresholds by radix descents (cluster_select.cuh), first by count,
// then by mass.  Masses are sums of fixed-point numbers w * 2^S (S = 62 -
// ceil(log2 V), at least 42 bits behind the point), so they do not depend on
// the order of the additions, and atomics give the same bits every time.
// A drawn token hangs on which side of a sum u * total falls: fp32 exponentials
// would move one draw in a few thousand, so w is computed in fp64 to 2^-46
// relative, by table and polynomial: with n = rint(z * 512 / ln 2) and
// r = z - n ln 2 / 512, |r| <= 6.8e-4,
//   exp(z) = 2^(n div 512) * 2^((n mod 512) / 512) * (1 + r + r^2/2 + r^3/6)
// (Tang, Table-driven implementation of the exponential function, 1989).
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
constexpr int kMassBins = 2048;

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
    int slice;    // elements of a row per CTA
    bool cached;  // the slice is kept in shared memory
    int S;        // fixed-point bits
};

template <class T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

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

struct Extra {
    double tab[kTab];
    float best;
    uint32_t best_at;
    float cta_best;       // of this CTA, read by the cluster
    uint32_t cta_best_at;
};

// w * 2^S as an integer.
struct Mass {
    const double *tab;
    double best, inv_t;
    int S;
    __device__ __forceinline__ uint64_t operator()(float x) const {
        if (x == (float)best) return 1ull << S;
        const double z = ((double)x - best) * inv_t;
        if (!(z > -44.0)) return 0;  // below 2^-63, and -inf
        constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
        const double t = fma(z, kTab / 0.693147180559945309417, kMagic);
        const int n = __double2loint(t);
        const double m = t - kMagic;
        const double r = fma(m, -0.693147180559945309417 / kTab, z);  // |m ln2/512| < 44: off by 2^-47 at most
        const double p = fma(r, fma(r, fma(r, 1.0 / 6.0, 0.5), 1.0), 1.0);
        const double w = p * tab[n & (kTab - 1)];
        // 2^S * 2^(n div 512) enters through the exponent; the rounding to an integer by adding 2^52
        const double scaled = __hiloint2double(__double2hiint(w) + ((S + (n >> 9)) << 20), __double2loint(w));
        return (uint64_t)__double_as_longlong(scaled + 4503599627370496.0) & 0xfffffffffffffull;
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

template <class T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const __grid_constant__ Args a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ Shared sh;
    __shared__ Extra ex;
    // masses by bin, read by the cluster: in the place of a count descent's bins
    unsigned long long *mass_bins = reinterpret_cast<unsigned long long *>(sh.hist);
    static_assert(sizeof(sh.hist) >= kMassBins * 8, "room for the masses");
    cg::cluster_group cl = cg::this_cluster();
    const int C = cl.num_blocks(), rank = cl.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C;
    for (int i = tid; i < kTab; i += kThreads) ex.tab[i] = exp2((double)i / kTab);
    pdl_trigger();
    pdl_wait();

    const T *x_row = reinterpret_cast<const T *>(a.logits) + (int64_t)row * a.row_stride;
    const int base = min(a.V, rank * a.slice), n = min(a.V, base + a.slice) - base;
    const T *x_g = x_row + base;
    T *x_s = reinterpret_cast<T *>(dyn);
    const bool cached = a.cached;
    auto load = [&](int i) {
        const float x = to_float<T>(cached ? x_s[i] : x_g[i]);
        return x != x ? -INFINITY : x;
    };

    // ---- the row, its maximum and the maximum's first place
    float best = -INFINITY;
    uint32_t best_at = 0xffffffffu;
    if (cached) {
        constexpr int kVec = 16 / sizeof(T);
        const bool wide = ((uintptr_t)x_g & 15) == 0;
        const int n_wide = wide ? n / kVec : 0;
        for (int i = tid; i < n_wide; i += kThreads)
            reinterpret_cast<uint4 *>(x_s)[i] = __ldg(reinterpret_cast<const uint4 *>(x_g) + i);
        for (int i = n_wide * kVec + tid; i < n; i += kThreads) x_s[i] = x_g[i];
        __syncthreads();
    }
    for (int i = tid; i < n; i += kThreads) {
        const float x = load(i);
        if (x > best) best = x, best_at = base + i;  // ascending i: the first of equals
    }
    auto better = [](float x, uint32_t i, float &bx, uint32_t &bi) {
        if (x > bx || (x == bx && i < bi)) bx = x, bi = i;
    };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_at, o), best, best_at);
    if (lane == 0) sh.warp_a[warp] = __float_as_uint(best), sh.warp_b[warp] = best_at;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWarps; ++w) better(__uint_as_float(sh.warp_a[w]), sh.warp_b[w], best, best_at);
        ex.cta_best = best;
        ex.cta_best_at = best_at;
    }
    cl.sync();
    if (tid == 0) {
        for (int r = 0; r < C; ++r) better(*of_rank(cl, &ex.cta_best, r), *of_rank(cl, &ex.cta_best_at, r), best, best_at);
        ex.best = best;
        ex.best_at = best_at;
    }
    cl.sync();  // also: nobody reads a CTA's shared memory after it may have left
    best = ex.best;
    best_at = ex.best_at;
    const float temp = a.temperature ? __ldg(a.temperature + row) : a.temperature0;
    if (best == -INFINITY || !(temp > 0.0f)) {  // cluster-uniform
        if (rank == 0 && tid == 0) {
            a.token[row] = best == -INFINITY ? -1 : (int64_t)best_at;
            if (a.logprob) a.logprob[row] = best == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    const Mass mass{ex.tab, (double)best, 1.0 / (double)temp, a.S};

    // ---- top-k: keys above `kth` are kept, equal ones below the row position `cut`
    uint32_t kth = 0, cut = 0xffffffffu;
    auto key = [&](int i) { return value_key<T>(load(i)); };
    const int k = a.top_k ? __ldg(a.top_k + row) : a.top_k0;
    if (k > 0 && k < a.V) {
        uint32_t ties, equal;
        kth = kth_largest(sh, cl, key, n, (uint32_t)k, key_low<T>(), &ties, &equal);
        if (ties < equal) cut = tie_cut(sh, cl, n, base, ties, [&](int i) { return key(i) == kth; });
    }
    auto keep = [&](uint32_t x, int i) { return x > kth || (x == kth && (uint32_t)(base + i) < cut); };

    // ---- top-p
    const float p = a.top_p ? __ldg(a.top_p + row) : a.top_p0;
    if (p < 1.0f) {
        // First by the distance from the maximum in bins of 1/64 (monotone in x, and spread however the
        // logits lie), then by the bits of the key among those of the bin that holds the threshold.
        const float inv_bin = 64.0f / temp;
        auto bin_of = [&](float x) {
            const float d = (best - x) * inv_bin;  // NaN when x is the infinite maximum
            return x == best ? 0 : d < (float)(kMassBins - 1) ? (int)d : kMassBins - 1;
        };
        int bin = -1;
        uint32_t prefix = 0, mask = 0;
        uint64_t above = 0, at = 0;  // mass above the bin, of the bin
        uint64_t want = 0;           // ceil(p * total): whole masses below it are below p * total
        int top = 33;
        while (true) {
            const int low = key_low<T>(), bits = top == 33 ? 11 : min(11, top - low), shift = top - bits;
            for (int i = tid; i < kMassBins; i += kThreads) mass_bins[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float x = load(i);
                const uint32_t kx = value_key<T>(x);
                if (!keep(kx, i)) continue;
                const int mine = bin_of(x);
                // bin 0 of the mass array is the top one in either kind of pass
                int slot;
                if (bin < 0) {
                    slot = mine;
                } else {
                    if (mine != bin || (kx & mask) != prefix) continue;
                    slot = kMassBins - 1 - (int)((kx >> shift) & ((1u << bits) - 1));
                }
                const uint64_t w = mass(x);
                if (w) atomicAdd(&mass_bins[slot], (unsigned long long)w);
            }
            cl.sync();
            uint64_t c[kPerThread], mine = 0;
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) {
                c[j] = 0;
                for (int r = 0; r < C; ++r) c[j] += of_rank(cl, mass_bins, r)[tid * kPerThread + j];
                mine += c[j];
            }
            uint64_t all;
            uint64_t before = block_exclusive(mine, sh.warp64, &all);
            if (bin < 0) {
                bool more = true;
                want = p > 0.0f ? share_of(p, all, &more) : 0;  // p <= 0: the first token alone
                want += more ? 1 : 0;
            }
            before += above;
#pragma unroll
            for (int j = 0; j < kPerThread; ++j) {
                // the bin before which less than the wanted mass lies, and after which not
                if (before < want && want <= before + c[j]) {
                    sh.found[0] = tid * kPerThread + j;
                    sh.found64[0] = before;
                    sh.found64[1] = c[j];
                }
                before += c[j];
            }
            cl.sync();
            above = sh.found64[0];
            at = sh.found64[1];
            if (bin < 0) {
                bin = sh.found[0];
                top = 32;
            } else {
                prefix |= (uint32_t)(kMassBins - 1 - sh.found[0]) << shift;
                mask |= ((1u << bits) - 1) << shift;
                top = shift;
            }
            __syncthreads();
            if (top <= low) break;
        }
        // every kept token with the threshold's key has the same mass
        const uint32_t key_p = prefix;
        const uint64_t w = max((uint64_t)1, mass(key_value<T>(key_p)));
        const uint64_t count = at / w;
        // how many of them: the smallest m with above + m w >= want > above
        const uint64_t m = (want - above + w - 1) / w;
        uint32_t cut_p = key_p == kth ? cut : 0xffffffffu;
        if (m < count) {
            const uint32_t old = cut_p;
            cut_p = tie_cut(sh, cl, n, base, (uint32_t)m,
                            [&](int i) { return key(i) == key_p && (uint32_t)(base + i) < old; });
        }
        kth = key_p;
        cut = cut_p;
    }

    // ---- the draw: masses of the warps' parts, then the part that holds the number
    const float mp = a.min_p ? __ldg(a.min_p + row) : a.min_p0;
    const double least = (double)mp * (double)(1ull << a.S);
    auto kept_mass = [&](int i) -> uint64_t {
        const float x = load(i);
        if (!keep(value_key<T>(x), i)) return 0;
        const uint64_t w = mass(x);
        return (double)w >= least || x == best ? w : 0;
    };
    int lo, hi;
    warp_part(n, lo, hi);
    uint64_t part = 0;
    for (int i = lo + lane; i < hi; i += 32) part += kept_mass(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    uint64_t cta_all;
    uint64_t before = block_exclusive(lane == 0 ? part : 0, sh.warp64, &cta_all);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (tid == 0) sh.cta64 = cta_all;
    cl.sync();
    uint64_t total = 0;
    for (int r = 0; r < C; ++r) {
        const uint64_t c = *of_rank(cl, &sh.cta64, r);
        before += r < rank ? c : 0;
        total += c;
    }
    cl.sync();  // no remote reads after this
    // cumulative mass > u * total, of whole masses: > floor(u * total); a number of 1 or more takes the last
    // kept token, one that is not above 0 the first
    const float u = __ldg(a.u + row);
    bool ignored;
    const uint64_t need = !(u > 0.0f) ? 0 : u < 1.0f ? share_of(u, total, &ignored) : total - 1;
    if (part && before <= need && need < before + part) {  // this warp holds it
        uint64_t seen = before;
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const uint64_t w = i0 + lane < hi ? kept_mass(i0 + lane) : 0;
            uint64_t inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, seen + inc > need);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    a.token[row] = base + i0 + lane;
                    if (a.logprob) a.logprob[row] = (float)log((double)w / (double)total);
                }
                break;
            }
            seen += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
}

template <class T>
static int launch(Args &a, cudaStream_t s) {
    // static shared memory of the kernel beside the row's slice
    constexpr size_t kRoom = 227 * 1024 - sizeof(Shared) - sizeof(Extra) - 1024;
    const int sms = sm_count();
    int C = cluster_size(a.B, sms, 8);
    while (C < 8 && (size_t)(a.V + C - 1) / C * sizeof(T) > kRoom) C *= 2;
    a.slice = ((a.V + C - 1) / C + 15) / 16 * 16;  // slices start 16-byte aligned when the row does
    a.cached = (size_t)a.slice * sizeof(T) <= kRoom;
    const size_t smem = a.cached ? (size_t)a.slice * sizeof(T) : 0;
    if (launch_cluster(sample_kernel<T>, C, a.B, smem, s, a) != cudaSuccess) return ECC_ERR_LAUNCH;
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
    int lg = 0;
    while ((1ll << lg) < V) ++lg;
    // the fixed-point value of one weight fits the 52 bits of the fp64 rounding, a row's sum 63 bits
    a.S = std::min(51, 62 - lg);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case ECC_SAMPLE_F16: return samp::launch<__half>(a, s);
        case ECC_SAMPLE_BF16: return samp::launch<__nv_bfloat16>(a, s);
        default: return samp::launch<float>(a, s);
    }
}
