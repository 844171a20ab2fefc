// cluster_select.cuh -- selection over one long row by a cluster of CTAs
// (sm_100a): each CTA holds a contiguous slice of the row, the counts of the
// slices are joined through distributed shared memory and the hardware
// cluster barrier.  Used by the cache eviction and by sampling.
//
// The k largest 32-bit keys of a row are found by a radix descent: per pass
// the keys that match the prefix so far are counted by their next digit (up
// to 11 bits), the cluster's counts are summed, and the digit in which the
// k-th key falls extends the prefix.  Shared-memory atomics of one warp on
// one address are serialised, so each bin has four copies, picked by lane.
#pragma once
#include <cooperative_groups.h>

#include <atomic>

#include "ecc_common.cuh"

namespace ecc {
namespace sel {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kCopies = 4;
constexpr int kPerThread = kBins / kThreads;
constexpr int kMaxCluster = 16;

// The cluster of this CTA; one of a single CTA meets at the block's barrier.
class Cluster {
    int n_, rank_;

public:
    __device__ __forceinline__ Cluster()
        : n_((int)cg::this_cluster().num_blocks()), rank_((int)cg::this_cluster().block_rank()) {}
    __device__ __forceinline__ int num_blocks() const { return n_; }
    __device__ __forceinline__ int block_rank() const { return rank_; }
    __device__ __forceinline__ void sync() const {
        if (n_ == 1) __syncthreads();
        else cg::this_cluster().sync();
    }
    template <class T>
    __device__ __forceinline__ T *map_shared_rank(T *p, unsigned rank) const {
        return cg::this_cluster().map_shared_rank(p, rank);
    }
};

struct Crossing {  // see crossing()
    uint32_t slot;
    uint64_t before, here;
};
struct CrossingShared {
    uint64_t share[kMaxCluster];  // the CTAs' sums of their bins, written by each of them
    Crossing found[2];            // written by the CTA that finds it
};

struct alignas(16) Shared {
    uint32_t hist[kBins * kCopies];
    uint32_t sum[kBins];  // this CTA's counts of a pass, read by the cluster
    uint32_t tot[kBins];  // the cluster's, this CTA's share of the bins
    uint32_t warp_a[kWarps], warp_b[kWarps];
    uint64_t warp64[kWarps];
    uint32_t cta_a, cta_b;  // totals of this CTA, read by the cluster
    uint64_t cta64;
    CrossingShared cross;
    uint32_t cut;     // written by the CTA that finds it
    uint32_t listed;  // entries of the first CTA's list
};

// Ascending order of floats as ascending unsigned order; -0 equals +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <class T>
__device__ __forceinline__ T *of_rank(const Cluster &cl, T *p, unsigned rank) {
    return cl.map_shared_rank(p, rank);
}

// Exclusive prefix of v over the block's threads; *total = the sum.
template <class T>
__device__ __forceinline__ T block_exclusive(T v, T *warp_sums, T *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    __syncthreads();  // earlier readers of warp_sums are done
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    // every warp adds up the warps' sums by itself: a scan over 32 lanes
    static_assert(kWarps == 32, "a lane per warp");
    const T w = warp_sums[lane];
    T upto = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    const T before = __shfl_sync(0xffffffffu, upto - w, warp), all = __shfl_sync(0xffffffffu, upto, 31);
    *total = all;
    return before + inc - v;
}

// Sums over the cluster, spread over it: CTA r gets the sums of from[r W ..
// r W + W), W = kBins / CTAs, in to[0 .. W).  All CTAs must have passed a
// cluster barrier since their `from` was written, and pass one (crossing()
// does) before it is written again.
template <class T, class U>
__device__ __forceinline__ void cluster_share(const Cluster &cl, T *from, U *to) {
    const int ranks = (int)cl.num_blocks(), W = kBins / ranks, at = (int)cl.block_rank() * W;
    for (int i = threadIdx.x; i < W; i += kThreads) {
        T c = 0;
        for (int r = 0; r < ranks; r += 8) {
            T v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = r + q < ranks ? of_rank(cl, from, r + q)[at + i] : 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) c += v[q];
        }
        to[i] = c;
    }
    __syncthreads();
}

// The sum of all bins; every CTA's cs.share is filled.
template <class T>
__device__ __forceinline__ uint64_t share_sums(CrossingShared &cs, const Cluster &cl, const T *bins,
                                               uint64_t *warp_sums) {
    const int ranks = (int)cl.num_blocks(), W = kBins / ranks;
    uint64_t v = 0;
    for (int i = threadIdx.x; i < W; i += kThreads) v += bins[i];
    uint64_t mine;
    block_exclusive(v, warp_sums, &mine);
    if (threadIdx.x < ranks) of_rank(cl, cs.share, threadIdx.x)[cl.block_rank()] = mine;
    cl.sync();
    uint64_t all = 0;
    for (int r = 0; r < ranks; ++r) all += cs.share[r];
    return all;
}
// Where the running sum over the spread bins, whose share_sums() are known,
// reaches want[j] (1 <= want[j] <= the sum of all): the bin, the sum before it
// and its own, the same in every CTA.  Ends with a cluster barrier.
template <class T, int K>
__device__ __forceinline__ void crossings(CrossingShared &cs, const Cluster &cl, const T *bins,
                                          const uint64_t (&want)[K], Crossing (&found)[K], uint64_t *warp_sums) {
    const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank(), W = kBins / ranks;
    uint64_t before = 0;
    for (int r = 0; r < rank; ++r) before += cs.share[r];
    const uint64_t mine = cs.share[rank];
    bool here = false;
#pragma unroll
    for (int j = 0; j < K; ++j) here = here || (before < want[j] && want[j] <= before + mine);
    if (here) {  // block-uniform
        const int per = (W + kThreads - 1) / kThreads;
        uint64_t v[kPerThread], sum = 0;
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            const int i = threadIdx.x * per + j;
            v[j] = j < per && i < W ? bins[i] : 0;
            sum += v[j];
        }
        uint64_t all;
        before += block_exclusive(sum, warp_sums, &all);
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
#pragma unroll
            for (int q = 0; q < K; ++q)
                if (before < want[q] && want[q] <= before + v[j])
                    for (int r = 0; r < ranks; ++r)
                        of_rank(cl, &cs, r)->found[q] = {(uint32_t)(rank * W + threadIdx.x * per + j), before, v[j]};
            before += v[j];
        }
    }
    cl.sync();
#pragma unroll
    for (int j = 0; j < K; ++j) {
        found[j] = cs.found[j];
        found[j].slot &= kBins - 1;  // a bin in any case
    }
}
template <class T>
__device__ __forceinline__ Crossing crossing(CrossingShared &cs, const Cluster &cl, const T *bins, uint64_t want,
                                             uint64_t *warp_sums) {
    const uint64_t w[1] = {want};
    Crossing f[1];
    crossings(cs, cl, bins, w, f, warp_sums);
    return f[0];
}

// The k-th largest key of the cluster's row, 1 <= k <= keys of the row.
// keys(i), i < n, are this CTA's; passes of `bits` bits from bit 31 down to
// bit `low` (the bits below are zero in every key).  *ties: how many of the
// keys equal to it belong to the k largest; *equal: how many there are.
template <class Keys>
__device__ __forceinline__ uint32_t kth_largest(Shared &sh, const Cluster &cl, const Keys &keys, int n, uint32_t k,
                                                int low, uint32_t *ties, uint32_t *equal) {
    const int tid = threadIdx.x;
    const unsigned ranks = cl.num_blocks();
    uint32_t prefix = 0, mask = 0;
    int top = 32;
    while (top > low) {
        const int bits = min(11, top - low), shift = top - bits;
        const uint32_t bins = 1u << bits;
        for (int i = tid; i < kBins * kCopies / 4; i += kThreads)
            reinterpret_cast<uint4 *>(sh.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < n; i += kThreads) {
            const uint32_t x = keys(i);
            if ((x & mask) == prefix) atomicAdd(&sh.hist[((x >> shift) & (bins - 1)) * kCopies + (tid & (kCopies - 1))], 1u);
        }
        __syncthreads();
        // bins from the top, so that a prefix counts the larger keys
        for (int i = tid; i < kBins; i += kThreads) {
            const uint4 c = reinterpret_cast<const uint4 *>(sh.hist)[kBins - 1 - i];
            sh.sum[i] = (c.x + c.y) + (c.z + c.w);
        }
        cl.sync();
        cluster_share(cl, sh.sum, sh.tot);
        share_sums(sh.cross, cl, sh.tot, sh.warp64);
        const Crossing f = crossing(sh.cross, cl, sh.tot, k, sh.warp64);
        prefix |= (kBins - 1 - f.slot) << shift;
        mask |= (bins - 1) << shift;
        k -= (uint32_t)f.before;
        *equal = (uint32_t)f.here;
        top = shift;
    }
    *ties = k;
    return prefix;
}

// A warp's contiguous part of the CTA's n elements, and the warp of element i.
__device__ __forceinline__ int part_size(int n) { return ((n + kWarps - 1) / kWarps + 31) / 32 * 32; }
__device__ __forceinline__ int part_of(int n, int i) { return i / part_size(n); }
__device__ __forceinline__ void warp_part(int n, int &lo, int &hi) {
    const int per = part_size(n);
    lo = min(n, (int)(threadIdx.x >> 5) * per);
    hi = min(n, lo + per);
}

// Number of this warp's elements that satisfy p(i).
template <class Pred>
__device__ __forceinline__ uint32_t warp_count(int lo, int hi, const Pred &p) {
    uint32_t c = 0;
    for (int i = lo + (int)(threadIdx.x & 31); i < hi; i += 32) c += p(i) ? 1u : 0u;
    return __reduce_add_sync(0xffffffffu, c);
}

// Cluster-wide exclusive prefix of one count per warp, in row order.
__device__ __forceinline__ uint32_t cluster_exclusive(Shared &sh, const Cluster &cl, uint32_t warp_value) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) sh.warp_a[warp] = warp_value;
    __syncthreads();
    const uint32_t x = sh.warp_a[threadIdx.x & 31], all = __reduce_add_sync(0xffffffffu, x);
    uint32_t before = __reduce_add_sync(0xffffffffu, (int)(threadIdx.x & 31) < warp ? x : 0);
    if (threadIdx.x == 0) sh.cta_a = all;
    cl.sync();
    for (unsigned r = 0; r < cl.block_rank(); ++r) before += *of_rank(cl, &sh.cta_a, r);
    cl.sync();  // cta_a may be written again
    return before;
}

// Row position behind the `ties`-th element (in row order) that satisfies
// p(i): elements of equal key are kept below it.  base: row position of this
// CTA's element 0.
template <class Pred>
__device__ __forceinline__ uint32_t tie_cut(Shared &sh, const Cluster &cl, int n, int base, uint32_t ties,
                                            const Pred &p) {
    int lo, hi;
    warp_part(n, lo, hi);
    const uint32_t c = warp_count(lo, hi, p);
    const uint32_t before = cluster_exclusive(sh, cl, c);
    if (before < ties && ties <= before + c) {  // this warp holds it
        const int lane = threadIdx.x & 31;
        uint32_t seen = before;
        for (int i0 = lo; i0 < hi; i0 += 32) {
            const bool hit = i0 + lane < hi && p(i0 + lane);
            const uint32_t m = __ballot_sync(0xffffffffu, hit);
            if (hit && seen + __popc(m & ((1u << lane) - 1u)) + 1 == ties)
                for (unsigned r = 0; r < cl.num_blocks(); ++r) *of_rank(cl, &sh.cut, r) = (uint32_t)(base + i0 + lane + 1);
            seen += __popc(m);
        }
    }
    cl.sync();
    const uint32_t cut = sh.cut;
    __syncthreads();
    return cut;
}

// Entries of a list of 64-bit words in the place of a pass's bins.
constexpr int kList = sizeof(Shared::hist) / 8;

// Moves the entries that every CTA put into its own list (room for kList, their
// number in *listed) behind one another into the first CTA's.  All CTAs have
// passed a cluster barrier since their last entry; ends with one.  Returns the
// number of all entries; nothing is moved when that is more than kList.
__device__ __forceinline__ uint32_t join_lists(const Cluster &cl, unsigned long long *list, const uint32_t *listed) {
    const int ranks = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    uint32_t before = 0, mine = 0, all = 0;
    for (int r = 0; r < ranks; ++r) {
        const uint32_t c = *of_rank(cl, const_cast<uint32_t *>(listed), r);
        if (r < rank) before += c;
        if (r == rank) mine = c;
        all += c;
    }
    if (rank > 0 && all <= (uint32_t)kList)
        for (int i = threadIdx.x; i < (int)mine; i += kThreads) of_rank(cl, list, 0)[before + i] = list[i];
    cl.sync();
    return all;
}

// Cluster size for `clusters` clusters that share a row of `n` elements each: the
// largest power of two up to 8 with which all of them run at the same time and
// every CTA has `least` elements.  A cluster lives inside one GPC, so fewer fit
// than the SMs would hold (16 rows in clusters of 8: 21 us in two waves where
// clusters of 4 take 14).  Asked once per device; kernels of one signature share
// the answer (a CTA of kThreads with this much shared memory has an SM to itself).
constexpr size_t kMostShared = 227 * 1024;
template <typename... KArgs>
static inline int cluster_size(void (*kernel)(KArgs...), int64_t clusters, int64_t n, int least) {
    static std::atomic<int> fit[64][4];  // by device and log2 of the size: clusters at a time, plus 1
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    int c = 1;
    for (int lg = 1; lg < 4 && n >= (int64_t)least << lg; ++lg) {
        int v = fit[dev][lg].load(std::memory_order_relaxed);
        if (v == 0) {
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared);
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1u << lg);
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = kMostShared;  // one CTA per SM
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim = {1u << lg, 1, 1};
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int most = 0;
            if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                most = 0;
            }
            v = most + 1;
            fit[dev][lg].store(v, std::memory_order_relaxed);
        }
        if (clusters > v - 1) break;
        c = 1 << lg;
    }
    return c;
}

// Bitonic sort of `size` entries, a power of two from 32 E to 1024 E, by size /
// E threads that hold E neighbouring entries each (0 behind entry n).  Partners
// in a thread are exchanged in registers, those in a warp by shuffles; strides
// of 32 E and more go through shared memory.
template <int E>
__device__ __forceinline__ void sort_bitonic(unsigned long long *x, int n, int size) {
    const int t = threadIdx.x, threads = size / E;
    if (t >= threads) return;
    unsigned long long v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = t * E + e < n ? x[t * E + e] : 0ull;
    for (int k = 2; k <= size; k *= 2) {
        for (int j = k / 2; j > 0; j /= 2) {
            if (j < E) {
#pragma unroll
                for (int s = E / 2; s > 0; s /= 2) {
                    if (j != s) continue;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (e & s) continue;
                        const unsigned long long p = v[e], q = v[e + s];
                        const bool swap = (p < q) == (((t * E + e) & k) == 0);
                        v[e] = swap ? q : p;
                        v[e + s] = swap ? p : q;
                    }
                }
                continue;
            }
            const int w = j / E;  // in threads
            const bool larger = ((t & w) == 0) == ((t * E & k) == 0);  // (k > j >= E)
            unsigned long long u[E];
            if (w < 32) {
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] = __shfl_xor_sync(0xffffffffu, v[e], w);
            } else {
                asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");  // earlier readers are done
#pragma unroll
                for (int e = 0; e < E; ++e) x[t * E + e] = v[e];
                asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] = x[(t ^ w) * E + e];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = larger == (v[e] < u[e]) ? u[e] : v[e];
        }
    }
    asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
#pragma unroll
    for (int e = 0; e < E; ++e) x[t * E + e] = v[e];
}

// Descending sort of the first n <= 4096 entries of `x`, all different, by the
// whole block; entries from n up to the next power of two may be overwritten.
// Up to 128 an entry's place is the number of larger ones, counted by 8 to 32
// threads (100: 1.0 us, by exchanges 1.6); more are sorted by exchanges: 500 in
// 3.6 us, 1000 in 6.8, 4096 in 23 (by merges of ranked runs 2.9, 5.7 and 26).
__device__ __forceinline__ void sort_descending(unsigned long long *x, int n) {
    const int t = threadIdx.x;
    if (n <= 128) {
        const int lg = n <= 32 ? 5 : n <= 64 ? 4 : 3;  // 2^lg threads an entry
        const int i = t >> lg, each = 1 << lg, threads = ((n << lg) + 31) / 32 * 32;
        if (t < threads) {
            const unsigned long long v = i < n ? x[i] : 0ull;
            int larger = 0;
            for (int q = t & (each - 1); q < n; q += each) larger += x[q] > v ? 1 : 0;
            for (int o = 1; o < each; o *= 2) larger += __shfl_xor_sync(0xffffffffu, larger, o);
            asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory");
            if (i < n && (t & (each - 1)) == 0) x[larger] = v;
        }
    } else {
        int size = 256;
        while (size < n) size *= 2;
        if (size <= 512) sort_bitonic<1>(x, n, size);
        else sort_bitonic<4>(x, n, size);
    }
    __syncthreads();
}

// Launch with a cluster of `c` neighbouring CTAs per row, as a dependent of the
// kernel before it on the stream.
template <typename... KArgs, typename... Args>
static inline cudaError_t launch_cluster(void (*kernel)(KArgs...), int c, int64_t rows, size_t smem, cudaStream_t s,
                                         Args &&...args) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(c * rows));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {(unsigned)c, 1, 1};
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace sel
}  // namespace ecc
