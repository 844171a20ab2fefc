// evict.cu -- thinning out a paged block cache by accumulated attention weight
// (sm_100a), out of place: a sequence of L tokens keeps, per kv head, its
// first `sinks`, its last `recent` and the budget - sinks - recent others with
// the largest weights (equal weights: the earlier token), in their order; the
// kept blocks are copied into other pages, the weights go along.
//
// Two launches.  evict_select_kernel: one cluster per (sequence, kv head)
// finds the threshold weight (cluster_select.cuh), ranks the kept tokens by
// counting and writes their positions and weights; one more cluster checks
// that no page is written twice or read and written.  evict_move_kernel
// copies the blocks.
//
// Measured at 8 sequences x 8 kv heads, 32768 -> 16384 tokens: selection 26 us
// (5 reading the weights, 5 writing positions and weights, the rest the
// barriers of its phases), move 87 us, 6.1 TB/s of the 0.54 GB read and written
// (bound by memory).  One sequence of 5001 tokens to 1024: 12 + 3 us; three
// digit descents instead of the binned pass took 24 + 5.
#include <algorithm>

#include "cluster_select.cuh"
#include "paged.cuh"

namespace ecc {

int launch_status();
int sm_count();

namespace paged {

struct EvictArgs {
    PageTable src, dst;
    const int *lens;
    const float *w;
    int64_t w_b, w_h;
    float *ow;
    int64_t ow_b, ow_h;
    int ow_len;  // columns of the output weights
    int *kept;   // [B][Hkv][budget]
    int B, Hkv, budget, sinks, recent;
    uint32_t *bitmap;  // of the pool's pages
    int *clash;        // set when the tables clash
    int cache_keys;    // keys of a slice kept in shared memory
};

// Weight -> key: NaN above everything, as a sort has it.
__device__ __forceinline__ uint32_t weight_key(float x) { return x != x ? 0xffffffffu : sel::key_of(x); }

__device__ __forceinline__ float key_weight(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);  // the NaN key gives a NaN
}

__device__ void check_tables(const EvictArgs &a, const sel::Cluster &cl) {
    const int t0 = cl.block_rank() * sel::kThreads + threadIdx.x, step = cl.num_blocks() * sel::kThreads;
    for (int i = t0; i < (a.src.n_pages + 31) / 32; i += step) a.bitmap[i] = 0;
    if (t0 == 0) *a.clash = 0;
    cl.sync();
    int bad = 0;
    const auto each = [&](const PageTable &t, int most, auto &&f) {
        for (int64_t i = t0; i < (int64_t)a.B * t.width; i += step) {
            const int b = (int)(i / t.width), c = (int)(i - (int64_t)b * t.width);
            const int n = min(max(0, min(__ldg(a.lens + b), a.src.capacity)), most);
            if ((int64_t)c * t.page_size >= n) continue;
            const int p = __ldg(t.table + b * t.stride + c);
            if ((uint32_t)p < (uint32_t)t.n_pages) f(p);
        }
    };
    each(a.dst, a.budget, [&](int p) { bad |= (atomicOr(a.bitmap + (p >> 5), 1u << (p & 31)) >> (p & 31)) & 1; });
    cl.sync();
    each(a.src, a.src.capacity, [&](int p) { bad |= (__ldcg(a.bitmap + (p >> 5)) >> (p & 31)) & 1; });
    if (bad) {
        atomicExch(a.clash, 1);
        atomicExch(&g_paged_error, 5);
    }
}

__global__ void __launch_bounds__(sel::kThreads, 1) evict_select_kernel(const __grid_constant__ EvictArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    sel::Shared &sh = *reinterpret_cast<sel::Shared *>(dyn);
    uint32_t *cache = reinterpret_cast<uint32_t *>(dyn + sizeof(sel::Shared));
    const sel::Cluster cl;
    const int C = cl.num_blocks(), rank = cl.block_rank(), tid = threadIdx.x, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x / C;
    if (row == a.B * a.Hkv) {  // the last cluster
        check_tables(a, cl);
        return;
    }
    const int b = row / a.Hkv, h = row - b * a.Hkv;
    // one thread reads the length for the whole cluster, which branches on it together
    if (tid == 0) sh.listed = (uint32_t)__ldg(a.lens + b);
    cl.sync();
    int L = (int)*sel::of_rank(cl, &sh.listed, 0);
    cl.sync();
    if (L < 0 || L > a.src.capacity) {
        if (tid == 0 && rank == 0) atomicExch(&g_paged_error, 5);
        L = max(0, min(L, a.src.capacity));
    }
    const float *w = a.w + b * a.w_b + h * a.w_h;
    float *ow = a.ow + b * a.ow_b + h * a.ow_h;
    int *kept = a.kept + (int64_t)row * a.budget;
    const int n_out = min(L, a.budget);
    // behind the last kept token: no positions, weights zero
    for (int i = n_out + rank * sel::kThreads + tid; i < max(a.budget, a.ow_len); i += C * sel::kThreads) {
        if (i < a.budget) kept[i] = -1;
        if (i < a.ow_len) ow[i] = 0.0f;
    }
    auto put_as = [&](int i, int t, float x) {
        kept[i] = t;
        if (i < a.ow_len) ow[i] = x;
    };
    auto put = [&](int i, int t) { put_as(i, t, w[t]); };
    if (L <= a.budget) {  // cluster-uniform
        for (int i = rank * sel::kThreads + tid; i < L; i += C * sel::kThreads) put(i, i);
        return;
    }
    for (int i = rank * sel::kThreads + tid; i < a.sinks; i += C * sel::kThreads) put(i, i);
    for (int i = rank * sel::kThreads + tid; i < a.recent; i += C * sel::kThreads)
        put(a.budget - a.recent + i, L - a.recent + i);
    const int k = a.budget - a.sinks - a.recent;
    if (k == 0) return;

    // this CTA's slice of the tokens that compete
    const int n_all = L - a.sinks - a.recent, per = (n_all + C - 1) / C;
    const int base = a.sinks + min(n_all, rank * per), n = min(n_all, (rank + 1) * per) - min(n_all, rank * per);
    const bool cached = n <= a.cache_keys;
    if (cached) {
#pragma unroll 8
        for (int i = tid; i < n; i += sel::kThreads) cache[i] = weight_key(__ldg(w + base + i));
        __syncthreads();
    }
    auto key = [&](int i) { return cached ? cache[i] : weight_key(__ldg(w + base + i)); };
    // What is kept: keys above kth, equal ones below the position cut.  One pass counts the keys by exponent and
    // six bits of mantissa, from 2^-23 to 2^8 (what lies outside falls into the end bins: the order is kept);
    // the bin that holds the k-th key is then listed and sorted in the cluster's first CTA.  A bin that does not
    // fit the list (many equal weights) is descended digit by digit.
    uint32_t kth, cut = 0xffffffffu;
    constexpr uint32_t kLowest = 0x80000000u + ((127u - 23u) << 23);
    auto bin_of = [](uint32_t x) {  // 0: the largest
        return sel::kBins - 1 - (int)min((uint32_t)sel::kBins - 1, x > kLowest ? (x - kLowest) >> 17 : 0u);
    };
    for (int i = tid; i < sel::kBins; i += sel::kThreads) sh.hist[i] = 0;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < n; i += sel::kThreads) atomicAdd(&sh.hist[bin_of(key(i))], 1u);
    cl.sync();
    sel::cluster_share(cl, sh.hist, sh.tot);
    sel::share_sums(sh.cross, cl, sh.tot, sh.warp64);
    const sel::Crossing at_k = sel::crossing(sh.cross, cl, sh.tot, (uint64_t)k, sh.warp64);
    if (at_k.here <= sel::kList) {
        // few entries go straight to the first CTA, which saves join_lists' barrier
        const bool at_rank0 = at_k.here <= 512;
        unsigned long long *list = reinterpret_cast<unsigned long long *>(sh.hist);
        unsigned long long *list_to = at_rank0 ? sel::of_rank(cl, list, 0) : list;
        uint32_t *listed_to = at_rank0 ? sel::of_rank(cl, &sh.listed, 0) : &sh.listed;
        for (int i0 = tid - lane; i0 < n; i0 += sel::kThreads) {
            const uint32_t x = i0 + lane < n ? key(i0 + lane) : 0;
            const bool hit = i0 + lane < n && bin_of(x) == (int)at_k.slot;
            const uint32_t m = __ballot_sync(0xffffffffu, hit);
            if (!m) continue;
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(listed_to, (uint32_t)__popc(m));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(m & ((1u << lane) - 1u));
            if (hit && at < sel::kList) list_to[at] = ((unsigned long long)x << 32) | (uint32_t)~(uint32_t)(base + i0 + lane);
        }
        cl.sync();
        const uint32_t all = at_rank0 ? sh.listed : sel::join_lists(cl, list, &sh.listed);
        if (rank == 0) {
            sel::sort_descending(list, (int)min(all, (uint32_t)sel::kList));
            if (tid < C) {
                const unsigned long long e = list[(k - (int)at_k.before - 1) & (sel::kList - 1)];
                *sel::of_rank(cl, &sh.cta_b, tid) = (uint32_t)(e >> 32);
                *sel::of_rank(cl, &sh.cut, tid) = ~(uint32_t)e + 1;
            }
        }
        cl.sync();
        kth = sh.cta_b;
        cut = sh.cut;
    } else {
        uint32_t ties, equal;
        kth = sel::kth_largest(sh, cl, key, n, (uint32_t)k, 0, &ties, &equal);
        if (ties < equal) cut = sel::tie_cut(sh, cl, n, base, ties, [&](int i) { return key(i) == kth; });
    }
    auto keep = [&](int i) {
        const uint32_t x = key(i);
        return x > kth || (x == kth && (uint32_t)(base + i) < cut);
    };
    int lo, hi;
    sel::warp_part(n, lo, hi);
    uint32_t at = a.sinks + sel::cluster_exclusive(sh, cl, sel::warp_count(lo, hi, keep));
#pragma unroll 4
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const bool hit = i0 + lane < hi && keep(i0 + lane);
        const uint32_t m = __ballot_sync(0xffffffffu, hit);
        const int to = (int)(at + __popc(m & ((1u << lane) - 1u))), t = base + i0 + lane;
        // the weight again out of its key (-0 comes back as +0)
        if (hit && to < a.budget - a.recent) put_as(to, t, cached ? key_weight(cache[i0 + lane]) : __ldg(w + t));
        at += __popc(m);
    }
}

// Copies the kept blocks: a group of R / 16 lanes per block, kBatch tokens of
// K and V in flight per group.
constexpr int kMoveThreads = 256;
constexpr int kBatch = 2;
struct MoveArgs {
    EvictArgs e;
    uint8_t *k, *v;
    int64_t kp, kh, vp, vh;  // strides of a page and a kv head, in bytes
};
template <int R>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ MoveArgs a, FastDiv div_n,
                                                                  FastDiv div_h) {
    constexpr int kLanes = R / 16, kGroups = 32 / kLanes;  // 8 or 6 lanes a block
    pdl_trigger();
    pdl_wait();
    if (*a.e.clash) return;
    const int lane = threadIdx.x & 31, grp = lane / kLanes, off = 16 * (lane - grp * kLanes);
    if (grp >= kGroups) return;
    const uint32_t total = (uint32_t)a.e.B * a.e.Hkv * a.e.budget;
    const uint32_t warp = (blockIdx.x * kMoveThreads + threadIdx.x) >> 5, warps = gridDim.x * (kMoveThreads / 32);
    for (uint32_t i0 = warp * (kGroups * kBatch); i0 < total; i0 += warps * (kGroups * kBatch)) {
        uint4 x[kBatch][2];
        uint8_t *to[kBatch][2];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const uint32_t i = i0 + j * kGroups + grp;
            to[j][0] = nullptr;
            if (i >= total) continue;
            const int t = __ldg(a.e.kept + i);
            if (t < 0) continue;
            if (t >= a.e.src.capacity) {  // the caller wrote to `kept` during the call
                atomicExch(&g_paged_error, 5);
                continue;
            }
            const uint32_t row = fdiv(i, div_n), b = fdiv(row, div_h);
            const int h = (int)(row - b * div_h.d), o = (int)(i - row * div_n.d);
            int ss, ds;
            const int sp = a.e.src.page((int)b, t, ss), dp = a.e.dst.page((int)b, o, ds);
            if (sp < 0 || dp < 0) continue;
            x[j][0] = __ldcs(reinterpret_cast<const uint4 *>(a.k + sp * a.kp + h * a.kh + (int64_t)ss * R + off));
            x[j][1] = __ldcs(reinterpret_cast<const uint4 *>(a.v + sp * a.vp + h * a.vh + (int64_t)ss * R + off));
            to[j][0] = a.k + dp * a.kp + h * a.kh + (int64_t)ds * R + off;
            to[j][1] = a.v + dp * a.vp + h * a.vh + (int64_t)ds * R + off;
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (!to[j][0]) continue;
            *reinterpret_cast<uint4 *>(to[j][0]) = x[j][0];
            *reinterpret_cast<uint4 *>(to[j][1]) = x[j][1];
        }
    }
}

}  // namespace paged

int evict_error(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, paged::g_paged_error, sizeof(int)) != cudaSuccess) return ECC_ERR_CUDA;
    if (reset) {
        const int z = 0;
        if (cudaMemcpyToSymbol(paged::g_paged_error, &z, sizeof(int)) != cudaSuccess) return ECC_ERR_CUDA;
    }
    return v;
}

}  // namespace ecc

using namespace ecc;

extern "C" size_t ecc_evict_paged_workspace_size(int64_t n_pages) {
    if (n_pages < 1 || n_pages >= (1ll << 31)) return 0;
    return (size_t)((n_pages + 31) / 32) * 4 + 4 + 256;
}

extern "C" int ecc_evict_paged(void *k_blocks, void *v_blocks, int64_t bs_p, int64_t bs_h, const ecc_pages_t *pages,
                               const int *seq_lens, const float *weights, int64_t ws_b, int64_t ws_h,
                               const ecc_pages_t *out_pages, float *out_weights, int64_t ows_b, int64_t ows_h,
                               int64_t out_len, int *kept, int B, int Hkv, int budget, int sinks, int recent,
                               int block_bytes, void *workspace, size_t workspace_bytes, ecc_stream_t stream) {
    using namespace paged;
    if (B == 0) return ECC_OK;
    if (!k_blocks || !v_blocks || !pages || !out_pages || !seq_lens || !weights || !out_weights || !kept)
        return ECC_ERR_NULL;
    if (B < 0 || Hkv < 1 || budget < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget || out_len < 0 ||
        out_len > (1ll << 30) || (block_bytes != 96 && block_bytes != kBlockBytes))
        return ECC_ERR_SHAPE;
    EvictArgs a{};
    int rc = make_table(*pages, &a.src);
    if (rc == ECC_OK) rc = make_table(*out_pages, &a.dst);
    if (rc != ECC_OK) return rc;
    if (pages->n_pages != out_pages->n_pages || pages->page_size != out_pages->page_size || a.dst.capacity < budget)
        return ECC_ERR_SHAPE;
    // 32-bit numbers of kept tokens (with the padding of the last step) and of clusters
    if (B > ECC_PAGED_MAX_BATCH || (int64_t)B * Hkv >= (1 << 20) || (int64_t)B * Hkv * budget >= (1ll << 31))
        return ECC_ERR_SHAPE;
    if ((uintptr_t)k_blocks % 16 || (uintptr_t)v_blocks % 16 || (uintptr_t)seq_lens % 4 || (uintptr_t)weights % 4 ||
        (uintptr_t)out_weights % 4 || (uintptr_t)kept % 4)
        return ECC_ERR_ALIGN;
    if (!workspace || workspace_bytes < ecc_evict_paged_workspace_size(pages->n_pages)) return ECC_ERR_WORKSPACE;
    a.lens = seq_lens;
    a.w = weights;
    a.w_b = ws_b;
    a.w_h = ws_h;
    a.ow = out_weights;
    a.ow_b = ows_b;
    a.ow_h = ows_h;
    a.ow_len = (int)out_len;
    a.kept = kept;
    a.B = B;
    a.Hkv = Hkv;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    uint8_t *ws = reinterpret_cast<uint8_t *>(((uintptr_t)workspace + 255) / 256 * 256);
    a.clash = reinterpret_cast<int *>(ws);
    a.bitmap = reinterpret_cast<uint32_t *>(ws + 4);

    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int64_t rows = (int64_t)B * Hkv;
    const int C = sel::cluster_size(evict_select_kernel, rows + 1, a.src.capacity, 4096);
    // the keys of a slice stay in shared memory when they fit beside the counts
    const int64_t slice = (a.src.capacity + C - 1) / C;
    a.cache_keys = (int)std::min<int64_t>(slice, (227 * 1024 - sizeof(sel::Shared)) / 4);
    if (sel::launch_cluster(evict_select_kernel, C, rows + 1, sizeof(sel::Shared) + (size_t)a.cache_keys * 4, s, a) != cudaSuccess)
        return ECC_ERR_LAUNCH;
    rc = launch_status();
    if (rc != ECC_OK) return rc;

    MoveArgs m{a, reinterpret_cast<uint8_t *>(k_blocks), reinterpret_cast<uint8_t *>(v_blocks), bs_p * block_bytes,
               bs_h * block_bytes, bs_p * block_bytes, bs_h * block_bytes};
    const int64_t per_cta = (kMoveThreads / 32) * (block_bytes == 96 ? 5 : 4) * kBatch;
    const int64_t grid = std::min<int64_t>((rows * budget + per_cta - 1) / per_cta, (int64_t)sm_count() * 8);
    const FastDiv dn = make_fastdiv((uint32_t)budget), dh = make_fastdiv((uint32_t)Hkv);
    const cudaError_t e =
        block_bytes == 96
            ? launch_pdl(evict_move_kernel<96>, dim3((unsigned)grid), dim3(kMoveThreads), 0, s, m, dn, dh)
            : launch_pdl(evict_move_kernel<128>, dim3((unsigned)grid), dim3(kMoveThreads), 0, s, m, dn, dh);
    if (e != cudaSuccess) return ECC_ERR_LAUNCH;
    return launch_status();
}
