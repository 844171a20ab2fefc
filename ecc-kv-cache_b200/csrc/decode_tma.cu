// decode_tma.cu -- TMA-fed tensor-core decode attention over 128-byte blocks
// (sm_100a), GQA groups of up to 8 query heads per kv head.
//
// Work split: the tiles (16 tokens of one (b, kv head) row) of all rows are
// laid end to end and cut into equal contiguous ranges, one per warp of the
// grid (persistent CTAs, one per SM, kWarps warps each).  A warp therefore
// sees at most a few row segments; for each it builds the query fragments in
// its own registers (loaded straight from global memory, WHT-rotated across
// the four lanes that hold one head) and writes one split partial (m, l, o)
// at the end.  Partial slot of a segment = warp - first warp of the row, so
// every row's partials are contiguous; the last warp of a row marks the
// row's unused slots empty.  No CTA-wide barrier is needed after set-up.
//
// Each warp streams its tiles through its own kStages-stage shared-memory
// ring: one lane issues four cp.async.bulk.tensor boxes per tile (K codes
// 16x64 B, K syndrome+meta 16x32 B, V codes, V syndrome+meta) on an mbarrier
// and later waits on it, then __syncwarp hands the data to the warp.  The
// tensor maps cover [0, seq_len) tokens, so rows past the sequence end come
// back as zeros; such tokens are masked to -inf.  QK: per 16-dim step, one
// m16n8k16 product for the centroids of 8 tokens (rows g / g+8 = fp16 hi /
// lo parts) per token half and one for the signs.  PV: per code byte of the
// lane (two dims in rows g / g+8), four products: centroids hi and lo
// against p*scale_v, centroids hi against its fp16 residual, signs against
// the sign weights.
//
// Every mbarrier wait is bounded (~2 s of clock64); on timeout the warp
// raises a device flag for ecc_device_status(), stops computing and drains
// its outstanding copies (bounded) before exiting.
#include <algorithm>

#include "decode_tile.cuh"

namespace ecc {

int launch_status();
int sm_count();

namespace tmak {

template <int G>
__global__ void __launch_bounds__(kThreads, 1)
decode_tma_kernel(const __grid_constant__ CUtensorMap mkc, const __grid_constant__ CUtensorMap mks,
                  const __grid_constant__ CUtensorMap mvc, const __grid_constant__ CUtensorMap mvs,
                  const __half *__restrict__ q, float *__restrict__ pm, float *__restrict__ pl,
                  float *__restrict__ po, int Hq, int Hkv, int64_t seq_len, int tpr, int64_t T, int nslots,
                  float scale_log2, int flags, const int *__restrict__ seq_len_dev,
                  const int *__restrict__ start_dev) {
    extern __shared__ __align__(1024) uint8_t sm[];
    // broadcast from lane 0 so that the compiler treats the warp index, and
    // the tile cursors derived from it, as warp-uniform values
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(sm);
    if (sbase != (uint32_t)kSmemReserve) {  // the table loads assume this base
        if (threadIdx.x == 0) atomicExch(&g_device_error, 2);
        return;
    }
    uint32_t *s_cent = reinterpret_cast<uint32_t *>(sm + kSmCent);
    const uint32_t ring = sbase + kSmRing + warp * kStages * kStageBytes;
    const uint32_t bars = sbase + kSmBar + warp * kStages * 8;

    if (threadIdx.x < 16) {
        const float cv = lm(threadIdx.x);
        const __half hi = __float2half_rn(cv);
        const __half lo = __float2half_rn(cv - __half2float(hi));
        s_cent[threadIdx.x] = (uint32_t)__half_as_ushort(hi) | ((uint32_t)__half_as_ushort(lo) << 16);
    }
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(bars + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    for (int v = warp; v < 256; v += kWarps) {
        const uint32_t e0 = s_cent[v & 15], e1 = s_cent[v >> 4];
        uint2 e;
        e.x = __byte_perm(e0, e1, 0x5410);
        e.y = __byte_perm(e0, e1, 0x7632);
        reinterpret_cast<uint32_t *>(sm + kSmLut + v * 256)[lane] = e.x;
        reinterpret_cast<uint32_t *>(sm + kSmLut + v * 256 + 128)[lane] = e.y;
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();  // everything above touched shared memory only

    if (seq_len_dev) {
        // Length in device memory (a launch recorded once and replayed as the
        // context grows): seq_len, tpr, T above describe the capacity the
        // tensor maps cover; the partition is rebuilt for the current length,
        // clamped to [1, capacity].
        const int64_t rows = T / tpr;
        seq_len = max((int64_t)1, min((int64_t)*seq_len_dev, seq_len));
        tpr = (int)((seq_len + kTile - 1) / kTile);
        T = rows * tpr;
    }
    // at most one warp per tile, so that every range is non-empty and the
    // partial slots of a row have no holes
    const int64_t NW = min((int64_t)gridDim.x * kWarps, T);
    const int64_t wid = (int64_t)blockIdx.x * kWarps + warp;
    if (wid >= NW) return;
    const int64_t tbeg = wid * T / NW;
    const int ntiles = (int)((wid + 1) * T / NW - tbeg);
    const int row_tok = tpr * kTile;  // tokens of a row rounded up to whole tiles

    // Producer cursor: (token base, kv head, batch) of the next tile to issue.
    // Kept by every lane (uniform arithmetic, no divisions per tile); lane 0
    // issues.
    int p_tb, p_kvh, p_b;
    {
        const int64_t r0 = tbeg / tpr;
        p_tb = (int)(tbeg - r0 * tpr) * kTile;
        p_kvh = (int)(r0 % Hkv);
        p_b = (int)(r0 / Hkv);
    }
    auto issue_next = [&](int s) {
        if (lane == 0) {
            const uint32_t bar = bars + 8 * s, dst = ring + s * kStageBytes;
            fence_proxy_async();  // this warp's earlier reads of the stage precede the overwrite
            mbar_expect_tx(bar, kStageBytes);
            tma_4d(dst + kOffKC, &mkc, 0, p_tb, p_kvh, p_b, bar);
            tma_4d(dst + kOffKS, &mks, 64, p_tb, p_kvh, p_b, bar);
            tma_4d(dst + kOffVC, &mvc, 0, p_tb, p_kvh, p_b, bar);
            tma_4d(dst + kOffVS, &mvs, 64, p_tb, p_kvh, p_b, bar);
        }
        p_tb += kTile;
        if (p_tb >= row_tok) {
            p_tb = 0;
            if (++p_kvh == Hkv) {
                p_kvh = 0;
                ++p_b;
            }
        }
    };
    Lane<G> L;
    L.g = lane >> 2;
    L.c = lane & 3;
    // Query words of lane (g, c): dims 32c..32c+31 of query head g of the
    // group (with the split columns, G <= 4, lanes g >= 4 repeat head g - 4,
    // so that the softmax state of columns 4..7, the V sign products, is that
    // of the head they belong to); zero for heads past the group.  The first
    // segment's words are requested before the first stages, so that they do
    // not queue behind the whole grid's first tiles.
    auto load_q = [&](uint4 (&qw)[4], int64_t row) {
        const int qh = (G <= 4) ? (L.g & 3) : L.g;
        const int b_ = (int)(row / Hkv), h0_ = (int)(row % Hkv) * G;
        const uint4 *src = reinterpret_cast<const uint4 *>(q + ((int64_t)b_ * Hq + h0_ + qh) * kD + 32 * L.c);
#pragma unroll
        for (int k = 0; k < 4; ++k) qw[k] = qh < G ? __ldg(src + k) : make_uint4(0u, 0u, 0u, 0u);
    };
    {
        uint4 qw[4];
        load_q(qw, tbeg / tpr);
        for (int s = 0; s < kStages && s < ntiles; ++s) issue_next(s);
        L.set_query(qw, (flags & ECC_DECODE_ROTATE_Q) != 0);
    }

    L.lane4 = (uint32_t)lane * 4u;
    L.sel_half = (L.g & 1) ? 0x7632u : 0x5410u;
    L.voff = 16u * (uint32_t)((L.g >> 1) ^ L.c) + 8u * (uint32_t)(L.g & 1);
    L.soff = 16u * (uint32_t)((L.g >> 2) & 1);
    L.scale_log2 = scale_log2;
    bool ok = true;
    int jfail = -1;        // first tile whose wait ran out
    int j = 0;             // tiles of this warp's range consumed so far
    int stage = 0;         // ring stage of tile j
    uint32_t phase = 0;    // mbarrier parity of tile j
    int64_t r = tbeg / tpr;                  // row of tile j
    int tok0 = (int)(tbeg - r * tpr) * kTile;  // first token of tile j within its row
    while (j < ntiles) {
        // ---------------- new row segment ----------------
        const int seg_tiles = min(ntiles - j, (row_tok - tok0) / kTile);
        const bool row_ends = (tok0 + seg_tiles * kTile == row_tok);
        const int kvh = (int)(r % Hkv), b = (int)(r / Hkv);
        const int h0 = kvh * G;
        // first attended token of the sequence (left padding before it)
        const int t_start = start_dev ? __ldg(start_dev + b) : 0;
        if (j > 0) {
            uint4 qw[4];
            load_q(qw, r);
            L.set_query(qw, (flags & ECC_DECODE_ROTATE_Q) != 0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) L.o[i][k] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            L.mrun[e] = -INFINITY;
            L.lrun[e] = 0.0f;
            L.zrun[e] = 0.0f;
        }
        // ---------------- tiles of the segment ----------------
        for (int u = 0; u < seg_tiles; ++u) {
            // every lane polls the stage's mbarrier once (one warp-wide
            // try_wait, no divergence); a warp that does not find the phase
            // complete in every lane takes the bounded wait in lane 0
            bool ready = ok;
            if (ok && !__all_sync(0xffffffffu, mbar_try(bars + 8 * stage, phase))) {
                bool r = true;
                if (lane == 0) r = mbar_wait(bars + 8 * stage, phase);
                ready = __shfl_sync(0xffffffffu, r, 0);
            }
            __syncwarp();  // orders the warp's reads of the stage after the wait
            if (ok && !ready) jfail = j;
            ok = ok && ready;
            if (ok)
                L.tile(ring + stage * kStageBytes, SeeRange{t_start - tok0, (int)min((int64_t)kTile, seq_len - tok0)});
            __syncwarp();
            if (ok && j + kStages < ntiles) issue_next(stage);
            ++j;
            tok0 += kTile;
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // ---------------- partial of the segment ----------------
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                L.lrun[e] += __shfl_xor_sync(0xffffffffu, L.lrun[e], off);
                L.zrun[e] += __shfl_xor_sync(0xffffffffu, L.zrun[e], off);
            }
        }
        const int slot = (int)(wid - owner_warp(r * tpr, T, NW));
        const int64_t prow = ((int64_t)b * Hq + h0) * nslots + slot;  // partial of head h0 of the group
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // accumulator i: rows g / g+8 = dims 16g + 2i / 16g + 2i + 1;
            // with the split columns the sign terms of heads 2c, 2c+1 are in
            // columns 4..7 of lane c + 2, each row with its power-of-two weight
            float sg[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (G <= 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    sg[k] = __shfl_down_sync(0xffffffffu, L.o[i][k], 2) * sign_unweight(k < 2 ? 2 * i : 2 * i + 1);
            }
            const int d0 = 16 * L.g + 2 * i;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int h = 2 * L.c + e;
                if (h >= G) continue;
                float2 *pod = reinterpret_cast<float2 *>(po + (prow + (int64_t)h * nslots) * kD + d0);
                *pod = make_float2(L.o[i][e] + (sg[e] + L.zrun[e]), L.o[i][2 + e] + (sg[2 + e] + L.zrun[e]));
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int h = 2 * L.c + e;
            if (h >= G) continue;
            const int64_t pr = ((int64_t)b * Hq + h0 + h) * nslots;
            if (L.g == 0) {
                pm[pr + slot] = (L.mrun[e] == -INFINITY) ? -INFINITY : L.mrun[e] * kLn2f;
                pl[pr + slot] = L.lrun[e];
                if (row_ends) {  // last segment of the row: the rest are empty
                    for (int k = slot + 1; k < nslots; ++k) {
                        pm[pr + k] = -INFINITY;
                        pl[pr + k] = 0.0f;
                    }
                }
            }
        }
        if (row_ends) {
            ++r;
            tok0 = 0;
        }
    }
    if (!ok && lane == 0) {
        // drain the copies still in flight before the warp exits: tiles
        // jfail .. min(ntiles, jfail + kStages) - 1 were issued and not consumed
        for (int k = jfail; k < min(ntiles, jfail + kStages); ++k) {
            const uint32_t bar = bars + 8 * (k % kStages);
            const long long c0 = clock64();
            while (!mbar_try(bar, (uint32_t)((k / kStages) & 1)) && clock64() - c0 < kWaitCycles) {
            }
        }
    }
}

// ---- host ----
template <int G>
static int launch_g(const CUtensorMap &kc, const CUtensorMap &ks, const CUtensorMap &vc, const CUtensorMap &vs,
                    const void *q, float *pm, float *pl, float *po, int Hq, int Hkv, int64_t seq_len, int tpr,
                    int64_t T, int grid, int ns, float scale_log2, int flags, cudaStream_t s,
                    const int *seq_len_dev = nullptr, const int *start_dev = nullptr) {
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        if (cudaFuncSetAttribute(decode_tma_kernel<G>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmBytes) !=
            cudaSuccess)
            return ECC_ERR_CUDA;
        configured[dev] = true;
    }
    if (launch_pdl(decode_tma_kernel<G>, dim3(grid), dim3(kThreads), kSmBytes, s, kc, ks, vc, vs,
                   reinterpret_cast<const __half *>(q), pm, pl, po, Hq, Hkv, seq_len, tpr, T, ns, scale_log2,
                   flags, seq_len_dev, start_dev) != cudaSuccess)
        return ECC_ERR_LAUNCH;
    return launch_status();
}

// Grid and partial-slot count of the balanced tile partition for a shape.
struct Plan {
    int grid;
    int64_t tpr, T;
    int nslots;
};
static Plan make_plan(int B, int Hkv, int64_t seq_len) {
    Plan p;
    p.tpr = (std::max<int64_t>(seq_len, 1) + kTile - 1) / kTile;
    const int64_t rows = (int64_t)B * Hkv;
    p.T = rows * p.tpr;
    p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(sm_count(), (p.T + kWarps - 1) / kWarps));
    const int64_t NW = std::min<int64_t>((int64_t)p.grid * kWarps, p.T);
    int64_t mx = 1;
    for (int64_t r = 0; r < rows; ++r) {
        const int64_t n = owner_warp(r * p.tpr + p.tpr - 1, p.T, NW) - owner_warp(r * p.tpr, p.T, NW) + 1;
        mx = std::max(mx, n);
    }
    p.nslots = (int)mx;
    return p;
}

}  // namespace tmak

// Partial slots per (b, query head) of the balanced partition: the split
// count ecc_decode uses by default.
int tma_default_splits(int B, int Hkv, int64_t seq_len) { return tmak::make_plan(B, Hkv, seq_len).nslots; }

// Returns ECC_OK when launched, a positive value when the shape is not one the
// TMA kernel handles (the caller then uses another kernel), or an error.
int launch_decode_tma(const void *q, const void *kb, const void *vb, int64_t bs_b, int64_t bs_h, float *pm,
                      float *pl, float *po, int B, int Hq, int Hkv, int64_t seq_len, int64_t chunk, int ns,
                      float scale_log2, int flags, cudaStream_t s, const int *start_dev) {
    using namespace tmak;
    (void)chunk;
    const int G = Hq / Hkv;
    if (G < 1 || G > 8 || seq_len < 1 || seq_len > (1ll << 30)) return 1;
    if (((uintptr_t)kb % 16) || ((uintptr_t)vb % 16) || ((uintptr_t)q % 16)) return 1;
    const Plan plan = make_plan(B, Hkv, seq_len);
    if (ns < plan.nslots) return 1;  // fewer partial slots than the partition writes
    if (!reserve_matches()) return 1;
    if (get_encode() != ECC_OK) return 1;
    const int rb = (flags & ECC_DECODE_BLOCK96) ? 96 : kBlockBytes;
    flags &= ECC_DECODE_ROTATE_Q;
    CUtensorMap kc, ks, vc, vs;
    if (make_maps(&kc, &ks, &vc, &vs, kb, vb, seq_len, Hkv, B, bs_h, bs_b, rb) != ECC_OK) return 1;
    switch (G) {
#define ECC_TMA_CASE(N) \
    case N: return launch_g<N>(kc, ks, vc, vs, q, pm, pl, po, Hq, Hkv, seq_len, (int)plan.tpr, plan.T, plan.grid, ns, scale_log2, flags, s, nullptr, start_dev);
        ECC_TMA_CASE(1) ECC_TMA_CASE(2) ECC_TMA_CASE(3) ECC_TMA_CASE(4)
        ECC_TMA_CASE(5) ECC_TMA_CASE(6) ECC_TMA_CASE(7)
        default: return launch_g<8>(kc, ks, vc, vs, q, pm, pl, po, Hq, Hkv, seq_len, (int)plan.tpr, plan.T, plan.grid, ns,
                                    scale_log2, flags, s, nullptr, start_dev);
#undef ECC_TMA_CASE
    }
}

// Partial slots that cover the balanced partition of every length up to
// max_len with the grid used for max_len: a row's tiles touch fewer than
// NW / rows + 2 warps (NW <= grid * kWarps), and never more than its tiles.
void tma_dev_plan(int B, int Hkv, int64_t max_len, int *grid, int *nslots) {
    using namespace tmak;
    const Plan p = make_plan(B, Hkv, max_len);
    const int64_t rows = (int64_t)B * Hkv;
    *grid = p.grid;
    *nslots = (int)std::min<int64_t>(p.tpr, (int64_t)p.grid * kWarps / rows + 2);
}

// The TMA decode with the length read from device memory at *seq_len_dev
// (clamped to [1, max_len]); tensor maps over max_len tokens.  Returns ECC_OK,
// a positive value when the shape is not one the TMA kernel handles, or an
// error.
int launch_decode_tma_dev(const void *q, const void *kb, const void *vb, int64_t bs_b, int64_t bs_h, float *pm,
                          float *pl, float *po, int B, int Hq, int Hkv, int64_t max_len, const int *seq_len_dev,
                          int ns, float scale_log2, int flags, cudaStream_t s) {
    using namespace tmak;
    const int G = Hq / Hkv;
    if (G < 1 || G > 8 || max_len < 1 || max_len > (1ll << 30)) return 1;
    if (((uintptr_t)kb % 16) || ((uintptr_t)vb % 16) || ((uintptr_t)q % 16)) return 1;
    int grid = 0, need = 0;
    tma_dev_plan(B, Hkv, max_len, &grid, &need);
    if (ns < need) return 1;
    const Plan plan = make_plan(B, Hkv, max_len);
    if (!reserve_matches()) return 1;
    if (get_encode() != ECC_OK) return 1;
    const int rb = (flags & ECC_DECODE_BLOCK96) ? 96 : kBlockBytes;
    flags &= ECC_DECODE_ROTATE_Q;
    CUtensorMap kc, ks, vc, vs;
    if (make_maps(&kc, &ks, &vc, &vs, kb, vb, max_len, Hkv, B, bs_h, bs_b, rb) != ECC_OK) return 1;
    switch (G) {
#define ECC_TMA_CASE(N) \
    case N: return launch_g<N>(kc, ks, vc, vs, q, pm, pl, po, Hq, Hkv, max_len, (int)plan.tpr, plan.T, grid, ns, scale_log2, flags, s, seq_len_dev);
        ECC_TMA_CASE(1) ECC_TMA_CASE(2) ECC_TMA_CASE(3) ECC_TMA_CASE(4)
        ECC_TMA_CASE(5) ECC_TMA_CASE(6) ECC_TMA_CASE(7)
        default: return launch_g<8>(kc, ks, vc, vs, q, pm, pl, po, Hq, Hkv, max_len, (int)plan.tpr, plan.T, grid, ns,
                                    scale_log2, flags, s, seq_len_dev);
#undef ECC_TMA_CASE
    }
}

}  // namespace ecc

namespace ecc {
namespace tmak {
// Self-test of the bounded wait: one warp arms an mbarrier for bytes that no
// copy will deliver and waits on it with mbar_wait (the decode's wait) and a
// short limit.  The wait runs out, raises the device flag and the kernel
// returns; *out = 1 when the warp saw the wait give up.
__global__ void wait_timeout_selftest_kernel(long long limit, int *out) {
    __shared__ __align__(8) uint64_t bar;
    const uint32_t b = smem_u32(&bar);
    if (threadIdx.x == 0) {
        mbar_init(b, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(b, 16);  // 16 bytes that never arrive: the phase never completes
    }
    __syncwarp();
    bool ok = true;
    if (threadIdx.x == 0) ok = mbar_wait(b, 0, limit);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (threadIdx.x == 0) *out = ok ? 0 : 1;
}
}  // namespace tmak
}  // namespace ecc

extern "C" int ecc_selftest_wait_timeout(long long limit_cycles, int *host_gave_up) {
    if (!host_gave_up || limit_cycles <= 0 || limit_cycles > (4ll << 30)) return ECC_ERR_SHAPE;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ECC_ERR_DEVICE;
    int *d = nullptr;
    if (cudaMalloc(&d, sizeof(int)) != cudaSuccess) return ECC_ERR_CUDA;
    ecc::tmak::wait_timeout_selftest_kernel<<<1, 32>>>(limit_cycles, d);
    int rc = ecc::launch_status();
    if (rc == ECC_OK && cudaMemcpy(host_gave_up, d, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess)
        rc = ECC_ERR_CUDA;
    cudaFree(d);
    return rc;
}

namespace ecc {
int compress_device_error(int reset);
int exchange_device_error(int reset);
int compress_paged_error(int reset);
int paged_decode_error(int reset, int *wait_error);
int paged_cache_error(int reset);
int evict_error(int reset);
}

extern "C" int ecc_device_status(int reset) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, ecc::g_device_error, sizeof(int)) != cudaSuccess) return ECC_ERR_CUDA;
    if (reset) {
        const int z = 0;
        if (cudaMemcpyToSymbol(ecc::g_device_error, &z, sizeof(int)) != cudaSuccess) return ECC_ERR_CUDA;
    }
    const int c = ecc::compress_device_error(reset);
    if (c < 0) return c;
    const int x = ecc::exchange_device_error(reset);
    if (x < 0) return x;
    int w = 0;
    int p = 0;
    for (int e : {ecc::paged_decode_error(reset, &w), ecc::compress_paged_error(reset), ecc::paged_cache_error(reset),
                  ecc::evict_error(reset)}) {
        if (e < 0) return e;
        p = p ? p : e;
    }
    if (!v) v = w;
    return v ? v : c ? c : x ? x : p;
}
