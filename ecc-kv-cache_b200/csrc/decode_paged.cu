// decode_paged.cu -- decode attention of one new token per sequence over a
// paged block cache (sm_100a): ragged lengths in device memory, an optional
// sliding window with sinks, and the attention weight of every cached token.
//
// Math per (sequence b, query head h), kv head = h / (Hq / Hkv), over the
// visible tokens t < L_b with (no window) or t >= L_b - window or t < sinks:
//   k_t, v_t = (C[q_t] scale_t + zero_t) + alpha_t s_t
//   s_t = sm_scale <q, k_t>,  out = sum_t softmax(s)_t v_t,  lse = log sum_t e^s_t
//   weights[b, kv head, t] += sum over the group's heads of softmax(s)_t
//
// The arithmetic of a 32-token stage is decode_tile.cuh's; this file gives it
// tiles out of pages.  A sequence's tiles are those that hold a visible
// token: the first ceil(sinks / 32) and those from the window's start on.  The
// tiles of all (sequence, kv head) rows, end to end, are cut into one equal
// range per warp of a persistent grid, so ragged lengths stay balanced however
// they are spread; the cut is made on the device from the lengths, so one
// recorded launch serves a growing cache.
//
// A warp that works on row r as range w writes its partial to slot w + r:
// along the tiles w or r grows by one at every new (range, row) pair, so the
// slots are distinct, a row's slots are contiguous, and NW + rows slots
// suffice for every distribution of lengths.  paged_merge_kernel joins them.
//
// Measured at 8 sequences x 65531 tokens, 32 query and 8 kv heads, pages of 128
// tokens (1.07 GB of blocks): 229 us with the merge, 4.7 TB/s; the loads alone
// take 169 us.  It is bound by the latency of dependent instructions at three
// warps of 168 registers per scheduler (ncu: issue 57 %, L1 62 %,
// ALU 52 %, tensor 37 %), and in runs of seconds by the 1000 W
// power cap.
#include <algorithm>

#include "decode_tile.cuh"
#include "paged.cuh"

namespace ecc {

int launch_status();
int sm_count();

namespace paged {

using namespace tmak;

// Room for the prefix sums of the sequences' tiles behind the ring.
constexpr int kMaxBatch = ECC_PAGED_MAX_BATCH;
constexpr int kSmPrefix = kSmBytes;                        // [kMaxBatch + 1] int
constexpr int kSmPaged = kSmPrefix + 4 * (kMaxBatch + 4);  // total
static_assert(kSmPaged <= 227 * 1024, "shared memory budget");
constexpr int kMaxRanges = 4096;  // warps of a launch at most (merge weights in shared memory)

struct DecodeArgs {
    const __half *q;
    PageTable t;
    const int *lens;
    int B, Hq, Hkv;
    int window, sinks;
    float scale_log2;
    int flags;
    float *pm, *pl, *po;
    int *row_first, *row_last;  // first and last range of a row
    float *raw;                 // log2-scaled scores [row][capacity][G], or null
    int64_t slots;              // partial slots of the workspace
};

// Tokens below x of a 32-token tile, as bits.
__device__ __forceinline__ uint32_t below(int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; }

// The tiles of one sequence: [0, nsink) hold sinks, the rest start at tile w0.
struct SeqTiles {
    int len, ws, nsink, w0, n;
    __device__ __forceinline__ SeqTiles() : len(0), ws(0), nsink(0), w0(0), n(0) {}
    __device__ __forceinline__ SeqTiles(int len_, int window, int sinks) : len(len_) {
        ws = window > 0 ? max(0, len - window) : 0;
        w0 = ws / kTile;
        nsink = min((min(sinks, ws) + kTile - 1) / kTile, w0);
        n = nsink + (len + kTile - 1) / kTile - w0;
    }
    __device__ __forceinline__ int base(int u) const { return kTile * (u < nsink ? u : u - nsink + w0); }
    __device__ __forceinline__ uint32_t visible(int tb, int sinks) const {
        return below(len - tb) & (below(sinks - tb) | ~below(ws - tb));
    }
};

__device__ __forceinline__ int seq_len_of(const DecodeArgs &a, int b) {
    const int n = __ldg(a.lens + b);
    return max(0, min(n, a.t.capacity));
}

// Hands the stage's scores to global memory: lane (g, c) holds tokens g, g + 8
// of both sub-tiles for heads 2c, 2c + 1.
template <int G>
struct StoreScores {
    float *dst;  // row and tile applied
    int g, c, n;  // n: tokens of the tile inside the sequence
    __device__ __forceinline__ void put(int tok, float a, float b) const {
        if (tok >= n) return;
        float *d = dst + (int64_t)tok * G + 2 * c;
        if constexpr (G % 2 == 0) {
            if (2 * c < G) *reinterpret_cast<float2 *>(d) = make_float2(a, b);
        } else {
            if (2 * c < G) d[0] = a;
            if (2 * c + 1 < G) d[1] = b;
        }
    }
    __device__ __forceinline__ void operator()(const float (&s0)[4], const float (&s1)[4]) const {
        put(g, s0[0], s0[1]);
        put(g + 8, s0[2], s0[3]);
        put(g + 16, s1[0], s1[1]);
        put(g + 24, s1[2], s1[3]);
    }
};

// Where a warp stands in the list of tiles: sequence b, kv head h, tile u.
struct Cursor {
    int b, h, u;
    SeqTiles st;
};

// kHalves: a stage is fetched as two 16-token boxes by two lanes, for pages that
// are no multiple of 32 tokens.  (A form of its own: with one box a stage every
// cursor is the same in all lanes, which the other form's loop pays 4 % for.)
template <int G, bool kScores, bool kHalves>
__global__ void __launch_bounds__(kThreads, 1)
decode_paged_kernel(const __grid_constant__ CUtensorMap mkc, const __grid_constant__ CUtensorMap mks,
                    const __grid_constant__ CUtensorMap mvc, const __grid_constant__ CUtensorMap mvs,
                    const __grid_constant__ DecodeArgs a) {
    extern __shared__ __align__(1024) uint8_t sm[];
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(sm);
    if (sbase != (uint32_t)kSmemReserve) {  // the table loads assume this base
        if (threadIdx.x == 0) atomicExch(&g_device_error, 2);
        return;
    }
    uint32_t *s_cent = reinterpret_cast<uint32_t *>(sm + kSmCent);
    int *s_pre = reinterpret_cast<int *>(sm + kSmPrefix);  // tiles of one kv head before sequence b
    const uint32_t ring = sbase + kSmRing + warp * kStages * kStageBytes;
    const uint32_t bars = sbase + kSmBar + warp * kStages * 8;

    if (threadIdx.x < 16) {
        const float cv = lm(threadIdx.x) * kCentScale;
        const __half hi = __float2half_rn(cv);
        const __half lo = __float2half_rn(cv - __half2float(hi));
        s_cent[threadIdx.x] = (uint32_t)__half_as_ushort(hi) | ((uint32_t)__half_as_ushort(lo) << 16);
    }
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(bars + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // a half-warp writes a row of the table, a lane the entries of two lanes (both of one half)
#pragma unroll 4
    for (int v = 2 * warp + (lane >> 4); v < 256; v += 2 * kWarps) {
        const uint2 e = lut_entry(s_cent, v, 2 * (lane & 15));
        reinterpret_cast<uint4 *>(sm + kSmLut + v * 256)[lane & 15] = make_uint4(e.x, e.y, e.x, e.y);
    }
    pdl_trigger();
    pdl_wait();  // everything above touched shared memory only

    // prefix sums of the sequences' tiles
    for (int b = threadIdx.x; b < a.B; b += kThreads) {
        const int n = __ldg(a.lens + b);
        if ((n < 0 || n > a.t.capacity) && blockIdx.x == 0) atomicExch(&g_paged_error, 5);
        s_pre[b + 1] = SeqTiles(max(0, min(n, a.t.capacity)), a.window, a.sinks).n;
    }
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int b0 = 0; b0 < a.B; b0 += 32) {
            int v = b0 + lane < a.B ? s_pre[b0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += x;
            }
            if (b0 + lane < a.B) s_pre[b0 + lane + 1] = carry + v;
            carry += __shfl_sync(0xffffffffu, v, 31);
        }
        if (lane == 0) s_pre[0] = 0;
    }
    __syncthreads();

    const int Hkv = a.Hkv;
    const uint32_t T = (uint32_t)s_pre[a.B] * Hkv;  // below 2^31 (check_shape)
    const uint32_t NW = min(gridDim.x * kWarps, T);
    // neighbouring ranges go to different SMs: a few tiles spread over the GPU
    const int64_t wid = (int64_t)warp * gridDim.x + blockIdx.x;
    if (wid >= NW) return;
    const uint32_t w32 = (uint32_t)wid;
    // range w starts at tile floor(w T / NW): with T = q NW + r that is w q + floor(w r / NW), w r < 2^24
    const uint32_t q_tiles = T / NW, r_tiles = T - q_tiles * NW;
    static_assert(kMaxRanges <= 4096, "products below 2^24");
    const int64_t tbeg = (int64_t)(w32 * q_tiles + w32 * r_tiles / NW);
    const int ntiles = (int)((int64_t)((w32 + 1) * q_tiles + (w32 + 1) * r_tiles / NW) - tbeg);

    // a sequence's tiles; their number is the one that the cut was made with
    auto tiles_of = [&](int b) {
        SeqTiles st(seq_len_of(a, b), a.window, a.sinks);
        st.n = s_pre[b + 1] - s_pre[b];
        return st;
    };
    Cursor cons;
    {
        int lo = 0, hi = a.B - 1;  // last sequence whose first tile is <= tbeg
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((int64_t)s_pre[mid] * Hkv <= tbeg) lo = mid;
            else hi = mid - 1;
        }
        cons.b = lo;
        cons.st = tiles_of(lo);
        const int rest = (int)(tbeg - (int64_t)s_pre[lo] * Hkv);
        cons.h = rest / cons.st.n;
        cons.u = rest - cons.h * cons.st.n;
    }
    Cursor prod = cons;
    auto advance_row = [&](Cursor &k) {  // to the next row's first tile
        k.u = 0;
        if (++k.h == Hkv) {
            k.h = 0;
            do ++k.b;
            while (k.b < a.B && s_pre[k.b + 1] == s_pre[k.b]);
            if (k.b < a.B) k.st = tiles_of(k.b);
        }
    };

    // The next tile to fetch: slot p_slot of page p_page (lane 1, with two boxes a stage: of its second 16
    // tokens), p_left tiles before the run of neighbouring tiles ends; the page after it is looked up early.
    int p_slot, p_page, p_next = 0, p_pi, p_left;
    const int *p_row;  // the sequence's row of the table
    auto page_at = [&](int pi) { return pi < a.t.width ? __ldg(p_row + pi) : -1; };
    auto start_run = [&]() {
        const int tb = prod.st.base(prod.u) + (kHalves ? 16 * (lane & 1) : 0);
        p_left = (prod.u < prod.st.nsink ? prod.st.nsink : prod.st.n) - prod.u;
        p_row = a.t.table + (int64_t)prod.b * a.t.stride;
        p_pi = (int)a.t.page_of(tb);
        p_slot = tb - p_pi * a.t.page_size;
        p_page = page_at(p_pi);
        if (!kHalves) p_next = page_at(p_pi + 1);
    };
    auto issue_next = [&](int s, bool more) {
        const uint32_t bar = bars + 8 * s;
        if (lane == 0) {
            fence_proxy_async();  // this warp's earlier reads of the stage precede the overwrite
            mbar_expect_tx(bar, kStageBytes);
        }
        if (kHalves) __syncwarp();
        if (lane == 0 || (kHalves && lane == 1)) {
            int page = p_page;
            if ((uint32_t)page >= (uint32_t)a.t.n_pages) {
                // no such page: the copy reads zeros out of the map's range.  The second half of
                // a sequence's last tile may lie behind its pages, which is no error.
                if (prod.st.base(prod.u) + 16 * lane < prod.st.len) atomicExch(&g_paged_error, 5);
                page = a.t.n_pages;
            }
            const uint32_t dst = ring + s * kStageBytes;
            if (kHalves) fence_proxy_async();
            tma_4d(dst + kOffKC + lane * kSubC, &mkc, 0, p_slot, prod.h, page, bar);
            tma_4d(dst + kOffKS + lane * kSubS, &mks, 64, p_slot, prod.h, page, bar);
            tma_4d(dst + kOffVC + lane * kSubC, &mvc, 0, p_slot, prod.h, page, bar);
            tma_4d(dst + kOffVS + lane * kSubS, &mvs, 64, p_slot, prod.h, page, bar);
        }
        if (!more) return;
        ++prod.u;
        if (--p_left == 0) {
            if (prod.u == prod.st.n) advance_row(prod);
            start_run();
        } else if (kHalves) {
            p_slot += kTile;
            if (p_slot >= a.t.page_size) {  // by one or two pages
                do {
                    p_slot -= a.t.page_size;
                    ++p_pi;
                } while (p_slot >= a.t.page_size);
                p_page = page_at(p_pi);
            }
        } else {
            p_slot += kTile;
            if (p_slot == a.t.page_size) {
                p_slot = 0;
                p_page = p_next;
                p_next = page_at(++p_pi + 1);
            }
        }
    };

    Lane<G, true> L;
    L.g = lane >> 2;
    L.c = lane & 3;
    L.scale_log2 = a.scale_log2;
    // query words of lane (g, c): dims 32c.. of query head g of the group (as in decode_tma_kernel)
    auto load_q = [&](uint4 (&qw)[4], int b, int h) {
        const int qh = (G <= 4) ? (L.g & 3) : L.g;
        const uint4 *src = reinterpret_cast<const uint4 *>(a.q + ((int64_t)b * a.Hq + h * G + qh) * kD + 32 * L.c);
#pragma unroll
        for (int k = 0; k < 4; ++k) qw[k] = qh < G ? __ldg(src + k) : make_uint4(0u, 0u, 0u, 0u);
    };
    {
        uint4 qw[4];
        load_q(qw, cons.b, cons.h);
        start_run();
        issue_next(0, ntiles > 1);
        L.set_query(qw, (a.flags & ECC_DECODE_ROTATE_Q) != 0);  // while the first copies are issued
        for (int s = 1; s < kStages && s < ntiles; ++s) issue_next(s, s + 1 < ntiles);
    }
    L.lane8 = (uint32_t)lane * 8u;
    L.lane_hi = lane_hi_of(lane);
    L.sel_half = (L.g & 1) ? 0x7632u : 0x5410u;
    L.voff = 16u * (uint32_t)((L.g >> 1) ^ L.c) + 8u * (uint32_t)(L.g & 1);
    L.soff = 16u * (uint32_t)((L.g >> 2) & 1);
    bool ok = true;
    int jfail = -1, j = 0, stage = 0;
    uint32_t phase = 0;
    while (j < ntiles) {
        // ---------------- new row segment ----------------
        const int seg_tiles = min(ntiles - j, cons.st.n - cons.u);
        const int row = cons.b * Hkv + cons.h;
        const bool begins = cons.u == 0, ends = cons.u + seg_tiles == cons.st.n;
        int tb = cons.st.base(cons.u);  // first token of the tile
        if (j > 0) {
            uint4 qw[4];
            load_q(qw, cons.b, cons.h);
            L.set_query(qw, (a.flags & ECC_DECODE_ROTATE_Q) != 0);
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
        L.vexp = 1;
        // ---------------- tiles of the segment ----------------
        for (int k = 0; k < seg_tiles; ++k) {
            bool ready = ok;
            if (ok && !__all_sync(0xffffffffu, mbar_try(bars + 8 * stage, phase))) {
                bool r = true;
                if (lane == 0) r = mbar_wait(bars + 8 * stage, phase);
                ready = __shfl_sync(0xffffffffu, r, 0);
            }
            __syncwarp();
            if (ok && !ready) jfail = j;
            ok = ok && ready;
            if (ok) {
                SeeBits see{0xffffffffu};
                if (tb + kTile > cons.st.len || tb < cons.st.ws) {
                    see.m = cons.st.visible(tb, a.sinks);
                    // Slots behind the last token hold whatever was there before: their V metadata (it may
                    // read as NaN or infinity) is cleared, so that 0 probability times it stays 0.  Lane =
                    // token; chunk 1 of its row in the swizzled box (see Lane::load_v).
                    if (!((see.m >> lane) & 1u))
                        *reinterpret_cast<uint2 *>(sm + (ring - sbase) + stage * kStageBytes + kOffVS + 32 * lane +
                                                   (16 ^ (16 * ((lane >> 2) & 1)))) = make_uint2(0u, 0u);
                    __syncwarp();
                }
                if constexpr (kScores)
                    L.tile(ring + stage * kStageBytes, see,
                           StoreScores<G>{a.raw + ((int64_t)row * a.t.capacity + tb) * G, L.g, L.c, cons.st.len - tb});
                else
                    L.tile(ring + stage * kStageBytes, see);
            }
            __syncwarp();
            if (ok && j + kStages < ntiles) issue_next(stage, j + kStages + 1 < ntiles);
            ++j;
            tb += kTile;
            if (++cons.u == cons.st.nsink) tb = kTile * cons.st.w0;
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
        const int64_t slot = wid + row;
        const float down = L.v_down();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float sg[4] = {0.f, 0.f, 0.f, 0.f};  // sign terms in the split columns (see decode_tma_kernel)
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
                float2 *pod = reinterpret_cast<float2 *>(a.po + (slot * G + h) * kD + d0);
                *pod = make_float2(fmaf(L.o[i][e] + sg[e], down, L.zrun[e]), fmaf(L.o[i][2 + e] + sg[2 + e], down, L.zrun[e]));
            }
        }
        if (L.g == 0) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int h = 2 * L.c + e;
                if (h >= G) continue;
                a.pm[slot * G + h] = L.mrun[e];
                a.pl[slot * G + h] = L.lrun[e];
            }
        }
        if (lane == 0) {
            if (begins) a.row_first[row] = (int)wid;
            if (ends) a.row_last[row] = (int)wid;
        }
        if (ends) advance_row(cons);
    }
    if (!ok && lane == 0) {
        // drain the copies still in flight before the warp exits
        for (int k = jfail; k < min(ntiles, jfail + kStages); ++k) {
            const uint32_t bar = bars + 8 * (k % kStages);
            const long long c0 = clock64();
            while (!mbar_try(bar, (uint32_t)((k / kStages) & 1)) && clock64() - c0 < kWaitCycles) {
            }
        }
    }
}

// Joins a row's partials: M = max m_i, w_i = 2^(m_i - M), L = sum l_i w_i,
// out = (sum o_i w_i) / L; one CTA per (sequence, query head), kMergeGroups
// groups of 128 threads (a thread per dimension) each take every
// kMergeGroups-th partial, so a long row (up to one partial per warp of the
// GPU) is read with enough loads in flight.  Every sum has a fixed order.
template <int kMergeGroups>
__global__ void __launch_bounds__(kD *kMergeGroups)
paged_merge_kernel(const __grid_constant__ DecodeArgs a, __half *__restrict__ out, float *__restrict__ lse,
                   float *__restrict__ lse2) {
    __shared__ float s_w[kMaxRanges];
    __shared__ float s_red[2][kD * kMergeGroups / 32];
    __shared__ float s_o[kMergeGroups][kD];
    const int G = a.Hq / a.Hkv;
    const int b = blockIdx.x / a.Hq, hq = blockIdx.x - b * a.Hq;
    const int row = b * a.Hkv + hq / G, e = hq - (hq / G) * G;
    const int tid = threadIdx.x, d = tid & (kD - 1), grp = tid / kD, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    // a short context is a chain of loads: each is asked for as early as its address is known
    const int len = seq_len_of(a, b), first = a.row_first[row], last = a.row_last[row];
    int n = 0;
    int64_t base = 0;
    if (len > 0) {  // an empty sequence has no partials
        n = min(last - first + 1, kMaxRanges);
        base = (int64_t)first + row;
        // lengths that changed between the two kernels must not lead out of the workspace
        if (first < 0 || base + n > a.slots) n = 0, base = 0;
    }
    const float *pm = a.pm + base * G + e, *pl = a.pl + base * G + e, *po = a.po + (base * G + e) * kD + d;
    constexpr int kEarly = 8;
    float early[kEarly];
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
        early[k] = grp + k * kMergeGroups < n ? po[(int64_t)(grp + k * kMergeGroups) * G * kD] : 0.0f;
    const float early_l = tid < n ? pl[(int64_t)tid * G] : 0.0f;
    float mx = -INFINITY;
    for (int i = tid; i < n; i += kD * kMergeGroups) {
        const float m = pm[(int64_t)i * G];
        s_w[i] = m;
        mx = fmaxf(mx, m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) s_red[0][warp] = mx;
    __syncthreads();
    float M = s_red[0][0];
#pragma unroll
    for (int k = 1; k < kD * kMergeGroups / 32; ++k) M = fmaxf(M, s_red[0][k]);
    float ls = 0.0f;
    for (int i = tid; i < n; i += kD * kMergeGroups) {  // the entries this thread wrote
        const float w = M == -INFINITY ? 0.0f : exp2f(s_w[i] - M);
        s_w[i] = w;
        ls = fmaf(i == tid ? early_l : pl[(int64_t)i * G], w, ls);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
    if (lane == 0) s_red[1][warp] = ls;
    __syncthreads();
    float Ls = 0.0f;
#pragma unroll
    for (int k = 0; k < kD * kMergeGroups / 32; ++k) Ls += s_red[1][k];

    float acc = 0.0f;
#pragma unroll
    for (int k = 0; k < kEarly; ++k)
        if (grp + k * kMergeGroups < n) acc = fmaf(early[k], s_w[grp + k * kMergeGroups], acc);
#pragma unroll 8
    for (int i = grp + kEarly * kMergeGroups; i < n; i += kMergeGroups) acc = fmaf(po[(int64_t)i * G * kD], s_w[i], acc);
    s_o[grp][d] = acc;
    __syncthreads();
    if (grp == 0) {
        float v = s_o[0][d];
#pragma unroll
        for (int k = 1; k < kMergeGroups; ++k) v += s_o[k][d];
        v = Ls > 0.0f ? v / Ls : 0.0f;
        if (a.flags & ECC_DECODE_UNROTATE_OUT) {
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const float p = __shfl_xor_sync(0xffffffffu, v, s);
                v = (lane & s) ? p - v : v + p;
            }
            s_o[0][d] = v;  // (each thread reads its own sum only above)
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const float x0 = s_o[0][lane], x1 = s_o[0][lane + 32], x2 = s_o[0][lane + 64], x3 = s_o[0][lane + 96];
            const float y0 = (warp & 1) ? x0 - x1 : x0 + x1, y1 = (warp & 1) ? x2 - x3 : x2 + x3;
            v = ((warp & 2) ? y0 - y1 : y0 + y1) * kInvSqrt128;
        }
        out[(int64_t)blockIdx.x * kD + d] = __float2half_rn(v);
    }
    if (tid == 0 && (lse || lse2)) {
        const float l2 = Ls > 0.0f ? M + log2f(Ls) : -INFINITY;
        if (lse) lse[blockIdx.x] = l2 * kLn2f;
        if (lse2) lse2[blockIdx.x] = l2;
    }
}

// weights[b, h, t] += sum over the group's heads of 2^(score - lse) for the
// visible tokens: a thread per token, kWeightTake tiles of a warp in flight,
// the kept scores of a token are contiguous.  Bound by memory: 4 G bytes of
// scores and 8 bytes of weights a token.
constexpr int kWeightThreads = 256;
constexpr int kWeightTake = 4;
constexpr int kWeightTiles = kWeightTake * kWeightThreads / 32;  // per CTA and step
template <int G>
__global__ void __launch_bounds__(kWeightThreads)
paged_weights_kernel(const __grid_constant__ DecodeArgs a, const float *__restrict__ lse2, float *__restrict__ weights,
                     int64_t ws_b, int64_t ws_h, int chunks) {
    pdl_trigger();
    pdl_wait();
    const int rows = a.B * a.Hkv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int64_t item = blockIdx.x; item < (int64_t)rows * chunks; item += gridDim.x) {
        const int row = (int)(item / chunks), chunk = (int)(item - (int64_t)row * chunks);
        const int b = row / a.Hkv, h = row - b * a.Hkv;
        const SeqTiles st(seq_len_of(a, b), a.window, a.sinks);
        const int u0 = chunk * kWeightTiles + warp * kWeightTake;
        if (u0 >= st.n) continue;
        float l2[G];
#pragma unroll
        for (int k = 0; k < G; ++k) l2[k] = __ldg(lse2 + (int64_t)row * G + k);
        float x[kWeightTake][G], old[kWeightTake];
        float *w[kWeightTake];
#pragma unroll
        for (int j = 0; j < kWeightTake; ++j) {
            const int tb = st.base(u0 + j);
            w[j] = nullptr;
            if (u0 + j >= st.n || !((st.visible(tb, a.sinks) >> lane) & 1u)) continue;
            w[j] = weights + b * ws_b + h * ws_h + tb + lane;
            const float *s = a.raw + ((int64_t)row * a.t.capacity + tb + lane) * G;
            if constexpr (G % 4 == 0) {
#pragma unroll
                for (int k = 0; k < G; k += 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(s + k);
                    x[j][k] = v.x, x[j][k + 1] = v.y, x[j][k + 2] = v.z, x[j][k + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < G; ++k) x[j][k] = s[k];
            }
            old[j] = *w[j];
        }
#pragma unroll
        for (int j = 0; j < kWeightTake; ++j) {
            if (!w[j]) continue;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < G; ++k) sum += exp2f(x[j][k] - l2[k]);
            *w[j] = old[j] + sum;
        }
    }
}

// ---- host ----
struct Layout {  // of the workspace, in bytes
    size_t pm, pl, po, first, last, lse2, raw, total;
    int64_t slots;
    int grid;
};
static Layout layout(int B, int Hq, int Hkv, int64_t capacity, bool weights) {
    const int64_t rows = (int64_t)B * Hkv, G = Hq / Hkv;
    const int64_t tiles = rows * ((capacity + kTile - 1) / kTile);
    Layout l;
    l.grid = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(sm_count(), kMaxRanges / kWarps), tiles));
    const int64_t slots = l.slots = std::min<int64_t>((int64_t)l.grid * kWarps, tiles) + rows;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    l.pm = take(slots * G * 4);
    l.pl = take(slots * G * 4);
    l.po = take(slots * G * kD * 4);
    l.first = take(rows * 4);
    l.last = take(rows * 4);
    l.lse2 = take((size_t)B * Hq * 4);
    l.raw = take(weights ? (size_t)rows * capacity * G * 4 : 0);
    l.total = at + 256;
    return l;
}

static int check_shape(int B, int Hq, int Hkv, int64_t capacity) {
    if (B < 1 || B > kMaxBatch || Hq < 1 || Hkv < 1 || capacity < 1) return ECC_ERR_SHAPE;
    if (Hq % Hkv) return ECC_ERR_GQA;
    if (Hq / Hkv > 8) return ECC_ERR_SHAPE;
    // 32-bit tile and token numbers, TMA coordinates
    if (capacity > (1ll << 30) || (int64_t)B * Hkv * ((capacity + kTile - 1) / kTile) >= (1ll << 31) ||
        (int64_t)B * Hq >= (1ll << 31))
        return ECC_ERR_SHAPE;
    return ECC_OK;
}

template <int G, bool kScores, bool kHalves>
static int launch_form(const CUtensorMap (&m)[4], const DecodeArgs &a, int grid, cudaStream_t s) {
    static bool configured[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ECC_ERR_DEVICE;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        if (cudaFuncSetAttribute(decode_paged_kernel<G, kScores, kHalves>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kSmPaged) != cudaSuccess)
            return ECC_ERR_CUDA;
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    if (launch_pdl(decode_paged_kernel<G, kScores, kHalves>, dim3(grid), dim3(kThreads), kSmPaged, s, m[0], m[1], m[2], m[3],
                   a) != cudaSuccess)
        return ECC_ERR_LAUNCH;
    return launch_status();
}

template <int G>
static int launch(const CUtensorMap (&m)[4], const DecodeArgs &a, int grid, bool halves, cudaStream_t s) {
    if (a.raw)
        return halves ? launch_form<G, true, true>(m, a, grid, s) : launch_form<G, true, false>(m, a, grid, s);
    return halves ? launch_form<G, false, true>(m, a, grid, s) : launch_form<G, false, false>(m, a, grid, s);
}

template <int G>
static int launch_weights(const DecodeArgs &a, const float *lse2, float *w, int64_t ws_b, int64_t ws_h,
                          cudaStream_t s) {
    const int tiles = (a.t.capacity + kTile - 1) / kTile;
    const int chunks = (tiles + kWeightTiles - 1) / kWeightTiles;
    const int64_t items = (int64_t)a.B * a.Hkv * chunks;
    const int64_t grid = std::min<int64_t>(items, (int64_t)sm_count() * 8);
    if (launch_pdl(paged_weights_kernel<G>, dim3((unsigned)grid), dim3(kWeightThreads), 0, s, a, lse2, w, ws_b, ws_h,
                   chunks) != cudaSuccess)
        return ECC_ERR_LAUNCH;
    return launch_status();
}

}  // namespace paged

int paged_decode_error(int reset, int *wait_error) {
    // 5: a bad length or page; *wait_error: 1 / 2 as for the contiguous decode
    int v = 0, w = 0;
    if (cudaMemcpyFromSymbol(&v, paged::g_paged_error, sizeof(int)) != cudaSuccess ||
        cudaMemcpyFromSymbol(&w, g_device_error, sizeof(int)) != cudaSuccess)
        return ECC_ERR_CUDA;
    if (reset) {
        const int z = 0;
        if (cudaMemcpyToSymbol(paged::g_paged_error, &z, sizeof(int)) != cudaSuccess ||
            cudaMemcpyToSymbol(g_device_error, &z, sizeof(int)) != cudaSuccess)
            return ECC_ERR_CUDA;
    }
    *wait_error = w;
    return v;
}

}  // namespace ecc

using namespace ecc;

extern "C" size_t ecc_decode_paged_workspace_size(int B, int Hq, int Hkv, int64_t capacity, int with_weights) {
    if (paged::check_shape(B, Hq, Hkv, capacity) != ECC_OK) return 0;
    return paged::layout(B, Hq, Hkv, capacity, with_weights != 0).total;
}

extern "C" int ecc_decode_paged(const void *q_f16, const void *k_blocks, const void *v_blocks, int64_t bs_p,
                                int64_t bs_h, const ecc_pages_t *pages, const int *seq_lens, void *out_f16, float *lse,
                                float *weights, int64_t ws_b, int64_t ws_h, void *workspace, size_t workspace_bytes,
                                int B, int Hq, int Hkv, float sm_scale, int window, int sinks, int flags,
                                ecc_stream_t stream) {
    using namespace paged;
    if (B == 0) return ECC_OK;
    if (!q_f16 || !k_blocks || !v_blocks || !pages || !seq_lens || !out_f16) return ECC_ERR_NULL;
    if (flags & ~(ECC_DECODE_ROTATE_Q | ECC_DECODE_UNROTATE_OUT | ECC_DECODE_BLOCK96)) return ECC_ERR_SHAPE;
    const int rb = (flags & ECC_DECODE_BLOCK96) ? 96 : kBlockBytes;
    DecodeArgs a{};
    int rc = make_table(*pages, &a.t);
    if (rc != ECC_OK) return rc;
    rc = check_shape(B, Hq, Hkv, a.t.capacity);
    if (rc != ECC_OK) return rc;
    if (window < 0 || sinks < 0 || (sinks > 0 && window == 0)) return ECC_ERR_SHAPE;
    if (!std::isfinite(sm_scale)) return ECC_ERR_PARAM;
    // TMA: 16-byte aligned pools; 16-byte loads of the query
    if (((uintptr_t)k_blocks % 16) || ((uintptr_t)v_blocks % 16) || ((uintptr_t)q_f16 % 16) ||
        ((uintptr_t)seq_lens % 4) || ((uintptr_t)out_f16 % 2) || (lse && (uintptr_t)lse % 4) ||
        (weights && (uintptr_t)weights % 4))
        return ECC_ERR_ALIGN;
    const Layout l = layout(B, Hq, Hkv, a.t.capacity, weights != nullptr);
    if (!workspace || workspace_bytes < l.total) return ECC_ERR_WORKSPACE;
    if (!reserve_matches()) return ECC_ERR_DEVICE;
    if (get_encode() != ECC_OK) return ECC_ERR_CUDA;

    uint8_t *w = reinterpret_cast<uint8_t *>(((uintptr_t)workspace + 255) / 256 * 256);
    a.q = reinterpret_cast<const __half *>(q_f16);
    a.lens = seq_lens;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.window = window;
    a.sinks = sinks;
    a.scale_log2 = (sm_scale > 0.0f ? sm_scale : 1.0f / std::sqrt((float)kD)) * 1.4426950408889634f;
    a.flags = flags;
    const bool halves = a.t.width > 1 && a.t.page_size % kTile != 0;
    a.pm = reinterpret_cast<float *>(w + l.pm);
    a.pl = reinterpret_cast<float *>(w + l.pl);
    a.po = reinterpret_cast<float *>(w + l.po);
    a.row_first = reinterpret_cast<int *>(w + l.first);
    a.row_last = reinterpret_cast<int *>(w + l.last);
    a.slots = l.slots;
    float *lse2 = reinterpret_cast<float *>(w + l.lse2);
    a.raw = weights ? reinterpret_cast<float *>(w + l.raw) : nullptr;

    CUtensorMap m[4];
    if (make_maps(&m[0], &m[1], &m[2], &m[3], k_blocks, v_blocks, a.t.page_size, Hkv, a.t.n_pages, bs_h, bs_p, rb,
                  halves ? 16 : kTile) != ECC_OK)
        return ECC_ERR_ALIGN;  // strides a tensor map cannot describe
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int G = Hq / Hkv;
    switch (G) {
#define ECC_PAGED_CASE(N) \
    case N: rc = launch<N>(m, a, l.grid, halves, s); break;
        ECC_PAGED_CASE(1) ECC_PAGED_CASE(2) ECC_PAGED_CASE(3) ECC_PAGED_CASE(4)
        ECC_PAGED_CASE(5) ECC_PAGED_CASE(6) ECC_PAGED_CASE(7) ECC_PAGED_CASE(8)
#undef ECC_PAGED_CASE
    }
    if (rc != ECC_OK) return rc;
    // partials per row when the rows are alike; a CTA of one group joins a few of them as fast and three times as
    // many such CTAs fit an SM (B32 Hq32, 7 slots a row: 8.5 us against 14)
    const bool wide = l.slots / ((int64_t)B * Hkv) > 8;
    const cudaError_t e =
        wide ? launch_pdl(paged_merge_kernel<4>, dim3((unsigned)(B * Hq)), dim3(kD * 4), 0, s, a,
                          reinterpret_cast<__half *>(out_f16), lse, weights ? lse2 : nullptr)
             : launch_pdl(paged_merge_kernel<1>, dim3((unsigned)(B * Hq)), dim3(kD), 0, s, a,
                          reinterpret_cast<__half *>(out_f16), lse, weights ? lse2 : nullptr);
    if (e != cudaSuccess) return ECC_ERR_LAUNCH;
    rc = launch_status();
    if (rc != ECC_OK || !weights) return rc;
    switch (G) {
#define ECC_PAGED_CASE(N) case N: return launch_weights<N>(a, lse2, weights, ws_b, ws_h, s);
        ECC_PAGED_CASE(1) ECC_PAGED_CASE(2) ECC_PAGED_CASE(3) ECC_PAGED_CASE(4)
        ECC_PAGED_CASE(5) ECC_PAGED_CASE(6) ECC_PAGED_CASE(7) ECC_PAGED_CASE(8)
#undef ECC_PAGED_CASE
    }
    return ECC_ERR_SHAPE;
}
