// decode_tile.cuh -- what the TMA-fed decode kernels share (sm_100a): the
// per-warp ring of 32-token stages, the code-byte table, the tensor-core
// arithmetic of one stage (Lane), the cut of a list of tiles into one range
// per warp, and the tensor maps.  Used by decode_tma.cu (one contiguous row
// per sequence) and decode_paged.cu (pages, ragged lengths, windows).
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cmath>
#include <mutex>

#include "ecc_common.cuh"

namespace ecc {

// raised by a bounded wait that ran out (one flag per translation unit;
// ecc_device_status reads them all)
static __device__ int g_device_error;

namespace tmak {

constexpr int kWarps = 12;          // warps per CTA (384 threads)
constexpr int kStages = 2;          // ring stages per warp
constexpr int kTile = 32;           // tokens per stage (two 16-token MMA sub-tiles)
constexpr int kStageBytes = 6144;
constexpr int kOffKC = 0, kOffKS = kOffKC + 32 * 64, kOffVC = kOffKS + 32 * 32, kOffVS = kOffVC + 32 * 64;
constexpr int kSubC = 1024, kSubS = 512;  // offset of sub-tile 1 in the code / syndrome boxes
constexpr int kThreads = kWarps * 32;
constexpr int kLutBytes = 65536;
constexpr float kLn2f = 0.6931471805599453f;
constexpr long long kWaitCycles = 4000000000ll;

constexpr int kSmemReserve = 1024;  // shared-window offset of dynamic shared memory
constexpr int kSmLut = 0;
constexpr int kSmRing = kSmLut + kLutBytes;                        // [kWarps][kStages][kStageBytes]
constexpr int kSmCent = kSmRing + kWarps * kStages * kStageBytes;  // [16] u32
constexpr int kSmBar = kSmCent + 16 * 4;                           // [kWarps][kStages] u64
constexpr int kSmBytes = kSmBar + kWarps * kStages * 8;
static_assert(kSmRing % 1024 == 0 && kStageBytes % 128 == 0, "TMA destinations 128-B aligned");
static_assert(kSmBar % 8 == 0, "mbarriers 8-B aligned");
static_assert(kSmBytes <= 227 * 1024, "shared memory budget");

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait by one lane; false when it ran out (the device flag is raised).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, long long limit = kWaitCycles) {
    if (mbar_try(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try(bar, parity)) {
        if (clock64() - t0 > limit) {
            atomicExch(&g_device_error, 1);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w,
                                       uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
    return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
    return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 transpose of 16-bit elements across the warp: lane (g, c) passes row g,
// columns 2c, 2c+1 and receives row g, columns 2c, 2c+1 of the transpose.
__device__ __forceinline__ uint32_t movtrans(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}
// Code-byte table lookup: for code byte v (codes v & 15, v >> 4) the fp16x2
// word of their hi parts and the fp16x2 word of their lo parts.  Row v of the
// table is 256 bytes: the hi words of the 32 lanes' private copies at v*256 +
// 4*lane, the lo words 128 bytes further.  Every 32-bit load of a warp then
// hits 32 distinct banks, and the two halves arrive in separate registers, so
// the centroid MMA operands (hi words of four lookups in one register quad,
// lo words in another) need no moves.  The offset v*256 + 4*lane is one prmt.
// The table sits at the start of the dynamic shared memory, whose
// shared-window address is the per-block reserve kSmemReserve (checked on the
// host against cudaDevAttrReservedSharedMemoryPerBlock and again by the
// kernel), so the base folds into the loads' immediate offsets.  The table is
// constant after the kernel's set-up barrier, so the loads are not volatile
// and may be scheduled freely.
__device__ __forceinline__ uint2 lut(uint32_t word, int byte_idx, uint32_t lane4) {
    uint2 r;
    const uint32_t a = __byte_perm(word, lane4, 0x5504u | ((uint32_t)byte_idx << 4));
    asm("ld.shared.u32 %0, [%1+%2];" : "=r"(r.x) : "r"(a), "n"(kSmemReserve + kSmLut));
    asm("ld.shared.u32 %0, [%1+%2];" : "=r"(r.y) : "r"(a), "n"(kSmemReserve + kSmLut + 128));
    return r;
}
// +-1 pair from bits p and p+16 of w (bit 1 -> +1.0)
__device__ __forceinline__ uint32_t sign_pair(uint32_t w, int p) {
    const uint32_t x = w << (15 - p);
    return (~x & 0x80008000u) | 0x3C003C00u;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float h_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
__device__ __forceinline__ float h_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }

// Sign bit p of both fp16 halves of x kept in place: each half is 0 or the
// fp16 value whose only set bit is p (p <= 14), a power of two sign_weight(p).
// Bit 15 is the fp16 sign bit, so that one moves to bit 14 first.
__device__ __forceinline__ uint32_t sign_bits(uint32_t x, int p) {
    return p == 15 ? ((x >> 1) & 0x40004000u) : (x & (0x00010001u << p));
}
// 1 / (value of the fp16 with only bit p set), bit 15 taken as bit 14
__host__ __device__ constexpr float sign_unweight(int p) {
    return p == 15 ? 0.5f
         : p == 14 ? 0.5f
         : p == 13 ? 128.0f
         : p == 12 ? 2048.0f
         : p == 11 ? 8192.0f
         : p == 10 ? 16384.0f
                   : (float)(1u << (24 - p));  // subnormal 2^(p-24)
}

// K sign bits kept as 0/1 in the exponent field: bit pair (p, p+16) of the
// syndrome word w lands at bit positions (q, q+16), q = kpos(p) in 10..14,
// each half then being 0 or the fp16 2^kexp(p).  x5 = w << 5, x10 = w << 10,
// x1 = w >> 1 are shared by the 16 pairs of a word (3 shifts + 16 masks
// instead of 2 operations per pair).
__host__ __device__ constexpr int kpos(int p) { return p == 15 ? 14 : p >= 10 ? p : p >= 5 ? p + 5 : p + 10; }
__host__ __device__ constexpr int kexp(int p) {
    return kpos(p) == 10 ? -14 : kpos(p) == 11 ? -13 : kpos(p) == 12 ? -11 : kpos(p) == 13 ? -7 : 1;
}
__device__ __forceinline__ uint32_t kbits(uint32_t w, uint32_t x5, uint32_t x10, uint32_t x1, int p) {
    const uint32_t src = p == 15 ? x1 : p >= 10 ? w : p >= 5 ? x5 : x10;
    return src & (0x00010001u << kpos(p));
}

// The attended tokens of a stage: an interval of offsets, or a bit per token.
struct SeeRange {
    int lo, hi;
    __device__ __forceinline__ bool has(int t) const { return t >= lo && t < hi; }
    __device__ __forceinline__ SeeRange second() const { return {lo - 16, hi - 16}; }  // of the second sub-tile
};
struct SeeBits {
    uint32_t m;
    __device__ __forceinline__ bool has(int t) const { return (m >> t) & 1u; }
    __device__ __forceinline__ SeeBits second() const { return {m >> 16}; }
};
struct NoScores {
    __device__ __forceinline__ void operator()(const float (&)[4], const float (&)[4]) const {}
};

// ---- the paired table (Lane<G, true>) ---------------------------------------
// The centroids times kCentScale: of all factors, the one with which the eight
// magnitudes lie nearest to fp16 values (8.6e-5 relative at most, 6.0e-5 rms
// over normal data, where an fp16 rounding is 2^-11 at most and 2.2e-4 rms), so
// that the fp16 parts alone serve the values: the output is rounded to fp16
// once more anyway.  Keys take both parts.
//
// Row v (256 bytes) holds a pair of words per lane at v*256 + 8*lane, the hi
// words and the lo words of the two codes of byte v; lanes 16..31 have them the
// other way round.  One 64-bit load brings a key byte's pair into the registers
// of operand rows g and g + 8, whose products are added up, so their order does
// not matter; the 32-bit loads of the values' hi words (at lane_hi) then hit 32
// distinct banks as well.
constexpr float kCentScale = 0x1.61a50cp+0f;
__device__ __forceinline__ uint2 lut_pair(uint32_t word, int byte_idx, uint32_t lane8) {
    uint2 r;
    const uint32_t a = __byte_perm(word, lane8, 0x5504u | ((uint32_t)byte_idx << 4));
    asm("ld.shared.v2.u32 {%0, %1}, [%2+%3];" : "=r"(r.x), "=r"(r.y) : "r"(a), "n"(kSmemReserve + kSmLut));
    return r;
}
__device__ __forceinline__ uint32_t lut_hi(uint32_t word, int byte_idx, uint32_t lane_hi) {
    uint32_t r;
    const uint32_t a = __byte_perm(word, lane_hi, 0x5504u | ((uint32_t)byte_idx << 4));
    asm("ld.shared.u32 %0, [%1+%2];" : "=r"(r) : "r"(a), "n"(kSmemReserve + kSmLut));
    return r;
}
__device__ __forceinline__ uint32_t lane_hi_of(int lane) { return 8u * lane + (lane < 16 ? 0u : 4u); }
// This lane's pair of row v from the 16 packed centroids (hi | lo << 16).
__device__ __forceinline__ uint2 lut_entry(const uint32_t *cent, int v, int lane) {
    const uint32_t e0 = cent[v & 15], e1 = cent[v >> 4];
    const uint32_t hi = __byte_perm(e0, e1, 0x5410), lo = __byte_perm(e0, e1, 0x7632);
    return lane < 16 ? make_uint2(hi, lo) : make_uint2(lo, hi);
}

// Two e5m2 values (the top bytes of fp16 values) of bytes 2j, 2j + 1 of w as an fp16x2 word.
__device__ __forceinline__ uint32_t e5m2_pair(uint32_t w, int j) { return __byte_perm(w, 0u, j ? 0x3424u : 0x1404u); }

// Consumer lane state for one work item.  kFine: the paired table above, and
// a query that is scaled, head by head, to a largest magnitude in [1, 2) and, when it is
// rotated here, not rounded to fp16 but carried as fp16 plus remainder (for
// groups of up to 4 heads in the idle columns 4..7 of the QK operand,
// otherwise as e5m2 words).  For groups of at most 4 query heads
// the PV products use the idle columns 4..7 of the n8 operand for the V sign
// term: lanes g < 4 of the P operand carry p * vscale of head g (columns
// 0..3, centroid products), lanes g >= 4 carry 2 p * valpha of head g - 4
// (columns 4..7, sign-bit products with the bits masked in place, so each
// accumulator row has one power-of-two weight, removed at the end).
template <int G, bool kFine = false>
struct Lane {
    static constexpr bool kLoCols = kFine && G <= 4, kLoWords = kFine && G > 4;
    uint32_t qc[8][2];
    uint32_t ql[kLoWords ? 8 : 1];  // remainders of the four values of qc[m], e5m2
    uint32_t qs[8][2];  // q of the sign products, k slot of bit p scaled by 2^-(ssh + kexp(p))
    float sgn2;         // 2^(ssh + 1): q.s = sgn2 * (sign product) - sum(q); kFine: 2
    float qsum[2];
    // PV accumulators: o[i] rows g / g+8 = dims 16g + 2i / 16g + 2i + 1 (code
    // byte i of the lane's 8 V code bytes), columns = the n8 operand columns
    float o[8][4];
    float mrun[2], lrun[2], zrun[2];
    uint32_t lane4, sel_half;
    uint32_t voff;  // this lane's byte offset in the swizzled V code box (see load_v)
    uint32_t soff;  // this lane's byte offset in the swizzled syndrome boxes (see qk, load_v)
    int g, c;
    float scale_log2;   // of the scores; kFine: without the query's scaling
    float scale_up[2];  // kFine: with it, of heads 2c, 2c + 1
    uint32_t lane8, lane_hi;  // kFine: offsets in the paired table
    int vexp;  // kFine: exponent field of the largest V scale or 2 alpha so far, 1..31 (see tile)
    __device__ __forceinline__ float v_up() const { return kFine ? __int_as_float((127 + 29 - vexp) << 23) : 1.0f; }
    __device__ __forceinline__ float v_down() const { return kFine ? __int_as_float((127 - 29 + vexp) << 23) : 1.0f; }

    // Query fragments of a row segment from the lane's fp16 query words qw
    // (dims 32c..32c+31 of its head): the centroid operand qc, the sign
    // operand qs with its exponent sgn2, and the per-head sums qsum.
    __device__ __forceinline__ void set_query(const uint4 (&qw)[4], bool rotate) {
        float x[32];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t wv[4] = {qw[k].x, qw[k].y, qw[k].z, qw[k].w};
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                x[8 * k + 2 * m] = h_lo(wv[m]);
                x[8 * k + 2 * m + 1] = h_hi(wv[m]);
            }
        }
        if (rotate) {  // q_rot = fp16(WHT(q)), like patch.py:106
#pragma unroll
            for (int s = 1; s < 32; s <<= 1)
#pragma unroll
                for (int k = 0; k < 32; ++k)
                    if ((k & s) == 0) {
                        const float a = x[k], bb = x[k + s];
                        x[k] = __fadd_rn(a, bb);
                        x[k + s] = __fsub_rn(a, bb);
                    }
#pragma unroll
            for (int s = 1; s <= 2; s <<= 1) {  // strides 32, 64: partner lane c ^ s
                const float sgn = (c & s) ? -1.0f : 1.0f;
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    const float p = __shfl_xor_sync(0xffffffffu, x[k], s);
                    x[k] = __fmaf_rn(sgn, x[k], p);
                }
            }
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const float v = x[k];
                const float q0 = __fmul_rn(v, kInvSqrt128);
                const float rem = __fmaf_rn(-q0, kSqrt128, v);
                x[k] = __fmaf_rn(rem, kInvSqrt128, q0);
                if (!kFine) x[k] = __half2float(__float2half_rn(x[k]));
            }
        }
        if constexpr (kFine) {
            float qmax = 0.0f;  // of the lane's head: the heads of a group may differ by any factor
#pragma unroll
            for (int k = 0; k < 32; ++k) qmax = fmaxf(qmax, fabsf(x[k]));
#pragma unroll
            for (int off = 1; off < 4; off <<= 1) qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, off));
            const int e2 = qmax > 0.0f ? max(-100, min(100, ((__float_as_int(qmax) >> 23) & 0xff) - 127)) : 0;
            const float down = __int_as_float((127 - e2) << 23), up = scale_log2 * __int_as_float((127 + e2) << 23);
            scale_up[0] = __shfl_sync(0xffffffffu, up, 4 * (2 * c));
            scale_up[1] = __shfl_sync(0xffffffffu, up, 4 * (2 * c + 1));
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] *= down;
        }
        if constexpr (kLoCols) {  // lanes g >= 4 hold the remainders of head g - 4
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const float hi = __half2float(__float2half_rn(x[k]));
                x[k] = g < 4 ? hi : x[k] - hi;
            }
        }
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            qc[m][0] = pack_h2(x[4 * m], x[4 * m + 1]);
            qc[m][1] = pack_h2(x[4 * m + 2], x[4 * m + 3]);
        }
        // sign-product operand: scale 2^-ssh keeps q * 2^(14 - ssh) < 2^15
        // for the largest |q| of the group (q is fp16, the scalings are
        // exact powers of two); kFine: |q| <= 2, so ssh = 0
        {
            int ssh = 0;
            if constexpr (!kFine) {
                float qmax = 0.0f;
#pragma unroll
                for (int k = 0; k < 32; ++k) qmax = fmaxf(qmax, fabsf(x[k]));
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, off));
                const int e2 = (qmax > 0.0f) ? ((__float_as_int(qmax) >> 23) & 0xff) - 127 : 0;
                ssh = max(0, e2);
                sgn2 = __int_as_float((ssh + 1 + 127) << 23);
            }
            if constexpr (kLoWords) {
                // a remainder is at most 2^-11; an e5m2 keeps three bits of it down to 2^-14 and steps of 2^-16
                // below, so at most 2^-14 of the fp16 rounding's 2^-11 is left
#pragma unroll
                for (int m = 0; m < 8; ++m) {
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v = x[4 * m + j];
                        // fp16, rounded to its top byte
                        const uint32_t hw = __half_as_ushort(__float2half_rn(v - __half2float(__float2half_rn(v))));
                        w |= ((hw + 0x7fu + ((hw >> 8) & 1u)) >> 8 & 0xffu) << (8 * j);
                    }
                    ql[m] = w;
                }
            }
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const float f0 = __int_as_float((127 - ssh - kexp(2 * m)) << 23);
                const float f1 = __int_as_float((127 - ssh - kexp(2 * m + 1)) << 23);
                qs[m][0] = pack_h2(x[2 * m] * f0, x[2 * m + 16] * f0);
                qs[m][1] = pack_h2(x[2 * m + 1] * f1, x[2 * m + 17] * f1);
            }
        }
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 32; ++k) sum += x[k];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qsum[0] = __shfl_sync(0xffffffffu, sum, 4 * (2 * c));       // head 2c
        qsum[1] = __shfl_sync(0xffffffffu, sum, 4 * (2 * c + 1));   // head 2c+1
    }

    // Raw V data of one 16-token sub-tile: tokens 2c, 2c+1, 2c+8, 2c+9 (code
    // bytes 8g..8g+7, syndrome word g/2) and the metadata of tokens g, g+8.
    //
    // The V code box (64-byte rows) is written with the 64-byte swizzle:
    // 16-byte chunk j of row r lands at chunk j ^ ((r >> 1) & 3).  Lane (g,
    // c) reads chunk g/2 of rows 2c + {0, 1, 8, 9}, whose (r >> 1) & 3 is c,
    // so its offset within a row is the lane constant 16 ((g/2) ^ c) + 8 (g &
    // 1) (voff): a half-warp's reads then fall on 16 banks instead of 8.  The
    // syndrome/metadata boxes (32-byte rows) use the 32-byte swizzle: chunk
    // j of row r at chunk j ^ ((r >> 2) & 1) (soff: 16 ((r >> 2) & 1) for the
    // rows a lane reads), which makes the syndrome-word and metadata reads
    // conflict-free.
    struct VRaw {
        uint2 vc[4];
        uint32_t vs[4];
        uint2 vma, vmb;
    };
    __device__ __forceinline__ VRaw load_v(uint32_t vcb, uint32_t vsb) const {
        VRaw v;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int tok = 2 * c + (u & 1) + 8 * (u >> 1);
            v.vc[u] = lds64(vcb + 64 * tok + voff);
            // row tok: (tok >> 2) & 1 = c >> 1
            v.vs[u] = lds32(vsb + 32 * tok + 16 * (c >> 1) + 4 * (g >> 1));
        }
        // metadata: chunk 1 of rows g and g + 8, (row >> 2) & 1 = g >> 2
        v.vma = lds64(vsb + 32 * g + (16 ^ soff));
        v.vmb = lds64(vsb + 32 * (g + 8) + (16 ^ soff));
        return v;
    }

    // log2-scaled scores of one 16-token sub-tile (K codes at kcb, syndrome +
    // metadata at ksb): s2[e] token g, s2[2+e] token g+8, head 2c+e; tokens
    // (sub-tile offsets) that are not in `see` are -inf.
    template <class See>
    __device__ __forceinline__ void qk(uint32_t kcb, uint32_t ksb, See see, float (&s2)[4]) const {
        const uint4 kca = lds128(kcb + 64 * g + 16 * c);
        const uint4 kcb8 = lds128(kcb + 64 * (g + 8) + 16 * c);
        // syndrome box with the 32-byte swizzle (see load_v): rows g, g + 8
        const uint32_t ksa = lds32(ksb + 32 * g + soff + 4 * c);
        const uint32_t ksb8 = lds32(ksb + 32 * (g + 8) + soff + 4 * c);
        const uint32_t ka5 = ksa << 5, ka10 = ksa << 10, ka1 = ksa >> 1;
        const uint32_t kb5 = ksb8 << 5, kb10 = ksb8 << 10, kb1 = ksb8 >> 1;
        const uint2 kma = lds64(ksb + 32 * g + (16 ^ soff));
        const uint2 kmb = lds64(ksb + 32 * (g + 8) + (16 ^ soff));
        const bool va = see.has(g), vb8 = see.has(g + 8);

        // Centroid products: rows g / g+8 of the A operand carry the fp16 hi /
        // lo parts of one token's centroids, so each table entry (hi, lo)
        // lands in the operand registers as loaded; one product per 8 tokens.
        float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f}, ss[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t kwa[4] = {kca.x, kca.y, kca.z, kca.w};
        const uint32_t kwb[4] = {kcb8.x, kcb8.y, kcb8.z, kcb8.w};
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            const int w = m >> 1, by = 2 * (m & 1);
            // token g, k slots 2c, 2c+1 and 2c+8, 2c+9, then token g+8
            const uint2 xa = kFine ? lut_pair(kwa[w], by, lane8) : lut(kwa[w], by, lane4);
            const uint2 ya = kFine ? lut_pair(kwa[w], by + 1, lane8) : lut(kwa[w], by + 1, lane4);
            const uint2 xb = kFine ? lut_pair(kwb[w], by, lane8) : lut(kwb[w], by, lane4);
            const uint2 yb = kFine ? lut_pair(kwb[w], by + 1, lane8) : lut(kwb[w], by + 1, lane4);
            mma16816(sa, xa.x, xa.y, ya.x, ya.y, qc[m][0], qc[m][1]);
            mma16816(sb, xb.x, xb.y, yb.x, yb.y, qc[m][0], qc[m][1]);
            if constexpr (kLoWords) {
                const uint32_t l0 = e5m2_pair(ql[m], 0), l1 = e5m2_pair(ql[m], 1);
                mma16816(sa, xa.x, xa.y, ya.x, ya.y, l0, l1);
                mma16816(sb, xb.x, xb.y, yb.x, yb.y, l0, l1);
            }
            mma16816(ss, kbits(ksa, ka5, ka10, ka1, 2 * m), kbits(ksb8, kb5, kb10, kb1, 2 * m),
                     kbits(ksa, ka5, ka10, ka1, 2 * m + 1), kbits(ksb8, kb5, kb10, kb1, 2 * m + 1), qs[m][0],
                     qs[m][1]);
        }
        // q.C of token g (head 2c+e) = hi row + lo row
        const float sc[4] = {sa[0] + sa[2], sa[1] + sa[3], sb[0] + sb[2], sb[1] + sb[3]};
        // score = scale q.C + alpha (2 q.b - sum q) + zero sum q  (s = 2b - 1)
        constexpr float kUnit = kFine ? 1.0f / kCentScale : 1.0f;  // of the table's centroids
        const float k_sa = h_lo(kma.x) * kUnit, k_za = h_hi(kma.x), k_aa = h_lo(kma.y);
        const float k_sb = h_lo(kmb.x) * kUnit, k_zb = h_hi(kmb.x), k_ab = h_lo(kmb.y);
        const float sgn = kFine ? 2.0f : sgn2, k_ga = k_aa * sgn, k_gb = k_ab * sgn, k_da = k_za - k_aa, k_db = k_zb - k_ab;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float xa = fmaf(k_sa, sc[e], fmaf(k_ga, ss[e], k_da * qsum[e]));
            float xb = fmaf(k_sb, sc[2 + e], fmaf(k_gb, ss[2 + e], k_db * qsum[e]));
            if constexpr (kLoCols) {  // linear in q: fp16 part plus remainder, in both lanes alike
                xa += __shfl_xor_sync(0xffffffffu, xa, 2);
                xb += __shfl_xor_sync(0xffffffffu, xb, 2);
            }
            const float sl = kFine ? scale_up[e] : scale_log2;
            s2[e] = va ? xa * sl : -INFINITY;
            s2[2 + e] = vb8 ? xb * sl : -INFINITY;
        }
    }

    // PV products of one 16-token sub-tile with probabilities p (same layout
    // as the scores: p[e] token g, p[2+e] token g+8, head 2c+e).
    //
    // The B operand (k = token, n = column) comes from the score layout (row =
    // token, columns 2c, 2c+1 in lane (g, c)) by one 8x8 transpose per token
    // half (movmatrix).  Its words: ws = p*scale_v with its fp16 residual
    // ws - fp16(ws) (a single fp16 rounding of ws is 2^-11 relative, close to
    // the 2e-3 output tolerance when a few large values dominate), and the
    // sign weights wa = p*alpha_v.  Groups of up to 4 heads use the idle
    // columns 4..7 for the sign products: the score columns 4..7 repeat heads
    // 0..3 (see the query set-up), lanes c >= 2 put 2*wa there, and the
    // sign bits are masked in place (each fp16 half is 0 or the power of two
    // whose only set bit is p), so every accumulator row has one known weight
    // that the epilogue divides out; s = 2b - 1 moves -alpha_v into the
    // zero-point sum.  Groups of 5..8 use +-1 sign operands against wa.
    //
    // Per code byte i of the lane (dims 16g + 2i, 16g + 2i + 1 in rows g,
    // g + 8 of accumulator i), four products: centroids hi x ws, centroids
    // lo x ws, centroids hi x residual, signs x sign weights.
    //
    // kFine: all weights are times v_up() = 2^k, with which the largest V scale
    // or 2 alpha met so far lies in [2^14, 2^15); the accumulators carry the
    // factor, tile() rescales them when k falls and the segment's end takes it
    // off.  fp16 and its residual end at 2^-25 absolute, so a weight is known to
    // 2^-22 relative or 2^-39 of (the largest probability x the largest scale),
    // where without the factor a token e^-12 below the largest with a scale of
    // 0.05 had two bits.
    __device__ __forceinline__ void pv(const VRaw &v, const float (&p)[4]) {
        const float up = v_up(), kUnit = kFine ? 1.0f / kCentScale * up : 1.0f;
        const float v_sa = h_lo(v.vma.x) * kUnit, v_aa = h_lo(v.vma.y);
        const float v_sb = h_lo(v.vmb.x) * kUnit, v_ab = h_lo(v.vmb.y);
        constexpr bool kSplitCols = G <= 4;
        // rows of the pre-transpose matrices: t = 0 token g, t = 1 token g+8
        uint32_t mw[2], mr[2], ma[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float sc = t ? v_sb : v_sa, al = (kSplitCols ? 2.0f : 1.0f) * up * (t ? v_ab : v_aa);
            const float w0 = p[2 * t] * sc, w1 = p[2 * t + 1] * sc;
            mw[t] = pack_h2(w0, w1);
            mr[t] = pack_h2(w0 - h_lo(mw[t]), w1 - h_hi(mw[t]));
            ma[t] = pack_h2(p[2 * t] * al, p[2 * t + 1] * al);
        }
        // B words: [0] tokens 2c, 2c+1, [1] tokens 2c+8, 2c+9 of column g
        uint32_t bw[2], br[2], bs[2];
        if constexpr (kSplitCols) {
            const bool cent = g < 4, lo_cols = c < 2;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t x = movtrans(lo_cols ? mw[t] : ma[t]);
                const uint32_t r = movtrans(mr[t]);
                bw[t] = cent ? x : 0u;
                bs[t] = cent ? 0u : x;
                br[t] = cent ? r : 0u;
            }
        } else {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                bw[t] = movtrans(mw[t]);
                br[t] = movtrans(mr[t]);
                bs[t] = movtrans(ma[t]);
            }
        }

        const uint32_t sA = __byte_perm(v.vs[0], v.vs[1], sel_half), sB = __byte_perm(v.vs[2], v.vs[3], sel_half);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t xa0 = w ? v.vc[0].y : v.vc[0].x, xa1 = w ? v.vc[1].y : v.vc[1].x;
            const uint32_t xb0 = w ? v.vc[2].y : v.vc[2].x, xb1 = w ? v.vc[3].y : v.vc[3].x;
            constexpr uint32_t kLo = 0x0F0F0F0Fu, kHi = 0xF0F0F0F0u;
            const uint32_t ia_e = (xa0 & kLo) | ((xa1 << 4) & kHi), ia_o = ((xa0 >> 4) & kLo) | (xa1 & kHi);
            const uint32_t ib_e = (xb0 & kLo) | ((xb1 << 4) & kHi), ib_o = ((xb0 >> 4) & kLo) | (xb1 & kHi);
            uint2 r0[4], r1[4], r2[4], r3[4];  // kFine: the hi words alone
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (kFine) {
                    r0[k].x = lut_hi(ia_e, k, lane_hi);
                    r1[k].x = lut_hi(ia_o, k, lane_hi);
                    r2[k].x = lut_hi(ib_e, k, lane_hi);
                    r3[k].x = lut_hi(ib_o, k, lane_hi);
                } else {
                    r0[k] = lut(ia_e, k, lane4);
                    r1[k] = lut(ia_o, k, lane4);
                    r2[k] = lut(ib_e, k, lane4);
                    r3[k] = lut(ib_o, k, lane4);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16816(o[4 * w + k], r0[k].x, r1[k].x, r2[k].x, r3[k].x, bw[0], bw[1]);
            if constexpr (!kFine) {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma16816(o[4 * w + k], r0[k].y, r1[k].y, r2[k].y, r3[k].y, bw[0], bw[1]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) mma16816(o[4 * w + k], r0[k].x, r1[k].x, r2[k].x, r3[k].x, br[0], br[1]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = 4 * w + k;
                if constexpr (kSplitCols)
                    mma16816(o[i], sign_bits(sA, 2 * i), sign_bits(sA, 2 * i + 1), sign_bits(sB, 2 * i),
                             sign_bits(sB, 2 * i + 1), bs[0], bs[1]);
                else
                    mma16816(o[i], sign_pair(sA, 2 * i), sign_pair(sA, 2 * i + 1), sign_pair(sB, 2 * i),
                             sign_pair(sB, 2 * i + 1), bs[0], bs[1]);
            }
        }
    }

    // One 32-token stage at `st` (two sub-tiles sharing one softmax update);
    // tokens (offsets within the stage) that are not in `see` are masked.
    // `scores` is handed the log2-scaled scores of the two sub-tiles.
    template <class See, class Scores = NoScores>
    __device__ __forceinline__ void tile(uint32_t st, See see, Scores scores = Scores()) {
        // kFine: the exponent field of the stage's largest V scale or 2 alpha, lane = token.  Asked for first (8 x 64k: 229
        // us; behind the scores, where it is needed, 235; without it 222)
        uint32_t top = 0;
        if constexpr (kFine) {
            const uint2 vm = lds64(st + kOffVS + 128 * g + 32 * c + (16 ^ (16 * (g & 1))));
            top = __reduce_max_sync(0xffffffffu, max(vm.x & 0x7fffu, (vm.y & 0x7fffu) + 0x400u));
        }
        const VRaw v0 = load_v(st + kOffVC, st + kOffVS);
        float s0[4], s1[4];
        qk(st + kOffKC, st + kOffKS, see, s0);
        qk(st + kOffKC + kSubC, st + kOffKS + kSubS, see.second(), s1);
        scores(s0, s1);

        // mb: the running maximum, or 0 while every token so far is masked
        // (left padding), so that masked scores give p = 0, not NaN
        float corr[2], mb[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(s0[e], s0[2 + e]), fmaxf(s1[e], s1[2 + e]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mnew = fmaxf(mrun[e], mx);
            mb[e] = mnew == -INFINITY ? 0.0f : mnew;
            corr[e] = ex2(mrun[e] - mb[e]);
            mrun[e] = mnew;
        }
        float corr_o[2] = {corr[0], corr[1]};
        if constexpr (kFine) {
            const int grown = max(vexp, (int)(top >> 10));
            const float f = __int_as_float((127 + vexp - grown) << 23);
            vexp = grown;
            corr_o[0] *= f;
            corr_o[1] *= f;
        }
        float p0[4], p1[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            p0[e] = ex2(s0[e] - mb[e]);
            p0[2 + e] = ex2(s0[2 + e] - mb[e]);
            p1[e] = ex2(s1[e] - mb[e]);
            p1[2 + e] = ex2(s1[2 + e] - mb[e]);
        }
        // unconditional rescale (32 multiplies): no branch in the middle of
        // the stage, so the compiler schedules the whole stage as one block
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            o[i][0] *= corr_o[0];
            o[i][1] *= corr_o[1];
            o[i][2] *= corr_o[0];
            o[i][3] *= corr_o[1];
        }
        const VRaw v1 = load_v(st + kOffVC + kSubC, st + kOffVS + kSubS);
        {
            // running sum and zero-point sum (with the split columns the sign
            // s = 2b - 1 moves -valpha into the zero point)
            constexpr bool kSplitCols = G <= 4;
            const float za0 = h_hi(v0.vma.x) - (kSplitCols ? h_lo(v0.vma.y) : 0.0f);
            const float zb0 = h_hi(v0.vmb.x) - (kSplitCols ? h_lo(v0.vmb.y) : 0.0f);
            const float za1 = h_hi(v1.vma.x) - (kSplitCols ? h_lo(v1.vma.y) : 0.0f);
            const float zb1 = h_hi(v1.vmb.x) - (kSplitCols ? h_lo(v1.vmb.y) : 0.0f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                lrun[e] = fmaf(lrun[e], corr[e], (p0[e] + p0[2 + e]) + (p1[e] + p1[2 + e]));
                zrun[e] = fmaf(zrun[e], corr[e],
                               fmaf(p0[e], za0, fmaf(p0[2 + e], zb0, fmaf(p1[e], za1, p1[2 + e] * zb1))));
            }
        }
        pv(v0, p0);
        pv(v1, p1);
    }
};

// warp that owns global tile t when T tiles are cut into NW equal ranges
// (range w = [floor(w*T/NW), floor((w+1)*T/NW)))
__host__ __device__ __forceinline__ int64_t owner_warp(int64_t t, int64_t T, int64_t NW) {
    return ((t + 1) * NW - 1) / T;
}

// ---- host ----
static PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
static std::mutex g_encode_mu;

static int get_encode() {
    std::lock_guard<std::mutex> lk(g_encode_mu);
    if (!g_encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr) != cudaSuccess ||
            qr != cudaDriverEntryPointSuccess || !fn)
            return ECC_ERR_CUDA;
        g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
    return ECC_OK;
}

// 4-D map over a block pool: (byte in record, token, kv head, batch); rb =
// bytes per record (128, or 96 without the pad sector).  The boxes read bytes
// 0..63 and 64..95 of a record, so both sizes take the same kernel.
static int make_map(CUtensorMap *m, const void *base, int64_t seq_len, int Hkv, int B, int64_t bs_h, int64_t bs_b,
                    uint32_t box_x, int rb, CUtensorMapSwizzle swz, int box_rows = kTile) {
    cuuint64_t dims[4] = {(cuuint64_t)rb, (cuuint64_t)seq_len, (cuuint64_t)Hkv, (cuuint64_t)B};
    cuuint64_t sh = (cuuint64_t)bs_h * rb, sb = (cuuint64_t)bs_b * rb;
    if (Hkv == 1) sh = (cuuint64_t)seq_len * rb;  // stride of an extent-1 dim is unused
    if (B == 1) sb = sh * (cuuint64_t)Hkv;
    cuuint64_t strides[3] = {(cuuint64_t)rb, sh, sb};
    cuuint32_t box[4] = {box_x, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const auto encode = [&]() {
        return g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void *>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swz, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (encode()) return ECC_OK;
    // The first CUDA call of a host thread: the driver's call, unlike the runtime's, does not make the device's
    // context current by itself.
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return ECC_ERR_CUDA;
    return encode() ? ECC_OK : ECC_ERR_CUDA;
}

// The four maps of a launch: K codes (64-byte rows, no swizzle: the K code
// reads are conflict-free as laid out), K syndrome + metadata (32-byte rows,
// 32-byte swizzle), V codes (64-byte swizzle), V syndrome + metadata (32-byte
// swizzle); the kernel's stage reads undo the swizzles.
static int make_maps(CUtensorMap *kc, CUtensorMap *ks, CUtensorMap *vc, CUtensorMap *vs, const void *kb,
                     const void *vb, int64_t len, int Hkv, int B, int64_t bs_h, int64_t bs_b, int rb,
                     int box_rows = kTile) {
    if (make_map(kc, kb, len, Hkv, B, bs_h, bs_b, 64, rb, CU_TENSOR_MAP_SWIZZLE_NONE, box_rows) != ECC_OK ||
        make_map(ks, kb, len, Hkv, B, bs_h, bs_b, 32, rb, CU_TENSOR_MAP_SWIZZLE_32B, box_rows) != ECC_OK ||
        make_map(vc, vb, len, Hkv, B, bs_h, bs_b, 64, rb, CU_TENSOR_MAP_SWIZZLE_64B, box_rows) != ECC_OK ||
        make_map(vs, vb, len, Hkv, B, bs_h, bs_b, 32, rb, CU_TENSOR_MAP_SWIZZLE_32B, box_rows) != ECC_OK)
        return ECC_ERR_CUDA;
    return ECC_OK;
}

// The table loads address shared memory with kSmemReserve folded in; the
// driver reports that reserve per device.
static bool reserve_matches() {
    static int known[64];  // 0 unknown, 1 matches, 2 differs
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (!known[dev]) {
        int v = -1;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrReservedSharedMemoryPerBlock, dev) != cudaSuccess) return false;
        known[dev] = (v == kSmemReserve) ? 1 : 2;
    }
    return known[dev] == 1;
}

}  // namespace tmak
}  // namespace ecc
