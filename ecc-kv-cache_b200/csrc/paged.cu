// paged.cu -- reading a paged block cache back as fp16 (sm_100a).
#include <algorithm>

#include "paged.cuh"

namespace ecc {

int launch_status();
int sm_count();

namespace paged {

// ---- read-back ---------------------------------------------------------------
// out = WHT(x) / sqrt(128) with x = C[q] scale + zero + alpha s per element, or
// x itself.  By linearity WHT(x) = scale WHT(C[q]) + alpha WHT(s) + zero WHT(1),
// and WHT(1) is 128 at element 0 alone; so the transforms run over the codes'
// centroids and the sign bits as they are stored, and scale and alpha come in
// per vector afterwards.
//
// The transform of 128 = 2^7 elements splits by the bits d0..d6 of the element
// number: bits {d0, d4, d5, d6} are contracted by tensor-core products with a
// 16 x 16 matrix of +-1, {d1, d2, d3} by butterflies between the eight products'
// results, which lie in the same lane: no exchange between lanes.  A warp
// takes 16 vectors; lane (g, c) holds the 16 code bytes 16c.. and the syndrome
// word c of vectors g and g + 8.
//   centroids, 8 vectors a product: operand rows g / g+8 = hi / lo fp16 parts of
//     vector g's centroids (22 bits; a code byte's pair of words is one 64-bit
//     load from a table with a copy per lane of a half-warp), k = (d0; d5, d6 =
//     c; d4 = code byte + 8).  The two result rows are added.
//   signs, 16 vectors a product: bits p and p + 16 of the syndrome word, moved
//     to bit 10, are fp16 0 or 2^-14: k = (d4; d5, d6 = c; d0), s = 2b - 1.
// Result columns 2c', 2c'+1 of tile j are bits (o0; o4, o5 = c'; o6 = j) of the
// output element, so a lane ends with 16 neighbouring outputs per tile.
//
// Measured at 2 x 4 x 8 x 10240 vectors out, 0.7 of them live: 53 us (3.2 TB/s of
// fp16 written), where filling the output with zeros alone takes 44 us.  A
// butterfly kernel with four lanes per vector (72 warp instructions and 21 L1
// wavefronts a vector, against 47 and 12) took 63 us, bound by L1; without the
// volatile order, 57 to 67 us.  In the stored basis (kRotate false) 53 us too.
constexpr int kReadWarps = 8;
constexpr int kReadVecs = 16;                       // per warp and step
constexpr int kReadTile = kReadWarps * kReadVecs;   // per CTA and step
constexpr int kReadTable = 65536;                   // bytes of its table

struct ReadJob {
    const uint8_t *blocks;
    int64_t bs_p, bs_h;
    __half *out;
};
struct ReadArgs {
    ReadJob j[2];
    PageTable t;
    const int *lens;
    FastDiv div_h, div_l;
    uint32_t n_vec;  // of one job
    int njobs, rec;
};

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __ffma2_rn(b, make_float2(-1.0f, -1.0f), a); }
// d = a b, with the accumulator's zero as an operand.  Volatile, like the loads
// of Share: in program order the next step's loads come first, and the
// compiler keeps them there instead of sinking them behind the products.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// fp16x2 of (-1)^e0, (-1)^e1
__device__ __forceinline__ uint32_t signs2(int e0, int e1) {
    return 0x3C003C00u | ((e0 & 1) ? 0x8000u : 0u) | ((e1 & 1) ? 0x80000000u : 0u);
}

// The record of vector vi of a job, or null behind the last token.
__device__ __forceinline__ const uint8_t *record_of(const ReadArgs &a, const ReadJob &jb, uint32_t vi) {
    if (vi >= a.n_vec) return nullptr;
    const uint32_t row = fdiv(vi, a.div_l);
    const int t = (int)(vi - row * a.div_l.d);
    const uint32_t b = fdiv(row, a.div_h);
    const int h = (int)(row - b * a.div_h.d);
    const int n = __ldg(a.lens + b);
    if (n < 0 || n > a.t.capacity) atomicExch(&g_paged_error, 5);
    if (t >= min(n, a.t.capacity)) return nullptr;
    int slot;
    const int page = a.t.page((int)b, t, slot);
    if (page < 0) return nullptr;
    return jb.blocks + ((int64_t)page * jb.bs_p + (int64_t)h * jb.bs_h + slot) * a.rec;
}

// A lane's share of a vector.
struct Share {
    uint4 codes;
    uint32_t sy;
    uint2 meta;
    __device__ __forceinline__ void load(const uint8_t *rec, int c) {
        codes = make_uint4(0u, 0u, 0u, 0u);
        sy = 0u;
        meta = make_uint2(0u, 0u);  // all zero: the output is zero
        if (!rec) return;
        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(codes.x), "=r"(codes.y), "=r"(codes.z), "=r"(codes.w)
                     : "l"(rec + 16 * c));
        asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(sy) : "l"(rec + kSynOff + 4 * c));
        asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(meta.x), "=r"(meta.y) : "l"(rec + kScaleOff));
    }
    __device__ __forceinline__ float scale() const { return __half2float(__ushort_as_half((unsigned short)meta.x)); }
    __device__ __forceinline__ float zero() const { return __half2float(__ushort_as_half((unsigned short)(meta.x >> 16))); }
    __device__ __forceinline__ float alpha() const { return __half2float(__ushort_as_half((unsigned short)meta.y)); }
};

template <bool kRotate>
__global__ void __launch_bounds__(kReadWarps * 32, 2) dequant_paged_kernel(const __grid_constant__ ReadArgs a) {
    // entry v, copy l (l = lane mod 16): (hi, lo) fp16x2 words of the codes v & 15, v >> 4, or their fp32 values, at
    // 256 v + 8 l: the offset is one byte permutation
    extern __shared__ __align__(16) uint8_t tab[];
    static_assert(kReadWarps * 32 == 256, "a thread has one low code, one copy and all high codes");
    float lo = lm(0);
#pragma unroll
    for (int k = 1; k < 16; ++k) lo = (threadIdx.x >> 4) == k ? lm(k) : lo;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const float hi = lm(k);
        uint2 *const to = reinterpret_cast<uint2 *>(tab + 256 * (16 * k + (threadIdx.x >> 4))) + (threadIdx.x & 15);
        if (kRotate) {
            const __half2 x = __floats2half2_rn(lo, hi);
            const __half2 y = __floats2half2_rn(lo - __low2float(x), hi - __high2float(x));
            *to = make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
        } else {
            *to = make_uint2(__float_as_uint(lo), __float_as_uint(hi));
        }
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const uint32_t lane8 = 8u * (lane & 15), tab_at = (uint32_t)__cvta_generic_to_shared(tab);
    const uint32_t tiles = (a.n_vec + kReadTile - 1) / kReadTile, steps = tiles * a.njobs;
    // the +-1 matrices: column o = (g & 1, g >> 1 & 1, g >> 2, j), rows as above
    uint32_t bc[2][2], bs[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int o0 = g & 1, o4 = (g >> 1) & 1, fixed = (c & 1 & (g >> 2)) + ((c >> 1) & j);
        bc[j][0] = signs2(fixed, fixed + o0);
        bc[j][1] = signs2(fixed + o4, fixed + o4 + o0);
        bs[j][0] = signs2(fixed, fixed + o4);
        bs[j][1] = signs2(fixed + o0, fixed + o0 + o4);
    }
    Share next[2];
    auto request = [&](uint32_t it) {
        const ReadJob &jb = it < tiles ? a.j[0] : a.j[1];
        const uint32_t v0 = (it < tiles ? it : it - tiles) * kReadTile + warp * kReadVecs + g;
#pragma unroll
        for (int q = 0; q < 2; ++q) next[q].load(record_of(a, jb, v0 + 8 * q), c);
    };
    if (blockIdx.x < steps) request(blockIdx.x);
    for (uint32_t it = blockIdx.x; it < steps; it += gridDim.x) {
        const Share cur[2] = {next[0], next[1]};
        if (it + gridDim.x < steps) request(it + gridDim.x);  // while this step is worked on
        const uint32_t v0 = (it < tiles ? it : it - tiles) * kReadTile + warp * kReadVecs + g;
        __half *const out = it < tiles ? a.j[0].out : a.j[1].out;
        auto store = [&](int q, int at, const uint32_t (&w)[8]) {  // 16 outputs from element `at`
            if (v0 + 8 * q >= a.n_vec) return;
            uint4 *dst = reinterpret_cast<uint4 *>(out + (int64_t)(v0 + 8 * q) * kD + at);
            dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
            dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        };
        auto half2_of = [](float2 x) {
            const __half2 h = __floats2half2_rn(x.x, x.y);
            return *reinterpret_cast<const uint32_t *>(&h);
        };
        auto entry = [&](uint32_t word, int byte) {
            uint2 r;  // the table is constant after the set-up barrier
            asm("ld.shared.v2.u32 {%0, %1}, [%2];"
                : "=r"(r.x), "=r"(r.y)
                : "r"(tab_at + __byte_perm(word, lane8, 0x5504u | ((uint32_t)byte << 4))));
            return r;
        };
        if constexpr (kRotate) {
            float2 x[2][2][8];  // [vector][tile][block]
            float2 sc[2], al[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float s = cur[q].scale() * kInvSqrt128, t = cur[q].alpha() * (kInvSqrt128 * 32768.0f);
                sc[q] = make_float2(s, s);
                al[q] = make_float2(t, t);  // of the bits' weight 2^-14, twice
            }
#pragma unroll
            for (int blk = 0; blk < 8; ++blk) {
                float ss[2][4];
                const int p = 2 * blk;
                // bits p (d0 = 0) and p + 1 (d0 = 1) of both halves to bit 10
                uint32_t w[2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int d0 = 0; d0 < 2; ++d0) {
                        const int sh = 10 - p - d0;
                        w[q][d0] = (sh >= 0 ? cur[q].sy << sh : cur[q].sy >> -sh) & 0x04000400u;
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    mma16816(ss[j], w[0][0], w[1][0], w[0][1], w[1][1], bs[j][0], bs[j][1]);
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint32_t w0 = blk < 4 ? cur[q].codes.x : cur[q].codes.y;
                    const uint32_t w1 = blk < 4 ? cur[q].codes.z : cur[q].codes.w;
                    const uint2 e0 = entry(w0, blk & 3), e1 = entry(w1, blk & 3);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float d[4];
                        mma16816(d, e0.x, e0.y, e1.x, e1.y, bc[j][0], bc[j][1]);
                        const float2 v = add2(make_float2(d[0], d[1]), make_float2(d[2], d[3]));
                        const float2 u = make_float2(ss[j][2 * q], ss[j][2 * q + 1]);
                        x[q][j][blk] = __ffma2_rn(v, sc[q], __fmul2_rn(u, al[q]));
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int s = 1; s < 8; s <<= 1)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (!(k & s)) {
                                const float2 y = x[q][j][k], z = x[q][j][k + s];
                                x[q][j][k] = add2(y, z);
                                x[q][j][k + s] = sub2(y, z);
                            }
                    // zero and the signs' -1: element 0 alone
                    if (j == 0 && c == 0) x[q][0][0].x += (cur[q].zero() - cur[q].alpha()) * (128.0f * kInvSqrt128);
                    uint32_t w[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] = half2_of(x[q][j][k]);
                    store(q, 64 * j + 16 * c, w);
                }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float sc = cur[q].scale(), zr = cur[q].zero();
                const uint32_t al = __float_as_uint(cur[q].alpha()), off = ~cur[q].sy;
                const uint32_t cw[4] = {cur[q].codes.x, cur[q].codes.y, cur[q].codes.z, cur[q].codes.w};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t w[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int i = 16 * half + 2 * k;  // of the lane's 32 elements
                        const uint2 e = entry(cw[2 * half + (k >> 2)], k & 3);
                        const float2 s = make_float2(__uint_as_float(al ^ ((off << (31 - i)) & 0x80000000u)),
                                                     __uint_as_float(al ^ ((off << (30 - i)) & 0x80000000u)));
                        const float2 y = make_float2(__uint_as_float(e.x), __uint_as_float(e.y));
                        w[k] = half2_of(add2(__ffma2_rn(y, make_float2(sc, sc), make_float2(zr, zr)), s));
                    }
                    store(q, 32 * c + 16 * half, w);
                }
            }
        }
    }
}

}  // namespace paged

int paged_cache_error(int reset) {
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

static inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }

extern "C" int ecc_dequantize_paged(const void *blocks0, int64_t b0s_p, int64_t b0s_h, void *out0_f16,
                                    const void *blocks1, int64_t b1s_p, int64_t b1s_h, void *out1_f16, int B, int H,
                                    int64_t max_len, const ecc_pages_t *pages, const int *seq_lens, int mode,
                                    ecc_stream_t stream) {
    using namespace paged;
    if (mode & ~(ECC_DEQUANT_UNROTATE | ECC_DEQUANT_BLOCK96)) return ECC_ERR_SHAPE;
    if (B < 0 || H < 0 || max_len < 0) return ECC_ERR_SHAPE;
    if ((int64_t)B * H == 0 || max_len == 0) return ECC_OK;
    if (!pages || !seq_lens || !blocks0 || !out0_f16 || (!blocks1 != !out1_f16)) return ECC_ERR_NULL;
    ReadArgs a{};
    const int rc = make_table(*pages, &a.t);
    if (rc != ECC_OK) return rc;
    // 32-bit vector numbers
    if (max_len > (1ll << 30) || (int64_t)B * H >= (1ll << 31) / max_len) return ECC_ERR_SHAPE;
    a.rec = (mode & ECC_DEQUANT_BLOCK96) ? 96 : kBlockBytes;
    if (!aligned(blocks0, 16) || !aligned(blocks1, 16) || !aligned(out0_f16, 16) || !aligned(out1_f16, 16) ||
        !aligned(seq_lens, 4))
        return ECC_ERR_ALIGN;
    a.j[0] = {reinterpret_cast<const uint8_t *>(blocks0), b0s_p, b0s_h, reinterpret_cast<__half *>(out0_f16)};
    a.j[1] = {reinterpret_cast<const uint8_t *>(blocks1), b1s_p, b1s_h, reinterpret_cast<__half *>(out1_f16)};
    a.njobs = blocks1 ? 2 : 1;
    a.lens = seq_lens;
    a.div_h = make_fastdiv((uint32_t)H);
    a.div_l = make_fastdiv((uint32_t)max_len);
    a.n_vec = (uint32_t)((int64_t)B * H * max_len);
    const int64_t tiles = (int64_t)(a.n_vec + kReadTile - 1) / kReadTile * a.njobs;
    const dim3 grid((unsigned)std::min<int64_t>(tiles, (int64_t)sm_count() * 2)), block(kReadWarps * 32);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const auto kernel = (mode & ECC_DEQUANT_UNROTATE) ? dequant_paged_kernel<true> : dequant_paged_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kReadTable);
    if (e == cudaSuccess) e = launch_pdl(kernel, grid, block, kReadTable, s, a);
    if (e != cudaSuccess) return ECC_ERR_LAUNCH;
    return launch_status();
}
