// paged.cu -- reading a paged block cache back as fp16 (sm_100a).
#include <algorithm>

#include "paged.cuh"

namespace ecc {

int launch_status();
int sm_count();

namespace paged {

// ---- read-back ---------------------------------------------------------------
// x = (C[q] scale + zero) + alpha s per element, then (optionally) the inverse
// rotation: the normalised WHT, whose factor 1/sqrt(128) is folded into scale,
// zero and alpha once per vector.  Four lanes hold a vector, lane g elements
// 32c + 8g + i: strides 1, 2, 4, 32, 64 of the transform stay in registers,
// 8 and 16 are lane exchanges.  Pairs of elements are packed fp32x2.  A code
// byte's two centroids come from a 256-entry table, one copy per lane of a
// half-warp (64-bit loads of a half-warp then hit distinct banks).
constexpr int kReadWarps = 8;
constexpr int kReadTile = kReadWarps * 8;  // vectors per CTA and step

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
    float norm;  // 1/sqrt(128), or 1 without the rotation
};

__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return __ffma2_rn(b, make_float2(-1.0f, -1.0f), a); }

template <bool kRotate>
__global__ void __launch_bounds__(kReadWarps * 32, 3) dequant_paged_kernel(const __grid_constant__ ReadArgs a) {
    __shared__ float2 tab[256 * 16];
    for (int i = threadIdx.x; i < 256 * 16; i += blockDim.x) {
        const int v = i >> 4;
        float lo = lm(0), hi = lm(0);
#pragma unroll
        for (int k = 1; k < 16; ++k) {
            lo = (v & 15) == k ? lm(k) : lo;
            hi = (v >> 4) == k ? lm(k) : hi;
        }
        tab[i] = make_float2(lo, hi);
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & 3;
    const float2 *mytab = tab + (lane & 15);
    const uint32_t tiles = (a.n_vec + kReadTile - 1) / kReadTile;
    // A lane's share of a vector: its code words, the syndrome, the metadata; a step's are requested before the
    // step in front of it is worked on.
    struct Raw {
        uint32_t cw[4];
        uint4 sy;
        uint2 meta;
        bool live;  // else: behind the sequence's last token
    };
    auto request = [&](uint32_t it, Raw &r) {
        const ReadJob &jb = it < tiles ? a.j[0] : a.j[1];
        const uint32_t vi = (it < tiles ? it : it - tiles) * kReadTile + warp * 8 + (lane >> 2);
        r.live = false;
        if (vi >= a.n_vec) return;
        const uint32_t row = fdiv(vi, a.div_l);
        const int t = (int)(vi - row * a.div_l.d);
        const uint32_t b = fdiv(row, a.div_h);
        const int h = (int)(row - b * a.div_h.d);
        const int n = __ldg(a.lens + b);
        if (n < 0 || n > a.t.capacity) atomicExch(&g_paged_error, 5);
        if (t >= min(n, a.t.capacity)) return;
        int slot;
        const int page = a.t.page((int)b, t, slot);
        if (page < 0) return;
        const uint8_t *src = jb.blocks + ((int64_t)page * jb.bs_p + (int64_t)h * jb.bs_h + slot) * a.rec;
#pragma unroll
        for (int c = 0; c < 4; ++c) r.cw[c] = __ldg(reinterpret_cast<const uint32_t *>(src) + 4 * c + g);
        r.sy = __ldg(reinterpret_cast<const uint4 *>(src + kSynOff));
        r.meta = __ldg(reinterpret_cast<const uint2 *>(src + kScaleOff));
        r.live = true;
    };
    const uint32_t steps = tiles * a.njobs;
    Raw next;
    if (blockIdx.x < steps) request(blockIdx.x, next);
    for (uint32_t it = blockIdx.x; it < steps; it += gridDim.x) {
        const Raw cur = next;
        if (it + gridDim.x < steps) request(it + gridDim.x, next);
        const uint32_t v = (it < tiles ? it : it - tiles) * kReadTile + warp * 8 + (lane >> 2);
        const bool valid = v < a.n_vec;
        __half *const out = it < tiles ? a.j[0].out : a.j[1].out;
        float2 P[4][4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) P[c][j] = make_float2(0.0f, 0.0f);
        if (cur.live) {
            const uint32_t sy[4] = {cur.sy.x, cur.sy.y, cur.sy.z, cur.sy.w};
            const float sc = __half2float(__ushort_as_half((unsigned short)(cur.meta.x & 0xffffu))) * a.norm;
            const float zr = __half2float(__ushort_as_half((unsigned short)(cur.meta.x >> 16))) * a.norm;
            const uint32_t al =
                __float_as_uint(__half2float(__ushort_as_half((unsigned short)(cur.meta.y & 0xffffu))) * a.norm);
            const float2 sc2 = make_float2(sc, sc), zr2 = make_float2(zr, zr);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t off = ~(sy[c] >> (8 * g));  // bit i set: s = -1
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 cen = mytab[((cur.cw[c] >> (8 * j)) & 0xffu) * 16];
                    const float2 s = make_float2(__uint_as_float(al ^ ((off << (31 - 2 * j)) & 0x80000000u)),
                                                 __uint_as_float(al ^ ((off << (30 - 2 * j)) & 0x80000000u)));
                    P[c][j] = add2(__ffma2_rn(cen, sc2, zr2), s);
                }
            }
        }
        if (kRotate) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
                for (int j = 0; j < 4; ++j) P[c][j] = make_float2(P[c][j].x + P[c][j].y, P[c][j].x - P[c][j].y);
#pragma unroll
                for (int j = 0; j < 4; j += 2) {  // stride 2
                    const float2 x = P[c][j], y = P[c][j + 1];
                    P[c][j] = add2(x, y);
                    P[c][j + 1] = sub2(x, y);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // stride 4
                    const float2 x = P[c][j], y = P[c][j + 2];
                    P[c][j] = add2(x, y);
                    P[c][j + 2] = sub2(x, y);
                }
            }
#pragma unroll
            for (int s = 1; s <= 2; s <<= 1) {  // strides 8, 16: partner lane g ^ s
                const float sg = (g & s) ? -1.0f : 1.0f;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 p = make_float2(__shfl_xor_sync(0xffffffffu, P[c][j].x, s),
                                                     __shfl_xor_sync(0xffffffffu, P[c][j].y, s));
                        P[c][j] = __ffma2_rn(make_float2(sg, sg), P[c][j], p);
                    }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // strides 32, 64
                float2 x = P[0][j], y = P[1][j];
                P[0][j] = add2(x, y);
                P[1][j] = sub2(x, y);
                x = P[2][j], y = P[3][j];
                P[2][j] = add2(x, y);
                P[3][j] = sub2(x, y);
                x = P[0][j], y = P[2][j];
                P[0][j] = add2(x, y);
                P[2][j] = sub2(x, y);
                x = P[1][j], y = P[3][j];
                P[1][j] = add2(x, y);
                P[3][j] = sub2(x, y);
            }
        }
        if (valid) {
            __half *dst = out + (int64_t)v * kD + 8 * g;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __half2 x = __floats2half2_rn(P[c][j].x, P[c][j].y);
                    w[j] = *reinterpret_cast<const uint32_t *>(&x);
                }
                *reinterpret_cast<uint4 *>(dst + 32 * c) = make_uint4(w[0], w[1], w[2], w[3]);
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
    a.norm = (mode & ECC_DEQUANT_UNROTATE) ? kInvSqrt128 : 1.0f;
    const int64_t tiles = (int64_t)(a.n_vec + kReadTile - 1) / kReadTile * a.njobs;
    const dim3 grid((unsigned)std::min<int64_t>(tiles, (int64_t)sm_count() * 3)), block(kReadWarps * 32);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = (mode & ECC_DEQUANT_UNROTATE) ? launch_pdl(dequant_paged_kernel<true>, grid, block, 0, s, a)
                                                        : launch_pdl(dequant_paged_kernel<false>, grid, block, 0, s, a);
    if (e != cudaSuccess) return ECC_ERR_LAUNCH;
    return launch_status();
}
