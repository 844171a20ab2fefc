// call.cu -- the paged and sampling entry points with their arguments in one
// array of words: a binding that converts every argument by itself (ctypes: 0.1
// us each, of 22 for the decode) pays 2 us a call for them, and 0.6 us for one
// packed array.
#include <cstring>

#include "../../include/ecc_kv_b200.h"

namespace {

struct Words {
    const int64_t *w;
    bool ok = true;  // every 32-bit argument fits
    template <class T>
    T *ptr() {
        return reinterpret_cast<T *>((uintptr_t)*w++);
    }
    int64_t i64() { return *w++; }
    int i32() {
        const int64_t v = *w++;
        ok = ok && v == (int64_t)(int)v;
        return (int)v;
    }
    float f32() {
        double d;
        std::memcpy(&d, w++, sizeof d);
        return (float)d;
    }
    ecc_pages_t pages() {
        ecc_pages_t p;
        p.table = ptr<const int>();
        p.table_stride = i64();
        p.width = i32();
        p.page_size = i32();
        p.n_pages = i64();
        return p;
    }
};

int compress(Words a) {
    const void *x0 = a.ptr<const void>();
    const int64_t x0b = a.i64(), x0h = a.i64(), x0l = a.i64();
    void *y0 = a.ptr<void>();
    const int64_t y0p = a.i64(), y0h = a.i64();
    const void *x1 = a.ptr<const void>();
    const int64_t x1b = a.i64(), x1h = a.i64(), x1l = a.i64();
    void *y1 = a.ptr<void>();
    const int64_t y1p = a.i64(), y1h = a.i64();
    const int B = a.i32(), H = a.i32();
    const int64_t L = a.i64();
    const ecc_pages_t pages = a.pages();
    const int *pos = a.ptr<const int>(), *new_lens = a.ptr<const int>();
    const int mode = a.i32();
    ecc_stream_t s = reinterpret_cast<ecc_stream_t>(a.ptr<void>());
    if (!a.ok) return ECC_ERR_SHAPE;
    return ecc_compress_paged(x0, x0b, x0h, x0l, y0, y0p, y0h, x1, x1b, x1h, x1l, y1, y1p, y1h, B, H, L, &pages, pos,
                              new_lens, mode, s);
}

int dequantize(Words a) {
    const void *x0 = a.ptr<const void>();
    const int64_t x0p = a.i64(), x0h = a.i64();
    void *y0 = a.ptr<void>();
    const void *x1 = a.ptr<const void>();
    const int64_t x1p = a.i64(), x1h = a.i64();
    void *y1 = a.ptr<void>();
    const int B = a.i32(), H = a.i32();
    const int64_t max_len = a.i64();
    const ecc_pages_t pages = a.pages();
    const int *lens = a.ptr<const int>();
    const int mode = a.i32();
    ecc_stream_t s = reinterpret_cast<ecc_stream_t>(a.ptr<void>());
    if (!a.ok) return ECC_ERR_SHAPE;
    return ecc_dequantize_paged(x0, x0p, x0h, y0, x1, x1p, x1h, y1, B, H, max_len, &pages, lens, mode, s);
}

int decode(Words a) {
    const void *q = a.ptr<const void>(), *k = a.ptr<const void>(), *v = a.ptr<const void>();
    const int64_t sp = a.i64(), sh = a.i64();
    const ecc_pages_t pages = a.pages();
    const int *lens = a.ptr<const int>();
    void *out = a.ptr<void>();
    float *lse = a.ptr<float>(), *weights = a.ptr<float>();
    const int64_t wb = a.i64(), wh = a.i64();
    void *ws = a.ptr<void>();
    const size_t ws_bytes = (size_t)a.i64();
    const int B = a.i32(), Hq = a.i32(), Hkv = a.i32();
    const float scale = a.f32();
    const int window = a.i32(), sinks = a.i32(), flags = a.i32();
    ecc_stream_t s = reinterpret_cast<ecc_stream_t>(a.ptr<void>());
    if (!a.ok) return ECC_ERR_SHAPE;
    return ecc_decode_paged(q, k, v, sp, sh, &pages, lens, out, lse, weights, wb, wh, ws, ws_bytes, B, Hq, Hkv, scale,
                            window, sinks, flags, s);
}

int evict(Words a) {
    void *k = a.ptr<void>(), *v = a.ptr<void>();
    const int64_t sp = a.i64(), sh = a.i64();
    const ecc_pages_t pages = a.pages();
    const int *lens = a.ptr<const int>();
    const float *w = a.ptr<const float>();
    const int64_t wb = a.i64(), wh = a.i64();
    const ecc_pages_t outs = a.pages();
    float *ow = a.ptr<float>();
    const int64_t ob = a.i64(), oh = a.i64(), out_len = a.i64();
    int *kept = a.ptr<int>();
    const int B = a.i32(), Hkv = a.i32(), budget = a.i32(), sinks = a.i32(), recent = a.i32(), rec = a.i32();
    void *ws = a.ptr<void>();
    const size_t ws_bytes = (size_t)a.i64();
    ecc_stream_t s = reinterpret_cast<ecc_stream_t>(a.ptr<void>());
    if (!a.ok) return ECC_ERR_SHAPE;
    return ecc_evict_paged(k, v, sp, sh, &pages, lens, w, wb, wh, &outs, ow, ob, oh, out_len, kept, B, Hkv, budget,
                           sinks, recent, rec, ws, ws_bytes, s);
}

int sample(Words a) {
    const void *x = a.ptr<const void>();
    const int64_t stride = a.i64();
    const int dtype = a.i32(), B = a.i32();
    const int64_t V = a.i64();
    const float *u = a.ptr<const float>(), *t = a.ptr<const float>();
    const float t0 = a.f32();
    const int *k = a.ptr<const int>();
    const int k0 = a.i32();
    const float *p = a.ptr<const float>();
    const float p0 = a.f32();
    const float *m = a.ptr<const float>();
    const float m0 = a.f32();
    int64_t *token = a.ptr<int64_t>();
    float *logprob = a.ptr<float>();
    ecc_stream_t s = reinterpret_cast<ecc_stream_t>(a.ptr<void>());
    if (!a.ok) return ECC_ERR_SHAPE;
    return ecc_sample(x, stride, dtype, B, V, u, t, t0, k, k0, p, p0, m, m0, token, logprob, s);
}

}  // namespace

extern "C" int ecc_call(int entry, const int64_t *words) {
    if (!words) return ECC_ERR_NULL;
    switch (entry) {
        case ECC_CALL_COMPRESS_PAGED: return compress(Words{words});
        case ECC_CALL_DEQUANTIZE_PAGED: return dequantize(Words{words});
        case ECC_CALL_DECODE_PAGED: return decode(Words{words});
        case ECC_CALL_EVICT_PAGED: return evict(Words{words});
        case ECC_CALL_SAMPLE: return sample(Words{words});
        default: return ECC_ERR_SHAPE;
    }
}
