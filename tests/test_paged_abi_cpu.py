"""The paged and sampling entry points refuse bad arguments before any device
call; the Python wrappers refuse CPU tensors."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, NULL, SHAPE, ALIGN, GQA, WORKSPACE, PARAM = 0, -1, -2, -3, -4, -5, -10


class Pages(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("width", ctypes.c_int),
                ("page_size", ctypes.c_int), ("n_pages", ctypes.c_int64)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(ROOT, "ecc-kv-cache_b200", "custom_ecc_cuda", "libeccb200.so"))
    p, i64, i32, f32, sz, pg = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t,
                                ctypes.POINTER(Pages))
    lib.ecc_compress_paged.argtypes = [p, i64, i64, i64, p, i64, i64, p, i64, i64, i64, p, i64, i64, i32, i32, i64, pg, p,
                                       p, i32, p]
    lib.ecc_dequantize_paged.argtypes = [p, i64, i64, p, p, i64, i64, p, i32, i32, i64, pg, p, i32, p]
    lib.ecc_decode_paged_workspace_size.argtypes = [i32, i32, i32, i64, i32]
    lib.ecc_decode_paged_workspace_size.restype = sz
    lib.ecc_decode_paged.argtypes = [p, p, p, i64, i64, pg, p, p, p, p, i64, i64, p, sz, i32, i32, i32, f32, i32, i32,
                                     i32, p]
    lib.ecc_evict_paged_workspace_size.argtypes = [i64]
    lib.ecc_evict_paged_workspace_size.restype = sz
    lib.ecc_evict_paged.argtypes = [p, p, i64, i64, pg, p, p, i64, i64, pg, p, i64, i64, i64, p, i32, i32, i32, i32, i32,
                                    i32, p, sz, p]
    lib.ecc_sample.argtypes = [p, i64, i32, i32, i64, p, p, f32, p, i32, p, f32, p, f32, p, p, p]
    return lib


GOOD = dict(table=4096, table_stride=4, width=4, page_size=16, n_pages=10)


def pages(**kw):
    return Pages(**{**GOOD, **kw})


BAD_PAGES = [(dict(table=None), NULL), (dict(width=0), SHAPE), (dict(page_size=0), SHAPE), (dict(n_pages=0), SHAPE),
             (dict(page_size=24), SHAPE), (dict(n_pages=1 << 31), SHAPE), (dict(width=1 << 20, page_size=1 << 11), SHAPE),
             (dict(table=4098), ALIGN)]


@pytest.mark.parametrize("kw,code", BAD_PAGES, ids=str)
def test_bad_page_tables(lib, kw, code):
    pg = pages(**kw)
    assert lib.ecc_compress_paged(4096, 0, 0, 128, 4096, 32, 16, None, 0, 0, 0, None, 0, 0, 1, 1, 4, pg, 4096, None, 1,
                                  None) == code
    assert lib.ecc_dequantize_paged(4096, 32, 16, 4096, None, 0, 0, None, 1, 1, 4, pg, 4096, 0, None) == code
    assert lib.ecc_decode_paged(4096, 4096, 4096, 32, 16, pg, 4096, 4096, None, None, 0, 0, 4096, 1 << 30, 1, 2, 1, 0.0,
                                0, 0, 0, None) == code
    assert lib.ecc_evict_paged(4096, 4096, 32, 16, pg, 4096, 4096, 64, 64, pages(table=8192), 4096, 64, 64, 64, 4096, 1, 1,
                               8, 0, 0, 128, 4096, 1 << 20, None) == code


def test_compress_paged_refusals(lib):
    def call(x=4096, blocks=4096, B=1, H=1, L=4, pg=pages(), pos=4096, new=None, mode=1, strides=(0, 0, 128), x1=None):
        return lib.ecc_compress_paged(x, *strides, blocks, 32, 16, x1, 0, 0, 128, None, 32, 16, B, H, L, pg, pos, new,
                                      mode, None)
    assert call(L=0) == OK and call(B=0) == OK
    for kw, code in ((dict(x=None), NULL), (dict(blocks=None), NULL), (dict(pos=None), NULL), (dict(pg=None), NULL),
                     (dict(x=4104), ALIGN), (dict(blocks=4112), ALIGN), (dict(pos=4098), ALIGN), (dict(new=4097), ALIGN),
                     (dict(strides=(0, 0, 129)), ALIGN), (dict(B=-1), SHAPE), (dict(L=-1), SHAPE), (dict(mode=4), SHAPE),
                     (dict(L=(1 << 30) + 1), SHAPE), (dict(x1=4096), NULL)):
        assert call(**kw) == code, kw


def test_dequantize_paged_refusals(lib):
    def call(b0=4096, o0=4096, b1=None, o1=None, B=1, H=1, n=4, pg=pages(), lens=4096, mode=0):
        return lib.ecc_dequantize_paged(b0, 32, 16, o0, b1, 32, 16, o1, B, H, n, pg, lens, mode, None)
    assert call(n=0) == OK and call(B=0) == OK
    for kw, code in ((dict(b0=None), NULL), (dict(o0=None), NULL), (dict(b1=4096), NULL), (dict(o1=4096), NULL),
                     (dict(lens=None), NULL), (dict(pg=None), NULL), (dict(b0=4104), ALIGN), (dict(o0=4098), ALIGN),
                     (dict(mode=4), SHAPE), (dict(B=-1), SHAPE), (dict(n=1 << 31), SHAPE),
                     (dict(B=1 << 10, H=1 << 10, n=1 << 20), SHAPE)):
        assert call(**kw) == code, kw


def test_decode_paged_refusals(lib):
    need = lib.ecc_decode_paged_workspace_size(2, 8, 2, 64, 0)
    assert 0 < need < lib.ecc_decode_paged_workspace_size(2, 8, 2, 64, 1)
    for bad in ((0, 8, 2, 64), (2, 7, 2, 64), (2, 18, 2, 64), (2, 8, 2, 0), (5000, 8, 2, 64), (2, 8, 2, (1 << 30) + 1)):
        assert lib.ecc_decode_paged_workspace_size(*bad, 0) == 0

    def call(q=4096, k=4096, v=4096, pg=pages(), lens=4096, out=4096, lse=None, w=None, ws=4096, nws=need, B=2, hq=8, hkv=2,
             sm=0.0, window=0, sinks=0, flags=0):
        return lib.ecc_decode_paged(q, k, v, 32, 16, pg, lens, out, lse, w, 64, 64, ws, nws, B, hq, hkv, sm, window, sinks,
                                    flags, None)
    assert call(B=0) == OK
    for kw, code in ((dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(lens=None), NULL),
                     (dict(out=None), NULL), (dict(pg=None), NULL), (dict(ws=None), WORKSPACE), (dict(nws=need - 1), WORKSPACE),
                     (dict(w=4096), WORKSPACE), (dict(hq=7), GQA), (dict(hq=18), SHAPE), (dict(B=-1), SHAPE),
                     (dict(window=-1), SHAPE), (dict(sinks=1), SHAPE), (dict(window=1, sinks=-1), SHAPE),
                     (dict(flags=4), SHAPE), (dict(sm=float("nan")), PARAM), (dict(sm=float("inf")), PARAM),
                     (dict(q=4104), ALIGN), (dict(k=4104), ALIGN), (dict(out=4097), ALIGN), (dict(lse=4098), ALIGN),
                     (dict(w=4098), ALIGN)):
        assert call(**kw) == code, kw


def test_evict_paged_refusals(lib):
    need = lib.ecc_evict_paged_workspace_size(10)
    assert need > 0 and lib.ecc_evict_paged_workspace_size(0) == 0 and lib.ecc_evict_paged_workspace_size(1 << 31) == 0

    def call(k=4096, pg=pages(), lens=4096, w=4096, og=pages(table=8192), ow=4096, kept=4096, B=1, hkv=1, budget=8, sinks=0,
             recent=0, rb=128, ws=4096, nws=need, out_len=64):
        return lib.ecc_evict_paged(k, 4096, 32, 16, pg, lens, w, 64, 64, og, ow, 64, 64, out_len, kept, B, hkv, budget,
                                   sinks, recent, rb, ws, nws, None)
    assert call(B=0) == OK
    for kw, code in ((dict(k=None), NULL), (dict(lens=None), NULL), (dict(w=None), NULL), (dict(ow=None), NULL),
                     (dict(kept=None), NULL), (dict(pg=None), NULL), (dict(og=None), NULL), (dict(ws=None), WORKSPACE),
                     (dict(nws=need - 1), WORKSPACE), (dict(budget=0), SHAPE), (dict(sinks=-1), SHAPE),
                     (dict(recent=-1), SHAPE), (dict(sinks=5, recent=4), SHAPE), (dict(budget=65), SHAPE),
                     (dict(rb=64), SHAPE), (dict(out_len=-1), SHAPE), (dict(B=-1), SHAPE), (dict(hkv=0), SHAPE),
                     (dict(og=pages(table=8192, n_pages=9)), SHAPE), (dict(og=pages(table=8192, page_size=32)), SHAPE),
                     (dict(k=4104), ALIGN), (dict(w=4098), ALIGN), (dict(kept=4097), ALIGN)):
        assert call(**kw) == code, kw


def test_sample_refusals(lib):
    def call(x=4096, stride=100, dtype=2, B=2, V=100, u=4096, t=(None, 1.0), k=(None, 0), p=(None, 1.0), m=(None, 0.0),
             tok=4096, lp=None):
        return lib.ecc_sample(x, stride, dtype, B, V, u, *t, *k, *p, *m, tok, lp, None)
    assert call(B=0) == OK
    nan = float("nan")
    for kw, code in ((dict(x=None), NULL), (dict(u=None), NULL), (dict(tok=None), NULL), (dict(B=-1), SHAPE),
                     (dict(V=0), SHAPE), (dict(V=(1 << 20) + 1), SHAPE), (dict(dtype=3), SHAPE), (dict(dtype=-1), SHAPE),
                     (dict(stride=-1), SHAPE), (dict(t=(None, -1.0)), PARAM), (dict(t=(None, nan)), PARAM),
                     (dict(k=(None, -1)), PARAM), (dict(p=(None, 0.0)), PARAM), (dict(p=(None, nan)), PARAM),
                     (dict(m=(None, -0.1)), PARAM), (dict(m=(None, 1.1)), PARAM), (dict(x=4098), ALIGN),
                     (dict(x=4097, dtype=0), ALIGN), (dict(u=4098), ALIGN), (dict(tok=4100), ALIGN), (dict(lp=4098), ALIGN),
                     (dict(t=(4097, 0.0)), ALIGN), (dict(k=(4097, 0)), ALIGN), (dict(p=(4097, 0.0)), ALIGN),
                     (dict(m=(4097, 0.0)), ALIGN)):
        assert call(**kw) == code, kw


def test_wrappers_refuse_cpu_tensors():
    import custom_ecc_cuda as ops
    pool = torch.zeros(4, 2, 16, 128, dtype=torch.uint8)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 128, dtype=torch.float16)
    for call in (lambda: ops.compress_pair_paged(x, x, pool, pool, table, n),
                 lambda: ops.dequantize_paged(pool, pool, table, n, 4),
                 lambda: ops.decode_attention_paged(x, pool, pool, table, n),
                 lambda: ops.evict_paged(pool, pool, table, n, torch.zeros(1, 2, 32), table, 8),
                 lambda: ops.sample_tokens(torch.zeros(2, 8), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_paged_cache_refuses_cpu_device():
    import types
    from custom_kv import PagedErrorCorrectedCache
    cfg = types.SimpleNamespace(num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2, hidden_size=256)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedErrorCorrectedCache(cfg, device="cpu")


@pytest.mark.parametrize("call,arg", [("crop", 3), ("reorder_cache", torch.tensor([1, 0])), ("batch_repeat_interleave", 2),
                                      ("batch_select_indices", torch.tensor([1]))])
def test_paged_cache_refuses_what_it_cannot_do(call, arg):
    """transformers' Cache does these to its layers; this cache has none, so they would pass without doing anything."""
    from custom_kv import PagedErrorCorrectedCache
    cache = object.__new__(PagedErrorCorrectedCache)
    cache.layers = []
    with pytest.raises(RuntimeError, match="PagedErrorCorrectedCache"):
        getattr(cache, call)(arg)


def test_written_weights_must_not_overlap():
    import custom_ecc_cuda as ops
    cpu = torch.device("cpu")

    def look(t, B, H, **kw):
        return ops._weights_like(t, "weights", B, H, 32, cpu, **kw)

    whole = torch.zeros(3, 2, 40)
    for t in (whole, whole[:, :, 4:], whole[:2], whole.transpose(0, 1).contiguous().transpose(0, 1), whole[:, :1], whole[:1],
              torch.zeros(6, 2, 40)[::2], torch.zeros(1, 1, 32).expand(1, 1, 32)):
        assert look(t, t.shape[0], t.shape[1]) == (t.data_ptr(), t.stride(0), t.stride(1))
    for t in (torch.zeros(1, 2, 40).expand(3, 2, 40), torch.zeros(3, 1, 40).expand(3, 2, 40),
              torch.zeros(1, 1, 40).expand(3, 1, 40), torch.zeros(200).as_strided((3, 2, 40), (40, 39, 1)),
              torch.zeros(300).as_strided((3, 2, 40), (79, 40, 1)), torch.zeros(300).as_strided((3, 2, 40), (40, 119, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            look(t, t.shape[0], t.shape[1])
        look(t, t.shape[0], t.shape[1], written=False)  # to be read only


def test_arguments_as_words(lib):
    """ecc_call gives what the typed entry points give, up to the first device call."""
    import struct
    call = lib.ecc_call
    call.argtypes = [ctypes.c_int, ctypes.c_void_p]
    pg = (4096, 4, 4, 16, 10)

    def words(layout, *v):
        return struct.pack("=" + layout, *v)

    def compress(x=4096, B=1, L=4, pages=pg, mode=1):
        return call(0, words("26q", x, 0, 0, 128, 4096, 32, 16, 0, 0, 0, 128, 0, 32, 16, B, 1, L, *pages, 4096, 0, mode, 0))

    def dequantize(x=4096, B=1, n=4, pages=pg, mode=0):
        return call(1, words("19q", x, 32, 16, 4096, 0, 0, 0, 0, B, 1, n, *pages, 4096, mode, 0))

    def decode(q=4096, B=1, hq=2, scale=0.0, sinks=0, flags=0, pages=pg, room=1 << 30):
        return call(2, words("21qd4q", q, 4096, 4096, 32, 16, *pages, 4096, 4096, 0, 0, 0, 0, 4096, room, B, hq, 1, scale,
                             0, sinks, flags, 0))

    def evict(k=4096, B=1, budget=8, recent=0, rec=128, room=1 << 20, pages=pg):
        return call(3, words("32q", k, 4096, 32, 16, *pages, 4096, 4096, 64, 64, 8192, *pages[1:], 4096, 64, 64, 64, 4096, B,
                             1, budget, 0, recent, rec, 4096, room, 0))

    def sample(x=4096, dtype=0, B=1, V=8, t0=1.0, k0=0, p0=1.0, m0=0.0):
        return call(4, words("7qd3qdqd3q", x, 8, dtype, B, V, 4096, 0, t0, 0, k0, 0, p0, 0, m0, 4096, 0, 0))

    assert compress(B=0) == OK and dequantize(B=0) == OK and decode(B=0) == OK and evict(B=0) == OK and sample(B=0) == OK
    for got, code in ((compress(x=0), NULL), (compress(L=-1), SHAPE), (compress(mode=4), SHAPE), (compress(x=4104), ALIGN),
                      (compress(B=1 << 32), SHAPE), (compress(pages=(4096, 4, 4, 24, 10)), SHAPE),
                      (dequantize(x=0), NULL), (dequantize(n=-1), SHAPE), (dequantize(mode=4), SHAPE),
                      (dequantize(x=4104), ALIGN), (dequantize(pages=(4098, 4, 4, 16, 10)), ALIGN),
                      (decode(q=0), NULL), (decode(q=4104), ALIGN), (decode(hq=9), SHAPE), (decode(scale=float("nan")), PARAM),
                      (decode(scale=float("inf")), PARAM), (decode(scale=1e300), PARAM), (decode(sinks=1), SHAPE),
                      (decode(flags=64), SHAPE), (decode(hq=2 + (1 << 32)), SHAPE), (decode(pages=(0, 4, 4, 16, 10)), NULL),
                      (evict(k=0), NULL), (evict(recent=9), SHAPE), (evict(rec=64), SHAPE), (evict(room=0), WORKSPACE),
                      (evict(budget=8 - (1 << 32)), SHAPE),
                      (sample(x=0), NULL), (sample(x=4097), ALIGN), (sample(dtype=3), SHAPE), (sample(V=0), SHAPE),
                      (sample(t0=-1.0), PARAM), (sample(k0=-1), PARAM), (sample(k0=1 << 31), SHAPE), (sample(p0=0.0), PARAM),
                      (sample(m0=1.5), PARAM), (call(5, words("q", 0)), SHAPE), (call(0, None), NULL)):
        assert got == code
