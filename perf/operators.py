"""Measured cases of the paged-cache operators and of token sampling.

Each case is one pass of a serving path over an ECC-INT4 cache kept in pages:

* ``append``  a chunk of new K/V goes into the pages of each sequence and the whole context is read back as fp16
              (what a chunked prefill does between two chunks);
* ``decode``  one new token of every sequence attends to its pages, with or without a sliding window and sinks;
* ``weights`` the same, adding up the attention weight that every cached token received;
* ``evict``   each sequence is cut down to a budget of tokens by that weight, into fresh pages;
* ``sample``  the next token of every sequence is drawn from the logits and given uniform numbers.

``own = False`` computes them with elementary torch operations, ``own = True`` with the kernels.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

D = 128
# the 16 Lloyd-Max levels of the block format
LEVELS = [-2.4008, -1.8435, -1.4371, -1.0993, -0.7996, -0.5224, -0.2582, 0.0, 0.2582, 0.5224, 0.7996, 1.0993, 1.4371,
          1.8435, 2.4008, 3.1584]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# --------------------------------------------------------------------------- cases
def _case(kind, name=None, **kw):
    base = {
        "append": dict(B=1, hkv=8, len=1024, new=64, ps=64, rec=128),
        "decode": dict(B=1, hq=32, hkv=8, len=1024, ps=64, rec=128, window=0, sinks=0, ragged=False, empty=False),
        "weights": dict(B=1, hq=32, hkv=8, len=1024, ps=64, rec=128, window=0, sinks=0, ragged=False, empty=False),
        "evict": dict(B=1, hkv=8, len=1024, ps=64, rec=128, budget=512, sinks=4, recent=128, ragged=False),
        "sample": dict(B=1, V=128256, dtype="fp16", top_k=0, top_p=1.0, min_p=0.0, temperature=1.0, mixed=False),
    }[kind]
    c = dict(base, kind=kind, **kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a short chunk of a small model's prompt behind a few cached tokens
        _case("append", "append short chunk", B=1, hkv=2, len=33, new=17, ps=16),
        # a prompt chunk of four sequences at different places of their contexts
        _case("append", "append prompt chunks", B=4, hkv=8, len=8192, new=2048, ps=64),
        # one chat turn, early: the step is latency
        _case("decode", "decode one short", B=1, hq=32, hkv=8, len=517, ps=16),
        # a serving batch with contexts of every length and one slot that is free
        _case("decode", "decode ragged batch", B=32, hq=32, hkv=8, len=16384, ps=64, ragged=True, empty=True),
        # the long-context decode step of the framework's benchmark, in pages
        _case("decode", "decode 8 x 64k", B=8, hq=32, hkv=8, len=65531, ps=128),
        # a sliding-window layer without grouped heads, records without their pad sector
        _case("decode", "decode window and sinks", B=16, hq=8, hkv=8, len=32768, ps=32, rec=96, window=4096, sinks=4,
              ragged=True),
        # weights of a model with eight query heads to a cached one, pages that end inside a tile
        _case("weights", "weights one 4k", B=1, hq=16, hkv=2, len=4097, ps=48),
        # the step that collects weights in a batch of long contexts
        _case("weights", "weights batch 32k", B=8, hq=32, hkv=8, len=32768, ps=64, ragged=True),
        # one sequence is cut down
        _case("evict", "evict one 5k to 1k", B=1, hkv=8, len=5001, ps=16, budget=1024, sinks=4, recent=256),
        # a batch at its memory limit is halved
        _case("evict", "evict batch 32k to 16k", B=8, hkv=8, len=32768, ps=64, budget=16384, sinks=16, recent=2048),
        # one chat with the usual settings
        _case("sample", "sample one", B=1, dtype="fp16", top_k=50, top_p=0.9, temperature=0.7),
        # a serving batch, each sequence with settings of its own, most without top-k
        _case("sample", "sample batch", B=64, dtype="bf16", mixed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "weights", "evict", "sample"])
    ps = rng.choice([16, 32, 48, 64, 128, 256])
    rec = rng.choice([128, 128, 96])
    if kind == "append":
        B = _log_int(rng, 1, 16)
        total = 40000 // B
        length = _log_int(rng, 8, max(9, min(16384, total)))
        return _case(kind, B=B, hkv=rng.choice([1, 2, 4, 8]), len=length, new=_log_int(rng, 1, 2100), ps=ps, rec=rec)
    if kind in ("decode", "weights"):
        B = _log_int(rng, 1, 64)
        hkv = rng.choice([1, 2, 4, 8])
        g = rng.choice([1, 2, 3, 4, 5, 7, 8])
        most = 4_000_000 if kind == "decode" else 1_600_000
        length = _log_int(rng, 1, max(2, min(131072, most // (B * hkv))))
        window = rng.choice([0, 0, _log_int(rng, 1, 8192)])
        return _case(kind, B=B, hq=g * hkv, hkv=hkv, len=length, ps=ps, rec=rec, window=window,
                     sinks=rng.choice([0, 1, 4, 70]) if window else 0, ragged=rng.random() < 0.6,
                     empty=B > 1 and rng.random() < 0.3)
    if kind == "evict":
        B = _log_int(rng, 1, 16)
        hkv = rng.choice([1, 2, 4, 8])
        length = _log_int(rng, 64, max(65, min(65536, 2_000_000 // (B * hkv))))
        sinks = rng.choice([0, 1, 4, 16])
        budget = max(sinks + 1, int(length * rng.uniform(0.1, 0.95)))
        recent = rng.randint(0, budget - sinks)
        return _case(kind, B=B, hkv=hkv, len=length, ps=ps, rec=rec, budget=budget, sinks=sinks, recent=recent,
                     ragged=rng.random() < 0.5)
    B = _log_int(rng, 1, 64)
    return _case(kind, B=B, V=_log_int(rng, 1000, 131072), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                 top_k=rng.choice([0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5]),
                 min_p=rng.choice([0.0, 0.0, 0.05]), temperature=rng.choice([0.0, 0.6, 0.7, 1.0, 1.3]),
                 mixed=rng.random() < 0.3)


def _lens(c):
    """Context length of each sequence: all alike, or spread from the longest down to a quarter of it at odd sizes."""
    n, B = c["len"], c["B"]
    lens = [max(1, n - (3 * n * b) // (4 * B) - b % 7) for b in range(B)] if c.get("ragged") else [n] * B
    if c.get("empty"):
        lens[-1] = 0
    return lens


def _new_lens(c):
    """Tokens that each sequence appends: the first the whole chunk, the others less."""
    return [max(1, c["new"] - (c["new"] * b) // (2 * c["B"])) for b in range(c["B"])]


def _old_lens(c):
    """Tokens that each sequence holds before the append."""
    return [max(0, c["len"] - (c["len"] * b) // (2 * c["B"])) for b in range(c["B"])]


def _pages(n, ps):
    return -(-n // ps)


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _blocks(shape, rec, g, spread=1.0):
    """Records as the quantiser leaves them for normal data: levels with the frequencies of a normal variable, random
    residual signs, a scale per vector (one in a hundred three times larger), a small zero point, alpha = 0.11 scale."""
    dev = "cuda"
    lv = torch.tensor(LEVELS, dtype=torch.float64)
    cdf = 0.5 * (1 + torch.erf((lv[1:] + lv[:-1]) / 2 / math.sqrt(2)))
    nib = torch.bucketize((torch.arange(256, dtype=torch.float64) + 0.5) / 256, cdf)
    tab = (nib[None, :] | (nib[:, None] << 4)).reshape(-1).to(torch.uint8).to(dev)
    pool = torch.zeros(*shape, rec, dtype=torch.uint8, device=dev)
    pool[..., :64] = tab[torch.randint(0, 65536, (*shape, 64), generator=g, device=dev, dtype=torch.int32)]
    pool[..., 64:80] = torch.randint(0, 256, (*shape, 16), generator=g, device=dev, dtype=torch.uint8)
    r = torch.rand(*shape, 3, generator=g, device=dev)
    scale = spread * (0.6 + 0.8 * r[..., 0]) * torch.where(r[..., 1] < 0.01, 3.0, 1.0)
    meta = torch.stack([scale, 0.2 * (r[..., 2] - 0.5), 0.11 * scale], -1).to(torch.float16)
    pool[..., 80:86] = meta.view(torch.uint8)
    return pool


def _table(counts, width, free, g):
    """A page table whose rows hold `counts` pages each out of a shuffled pool (-1 behind them), from page `free` on."""
    total = sum(counts)
    perm = (torch.randperm(total, generator=g, device="cuda") + free).tolist() if total else []
    rows, at = [], 0
    for n in counts:
        rows.append(perm[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda").reshape(len(counts), width)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, g, kind = case, _gen(seed), case["kind"]
    if kind == "sample":
        B, V = c["B"], c["V"]
        x = torch.randn(B, V, generator=g, device="cuda") * 1.5
        # a few dozen likely tokens on top of a long tail, as a language model's logits have
        top = torch.randint(0, V, (B, 48), generator=g, device="cuda")
        x.scatter_(1, top, 4 + 6 * torch.rand(B, 48, generator=g, device="cuda"))
        x[:, V // 2:V // 2 + 5] = -math.inf  # tokens that a grammar or a ban list rules out
        s = {"kind": kind, "logits": x.to(DTYPES[c["dtype"]]), "u": torch.rand(B, generator=g, device="cuda")}
        if c["mixed"]:
            i = torch.arange(B, device="cuda")
            s["temperature"] = torch.tensor([0.7, 1.0, 0.0, 1.3], device="cuda")[i % 4]
            s["top_k"] = _i32([0, 0, 0, 40, 0])[i % 5]
            s["top_p"] = torch.tensor([0.9, 0.95, 1.0], device="cuda")[i % 3]
            s["min_p"] = torch.tensor([0.0, 0.0, 0.02, 0.0, 0.1], device="cuda")[i % 5]
        else:
            s.update(temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
        return s
    B, hkv, ps, rec = c["B"], c["hkv"], c["ps"], c["rec"]
    s = {"kind": kind}
    if kind == "append":
        old, new = _old_lens(c), _new_lens(c)
        lens = [a + b for a, b in zip(old, new)]
        width = _pages(max(lens), ps)
        s["table"] = _table([_pages(n, ps) for n in lens], width, 1, g)  # page 0 is nobody's
        n_pages = 1 + sum(_pages(n, ps) for n in lens)
        s["pos"], s["new_lens"], s["lens"], s["max_len"] = _i32(old), _i32(new), _i32(lens), max(lens)
        # projections come as [B, L, H, D]: the cache gets them transposed; a few channels are outliers
        amp = torch.where(torch.rand(hkv, 1, D, generator=g, device="cuda") < 0.03, 6.0, 1.0)
        for n in ("k", "v"):
            x = torch.randn(B, c["new"], hkv, D, generator=g, device="cuda").transpose(1, 2)
            s[n] = (x * amp if n == "k" else x).to(torch.float16)
            s[n + "_pool"] = _blocks((n_pages, hkv, ps), rec, g)
        return s
    lens = _lens(c)
    width = max(1, _pages(max(lens), ps))
    counts = [_pages(n, ps) for n in lens]
    out_pages = _pages(c["budget"], ps) * B if kind == "evict" else 0
    s["table"], s["lens"] = _table(counts, width, out_pages, g), _i32(lens)
    n_pages = max(1, sum(counts) + out_pages)
    s["k_pool"], s["v_pool"] = (_blocks((n_pages, hkv, ps), rec, g, a) for a in (1.5, 1.0))
    cap = width * ps
    if kind in ("decode", "weights"):
        s["q"] = torch.randn(B, c["hq"], 1, D, generator=g, device="cuda").to(torch.float16)
        s["window"], s["sinks"] = c["window"], c["sinks"]
        # the decode cases take the model's query, the others one that is rotated already
        s["rotate"] = kind == "decode"
    if kind in ("weights", "evict"):
        # a heavy tail, as attention leaves it, and many tokens that got nothing
        r = torch.rand(B, hkv, cap, generator=g, device="cuda")
        w = torch.where(r < 0.1, 0.0, (r - 0.1) ** 8)
        s["weights"] = torch.where(torch.arange(cap, device="cuda") < s["lens"][:, None, None], w, 0.0)
    if kind == "evict":
        s["out_table"] = torch.randperm(out_pages, generator=g, device="cuda").to(torch.int32).reshape(B, -1)
        s["budget"], s["sinks"], s["recent"] = c["budget"], c["sinks"], c["recent"]
    return s


# --------------------------------------------------------------------------- plain forms
@functools.lru_cache(None)
def _hadamard():
    e = torch.tensor([[1.0, 1.0], [1.0, -1.0]])
    return (functools.reduce(torch.kron, [e] * 7) / math.sqrt(D)).to("cuda")


@functools.lru_cache(None)
def _levels():
    return torch.tensor(LEVELS, dtype=torch.float32, device="cuda")


def _unpack(blocks):
    """[..., rec] u8 -> [..., 128] fp32: (C[q] scale + zero) + alpha s."""
    codes = blocks[..., :64]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int32)
    bits = (blocks[..., 64:80, None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
    meta = blocks[..., 80:86].contiguous().view(torch.float16).float()
    s = bits.flatten(-2).float() * 2 - 1
    return (_levels()[q] * meta[..., 0:1] + meta[..., 1:2]) + meta[..., 2:3] * s


def _gather(pool, table):
    """The records of every sequence in order, [B, H, tokens, rec]; pages of the table that are unset read page 0."""
    x = pool[table.clamp(min=0)]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _slots(table, pos, ps):
    """(page, slot) of token positions pos [B, n]."""
    return table.gather(1, (pos // ps).clamp(max=table.shape[1] - 1).long()).long(), (pos % ps).long()


def _compress(x, rec):
    """fp16 vectors [..., 128] -> records: rotation, 16-level codes of the vector's own statistics, residual signs. The
    sums run in the order of the format's definition (four accumulators of eight lanes), all in fp32 but the deviation."""
    v = x.float()
    for s in (1, 2, 4, 8, 16, 32, 64):
        a, b = v.unflatten(-1, (-1, 2, s)).unbind(-2)
        v = torch.stack([a + b, a - b], -2).flatten(-3)
    v = v / torch.tensor(math.sqrt(D), dtype=torch.float32, device="cuda")

    def total(t):
        t = t.unflatten(-1, (4, 4, 8))
        acc = ((t[..., 0, :, :] + t[..., 1, :, :]) + t[..., 2, :, :]) + t[..., 3, :, :]
        lane = ((acc[..., 0, :] + acc[..., 1, :]) + acc[..., 2, :]) + acc[..., 3, :]
        a, b, c, d, e, f, g, h = lane.unbind(-1)
        return (((((((a + b) + c) + d) + e) + f) + g) + h)[..., None]

    zero = total(v) / D
    dev = (v.double() - zero.double()).square().sum(-1, keepdim=True)
    scale = ((dev / (D - 1)).sqrt().float().double() + 1e-8).float()
    u = (v - zero) / scale
    lv = _levels()
    q = torch.bucketize(u, (lv[1:] + lv[:-1]) / 2)  # on a border the lower level, as the first of two equal distances
    res = v - (lv[q] * scale + zero)
    alpha = total(res.abs()) / D
    out = torch.zeros(*v.shape[:-1], rec, dtype=torch.uint8, device="cuda")
    out[..., :64] = (q[..., 0::2] | (q[..., 1::2] << 4)).to(torch.uint8)
    bit = (res >= 0).unflatten(-1, (16, 8)).to(torch.int32) << torch.arange(8, device="cuda", dtype=torch.int32)
    out[..., 64:80] = bit.sum(-1).to(torch.uint8)
    out[..., 80:86] = torch.cat([scale, zero, alpha], -1).to(torch.float16).view(torch.uint8)
    return out


def _append(s):
    table, ps, rec = s["table"], s["k_pool"].shape[2], s["k_pool"].shape[3]
    B, H, n, _ = s["k"].shape
    i = torch.arange(n, device="cuda")
    page, slot = _slots(table, s["pos"][:, None] + i, ps)
    page = torch.where(i < s["new_lens"][:, None], page, 0)  # what a sequence does not append lands on nobody's page
    h = torch.arange(H, device="cuda")[None, :, None]
    t = torch.arange(s["max_len"], device="cuda")
    live = (t < s["lens"][:, None])[:, None, :, None]
    out = []
    for x, pool in ((s["k"], s["k_pool"]), (s["v"], s["v_pool"])):
        pool[page[:, None, :], h, slot[:, None, :]] = _compress(x, rec)
        y = _unpack(_gather(pool, table)[:, :, :s["max_len"]]) @ _hadamard()
        out.append(torch.where(live, y, 0.0).to(torch.float16))
    return {"k": out[0], "v": out[1]}


def _attend(s):
    """(softmax weights [B, Hkv, G, T], output [B, Hq, 1, 128]) in fp32."""
    k = _unpack(_gather(s["k_pool"], s["table"]))
    B, H, T, _ = k.shape
    q = s["q"].float().view(B, H, -1, D)
    if s["rotate"]:
        q = q @ _hadamard()
    sc = (q @ k.transpose(-1, -2)) / math.sqrt(D)
    del k
    t, n = torch.arange(T, device="cuda"), s["lens"][:, None]
    see = t < n
    if s["window"]:
        see = see & ((t >= n - s["window"]) | (t < s["sinks"]))
    sc = torch.where(see[:, None, None, :], sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = p @ _unpack(_gather(s["v_pool"], s["table"]))
    if s["rotate"]:
        o = o @ _hadamard()
    return p, o.reshape(B, -1, 1, D)


def _evict(s):
    kp, vp, w, ps = s["k_pool"], s["v_pool"], s["weights"], s["k_pool"].shape[2]
    B, H, cap = w.shape
    n = s["budget"]
    pad = max(0, n - cap)
    t, L = torch.arange(cap + pad, device="cuda"), s["lens"][:, None, None]
    wide = torch.nn.functional.pad(w, (0, pad))
    safe = (t < s["sinks"]) | (t >= L - s["recent"]) | (L <= n)
    key = torch.where(t < L, torch.where(safe, math.inf, wide), -math.inf)
    at = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :n].sort(-1).values
    live = torch.arange(n, device="cuda") < L.clamp(max=n)
    kept = torch.where(live, at, -1).to(torch.int32)
    out_w = torch.zeros_like(w)
    out_w[..., :min(n, cap)] = torch.where(live, wide.gather(-1, at), 0.0)[..., :cap]
    dst_page, dst_slot = _slots(s["out_table"], torch.arange(n, device="cuda").expand(B, n), ps)
    src_page, src_slot = _slots(s["table"], at.clamp(max=cap - 1).flatten(1), ps)
    src_page, src_slot = src_page.view(B, H, n).clamp(min=0), src_slot.view(B, H, n)
    h = torch.arange(H, device="cuda")[None, :, None]
    for pool in (kp, vp):
        old = pool[dst_page[:, None, :], h, dst_slot[:, None, :]]
        pool[dst_page[:, None, :], h, dst_slot[:, None, :]] = torch.where(live[..., None], pool[src_page, h, src_slot], old)
    return {"kept": kept, "weights": out_w, "k": kp, "v": vp}


def _column(v, B):
    """A setting, one for all or one for each sequence, as [B, 1]."""
    return (v if isinstance(v, torch.Tensor) else torch.full((B,), v, dtype=torch.float32, device="cuda")).double()[:, None]


def _sample(s):
    """In 64 bits: the drawn token hangs on sums that stand next to the given numbers."""
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    B, V = x.shape
    T, k, p, mp = (_column(s[n], B) for n in ("temperature", "top_k", "top_p", "min_p"))
    xs, at = torch.sort(x, dim=-1, descending=True, stable=True)
    top = xs[:, :1]
    w = torch.exp(torch.where(xs == top, 0.0, (xs - top) / torch.where(T > 0, T, 1.0)))
    rank = torch.arange(V, device="cuda")
    w = torch.where((rank < torch.where(k > 0, k, V)) & ((T > 0) | (rank == 0)), w, 0.0)
    before = w.cumsum(-1) - w
    w = torch.where((before < p * w.sum(-1, keepdim=True)) & (w >= mp) | (rank == 0), w, 0.0)
    mass = torch.zeros_like(w).scatter_(1, at, w)
    cum = mass.cumsum(-1)
    total = cum[:, -1:]
    token = (cum <= s["u"].double()[:, None] * total).sum(-1).clamp(max=V - 1)
    logp = torch.log(mass.gather(1, token[:, None]) / total)[:, 0]
    none = top[:, 0] == -math.inf
    return {"token": torch.where(none, -1, token), "logprob": torch.where(none, -math.inf, logp).float()}


# --------------------------------------------------------------------------- the framework's calls
def _ops():
    path = os.path.join(os.getcwd(), "ecc-kv-cache_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import custom_ecc_cuda
    return custom_ecc_cuda


def run(state):
    s, kind = state, state["kind"]
    if kind == "append":
        if own:
            ops = _ops()
            ops.compress_pair_paged(s["k"], s["v"], s["k_pool"], s["v_pool"], s["table"], s["pos"], new_lens=s["new_lens"])
            k, v = ops.dequantize_paged(s["k_pool"], s["v_pool"], s["table"], s["lens"], s["max_len"])
            return {"k": k, "v": v}
        return _append(s)
    if kind == "decode":
        if own:
            return _ops().decode_attention_paged(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"],
                                                 window=s["window"], sinks=s["sinks"], rotate_q=True, unrotate_out=True)
        return _attend(s)[1].to(torch.float16)
    if kind == "weights":
        w = s["weights"].clone()  # a cache adds to its own; here every pass starts from the same
        if own:
            o = _ops().decode_attention_paged(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"],
                                              window=s["window"], sinks=s["sinks"], weights=w)
            return {"out": o, "weights": w}
        p, o = _attend(s)
        return {"out": o.to(torch.float16), "weights": w.add_(p.sum(2))}
    if kind == "evict":
        if own:
            w, kept = _ops().evict_paged(s["k_pool"], s["v_pool"], s["table"], s["lens"], s["weights"], s["out_table"],
                                         budget=s["budget"], sinks=s["sinks"], recent=s["recent"])
            return {"kept": kept, "weights": w, "k": s["k_pool"], "v": s["v_pool"]}
        return _evict(s)
    if own:
        token, logprob = _ops().sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                              top_p=s["top_p"], min_p=s["min_p"], return_logprobs=True)
        return {"token": token, "logprob": logprob}
    return _sample(s)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, kind = case, case["kind"]
    if kind == "sample":
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": c["B"] * (c["V"] * size + 16), "flops": 4 * c["B"] * c["V"]}
    hkv, rec = c["hkv"], c["rec"]
    content = 96  # the 32-byte sectors of a record that hold something
    if kind == "append":
        new, every = sum(_new_lens(c)), sum(_new_lens(c)) + sum(_old_lens(c))
        rows = c["B"] * (max(a + b for a, b in zip(_old_lens(c), _new_lens(c))))
        return {"bytes": 2 * hkv * (new * (2 * D + rec) + (every - new) * content + rows * 2 * D),
                "flops": 2 * hkv * (new + every) * 7 * D}
    lens = _lens(c)
    if kind == "evict":
        kept = sum(min(n, c["budget"]) for n in lens)
        rows = c["B"] * _pages(max(lens), c["ps"]) * c["ps"]
        return {"bytes": hkv * (sum(lens) * 4 + kept * 2 * (content + rec) + rows * 4 + c["B"] * c["budget"] * 4), "flops": 0}
    seen = sum(min(n, c["window"] + min(c["sinks"], max(0, n - c["window"]))) if c["window"] else n for n in lens)
    q = c["B"] * c["hq"] * 2 * D * 2
    extra = 8 * hkv * seen if kind == "weights" else 0
    return {"bytes": seen * hkv * 2 * content + q + extra, "flops": 4 * seen * c["hq"] * D}


# --------------------------------------------------------------------------- from the definitions, in 64 bits
def _wht64(x):
    """The normalised transform of the last axis by butterflies."""
    for k in range(7):
        y = x.unflatten(-1, (D >> (k + 1), 2, 1 << k))
        x = torch.stack([y.select(-2, 0) + y.select(-2, 1), y.select(-2, 0) - y.select(-2, 1)], -2).flatten(-3)
    return x / 128.0 ** 0.5


def _values64(r):
    """Records [n, rec] -> values [n, 128], field by field."""
    lv = torch.tensor(LEVELS, dtype=torch.float64).float().double().cuda()
    v = torch.empty(r.shape[0], D, dtype=torch.float64, device="cuda")
    v[:, 0::2] = lv[(r[:, :64] % 16).long()]
    v[:, 1::2] = lv[torch.div(r[:, :64], 16, rounding_mode="floor").long()]
    f = r[:, 80:86].contiguous().view(torch.float16).double()
    v = v * f[:, :1] + f[:, 1:2]
    for j in range(8):
        on = torch.div(r[:, 64:80], 1 << j, rounding_mode="floor") % 2 == 1
        v[:, j::8] += torch.where(on, f[:, 2:], -f[:, 2:])
    return v


def _row64(pool, table, b, h, n):
    ps = pool.shape[2]
    return pool[table[b, :_pages(n, ps)].long(), h].reshape(-1, pool.shape[3])[:n]


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "evict":
        w = s["weights"].double().cpu()
        out = torch.zeros_like(w)
        for b, n in enumerate(s["lens"].tolist()):
            lo, hi = case["sinks"], n - case["recent"]
            for h in range(case["hkv"]):
                keep = list(range(n))
                if n > case["budget"]:
                    v = w[b, h, :n].tolist()
                    mid = sorted(range(lo, hi), key=lambda t: (-v[t], t))[:case["budget"] - lo - case["recent"]]
                    keep = list(range(lo)) + sorted(mid) + list(range(hi, n))
                out[b, h, :len(keep)] = w[b, h, keep]
        return {"kept": None, "weights": out, "k": None, "v": None}
    if kind == "sample":
        x = s["logits"].double().cpu().numpy()
        B, V = x.shape
        col = lambda v: (v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, np.float32(v), np.float64))  # noqa: E731
        T, K, P, M, U = (col(v) for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["u"]))
        token, logp = np.empty(B, np.int64), np.empty(B, np.float64)
        for b in range(B):
            best = x[b].max()
            if T[b] == 0:
                token[b], logp[b] = int(x[b].argmax()), 0.0
                continue
            order = np.lexsort((np.arange(V), -x[b]))
            order = order[:int(K[b])] if K[b] > 0 else order
            e = np.exp((x[b][order] - best) / T[b])
            e = e[:max(1, int(np.searchsorted(np.concatenate([[0.0], np.cumsum(e)[:-1]]), P[b] * e.sum(), "left")))]
            e = e[:max(1, int((e >= M[b]).sum()))]
            ids = np.sort(order[:len(e)])
            cdf = np.cumsum(np.exp((x[b][ids] - best) / T[b]))
            j = min(int(np.searchsorted(cdf, U[b] * cdf[-1], "right")), len(ids) - 1)
            token[b], logp[b] = ids[j], (x[b][ids[j]] - best) / T[b] - math.log(cdf[-1])
        return {"token": None, "logprob": torch.from_numpy(logp)}
    if kind == "append":
        # the codes are a choice that the format fixes in 32 bits; what is read back of them is a number
        _append(s)
        B, H = case["B"], case["hkv"]
        out = {}
        for n in ("k", "v"):
            y = torch.zeros(B, H, s["max_len"], D, dtype=torch.float64, device="cuda")
            for b, size in enumerate(s["lens"].tolist()):
                for h in range(H):
                    y[b, h, :size] = _wht64(_values64(_row64(s[n + "_pool"], s["table"], b, h, size)))
            out[n] = y
        return out
    B, H, hq = case["B"], case["hkv"], case["hq"]
    G = hq // H
    o = torch.zeros(B, hq, 1, D, dtype=torch.float64, device="cuda")
    w = s["weights"].double() if kind == "weights" else None
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        sink = min(case["sinks"], first)
        for h in range(H if n else 0):
            take = torch.cat([torch.arange(sink), torch.arange(first, n)]).cuda()
            k, v = (_values64(_row64(s[x + "_pool"], s["table"], b, h, n)[take]) for x in "kv")
            q = s["q"][b, h * G:(h + 1) * G, 0].double()
            q = _wht64(q) if s["rotate"] else q
            p = torch.softmax(q @ k.T / 128.0 ** 0.5, -1)
            y = p @ v
            o[b, h * G:(h + 1) * G, 0] = _wht64(y) if s["rotate"] else y
            if w is not None:
                w[b, h, take] += p.sum(0)
    return o if w is None else {"out": o, "weights": w}
