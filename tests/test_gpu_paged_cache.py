"""The paged operators together, as a serving loop uses them: ragged appends,
decode steps that collect weights, eviction, reuse of freed pages, sampling in
a recorded step; and PagedErrorCorrectedCache under transformers."""
import types

import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def config(layers=2, hq=4, hkv=2):
    return types.SimpleNamespace(num_hidden_layers=layers, num_attention_heads=hq, num_key_value_heads=hkv,
                                 hidden_size=128 * hq, head_dim=128)


def states(cache, B, L, g):
    shape = (B, L, cache.num_heads, 128)
    return [tuple(torch.randn(shape, generator=g, device="cuda").half().transpose(1, 2) for _ in range(2))
            for _ in range(len(cache))]


def check_step(cache, g, expect_w):
    """One decode step of every layer against the plain implementation on the cache's own blocks; `expect_w`: the
    weights so far, 64-bit, and their bounds."""
    B, hq = cache.batch_size, cache.num_attention_heads
    for layer in range(len(cache)):
        q = torch.randn(B, hq, 1, 128, generator=g, device="cuda").half()
        out = cache.decode_attention(q, layer)
        kp, vp = (p.cpu().numpy() for p in cache.layer_pools(layer))
        o, tol, _, _, w, w_tol = R.attend(q[:, :, 0].cpu().numpy(), kp, vp, cache.block_table.cpu().numpy(), cache.lengths,
                                          cache.window, cache.sinks, rotate=True)
        assert (np.abs(out[:, :, 0].cpu().numpy() - o) <= tol).all()
        expect_w[layer][0] += w
        expect_w[layer][1] += w_tol + 2.0 ** -24 * expect_w[layer][0]
        if cache.weights is not None:
            assert (np.abs(cache.weights[layer].cpu().numpy() - expect_w[layer][0]) <= expect_w[layer][1]).all()


@pytest.mark.parametrize("window,sinks,block_bytes", [(0, 0, 128), (40, 4, 96)])
def test_serving_loop(cuda_device, window, sinks, block_bytes):
    import custom_ecc_cuda as ops
    from custom_kv import PagedErrorCorrectedCache
    ops.device_status(reset=True)
    g = torch.Generator(device="cuda").manual_seed(window)
    cache = PagedErrorCorrectedCache(config(), batch_size=3, max_cache_len=256, num_pages=40, page_size=16,
                                     window=window, sinks=sinks, collect_weights=True, block_bytes=block_bytes)
    zero = np.zeros((3, 2, 256))
    want_w = [[zero.copy(), zero.copy()] for _ in range(2)]

    def append(new):
        for layer, (k, v) in enumerate(states(cache, 3, max(new), g)):
            cache.append(k, v, layer, new_lens=new)

    append([150, 33, 0])          # prompts of two sequences; the third slot is empty
    assert cache.lengths == [150, 33, 0] and cache.free_pages == 40 - 10 - 3
    check_step(cache, g, want_w)
    append([1, 1, 70])            # a step of two, the prompt of the third
    check_step(cache, g, want_w)
    for _ in range(3):
        append([1, 1, 1])
        check_step(cache, g, want_w)

    before = [(cache.weights[i].clone(), [x.clone() for x in cache.layer_pools(i)], cache.block_table.clone()) for i in
              range(2)]
    lens = cache.lengths
    assert cache.evict(60, sinks=4, recent=20) == [0, 2]
    assert cache.lengths == [60, 37, 60] and cache.get_seq_length() == 154
    assert cache.free_pages == 40 - 4 - 3 - 4
    for layer in range(2):
        w, pools, table = before[layer]
        for b in (0, 2):
            for h in range(2):
                row = w[b, h].cpu().numpy()
                mid = sorted(range(4, lens[b] - 20), key=lambda t: (-row[t], t))[:36]
                ids = list(range(4)) + sorted(mid) + list(range(lens[b] - 20, lens[b]))
                assert np.array_equal(cache.weights[layer, b, h].cpu().numpy()[:60], row[ids])
                assert not cache.weights[layer, b, h, 60:].any()
                for old, new in zip(pools, cache.layer_pools(layer)):
                    a = R.sequence(old.cpu().numpy(), table[b].cpu().numpy(), h, lens[b])[ids]
                    z = R.sequence(new.cpu().numpy(), cache.block_table[b].cpu().numpy(), h, 60)
                    assert np.array_equal(a, z)
                want_w[layer][0][b, h] = 0
                want_w[layer][0][b, h, :60] = row[ids]
                want_w[layer][1][b, h] = 0
    for _ in range(2):
        append([1, 1, 1])
        check_step(cache, g, want_w)
    cache.release([1])
    for layer in range(2):
        want_w[layer][0][1] = 0
        want_w[layer][1][1] = 0
    append([1, 90, 1])            # a new sequence in the freed slot
    check_step(cache, g, want_w)
    assert cache.lengths == [63, 90, 63]
    cache.release()
    assert cache.free_pages == 40 and cache.get_seq_length() == 0
    assert ops.device_status(reset=True) == 0


def test_context_reads_back_what_was_appended(cuda_device):
    from custom_kv import PagedErrorCorrectedCache
    for rotate in (True, False):
        cache = PagedErrorCorrectedCache(config(1), batch_size=2, max_cache_len=64, page_size=16, rotate_values=rotate)
        g = torch.Generator(device="cuda").manual_seed(1)
        (k, v), = states(cache, 2, 40, g)
        cache.append(k, v, 0, new_lens=[40, 9])
        for x, y in zip((k, v), cache.context(0)):
            assert y.shape == (2, 2, 40, 128) and not y[1, :, 9:].any()
            # 16 levels for normal data leave a tenth of the norm
            for b, n in ((0, 40), (1, 9)):
                assert (x[b, :, :n] - y[b, :, :n]).float().norm() < 0.2 * x[b, :, :n].float().norm()


def test_cache_refusals(cuda_device):
    from custom_kv import PagedErrorCorrectedCache
    for kw in (dict(page_size=24), dict(page_size=0), dict(block_bytes=64), dict(sinks=4), dict(num_pages=0),
               dict(device="cpu")):
        with pytest.raises(RuntimeError):
            PagedErrorCorrectedCache(config(), **{**dict(batch_size=1, max_cache_len=64), **kw})
    with pytest.raises(RuntimeError):
        PagedErrorCorrectedCache(config(hq=18, hkv=2))
    cache = PagedErrorCorrectedCache(config(1), batch_size=2, max_cache_len=64, num_pages=5, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    (k, v), = states(cache, 2, 40, g)
    with pytest.raises(RuntimeError, match="out of pages"):
        cache.append(k, v, 0)
    assert cache.free_pages == 5 and cache.lengths == [0, 0]
    for kw in (dict(new_lens=[41, 0]), dict(new_lens=[1]), dict(new_lens=[-1, 0])):
        with pytest.raises(RuntimeError):
            cache.append(k, v, 0, **kw)
    with pytest.raises(RuntimeError, match="overflow"):
        cache.append(torch.cat([k, k], 2), torch.cat([v, v], 2), 0, new_lens=[65, 0])
    cache.append(k, v, 0, new_lens=[40, 20])
    with pytest.raises(RuntimeError, match="collect_weights"):
        cache.evict(8)
    with pytest.raises(RuntimeError, match="one length"):
        cache.update(k[:, :, :2], v[:, :, :2], 0)
    mask = torch.ones(2, 1, 1, 40, dtype=torch.bool, device="cuda")
    q = torch.zeros(2, 4, 1, 128, dtype=torch.float16, device="cuda")
    cache.decode_attention(q, 0, attn_mask=mask)
    cache.append(k[:, :, :1], v[:, :, :1], 0)
    mask[0, ..., 0] = False
    with pytest.raises(RuntimeError, match="padding"):
        cache.decode_attention(q, 0, attn_mask=mask)


@pytest.mark.parametrize("rotate", [True, False])
def test_refused_append_leaves_the_cache_as_it_was(cuda_device, rotate):
    """Layer 0's states are refused by the operator (no contiguous rows, a base off 16 bytes, another device): lengths,
    pages and positions stay, and the next append goes where it would have gone."""
    from custom_kv import PagedErrorCorrectedCache
    caches = [PagedErrorCorrectedCache(config(2), batch_size=2, max_cache_len=96, num_pages=9, page_size=16,
                                       rotate_values=rotate) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(5)
    first, second = states(caches[0], 2, 20, g), states(caches[0], 2, 30, g)

    def look(c):
        return (c.lengths, c.free_pages, c.seq_lens.tolist(), c.block_table.tolist(), c._pos.tolist(), c.get_seq_length(),
                [list(p) for p in c._pages], list(c._free), list(c._seen))

    for i, cache in enumerate(caches):
        for step, (new, kv) in enumerate((([20, 7], first), ([9, 30], second))):
            if i == 0:
                k, v = kv[0]
                flat = torch.zeros(k.numel() + 1, dtype=torch.float16, device="cuda")
                off = flat[1:].view(k.shape)
                turned = torch.empty(*k.shape[:2], 128, k.shape[2], dtype=torch.float16, device="cuda").transpose(2, 3)
                was = look(cache)
                for bad in ((off, v), (k, off), (turned, v), (k, turned), (k.cpu(), v), (k, v.cpu())):
                    with pytest.raises(RuntimeError):
                        cache.append(*bad, 0, new_lens=new)
                    assert look(cache) == was
            for layer, (k, v) in enumerate(kv):
                cache.append(k, v, layer, new_lens=new)
                if i == 0 and step == 1 and layer == 0:  # a refusal of a later layer can be mended by a second call
                    with pytest.raises(RuntimeError):
                        cache.append(k.cpu(), v.cpu(), 1, new_lens=new)
    assert look(caches[0]) == look(caches[1])
    assert caches[0].lengths == [29, 37]
    for layer in range(2):
        for x, y in zip(caches[0].context(layer), caches[1].context(layer)):
            assert torch.equal(x, y)


def test_failed_eviction_leaves_the_cache_as_it_was(cuda_device, monkeypatch):
    """An error in the second layer's cut (no memory for its results, say): pages, lengths, weights and blocks of every
    layer stay, and the eviction can be asked for again."""
    import custom_ecc_cuda as ops
    from custom_kv import PagedErrorCorrectedCache
    cache = PagedErrorCorrectedCache(config(3), batch_size=2, max_cache_len=64, num_pages=11, page_size=16,
                                     collect_weights=True)
    g = torch.Generator(device="cuda").manual_seed(6)
    for layer, (k, v) in enumerate(states(cache, 2, 60, g)):
        cache.append(k, v, layer)
    cache.weights.copy_(torch.rand(cache.weights.shape, generator=g, device="cuda"))
    was = (cache.lengths, list(cache._free), cache.seq_lens.tolist(), cache.block_table.tolist())
    weights, context = cache.weights.clone(), [cache.context(i) for i in range(3)]
    real, calls = ops.evict_paged, []

    def failing(*args, **kw):
        calls.append(args)
        if len(calls) == 2:
            raise RuntimeError("no memory")
        return real(*args, **kw)

    monkeypatch.setattr(ops, "evict_paged", failing)
    with pytest.raises(RuntimeError, match="no memory"):
        cache.evict(30, sinks=2, recent=5)
    assert (cache.lengths, list(cache._free), cache.seq_lens.tolist(), cache.block_table.tolist()) == was
    assert torch.equal(cache.weights, weights)
    for i in range(3):
        assert all(torch.equal(x, y) for x, y in zip(cache.context(i), context[i]))
    assert cache.evict(30, sinks=2, recent=5) == [0, 1] and cache.lengths == [30, 30]
    for i in range(3):
        for b in range(2):
            for h in range(2):
                row = weights[i, b, h].cpu().numpy()
                mid = sorted(range(2, 55), key=lambda t: (-row[t], t))[:23]
                ids = list(range(2)) + sorted(mid) + list(range(55, 60))
                assert np.array_equal(cache.weights[i, b, h, :30].cpu().numpy(), row[ids])
                assert not cache.weights[i, b, h, 30:].any()
                for x, y in zip(cache.context(i), context[i]):
                    assert torch.equal(x[b, h], y[b, h, ids])


def test_every_layers_mask_is_looked_at(cuda_device):
    """A model's layers may have masks of their own (a sliding window in every other one)."""
    from custom_kv import PagedErrorCorrectedCache
    cache = PagedErrorCorrectedCache(config(3), batch_size=2, max_cache_len=64, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    for layer, (k, v) in enumerate(states(cache, 2, 40, g)):
        cache.append(k, v, layer)
    q = torch.randn(2, 4, 1, 128, generator=g, device="cuda").half()
    whole = torch.ones(2, 1, 1, 40, dtype=torch.bool, device="cuda")
    part = whole.clone()
    part[..., :8] = False
    for layer in range(3):
        assert torch.equal(cache.decode_attention(q, layer, attn_mask=whole), cache.decode_attention(q, layer))
        for mask in (part, torch.zeros(2, 1, 1, 40, device="cuda").masked_fill(~part, torch.finfo(torch.float32).min)):
            with pytest.raises(RuntimeError, match="padding"):
                cache.decode_attention(q, layer, attn_mask=mask)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [-1e4, -0.5, 1e-3, float("nan")])
def test_masks_that_add_to_the_scores_are_refused(cuda_device, dtype, value):
    """A finite stand-in for minus infinity, or a position bias: neither is dropped silently."""
    from custom_kv import PagedErrorCorrectedCache
    cache = PagedErrorCorrectedCache(config(1), batch_size=2, max_cache_len=64, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    (k, v), = states(cache, 2, 40, g)
    cache.append(k, v, 0)
    q = torch.randn(2, 4, 1, 128, generator=g, device="cuda").half()
    mask = torch.zeros(2, 1, 1, 40, dtype=dtype, device="cuda")
    mask[1, ..., 0] = -0.0
    assert torch.equal(cache.decode_attention(q, 0, attn_mask=mask), cache.decode_attention(q, 0))
    mask[1, ..., 3] = value
    with pytest.raises(RuntimeError, match="padding"):
        cache.decode_attention(q, 0, attn_mask=mask)


def _tiny_llama(seed=0, layers=2):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(seed)
    cfg = LlamaConfig(hidden_size=512, intermediate_size=1024, num_hidden_layers=layers, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, vocab_size=1000, max_position_embeddings=4096,
                      rope_theta=500000.0, attn_implementation="sdpa")
    return LlamaForCausalLM(cfg).half().cuda().eval()


def test_model_runs_on_the_paged_cache(cuda_device):
    """Prompt in two chunks, decode steps, an eviction in between; the first step's blocks are those of the contiguous
    cache, bit for bit."""
    from custom_kv import Sampler, ecc_cache, paged_ecc_cache
    model = _tiny_llama(1)
    ids = torch.randint(0, 1000, (2, 150), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        with ecc_cache(model, batch_size=2, max_cache_len=256) as ref:
            a = model(ids[:, :100], past_key_values=ref, use_cache=True).logits
            blocks = [[p[:, :, :100].clone() for p in ref.layer_pools(i)] for i in range(2)]
        with paged_ecc_cache(model, batch_size=2, max_cache_len=256, page_size=16, collect_weights=True) as cache:
            b = model(ids[:, :100], past_key_values=cache, use_cache=True).logits
            assert torch.equal(a, b)
            for i in range(2):
                for x, pool in zip(blocks[i], cache.layer_pools(i)):
                    for s in range(2):
                        got = pool[cache.block_table[s, :7].long()].transpose(0, 1).reshape(2, 112, 128)[:, :100]
                        assert torch.equal(got, x[s])
            logits = model(ids[:, 100:], past_key_values=cache, use_cache=True).logits[:, -1]
            assert cache.lengths == [150, 150]
            sampler = Sampler(temperature=0.8, top_k=40, top_p=0.95)
            for step in range(6):
                tok = sampler(logits)[:, None]
                assert tok.min() >= 0 and tok.max() < 1000
                logits = model(tok, past_key_values=cache, use_cache=True).logits[:, -1]
                assert torch.isfinite(logits).all()
                if step == 2:
                    assert cache.evict(100, sinks=4, recent=32) == [0, 1]
            assert cache.lengths == [103, 103] and cache.get_seq_length() == 156
            # every step and layer handed out one unit of weight per query head of the group
            assert float(cache.weights.sum()) <= 6 * 2 * 2 * 4 * (1 + 1e-4)


def test_slots_of_different_lengths_have_positions_of_their_own(cuda_device):
    """A step whose positions are one for all slots is refused and leaves the cache as it was; with the cache's position_ids
    the first layer's keys are, block for block, those of the same tokens in slots of one length."""
    from custom_kv import paged_ecc_cache
    model = _tiny_llama(2)
    g = torch.Generator().manual_seed(9)
    ids, toks = torch.randint(0, 1000, (2, 50), generator=g).cuda(), torch.randint(0, 1000, (3, 2, 1), generator=g).cuda()

    def block(cache, slot, t):  # the key of token t in the first layer
        return cache.layer_pools(0)[0][int(cache.block_table[slot, t // 16]), :, t % 16].clone()

    new = dict(batch_size=2, max_cache_len=96, page_size=16)
    with torch.no_grad():
        alone = model(ids, use_cache=False).logits
        with paged_ecc_cache(model, **new) as cache:  # slot 0 goes on at 50, as both slots do here
            model(ids, past_key_values=cache, use_cache=True)
            long = []
            for i in range(3):
                assert cache.position_ids().tolist() == [[50 + i], [50 + i]]
                model(toks[i], past_key_values=cache, use_cache=True)
                long.append(block(cache, 0, 50 + i))
        with paged_ecc_cache(model, **new) as cache:  # slot 1 begins at 0
            short = []
            for i in range(3):
                model(toks[i], past_key_values=cache, use_cache=True)
                short.append(block(cache, 1, i))
        with paged_ecc_cache(model, **new) as cache:
            model(ids, past_key_values=cache, use_cache=True)
            cache.release([1])
            for i in range(3):
                n = 50 + i
                for bad in (dict(), dict(position_ids=torch.tensor([[n]], device="cuda")),
                            dict(position_ids=torch.tensor([[n], [n]], device="cuda"))):
                    with pytest.raises(RuntimeError, match="position_ids"):
                        model(toks[i], past_key_values=cache, use_cache=True, **bad)
                    assert cache.lengths == [n, i]
                assert cache.position_ids().tolist() == [[n], [i]]
                model(toks[i], past_key_values=cache, use_cache=True, position_ids=cache.position_ids())
                assert torch.equal(block(cache, 0, n), long[i]) and torch.equal(block(cache, 1, i), short[i])
            assert torch.equal(model(ids, use_cache=False).logits, alone)  # a pass without the cache is no concern of it


def test_positions_a_model_shows_only_as_angles(cuda_device):
    from custom_kv import PagedErrorCorrectedCache
    cache = PagedErrorCorrectedCache(config(1), batch_size=2, max_cache_len=64, page_size=16)
    g = torch.Generator(device="cuda").manual_seed(1)
    (k, v), = states(cache, 2, 40, g)
    angles = torch.rand(2, 1, 128, generator=g, device="cuda")
    same = angles[:1].expand(2, 1, 128)
    for bad in (same, angles[:1]):
        cache.check_positions(None, (bad.cos(), bad.sin()))  # slots of one length
    cache.append(k, v, 0, new_lens=[40, 9])
    cache.check_positions(None, (angles.cos(), angles.sin()))
    cache.check_positions(None)
    for bad in (same, angles[:1]):
        with pytest.raises(RuntimeError, match="position_ids"):
            cache.check_positions(None, (bad.cos(), bad.sin()))


def test_recorded_settings_outlive_the_sampler(cuda_device):
    import custom_ecc_cuda as ops
    from custom_kv import Sampler, ecc_cache
    from custom_kv.graph import GraphDecoder
    model = _tiny_llama(3)
    ids = torch.randint(0, 1000, (2, 40), generator=torch.Generator().manual_seed(4)).cuda()
    with torch.no_grad(), ecc_cache(model, batch_size=2, max_cache_len=128) as cache:
        logits = model(ids, past_key_values=cache, use_cache=True).logits[:, -1]
        sampler = Sampler(temperature=torch.tensor([0.9, 0.5], device="cuda"))
        dec = GraphDecoder(model, cache, sampler(logits)[:, None], sampler=sampler)
        sampler.temperature = 1.0  # the record goes on with the tensor that it was made with
        torch.cuda.empty_cache()
        taken = [torch.full((2,), 7.0, device="cuda") for _ in range(64)]
        for u in ([0.1, 0.9], [0.7, 0.3]):
            u = torch.tensor(u, device="cuda")
            t = dec.step(u)
            assert torch.equal(t[:, 0], ops.sample_tokens(dec.logits, u, temperature=torch.tensor([0.9, 0.5], device="cuda")))
        assert len(taken) == 64


def test_graph_decoder_samples(cuda_device):
    import custom_ecc_cuda as ops
    from custom_kv import Sampler, ecc_cache
    from custom_kv.graph import GraphDecoder
    model = _tiny_llama(3)
    ids = torch.randint(0, 1000, (2, 60), generator=torch.Generator().manual_seed(2)).cuda()
    g = torch.Generator(device="cuda").manual_seed(7)
    with torch.no_grad(), ecc_cache(model, batch_size=2, max_cache_len=128) as cache:
        logits = model(ids, past_key_values=cache, use_cache=True).logits[:, -1]
        temp = torch.tensor([0.9, 0.5], device="cuda")
        sampler = Sampler(temperature=temp, top_k=30, top_p=0.9, generator=g)
        dec = GraphDecoder(model, cache, sampler(logits)[:, None], sampler=sampler)
        for step in range(5):
            if step == 3:
                temp.fill_(0.0)  # settings given as tensors may change between steps
            u = torch.rand(2, generator=g, device="cuda")
            t = dec.step(u) if step % 2 else dec.step()
            used = u if step % 2 else dec.uniform
            assert torch.equal(t[:, 0], ops.sample_tokens(dec.logits, used, temperature=temp, top_k=30, top_p=0.9))
            assert torch.equal(dec.ids, t)
            if step >= 3:
                assert torch.equal(t[:, 0], dec.logits.argmax(-1))
        greedy = GraphDecoder(model, cache, ids[:, :1]) if dec.sync_host_lengths() else None
        with pytest.raises(RuntimeError):
            greedy.step(u)
