"""Paged cache: append, read-back and decode attention (ragged lengths,
windows with sinks, attention weights) against plain 64-bit implementations."""
import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def cu(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def _clean_status(cuda_device):
    import custom_ecc_cuda as ops
    ops.device_status(reset=True)
    yield
    assert ops.device_status(reset=True) == 0


def check_decode(lens, hq, hkv, ps, rec, window=0, sinks=0, rotate=False, seed=0, width=None):
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(seed)
    kp, vp, table = R.make_pools(lens, ps, hkv, rec, rng, width=width)
    B = len(lens)
    q = rng.normal(size=(B, hq, 128)).astype(np.float16)
    cap = table.shape[1] * ps
    w0 = rng.uniform(0, 1, (B, hkv, cap + 3)).astype(np.float32)
    wt = cu(w0)
    out, lse = ops.decode_attention_paged(cu(q), cu(kp), cu(vp), cu(table), i32(lens), window=window, sinks=sinks,
                                          rotate_q=rotate, unrotate_out=rotate, weights=wt, return_lse=True)
    plain = ops.decode_attention_paged(cu(q), cu(kp), cu(vp), cu(table), i32(lens), window=window, sinks=sinks,
                                       rotate_q=rotate, unrotate_out=rotate)
    assert torch.equal(out, plain)  # the weights do not change the output
    o, tol, l, l_tol, ws, w_tol = R.attend(q, kp, vp, table, lens, window, sinks, rotate)
    got = out.cpu().numpy().astype(np.float64).reshape(B, hq, 128)
    assert np.isfinite(got).all()
    assert (np.abs(got - o) <= tol).all(), np.max(np.abs(got - o) / tol)
    gl = lse.cpu().numpy().astype(np.float64)
    empty = np.isneginf(l)
    assert (np.isneginf(gl) == empty).all()
    assert (np.abs(gl[~empty] - l[~empty]) <= l_tol[~empty]).all()
    gw = wt.cpu().numpy()
    base = w0[:, :, :cap].astype(np.float64)
    # one more rounding: the sum is added to the accumulator in fp32
    assert (np.abs(gw[:, :, :cap] - (base + ws)) <= w_tol + 2.0 ** -24 * (base + ws)).all()
    for b, n in enumerate(lens):
        hid = np.setdiff1d(np.arange(cap + 3), R.visible(n, window, sinks))
        assert np.array_equal(gw[b][:, hid], w0[b][:, hid])


@pytest.mark.parametrize("ps", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("rec", [128, 96])
def test_decode_ragged_lengths(ps, rec):
    check_decode([0, 1, 15, 16, 17, 31, 33, 130, 300, 0], 8, 2, ps, rec, seed=ps + rec)


@pytest.mark.parametrize("g", [1, 2, 3, 4, 5, 6, 7, 8])
def test_decode_groups(g):
    check_decode([77, 5, 200], 3 * g, 3, 32, 128, seed=g)
    check_decode([77, 5, 200], 2 * g, 2, 16, 128, rotate=True, seed=g)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 40), (64, 32), (100, 64), (5000, 9)])
@pytest.mark.parametrize("ps", [32, 48])
def test_decode_window_and_sinks(window, sinks, ps):
    check_decode([0, 1, 20, 32, 64, 65, 129, 500], 4, 1, ps, 128, window=window, sinks=sinks, seed=window + sinks)


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [5000], [4000] * 3, [1] * 70 + [900]])
def test_decode_batch_shapes(lens):
    check_decode(lens, 4, 2, 64, 128, rotate=True, seed=len(lens))


def peaked(n, at, nats, v_scale, sink_v, g, rec, ps, seed):
    """One kv head, n tokens of small keys and one, at `at`, that all heads' scores put `nats` above them; values of scale
    `v_scale` (a number or a function of the token), that token's `sink_v`.  Returns q, pools and table."""
    rng = np.random.default_rng(seed)
    kp, vp, table = R.make_pools([n], ps, 1, rec, rng)
    base = rng.normal(size=128)
    q = (base * rng.uniform(0.97, 1.03, (1, g, 1)) + 0.01 * rng.normal(size=(1, g, 128))).astype(np.float16)

    def metas(pool, scale):
        for t in range(n):
            m = np.array([scale[t], 0.0, 0.11 * scale[t]], np.float16)
            pool[table[0, t // ps], 0, t % ps, 80:86] = m.view(np.uint8)

    ks, vs = np.full(n, 0.05), np.array([v_scale(t) if callable(v_scale) else v_scale for t in range(n)], float)
    if nats:
        codes = np.where(q[0, 0] > 0, 14, 0).astype(np.uint8)  # the levels 2.4008 and -2.4008
        kp[table[0, at // ps], 0, at % ps, :64] = codes[0::2] | (codes[1::2] << 4)
        ks[at] = nats / (2.4008 * np.abs(q[0, 0].astype(float)).sum() * R.SM)
        vs[at] = sink_v
    metas(kp, ks)
    metas(vp, vs)
    return q, kp, vp, table


@pytest.mark.parametrize("g,rec", [(4, 128), (8, 128), (1, 96)])
@pytest.mark.parametrize("at,nats,v_scale,sink_v", [
    (0, 12, 0.2, 1e-6), (0, 12, 0.05, 0.0), (0, 12, 0.02, 1e-6), (4095, 12, 0.05, 1e-6), (1777, 14, 0.5, 1e-6), (0, 17, 8.0, 1e-4),
    (5, 8, 0.1, 1e-3), (0, 6, 1e-3, 1e-6), (0, 12, 0.05, 3.0), (0, 0, 1e-3, 0.0), (0, 0, lambda t: 10.0 ** (t % 47 / 9 - 3.5), 0.0),
    (0, 10, lambda t: 10.0 ** (t / 1024 - 3), 1e-6), (0, 10, lambda t: 10.0 ** (1 - t / 1024), 1e-6), (0, 0, 2e4, 0.0)],
    ids=lambda v: getattr(v, "__name__", str(v)))
def test_decode_small_values_beside_a_dominating_token(at, nats, v_scale, sink_v, g, rec):
    """Attention sinks with next to no value of their own: the output is made of probabilities far below the largest.
    Sequences share one context, so many that a warp takes thousands of tokens in one piece.

    The bound is attend()'s.  Its absolute 1e-7 holds what fp16 leaves of a weight: 2^-39 of (the largest probability x
    the largest scale), so n 2^-36 of the largest scale for n tokens (2^3 > the largest level, its factor and the signs):
    6e-8 of it, which the scales above 1 of these cases add here."""
    import custom_ecc_cuda as ops
    n, B = 4096, 1024
    q, kp, vp, table = peaked(n, at, nats, v_scale, sink_v, g, rec, 64, seed=at + g)
    o, tol, l, l_tol, _, _ = R.attend(q, kp, vp, table, [n])
    top = R.fields(R.sequence(vp, table[0], 0, n))[2][:, 0].max()
    tol = tol + n * 2.0 ** -36 * top
    out, lse = ops.decode_attention_paged(cu(q).expand(B, g, 128).contiguous(), cu(kp), cu(vp), cu(table).expand(B, -1),
                                          i32([n] * B), return_lse=True)
    got = out.cpu().numpy().astype(np.float64).reshape(B, g, 128)
    assert np.isfinite(got).all()
    assert (np.abs(got - o) <= tol).all(), np.max(np.abs(got - o) / tol)
    assert (np.abs(lse.cpu().numpy() - l) <= l_tol).all()


@pytest.mark.parametrize("g", [2, 4, 8])
@pytest.mark.parametrize("ratio,k_scale", [(1e-2, 50), (1e-3, 500), (1e-4, 5000), (1e-5, 5000), (3000.0, 0.01)])
def test_decode_heads_of_unlike_magnitude(g, ratio, k_scale):
    """One head of a group is 1 / ratio times the others: each keeps the precision of its own magnitude."""
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(g)
    kp, vp, table = R.make_pools([300], 64, 1, 128, rng)
    for t in range(300):
        meta = kp[table[0, t // 64], 0, t % 64, 80:86].view(np.float16)
        meta[:] = (meta.astype(np.float64) * k_scale).astype(np.float16)
    q = rng.normal(size=(1, g, 128))
    q[:, 1:] *= ratio
    q = q.astype(np.float16)
    for rotate in (False, True):
        o, tol, l, l_tol, _, _ = R.attend(q, kp, vp, table, [300], rotate=rotate)
        out, lse = ops.decode_attention_paged(cu(q), cu(kp), cu(vp), cu(table), i32([300]), rotate_q=rotate,
                                              unrotate_out=rotate, return_lse=True)
        assert (np.abs(out.cpu().numpy().astype(np.float64).reshape(1, g, 128) - o) <= tol).all()
        assert (np.abs(lse.cpu().numpy() - l) <= l_tol).all(), np.max(np.abs(lse.cpu().numpy() - l) / l_tol)


@pytest.mark.parametrize("lens,hq,rotate", [
    ([16500] + [(0, 1, 33, 0, 70)[b % 5] for b in range(299)], 4, False),  # few slots a row: one group of threads joins 516
    ([(0, 3, 0)[b % 3] for b in range(250)] + [9000, 7000] + [0] * 48, 2, True),
    ([40003], 4, True), ([40003], 8, False)],  # 1251 partials, four groups
    ids=["one long of 300", "two long of 300", "one of 40k", "one of 40k, group of 8"])
def test_decode_joins_many_partials(lens, hq, rotate):
    check_decode(lens, hq, 1, 64, 128, rotate=rotate, seed=len(lens) + hq)


def test_decode_one_page_per_sequence_of_any_size():
    # a contiguous pool is a paged one with one page per sequence
    check_decode([100, 37, 0, 1], 8, 4, 100, 128, seed=3, width=1)


def test_decode_weights_of_a_whole_context_sum_to_the_heads():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(5)
    lens = [3000, 64, 1]
    kp, vp, table = R.make_pools(lens, 64, 2, 128, rng)
    w = torch.zeros(3, 2, table.shape[1] * 64, device="cuda")
    q = cu(rng.normal(size=(3, 16, 128)).astype(np.float16))
    for _ in range(3):
        ops.decode_attention_paged(q, cu(kp), cu(vp), cu(table), i32(lens), weights=w)
    # 3 steps of 8 heads; a sum of softmax weights is 1 within the bound of its terms
    assert torch.allclose(w.sum(-1), torch.full((3, 2), 24.0, device="cuda"), rtol=2e-5, atol=0)


def test_decode_strides_and_shared_pages():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(9)
    lens, ps, hkv = [40, 40, 70], 16, 2
    kp, vp, table = R.make_pools(lens, ps, hkv, 128, rng)
    table[1, :2] = table[0, :2]  # a shared prefix
    q = rng.normal(size=(3, 4, 128)).astype(np.float16)
    P = kp.shape[0]
    big_k = torch.full((P, 2 * hkv + 1, ps + 2, 128), 255, dtype=torch.uint8, device="cuda")
    big_v = big_k.clone()
    k, v = big_k[:, 1::2][:, :, 1:1 + ps], big_v[:, 1::2][:, :, 1:1 + ps]
    k.copy_(cu(kp)), v.copy_(cu(vp))
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = cu(table)
    t = wide[:, 2:2 + table.shape[1]]
    qq = cu(np.repeat(q[:, :, None], 2, 2))[:, :, 1:2]  # not contiguous
    w = torch.zeros(hkv, 3, 200, device="cuda").transpose(0, 1)
    out = ops.decode_attention_paged(qq, k, v, t, i32(lens), weights=w)
    o, tol, _, _, ws, w_tol = R.attend(q, kp, vp, table, lens)
    assert (np.abs(out.cpu().numpy().reshape(3, 4, 128) - o) <= tol).all()
    assert (np.abs(w.cpu().numpy()[:, :, :ws.shape[2]] - ws) <= w_tol + 2.0 ** -24).all()


def test_decode_agrees_with_the_contiguous_decode():
    import custom_ecc_cuda as ops
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 2, 2, 640, 128, generator=g, device="cuda").half()
    kp = torch.zeros(2, 2, 640, 128, dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.compress_pair_into(x[0], x[1], kp, vp)
    q = torch.randn(2, 8, 1, 128, generator=g, device="cuda").half()
    a = ops.decode_attention(q, kp, vp, seq_len=600, rotate_q=True, unrotate_out=True)
    table = torch.arange(2, dtype=torch.int32, device="cuda")[:, None]
    b = ops.decode_attention_paged(q, kp, vp, table, i32([600, 600]), rotate_q=True, unrotate_out=True)
    # the same stages summed in another order: the fp16 results are a step apart at most
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -10 * a.float().abs().max()


def test_decode_bad_length_and_page_are_flagged():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(2)
    kp, vp, table = R.make_pools([40, 40], 16, 1, 128, rng)
    q = cu(rng.normal(size=(2, 2, 128)).astype(np.float16))
    good = ops.decode_attention_paged(q, cu(kp), cu(vp), cu(table), i32([40, 40]))
    for bad in (kp.shape[0], -1, 1 << 30):
        t = table.copy()
        t[1, 1] = bad
        out = ops.decode_attention_paged(q, cu(kp), cu(vp), cu(t), i32([40, 40]))
        assert ops.device_status(reset=True) == 5
        assert torch.equal(out[0], good[0]) and torch.isfinite(out).all()
    for n in (-3, 1000):
        out = ops.decode_attention_paged(q, cu(kp), cu(vp), cu(table), i32([40, n]))
        assert ops.device_status(reset=True) == 5
        assert torch.equal(out[0], good[0])


def test_decode_refusals():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(2)
    kp, vp, table = (cu(x) for x in R.make_pools([40, 40], 16, 2, 128, rng))
    q, n = torch.zeros(2, 4, 1, 128, dtype=torch.float16, device="cuda"), i32([40, 40])
    call = ops.decode_attention_paged
    bad = [
        dict(query=q.float()), dict(query=q[:1]), dict(query=q[:, :3]), dict(query=q.expand(2, 4, 2, 128)),
        dict(query=torch.zeros(2, 18, 1, 128, dtype=torch.float16, device="cuda")),
        dict(k_pool=kp[0]), dict(v_pool=vp[:, :1]), dict(k_pool=kp.half()), dict(v_pool=vp.cpu()),
        dict(block_table=table.long()), dict(block_table=table[0]), dict(block_table=table[:1]),
        dict(block_table=table.t().contiguous().t()), dict(seq_lens=n.long()), dict(seq_lens=n[:1]),
        dict(seq_lens=n.cpu()), dict(window=-1), dict(sinks=4), dict(window=4, sinks=-1),
        dict(weights=torch.zeros(2, 2, 47, device="cuda")), dict(weights=torch.zeros(2, 1, 48, device="cuda")),
        dict(weights=torch.zeros(2, 2, 48, dtype=torch.float16, device="cuda")),
        dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")), dict(sm_scale=float("nan")),
        dict(out=torch.zeros(2, 4, 1, 128, device="cuda")),
    ]
    args = dict(query=q, k_pool=kp, v_pool=vp, block_table=table, seq_lens=n)
    call(**args)
    for b in bad:
        with pytest.raises(RuntimeError):
            call(**{**args, **b})
    odd = torch.zeros(4, 2, 24, 128, dtype=torch.uint8, device="cuda")  # a page size that splits a 16-token group
    with pytest.raises(RuntimeError):
        call(q, odd, odd, table, n)


def test_decode_in_a_graph_follows_lengths_and_pages():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(4)
    lens = [500, 300, 77]
    kp, vp, table = R.make_pools(lens, 32, 2, 128, rng)
    kd, vd, td = cu(kp), cu(vp), cu(table)
    q = cu(rng.normal(size=(3, 8, 128)).astype(np.float16))
    cap = table.shape[1] * 32
    need = ops.decode_paged_workspace_size(3, 8, 2, cap, with_weights=True)
    states = []
    for _ in range(2):  # two graphs, each with a workspace of its own
        n = i32([1, 1, 1])
        w = torch.zeros(3, 2, cap, device="cuda")
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.decode_attention_paged(q, kd, vd, td, n, weights=w, workspace=ws)
        torch.cuda.current_stream().wait_stream(side)
        w.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.decode_attention_paged(q, kd, vd, td, n, weights=w, workspace=ws)
        states.append((graph, n, w, out))
    for step, now in enumerate(([500, 300, 77], [0, 1, 33], [499, 0, 64])):
        graph, n, w, out = states[step % 2]
        n.copy_(i32(now))
        w.zero_()
        graph.replay()
        w2 = torch.zeros_like(w)
        ref = ops.decode_attention_paged(q, kd, vd, td, i32(now), weights=w2)
        assert torch.equal(out, ref) and torch.equal(w, w2)


def test_decode_on_a_side_stream():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(6)
    kp, vp, table = R.make_pools([900, 900], 64, 2, 128, rng)
    q = cu(rng.normal(size=(2, 4, 128)).astype(np.float16))
    kd, vd, td, n = cu(kp), cu(vp), cu(table), i32([900, 900])
    ref = ops.decode_attention_paged(q, kd, vd, td, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for k in range(10):
        with torch.cuda.stream(streams[k % 2]):
            outs.append(ops.decode_attention_paged(q, kd, vd, td, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_decode_from_two_threads_on_one_stream():
    import threading
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(16)
    cases = []
    for lens, hkv in (([4000, 17, 900], 2), ([2500, 3100], 4)):
        kp, vp, table = R.make_pools(lens, 64, hkv, 128, rng)
        q = cu(rng.normal(size=(len(lens), 4 * hkv, 128)).astype(np.float16))
        args = (q, cu(kp), cu(vp), cu(table), i32(lens))
        cases.append((args, ops.decode_attention_paged(*args)))
    torch.cuda.synchronize()
    outs = [[], []]

    def run(i):
        for _ in range(200):
            outs[i].append(ops.decode_attention_paged(*cases[i][0]))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(outs[i]) == 200 and all(torch.equal(o, cases[i][1]) for o in outs[i])


@pytest.mark.parametrize("which", ["paged", "contiguous", "masked", "device length"])
def test_decode_as_the_first_call_of_a_thread(which):
    """A thread that has made no CUDA call yet: no context is current in it."""
    import threading
    import custom_ecc_cuda as ops
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(2, 2, 2, 300, 128, generator=g, device="cuda").half()
    kp = torch.zeros(2, 2, 300, 128, dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.compress_pair_into(x[0], x[1], kp, vp)
    q = torch.randn(2, 8, 1, 128, generator=g, device="cuda").half()
    table, n, start, one = torch.arange(2, dtype=torch.int32, device="cuda")[:, None], i32([300, 45]), i32([0, 99]), i32([300])
    ws = torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    call = {"paged": lambda: ops.decode_attention_paged(q, kp, vp, table, n, workspace=ws, out=out),
            "contiguous": lambda: ops.decode_attention(q, kp, vp, 300, workspace=ws, out=out),
            "masked": lambda: ops.decode_attention_masked(q, kp, vp, 300, start, workspace=ws, out=out),
            "device length": lambda: ops.decode_attention_dev(q, kp, vp, one, workspace=ws, out=out)}[which]
    want = call().clone()
    out.zero_()
    torch.cuda.synchronize()
    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_calls_that_share_a_workspace_issue_their_launches_one_at_a_time(monkeypatch):
    """The contiguous decodes take the workspace of the paged calls on their stream: every one of these entry points is
    called with the device's lock held, so no launch of another thread comes between its launches."""
    import custom_ecc_cuda as ops
    real, seen = ops._lib, []

    class Recording:
        def __getattr__(self, name):
            fn = getattr(real, name)
            if name not in ("ecc_call", "ecc_decode", "ecc_decode_masked", "ecc_decode_dev"):
                return fn

            def call(*args):
                seen.append((name, ops._launch_locks[0].locked()))
                return fn(*args)
            return call

    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(2, 2, 2, 64, 128, generator=g, device="cuda").half()
    kp = torch.zeros(2, 2, 64, 128, dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.compress_pair_into(x[0], x[1], kp, vp)
    q = torch.randn(2, 8, 1, 128, generator=g, device="cuda").half()
    table = torch.arange(2, dtype=torch.int32, device="cuda")[:, None]
    monkeypatch.setattr(ops, "_lib", Recording())
    outs = [ops.decode_attention(q, kp, vp, seq_len=60), ops.decode_attention_masked(q, kp, vp, 60, i32([0, 0])),
            ops.decode_attention_dev(q, kp, vp, i32([60])), ops.decode_attention_paged(q, kp, vp, table, i32([60, 60]))]
    assert seen == [("ecc_decode", True), ("ecc_decode_masked", True), ("ecc_decode_dev", True), ("ecc_call", True)]
    assert not ops._launch_locks[0].locked()
    for o in outs[1:]:
        assert (o.float() - outs[0].float()).abs().max() <= 2.0 ** -10 * outs[0].float().abs().max()


def test_contiguous_and_paged_decode_from_threads_on_one_stream():
    import threading
    import custom_ecc_cuda as ops
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 3, 2, 4000, 128, generator=g, device="cuda").half()
    kp = torch.zeros(3, 2, 4000, 128, dtype=torch.uint8, device="cuda")
    vp = torch.zeros_like(kp)
    ops.compress_pair_into(x[0], x[1], kp, vp)
    q = torch.randn(3, 8, 1, 128, generator=g, device="cuda").half()
    table, n, start = torch.arange(3, dtype=torch.int32, device="cuda")[:, None], i32([4000, 17, 900]), i32([0, 9, 700])
    calls = [lambda: ops.decode_attention_paged(q, kp, vp, table, n), lambda: ops.decode_attention(q, kp, vp, 3900),
             lambda: ops.decode_attention_masked(q, kp, vp, 3500, start),
             lambda: ops.decode_attention_dev(q, kp, vp, n[:1])]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    outs = [[] for _ in calls]

    def run(i):
        for _ in range(100):
            outs[i].append(calls[i]())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert len(o) == 100 and all(torch.equal(a, w) for a in o)


# ------------------------------------------------------------------ append and read-back
@pytest.mark.parametrize("L,hkv,ps,rec", [(1, 2, 16, 128), (17, 3, 32, 96), (40, 1, 48, 128), (700, 4, 64, 128),
                                          (700, 4, 64, 96)])
@pytest.mark.parametrize("rotate", [True, False])
def test_append_writes_the_blocks_of_compress_pair_into(L, hkv, ps, rec, rotate):
    import custom_ecc_cuda as ops
    B = 3
    g = torch.Generator(device="cuda").manual_seed(L)
    k, v = (torch.randn(B, L, hkv, 128, generator=g, device="cuda").half().transpose(1, 2) for _ in range(2))
    k[0, 0, 0] = 0  # a vector without spread
    pos, new = [0, ps - 1, 2 * ps], [L, max(0, L - 5), 0]
    rng = np.random.default_rng(L)
    lens = [p + n for p, n in zip(pos, new)]
    table, total = R.layout(lens, ps, 2, rng)
    kp = torch.randint(0, 256, (total, hkv, ps, rec), generator=g, device="cuda", dtype=torch.uint8)
    vp = torch.randint(0, 256, (total, hkv, ps, rec), generator=g, device="cuda", dtype=torch.uint8)
    want = []
    for x, pool in ((k, kp), (v, vp)):
        flat = torch.zeros(B, hkv, L, rec, dtype=torch.uint8, device="cuda")
        ops.compress_into(x, flat, rotate=rotate)
        w = pool.clone()
        for b in range(B):
            for i in range(new[b]):
                p = pos[b] + i
                w[int(table[b, p // ps]), :, p % ps] = flat[b, :, i]
        want.append(w)
    ops.compress_pair_paged(k, v, kp, vp, cu(table), i32(pos), new_lens=i32(new), rotate=rotate)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    only = kp.clone().random_(0, 255)
    keep = only.clone()
    ops.compress_pair_paged(k[:1], None, only, None, cu(table[:1]), i32(pos[:1]), rotate=rotate)
    for i in range(L):
        p = pos[0] + i
        keep[int(table[0, p // ps]), :, p % ps] = want[0][int(table[0, p // ps]), :, p % ps]
    assert torch.equal(only, keep)


@pytest.mark.parametrize("L", [3, 3000])
def test_append_out_of_range_writes_nothing(L):
    import custom_ecc_cuda as ops
    x = torch.randn(2, 2, L, 128, device="cuda").half()
    pool = torch.zeros(400, 2, 16, 128, dtype=torch.uint8, device="cuda")
    table = torch.arange(400, dtype=torch.int32, device="cuda").reshape(2, 200)
    for t, pos, new in ((table, [3200, -L], None), (table - 1000, [0, 0], None), (table + 400, [0, 0], None),
                        (table, [0, 0], [-1, -5])):
        ops.compress_pair_paged(x, x, pool, pool.clone(), t, i32(pos), new_lens=None if new is None else i32(new))
        assert ops.device_status(reset=True) == 5
        assert int(pool.max()) == 0
    one = pool.clone()
    ops.compress_pair_paged(x, None, one, None, table, i32([0, 0]), new_lens=i32([L + 1, 1]))  # the other goes on
    assert ops.device_status(reset=True) == 5
    assert not one[:200].any() and one[200, :, 0].any() and not one[200, :, 1:].any()


def test_pages_beyond_four_gigabytes():
    """Append, read-back, decode and eviction on pages whose byte offsets pass 32 bits."""
    import custom_ecc_cuda as ops
    hkv, ps = 4, 256
    per = hkv * ps * 128
    total = (1 << 32) // per + 40
    g = torch.Generator(device="cuda").manual_seed(0)
    big = [torch.empty(total, hkv, ps, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    small = [torch.empty(8, hkv, ps, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    far = torch.tensor([[total - 1, total - 7, 3]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[5, 1, 3]], dtype=torch.int32, device="cuda")
    x = [torch.randn(1, hkv, 700, 128, generator=g, device="cuda").half() for _ in range(2)]
    q = torch.randn(1, 8, 1, 128, generator=g, device="cuda").half()
    got = []
    for pools, table, out in ((big, far, far - 1), (small, near, near - 1)):
        ops.compress_pair_paged(x[0], x[1], *pools, table, i32([0]))
        w = torch.zeros(1, hkv, 768, device="cuda")
        o = ops.decode_attention_paged(q, *pools, table, i32([700]), weights=w)
        k, v = ops.dequantize_paged(*pools, table, i32([700]), 700)
        ow, kept = ops.evict_paged(*pools, table, i32([700]), w, out, 400, sinks=3, recent=50)
        ek, ev = ops.dequantize_paged(*pools, out, i32([400]), 400)
        got.append((o, w, k, v, ow, kept, ek, ev))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert (got[0][2] - x[0]).float().norm() < 0.2 * x[0].float().norm()


def test_append_refusals():
    import custom_ecc_cuda as ops
    x = torch.zeros(2, 2, 3, 128, dtype=torch.float16, device="cuda")
    pool = torch.zeros(8, 2, 16, 128, dtype=torch.uint8, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
    args = dict(k=x, v=x, k_pool=pool, v_pool=pool.clone(), block_table=table, pos=i32([0, 0]))
    ops.compress_pair_paged(**args)
    for b in (dict(k=x.float()), dict(v=x[:, :1]), dict(v=None), dict(v_pool=None), dict(k=x[..., :64]),
              dict(k=x.transpose(2, 3)), dict(k=x[0]), dict(pos=i32([0])), dict(pos=i32([0, 0]).long()),
              dict(new_lens=i32([1])), dict(block_table=table[:1]), dict(k_pool=pool[:, :1]),
              dict(v_pool=pool[..., :96]), dict(k=x.cpu()), dict(k=torch.zeros(2, 2, 3, 129, dtype=torch.float16,
                                                                                device="cuda")[..., 1:])):
        with pytest.raises(RuntimeError):
            ops.compress_pair_paged(**{**args, **b})


@pytest.mark.parametrize("rec,ps", [(128, 16), (96, 48), (128, 128)])
@pytest.mark.parametrize("unrotate", [True, False])
def test_read_back(rec, ps, unrotate):
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(ps)
    lens, hkv = [0, 1, 33, 300], 3
    kp, vp, table = R.make_pools(lens, ps, hkv, rec, rng)
    for max_len in (300, 333, 20):
        got = ops.dequantize_paged(cu(kp), cu(vp), cu(table), i32(lens), max_len, unrotate=unrotate)
        H = R.hadamard()
        for x, pool in zip(got, (kp, vp)):
            x = x.cpu().numpy()
            assert x.shape == (4, hkv, max_len, 128)
            for b, n in enumerate(lens):
                m = min(n, max_len)
                assert not x[b, :, m:].any()
                for h in range(hkv if m else 0):
                    y = R.values(R.sequence(pool, table[b], h, n)[:m])
                    # fp32: three roundings per value, seven per butterfly chain, of magnitudes up to the row's sum
                    e = 12 * 2.0 ** -24 * np.abs(y).sum(-1, keepdims=True) / (np.sqrt(128.0) if unrotate else 1.0)
                    y = y @ H if unrotate else y
                    assert (np.abs(x[b, h, :m] - y) <= 2.0 ** -11 * np.abs(y) + e + 2.0 ** -25).all()
    one = ops.dequantize_paged(cu(kp), None, cu(table), i32(lens), 300, unrotate=unrotate)
    assert torch.equal(one, ops.dequantize_paged(cu(kp), cu(vp), cu(table), i32(lens), 300, unrotate=unrotate)[0])


def test_read_back_refusals_and_flag():
    import custom_ecc_cuda as ops
    pool = torch.zeros(8, 2, 16, 128, dtype=torch.uint8, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
    n = i32([64, 64])
    for bad in (dict(max_len=-1), dict(seq_lens=n[:1]), dict(v_pool=pool[..., :96]),
                dict(out=(torch.zeros(2, 2, 5, 128, device="cuda"),) * 2), dict(block_table=table.long())):
        with pytest.raises(RuntimeError):
            ops.dequantize_paged(**{**dict(k_pool=pool, v_pool=pool, block_table=table, seq_lens=n, max_len=5), **bad})
    x, _ = ops.dequantize_paged(pool, pool, table + 5, n, 64)
    assert ops.device_status(reset=True) == 5 and not x.any()
