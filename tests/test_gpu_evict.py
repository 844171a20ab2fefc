"""Eviction from a paged cache by accumulated attention weight, against a
plain implementation: positions, weights and blocks are equal, not close."""
import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def cu(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def i32(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def keep_of(w, n, budget, sinks, recent):
    if n <= budget:
        return list(range(n))
    mid = range(sinks, n - recent)
    # NaN above everything, then larger weights, then the earlier token
    order = sorted(mid, key=lambda t: (not np.isnan(w[t]), -(w[t] if not np.isnan(w[t]) else 0.0), t))
    return list(range(sinks)) + sorted(order[:budget - sinks - recent]) + list(range(n - recent, n))


def check(lens, hkv, ps, rec, budget, sinks, recent, weights=None, seed=0, spare=3):
    import custom_ecc_cuda as ops
    ops.device_status(reset=True)
    rng = np.random.default_rng(seed)
    B = len(lens)
    out_w = -(-budget // ps)
    kp, vp, table = R.make_pools(lens, ps, hkv, rec, rng, extra=B * out_w + spare)
    kp[kp == 0xFF] = 7
    used = set(int(table[b, c]) for b, n in enumerate(lens) for c in range(-(-n // ps)))
    free = [p for p in range(kp.shape[0]) if p not in used]
    out_table = np.array(rng.permutation(free)[:B * out_w], np.int32).reshape(B, out_w)
    cap = table.shape[1] * ps
    w = weights(rng, B, hkv, cap) if weights else rng.random((B, hkv, cap))
    w = w.astype(np.float32)
    kd, vd = cu(kp), cu(vp)
    ow, kept = ops.evict_paged(kd, vd, cu(table), i32(lens), cu(w), cu(out_table), budget, sinks=sinks, recent=recent)
    assert ops.device_status(reset=True) == 0
    want_k, want_v, want_w = kp.copy(), vp.copy(), np.zeros_like(w)
    want_kept = np.full((B, hkv, budget), -1, np.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            ids = keep_of(w[b, h], n, budget, sinks, recent)
            want_kept[b, h, :len(ids)] = ids
            want_w[b, h, :len(ids)] = w[b, h, ids]
            for o, t in enumerate(ids):
                src, dst = (table[b, t // ps], h, t % ps), (out_table[b, o // ps], h, o % ps)
                want_k[dst], want_v[dst] = kp[src], vp[src]
    assert np.array_equal(kept.cpu().numpy(), want_kept)
    assert np.array_equal(ow.cpu().numpy(), want_w, equal_nan=True)
    assert np.array_equal(kd.cpu().numpy(), want_k) and np.array_equal(vd.cpu().numpy(), want_v)


@pytest.mark.parametrize("ps,rec", [(16, 128), (48, 96), (64, 128)])
def test_evict_ragged(ps, rec):
    check([0, 1, 50, 51, 77, 600, 300], 3, ps, rec, 50, 4, 10, seed=ps)


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (40, 20, 20), (199, 0, 0), (199, 3, 5),
                                                 (64, 0, 64), (64, 64, 0), (500, 4, 4)])
def test_evict_budgets(budget, sinks, recent):
    check([200, 64, 65], 2, 16, 128, budget, sinks, recent, seed=budget)


def _ties(rng, B, H, n):
    return rng.integers(0, 3, (B, H, n)) * 0.25


def _zeros(rng, B, H, n):
    return np.where(rng.random((B, H, n)) < 0.5, 0.0, -0.0)


def _special(rng, B, H, n):
    w = rng.random((B, H, n)) ** 8
    w[rng.random(w.shape) < 0.05] = np.inf
    w[rng.random(w.shape) < 0.05] = -np.inf
    w[rng.random(w.shape) < 0.05] = np.nan
    w[rng.random(w.shape) < 0.1] = -1.0
    w[rng.random(w.shape) < 0.1] = 1e-42
    return w


@pytest.mark.parametrize("weights", [_ties, _zeros, _special])
@pytest.mark.parametrize("budget", [30, 200])
def test_evict_equal_and_special_weights(weights, budget):
    check([700, 250], 2, 16, 128, budget, 2, 9, weights=weights, seed=budget)


def _one_value(rng, B, H, n):
    return np.full((B, H, n), 0.125)


def _three_values(rng, B, H, n):
    w = rng.integers(0, 3, (B, H, n)) * 0.25
    w[..., ::7] = rng.random((B, H, w[..., ::7].shape[-1]))
    return w


@pytest.mark.parametrize("weights", [_one_value, _three_values])
@pytest.mark.parametrize("B,hkv", [(1, 1), (20, 3)])  # one row by a cluster, one CTA per row
def test_evict_more_equal_weights_than_the_list_holds(weights, B, hkv):
    check([20011 - 100 * b for b in range(B)], hkv, 64, 96, 9000, 4, 100, weights=weights, seed=B, spare=1)


def test_evict_one_long_row():
    check([20011], 1, 16, 128, 9000, 4, 100, seed=1)


@pytest.mark.parametrize("rows", [(3, 5), (25, 3), (40, 4)])
def test_evict_cluster_sizes(rows):
    check([90 + 13 * b for b in range(rows[0])], rows[1], 16, 128, 64, 1, 7, seed=rows[0])


def test_evict_slice_that_does_not_fit_in_shared_memory():
    import custom_ecc_cuda as ops
    n, budget, ps, B = 45000, 20000, 64, 80  # 160 rows: one CTA each
    w = torch.rand(B, 2, -(-n // ps) * ps, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    pages, outs = -(-n // ps), -(-budget // ps)
    # one sequence's pages serve all of them as the source
    pool = torch.randint(0, 256, (pages + B * outs, 2, ps, 96), dtype=torch.uint8, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(B, pages).contiguous()
    out_table = (pages + torch.arange(B * outs, dtype=torch.int32, device="cuda")).view(B, outs)
    ow, kept = ops.evict_paged(pool, pool.clone(), table, i32([n] * B), w, out_table, budget, recent=50)
    assert ops.device_status(reset=True) == 0
    top = w[..., :n - 50].topk(budget - 50).indices.sort(-1).values
    assert torch.equal(kept[..., :budget - 50].long(), top)  # no equal weights at this border
    assert torch.equal(ow[..., :budget], w.gather(-1, kept.long()))
    for b in (0, 79):
        got = pool[out_table[b].long()].transpose(0, 1).reshape(2, -1, 96)[:, :budget]
        src = pool[:pages].transpose(0, 1).reshape(2, -1, 96)
        assert torch.equal(got, torch.stack([src[h, kept[b, h].long()] for h in range(2)]))


def test_evict_clashing_pages_move_nothing():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(0)
    kp, vp, table = R.make_pools([100, 100], 16, 2, 128, rng, extra=8)
    w = cu(rng.random((2, 2, 112)).astype(np.float32))
    used = set(table.reshape(-1).tolist())
    free = [p for p in range(kp.shape[0]) if p not in used][:8]
    good = np.array(free, np.int32).reshape(2, 4)
    same = good.copy()
    same[1, 2] = good[0, 0]          # twice
    taken = good.copy()
    taken[0, 1] = table[1, 3]        # holds a token
    for t in (same, taken):
        kd, vd = cu(kp), cu(vp)
        ops.evict_paged(kd, vd, cu(table), i32([100, 100]), w, cu(t), 60)
        assert ops.device_status(reset=True) == 5
        assert np.array_equal(kd.cpu().numpy(), kp) and np.array_equal(vd.cpu().numpy(), vp)
    for t, out in ((table + 1000, good), (table, good - 1000)):  # pages that do not exist
        kd, vd = cu(kp), cu(vp)
        ops.evict_paged(kd, vd, cu(t), i32([100, 100]), w, cu(out), 60)
        assert ops.device_status(reset=True) == 5
        assert np.array_equal(kd.cpu().numpy(), kp) and np.array_equal(vd.cpu().numpy(), vp)


def test_evict_refusals():
    import custom_ecc_cuda as ops
    pool = torch.zeros(20, 2, 16, 128, dtype=torch.uint8, device="cuda")
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    out = table + 8
    w, n = torch.zeros(2, 2, 64, device="cuda"), i32([64, 64])
    wide = torch.zeros(2, 2, 96, device="cuda")
    args = dict(k_pool=pool, v_pool=pool.clone(), block_table=table, seq_lens=n, weights=w, out_table=out, budget=40)
    ops.evict_paged(**args)
    both = torch.zeros(2, 2, 2, 64, device="cuda")  # two halves of one tensor are two tensors
    ops.evict_paged(**{**args, "weights": both[0], "out_weights": both[1]})
    for b in (dict(budget=0), dict(budget=65), dict(sinks=-1), dict(recent=-1), dict(sinks=30, recent=11),
              dict(out_table=table), dict(out_table=out[:1]), dict(out_table=out.long()), dict(weights=w.half()),
              dict(weights=w[..., :63]), dict(weights=w[:1]), dict(out_weights=w), dict(weights=wide[:, :, :64], out_weights=wide[:, :, 32:96]), dict(seq_lens=n[:1]),
              dict(kept=torch.zeros(2, 2, 39, dtype=torch.int32, device="cuda")), dict(k_pool=pool[..., :96]),
              dict(workspace=torch.zeros(4, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(RuntimeError):
            ops.evict_paged(**{**args, **b})


def test_evict_in_a_graph():
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(3)
    kp, vp, table = R.make_pools([300, 300], 16, 2, 128, rng, extra=20)
    used = set(table.reshape(-1).tolist())
    out = cu(np.array([p for p in range(kp.shape[0]) if p not in used][:16], np.int32).reshape(2, 8))
    kd, vd, td, n, w = cu(kp), cu(vp), cu(table), i32([1, 1]), torch.zeros(2, 2, 304, device="cuda")
    ws = torch.empty(4096, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.evict_paged(kd, vd, td, n, w, out, 100, sinks=2, recent=5, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ow, kept = ops.evict_paged(kd, vd, td, n, w, out, 100, sinks=2, recent=5, workspace=ws)
    for lens in ([300, 120], [0, 299]):
        n.copy_(i32(lens))
        w.copy_(cu(rng.random((2, 2, 304)).astype(np.float32)))
        graph.replay()
        want = [[keep_of(w[b, h].cpu().numpy(), lens[b], 100, 2, 5) for h in range(2)] for b in range(2)]
        got = kept.cpu().numpy()
        for b in range(2):
            for h in range(2):
                ids = want[b][h]
                assert got[b, h, :len(ids)].tolist() == ids and (got[b, h, len(ids):] == -1).all()
                assert torch.equal(ow[b, h, :len(ids)], w[b, h][torch.tensor(ids, dtype=torch.long, device="cuda")])
