"""Sampling from given uniform numbers against a plain implementation in 64
bits.  Tokens are equal: the kernel's masses are exact to 2^-45, so a draw can
differ only where a given number lies that close to a border."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def reference(x, u, T, k, p, mp):
    """One row, float64: (token, logprob, kept tokens)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    best = x.max()
    if best == -np.inf:
        return -1, -np.inf, []
    if not T > 0:
        return int(x.argmax()), 0.0, [int(x.argmax())]
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[:k] if k > 0 else order
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[order] == best, 1.0, np.exp((x[order] - best) / np.float64(T)))
    if p < 1:
        before = np.cumsum(w) - w
        c = max(1, int((before < p * w.sum()).sum()))
        order, w = order[:c], w[:c]
    ok = (w >= mp) & (w > 0)
    ok[0] = True
    ids, w = order[ok], w[ok]
    s = np.argsort(ids)
    ids, w = ids[s], w[s]
    cum = np.cumsum(w)
    j = min(int((cum <= u * cum[-1]).sum()), len(ids) - 1)
    return int(ids[j]), float(np.log(w[j] / cum[-1])), ids.tolist()


def check(x, u, T=1.0, k=0, p=1.0, mp=0.0):
    import custom_ecc_cuda as ops
    B = x.shape[0]
    tok, lp = ops.sample_tokens(x, u, temperature=T, top_k=k, top_p=p, min_p=mp, return_logprobs=True)
    assert torch.equal(tok, ops.sample_tokens(x, u, temperature=T, top_k=k, top_p=p, min_p=mp))
    col = lambda v: (v.cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, v, np.float32))  # noqa: E731
    T, k, p, mp, un = col(T), col(k), col(p), col(mp), u.cpu().numpy().astype(np.float64)
    xs = x.float().cpu().numpy()
    for b in range(B):
        t, l, _ = reference(xs[b], un[b], np.float64(T[b]), int(k[b]), np.float64(p[b]), np.float64(mp[b]))
        assert int(tok[b]) == t, (b, int(tok[b]), t)
        # the last rounding to fp32, and 2^-44 of the probabilities before it
        assert (l == float(lp[b])) or abs(float(lp[b]) - l) <= 2.0 ** -24 * abs(l) + 2.0 ** -40
    return tok


def rows(B, V, dtype, seed, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, V, generator=g, device="cuda") * spread
    top = torch.randint(0, V, (B, 20), generator=g, device="cuda")
    x.scatter_(1, top, 4 + 6 * torch.rand(B, 20, generator=g, device="cuda"))
    return x.to(TYPES[dtype]), torch.rand(B, generator=g, device="cuda")


SETTINGS = [dict(), dict(T=0.0), dict(T=0.6), dict(k=1), dict(k=7), dict(k=50, p=0.9, T=0.7), dict(p=0.5), dict(p=0.95),
            dict(p=0.01), dict(mp=0.05), dict(mp=1.0), dict(k=1000, p=0.99, mp=0.001, T=1.3), dict(T=5.0, p=0.9)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_sample_settings(dtype, setting):
    check(*rows(9, 5003, dtype, seed=len(str(setting))), **setting)


@pytest.mark.parametrize("V", [1, 2, 15, 16, 17, 31, 100, 513, 4096, 128256])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_sample_sizes(V, dtype):
    x, u = rows(3, V, dtype, seed=V)
    check(x, u)
    check(x, u, p=0.8, T=0.9)
    check(x, u, k=min(V, 40), p=0.9)


@pytest.mark.parametrize("B", [1, 5, 18, 40, 80, 300])
def test_sample_batches(B):
    check(*rows(B, 3001, "bf16", seed=B), p=0.9, T=0.8)


def test_sample_per_row_settings():
    x, u = rows(60, 2000, "fp16", seed=1)
    i = torch.arange(60, device="cuda")
    T = torch.tensor([0.7, 0.0, 1.0, 1e-30, 2.0, 1e30], device="cuda")[i % 6]
    k = torch.tensor([0, 1, 5, 3000, -2], dtype=torch.int32, device="cuda")[i % 5]
    p = torch.tensor([0.9, 1.0, 0.3, 2.0], device="cuda")[i % 4]
    mp = torch.tensor([0.0, 0.1, 0.0], device="cuda")[i % 3]
    check(x, u, T, k, p, mp)
    p = torch.tensor([0.0, -1.0], device="cuda")[i % 2].contiguous()  # the most likely token alone
    check(x, u, 0.5, 0, p, 0.0)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sample_equal_logits(dtype):
    u = torch.tensor([0.0, 0.1, 0.25, 0.4999999, 0.5, 0.75, 0.999999], device="cuda")
    x = torch.zeros(7, 1000, dtype=TYPES[dtype], device="cuda")
    for s in (dict(), dict(k=10), dict(p=0.5), dict(k=100, p=0.25), dict(mp=1.0), dict(mp=0.5, k=3)):
        check(x, u, **s)
    x[:, ::3] = -2.5  # two values, one of them negative, both many times
    x[:, 5] = -0.0
    for s in (dict(), dict(k=10), dict(k=700), dict(p=0.5), dict(p=0.97), dict(k=800, p=0.99), dict(T=0.3, p=0.9999)):
        check(x, u, **s)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sample_more_equal_logits_than_the_list_holds(dtype):
    u = torch.tensor([0.0, 0.1, 0.25, 0.4999999, 0.5, 0.75, 0.999999], device="cuda")
    x = torch.full((7, 30000), -1.5, dtype=TYPES[dtype], device="cuda")
    for s in (dict(), dict(k=10), dict(k=20000), dict(p=0.5), dict(k=20000, p=0.25), dict(mp=1.0), dict(T=0.0)):
        check(x, u, **s)
    x[:, ::3] = 0.75  # 10000 and 20000 of two values, and a few others
    x[:, 5::1001] = -0.0
    x[:, 7::999] = 3.0
    for s in (dict(), dict(k=10), dict(k=9000), dict(k=25000), dict(p=0.5), dict(p=0.97), dict(k=25000, p=0.99),
              dict(k=9000, p=0.999), dict(T=0.3, p=0.9999), dict(k=20000, p=0.6, mp=0.01)):
        check(x, u, **s)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sample_masks_infinities_and_nan(dtype):
    x, u = rows(8, 700, dtype, seed=3)
    inf = float("inf")
    x[0] = -inf
    x[1, 100:] = -inf
    x[2, :699] = -inf
    x[3] = float("nan")
    x[4, ::2] = float("nan")
    x[5, [7, 300, 650]] = inf
    x[6, 3] = inf
    x[6, 600:] = -inf
    x[7, :] = torch.finfo(x.dtype).min  # a mask by the type's lowest value, everywhere
    for s in (dict(), dict(T=0.0), dict(k=5), dict(k=690), dict(p=0.9), dict(p=0.5, k=2), dict(mp=0.1)):
        tok = check(x, u, **s)
        assert int(tok[0]) == -1 and int(tok[3]) == -1


def test_sample_extreme_numbers():
    x, _ = rows(6, 333, "fp32", seed=4)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan")], device="cuda")
    import custom_ecc_cuda as ops
    tok = ops.sample_tokens(x, u)
    check(x[:2], u[:2])
    kept = [reference(x[b].cpu().numpy(), 0.5, 1.0, 0, 1.0, 0.0)[2] for b in range(6)]
    assert int(tok[2]) == kept[2][-1] and int(tok[3]) == kept[3][-1] and int(tok[4]) == kept[4][0]
    assert 0 <= int(tok[5]) < 333


@pytest.mark.parametrize("scale", [1.0, 1e30])
@pytest.mark.parametrize("T", [1e-30, 1e-3, 1e30, 3e38, float("inf")])
def test_sample_extreme_temperatures(T, scale):
    x, u = rows(4, 2500, "fp32", seed=5)
    x *= scale
    x[1, 3] = torch.finfo(x.dtype).min  # finite: as likely as any other when the temperature is infinite
    for s in (dict(), dict(k=2000), dict(p=0.7), dict(mp=0.5), dict(k=400, p=0.3)):
        check(x, u, T=T, **s)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("V,allowed", [(9000, 100), (128256, 100), (128256, 4096), (128256, 5000), (60, 7)])
def test_sample_infinite_temperature_over_a_masked_row(V, allowed, dtype):
    """Every allowed token weighs the same, a masked one (-inf or NaN) nothing: with equal weights the kept tokens are
    the first by (logit, index) and the draw is token floor(u * kept) of them, ascending."""
    import custom_ecc_cuda as ops
    rng = np.random.default_rng(V + allowed)
    x = np.full((6, V), -np.inf, np.float32)
    ids = [np.sort(rng.choice(V, allowed, replace=False)) for _ in range(6)]
    for b in range(6):
        x[b, rng.choice(V, V // 8, replace=False)] = np.nan
        x[b, ids[b]] = rng.normal(size=allowed)
    xs = torch.from_numpy(x).to(TYPES[dtype])
    x = xs.float().numpy()
    u = np.array([0.0, 0.2, 0.4999, 0.71, 0.93, 0.99999], np.float32)
    inf = torch.full((6,), float("inf"), device="cuda")
    for k, p in ((0, 1.0), (50, 1.0), (0, 0.35), (50, 0.55), (3000, 1.0), (3000, 0.35), (V - 1, 1.0)):
        for T in (float("inf"), inf):
            out = torch.full((6,), -7, device="cuda")
            tok, lp = ops.sample_tokens(xs.cuda(), torch.from_numpy(u).cuda(), temperature=T, top_k=k, top_p=p,
                                        return_logprobs=True, out=out)
            for b in range(6):
                order = ids[b][np.lexsort((ids[b], -x[b, ids[b]]))]
                order = order[:k] if k else order
                if p < 1:
                    order = order[:int(np.ceil(np.float64(np.float32(p)) * len(order)))]
                want = np.sort(order)[int(np.float64(u[b]) * len(order))]
                assert int(tok[b]) == want, (k, p, b)
                l = np.log(len(order))
                assert abs(float(lp[b]) + l) <= 2.0 ** -24 * l + 2.0 ** -40


def exact_draws(x, u, p=1.0):
    """Tokens of one row of logits for many numbers, at temperature 1: integer sums of weights to 2^-100, rounded from 60
    decimal digits.  Also how far each number lies from the next border, as a part of the kept sum."""
    from bisect import bisect_left, bisect_right
    from decimal import Decimal, getcontext
    from itertools import accumulate
    getcontext().prec = 60
    best = Decimal(float(x.max()))
    weight = {v: int((Decimal(v) - best).exp() * (1 << 100)) for v in set(x.tolist())}
    w = [weight[v] for v in x.tolist()]
    ids = list(range(len(w)))
    gap = 1.0
    if p < 1:
        order = sorted(ids, key=lambda i: (-x[i], i))
        before = [0] + list(accumulate(w[i] for i in order))
        m, shift = int(np.float64(np.float32(p)) * (1 << 60)), 60  # (exact: 24 bits)
        border = -(-m * before[-1] >> shift)  # kept: what begins below p * total
        c = bisect_left(before, border, 0, len(order))
        gap = min(abs(b - border) for b in before[max(0, c - 1):c + 1]) / before[-1]
        ids = sorted(order[:c])
    cum = list(accumulate(w[i] for i in ids))
    tok, gaps = [], []
    for v in u.tolist():
        target = int(np.float64(v) * (1 << 60)) * cum[-1] >> 60
        j = bisect_right(cum, target)
        tok.append(ids[j])
        gaps.append(min(gap, min(abs(b - target) for b in cum[max(0, j - 1):j + 1]) / cum[-1]))
    return np.array(tok), np.array(gaps)


@pytest.mark.parametrize("dtype,V,low,high,p,B", [
    ("bf16", 1 << 20, -13.875, -13.875, 1.0, 20000), ("bf16", 1 << 20, -15.0, -15.0, 1.0, 20000),
    ("fp16", 1 << 20, -15.0, -13.0, 1.0, 20000), ("fp16", 128256, -11.75, -11.75, 1.0, 20000),
    ("bf16", 128256, -20.0, -11.0, 1.0, 20000), ("bf16", 1 << 20, -13.875, -13.875, 0.75, 4000),
    ("fp16", 128256, -12.0, -11.0, 0.9, 4000), ("fp32", 1 << 20, -14.0, -14.0, 1.0, 500),
    ("fp16", 1 << 20, -40.0, -30.0, 1.0, 4000)])
def test_sample_one_peak_and_a_long_flat_tail(dtype, V, low, high, p, B):
    """Each token of the tail weighs next to nothing, all of them as much as the peak: a rounding of every weight in the
    same direction would move the draws along the tail.  Running sums are off by at most V 2^-61 + 2^-45 of the whole
    (each weight by half a unit 2^-S < 2^-61 of the sum, and by 2^-45 of itself), the same again for the total that
    the number multiplies: draws that lie closer to a border are not compared, and there are few."""
    import custom_ecc_cuda as ops
    g = torch.Generator().manual_seed(V)
    steps = int(round((high - low) * 8))
    x = (low + torch.randint(0, steps + 1, (V,), generator=g) / 8.0).to(TYPES[dtype])
    x[V // 3] = 0.0
    u = torch.rand(B, generator=g)
    tok, lp = ops.sample_tokens(x.cuda()[None].expand(B, V), u.cuda(), top_p=p, return_logprobs=True)
    want, gaps = exact_draws(x.float().numpy(), u.numpy(), p)
    clear = gaps > 2 * (V * 2.0 ** -61 + 2.0 ** -45)
    assert clear.mean() > 0.999
    assert np.array_equal(tok.cpu().numpy()[clear], want[clear]), (tok.cpu().numpy() != want)[clear].sum()
    assert torch.isfinite(lp).all()


def test_sample_distribution():
    """Evenly spaced numbers draw every token in proportion to its probability, to one part in their count."""
    import custom_ecc_cuda as ops
    n = 4096
    x = torch.tensor([[2.0, 0.0, -1.0, 1.0, -30.0, 1.5]], device="cuda").expand(n, 6).contiguous()
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(ops.sample_tokens(x, u), minlength=6).double() / n
    assert (got - torch.softmax(x[0].double(), 0)).abs().max() <= 1.0 / n


def test_sample_strided_and_unaligned_rows():
    g = torch.Generator(device="cuda").manual_seed(0)
    wide = torch.randn(4, 3, 1001, generator=g, device="cuda").half()
    u = torch.rand(4, generator=g, device="cuda")
    check(wide[:, 1], u, p=0.9)         # rows 3003 elements apart: not 16-byte aligned
    check(wide[:, 2, 1:], u, k=9)
    check(wide[:1, 0].expand(4, 1001), u)  # one row for all


def test_sample_row_larger_than_shared_memory():
    check(*rows(2, 1 << 20, "fp32", seed=9), T=0.8, p=0.9)


def test_sample_in_a_graph_and_on_a_stream():
    import custom_ecc_cuda as ops
    x, u = rows(5, 4001, "bf16", seed=2)
    ops.sample_tokens(x, u, top_k=5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = ops.sample_tokens(x, u, temperature=0.9, top_k=50, top_p=0.9, return_logprobs=True)
    for s in range(3):
        nx, nu = rows(5, 4001, "bf16", seed=20 + s)
        x.copy_(nx), u.copy_(nu)
        graph.replay()
        assert torch.equal(tok, ops.sample_tokens(nx, nu, temperature=0.9, top_k=50, top_p=0.9))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = ops.sample_tokens(x, u)
    side.synchronize()
    assert torch.equal(a, ops.sample_tokens(x, u))


def test_sample_refusals():
    import custom_ecc_cuda as ops
    x, u = rows(4, 100, "fp32", seed=0)
    for kw in (dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=x.double()), dict(logits=x.t()),
               dict(logits=x[:, :0]), dict(uniform=u[:3]), dict(uniform=u.double()), dict(uniform=u.cpu()),
               dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=0.0), dict(top_p=-0.5),
               dict(min_p=1.5), dict(min_p=-0.1), dict(temperature=u[:2]), dict(top_k=u), dict(top_p=u.half()),
               dict(out=torch.zeros(4, dtype=torch.int32, device="cuda"))):
        with pytest.raises(RuntimeError):
            ops.sample_tokens(**{**dict(logits=x, uniform=u), **kw})
    with pytest.raises(RuntimeError):
        ops.sample_tokens(torch.zeros(1, (1 << 20) + 1, dtype=torch.float16, device="cuda"), u[:1])
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,)
