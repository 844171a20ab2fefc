"""Plain 64-bit implementations of the paged-cache operators (numpy), with the
error that the kernels' arithmetic may add to each value, from the inputs."""
import numpy as np

LEVELS = np.array([0xc019a6b5, 0xbfebf7cf, 0xbfb7f2e5, 0xbf8cb5dd, 0xbf4cb296, 0xbf05bc02, 0xbe8432ca, 0, 0x3e8432ca,
                   0x3f05bc02, 0x3f4cb296, 0x3f8cb5dd, 0x3fb7f2e5, 0x3febf7cf, 0x4019a6b5, 0x404a233a],
                  dtype=np.uint32).view(np.float32).astype(np.float64)
SM = 1.0 / np.sqrt(128.0)


def hadamard():
    h = np.ones((1, 1))
    for _ in range(7):
        h = np.block([[h, h], [h, -h]])
    return h / np.sqrt(128.0)


def records(n, rec, rng, garbage=False):
    """n records of random codes and signs with scale 0.5..1.5, small zero point, alpha ~ 0.1 scale; `garbage`: 0xFF in
    every byte (NaN metadata), as memory that was never written may read."""
    out = np.zeros((n, rec), np.uint8)
    if garbage:
        out[:] = 0xFF
        return out
    out[:, :80] = rng.integers(0, 256, (n, 80))
    meta = np.empty((n, 3), np.float16)
    meta[:, 0] = rng.uniform(0.5, 1.5, n)
    meta[:, 1] = rng.uniform(-0.2, 0.2, n)
    meta[:, 2] = 0.11 * meta[:, 0]
    out[:, 80:86] = meta.view(np.uint8).reshape(n, 6)
    return out


def fields(blocks):
    """(levels [n, 128], signs [n, 128], meta [n, 3]) of records [n, rec], float64."""
    c = np.empty((blocks.shape[0], 128))
    c[:, 0::2] = LEVELS[blocks[:, :64] & 15]
    c[:, 1::2] = LEVELS[blocks[:, :64] >> 4]
    s = np.unpackbits(blocks[:, 64:80], axis=1, bitorder="little").astype(np.float64) * 2 - 1
    return c, s, np.ascontiguousarray(blocks[:, 80:86]).view(np.float16).astype(np.float64)


def values(blocks):
    c, s, m = fields(blocks)
    return c * m[:, 0:1] + m[:, 1:2] + m[:, 2:3] * s


def sequence(pool, table_row, h, n):
    """Records of a sequence's first n tokens for kv head h."""
    ps = pool.shape[2]
    pages = -(-n // ps)
    return pool[table_row[:pages], h].reshape(-1, pool.shape[3])[:n]


def visible(n, window, sinks):
    t = np.arange(n)
    return t[(t >= n - window) | (t < sinks)] if window else t


def attend(q, k_pool, v_pool, table, lens, window=0, sinks=0, rotate=False):
    """q [B, Hq, 128] fp16 -> out [B, Hq, 128], lse [B, Hq], weights [B, Hkv, tokens] and the error bound of each.

    Bounds (u = 2^-11, half a step of fp16; w = 2^-22):
    * a score: the tensor-core sum of 128 products (hi + lo parts carry a level to w relative, eight chained steps each
      lose at most w of the magnitudes added), so 12 w sm sum |q| (|C| scale + 2 alpha + |zero|), plus w |s|; a query
      rotated inside is carried to 2^-14 at least (fp16 and a remainder of three bits), which adds u/8 sm sum |q||k|;
    * the values' centroids are carried as one fp16 each (of the level times a factor chosen for it): 8.6e-5 of
      |C| scale at most;
    * a probability: twice the largest score error, plus the 2^-21 of two base-2 exponentials, relative;
    * an output: the probabilities' error times sum p |v|, the fp16 sign weights u alpha, 16 w of the sums, and u |out|
      for the last rounding; the inverse rotation adds up the bounds of 128 elements over sqrt(128)."""
    B, Hq, _ = q.shape
    Hkv = k_pool.shape[1]
    G, H, u, w = Hq // Hkv, hadamard(), 2.0 ** -11, 2.0 ** -22
    cap = table.shape[1] * k_pool.shape[2]
    out, tol = np.zeros((B, Hq, 128)), np.zeros((B, Hq, 128))
    lse, lse_tol = np.full((B, Hq), -np.inf), np.zeros((B, Hq))
    wsum, w_tol = np.zeros((B, Hkv, cap)), np.zeros((B, Hkv, cap))
    for b in range(B):
        n = int(lens[b])
        t = visible(n, window, sinks)
        for h in range(Hkv if n else 0):
            kb, vb = sequence(k_pool, table[b], h, n)[t], sequence(v_pool, table[b], h, n)[t]
            k, v = values(kb), values(vb)
            kc, _, km = fields(kb)
            size = np.abs(kc) * km[:, 0:1] + 2 * km[:, 2:3] + np.abs(km[:, 1:2])
            alpha = fields(vb)[2][:, 2]
            for g in range(G):
                x = q[b, h * G + g].astype(np.float64)
                x = x @ H if rotate else x
                s = SM * (k @ x)
                e = 12 * w * SM * (size @ np.abs(x)) + w * np.abs(s)
                if rotate:
                    e = e + u / 8 * SM * (np.abs(k) @ np.abs(x))
                e = e.max()
                m = s.max()
                p = np.exp(s - m)
                lse[b, h * G + g] = m + np.log(p.sum())
                lse_tol[b, h * G + g] = e + 4 * w * (1 + abs(lse[b, h * G + g]))
                p /= p.sum()
                rel = 2 * e + 2.0 ** -21
                wsum[b, h, t] += p
                w_tol[b, h, t] += p * (rel + 4 * w) + 2.0 ** -40
                o = p @ v
                d = rel * (p @ np.abs(v)) + u * (p @ alpha) + 16 * w * (p @ np.abs(v)) + 1e-7
                vc, _, vm = fields(vb)
                d = d + 8.6e-5 * (p @ (np.abs(vc) * vm[:, 0:1]))
                if rotate:
                    o, d = o @ H, np.full(128, d.sum() / np.sqrt(128.0))
                out[b, h * G + g], tol[b, h * G + g] = o, d + u * np.abs(o) + 2.0 ** -25
    return out, tol, lse, lse_tol, wsum, w_tol


def layout(lens, ps, extra, rng, width=None):
    """A page table of shuffled pages for the lengths (garbage behind each row) and the number of pages."""
    counts = [-(-n // ps) for n in lens]
    total = sum(counts) + extra
    perm = rng.permutation(total)
    width = max([1] + counts) if width is None else width
    table = np.full((len(lens), width), -1, np.int32)
    table[:, -1:] = 1 << 30
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return table, total


def make_pools(lens, ps, hkv, rec, rng, extra=1, width=None):
    """(k pool, v pool, table): every slot that no sequence's token owns reads 0xFF."""
    table, total = layout(lens, ps, extra, rng, width)
    pools = []
    for _ in range(2):
        pool = np.full((total, hkv, ps, rec), 0xFF, np.uint8)
        for b, n in enumerate(lens):
            for t0 in range(0, n, ps):
                c = min(ps, n - t0)
                pool[table[b, t0 // ps], :, :c] = records(hkv * c, rec, rng).reshape(hkv, c, rec)
        pools.append(pool)
    return pools[0], pools[1], table
