"""Plain forms in 64 bits of what a paged cache does about its size: attention with the weights of the cached tokens, and eviction. And the
batches that the tests use."""
import numpy as np
import torch

DEVICE = "cuda"


class Batch:
    """A paged batch of the given lengths (tokens in the cache). Pages come from a shuffled pool whose other slots hold NaN; `holes`: (sequence, page)
    entries that are unmapped; `prefixes`: (first sequence, end, tokens) whose whole pages are shared."""

    def __init__(self, lens, *, hq=8, hkv=2, d=64, bs=16, dtype=torch.bfloat16, seed=0, holes=(), prefixes=(), extra_pages=2, size=1.0, stale=float("nan")):
        gen = torch.Generator(device=DEVICE).manual_seed(seed)
        order = np.random.default_rng(seed)
        self.lens_host = np.array(lens, np.int32)
        self.hq, self.hkv, self.d, self.bs, self.dtype = hq, hkv, d, bs, dtype
        counts = -(-np.maximum(self.lens_host, 0) // bs)
        shared = np.zeros(len(lens), np.int64)
        for first, end, tokens in prefixes:
            shared[first + 1:end] = tokens // bs
        taken = np.maximum(counts - shared, 0)
        blocks = int(taken.sum()) + 3
        ids = order.permutation(blocks).astype(np.int32)
        self.blocks, self.width = blocks, max(1, int(counts.max()) + extra_pages)
        table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for i in range(len(lens)):
            table[i, :min(shared[i], counts[i])] = table[i - 1, :min(shared[i], counts[i])]
            table[i, shared[i]:max(counts[i], shared[i])] = ids[at:at + taken[i]]
            at += taken[i]
        for s, page in holes:
            table[s, page] = -1
        self.table_host = table
        pool = lambda: (size * torch.randn((blocks, bs, hkv, d), generator=gen, device=DEVICE)).to(dtype)
        self.k, self.v = pool(), pool()
        if stale is not None:  # slots that no sequence has
            owned = np.zeros((blocks, bs), bool)
            for i, n in enumerate(lens):
                for j in range(n):
                    if table[i, j // bs] >= 0:
                        owned[table[i, j // bs], j % bs] = True
            spare = torch.from_numpy(~owned).to(DEVICE)
            for x in (self.k, self.v):
                x[spare] = stale
        self.table, self.lens = torch.from_numpy(table).to(DEVICE), torch.from_numpy(self.lens_host).to(DEVICE)
        self.q = torch.randn((len(lens), hq, 1, d), generator=gen, device=DEVICE).to(dtype)
        # what earlier steps have left; behind a sequence's last token too, where nothing may touch it
        self.weights = torch.rand((len(lens), hkv, self.width * bs), generator=gen, device=DEVICE)
        self.gen = gen

    def keys(self, s):
        """Tokens of sequence s that are on mapped pages, and their K and V in 64 bits, [tokens, kv heads, D]."""
        n = int(self.lens_host[s])
        at = np.array([j for j in range(n) if self.table_host[s, j // self.bs] >= 0], np.int64)
        slots = torch.from_numpy(self.table_host[s, at // self.bs].astype(np.int64) * self.bs + at % self.bs).to(DEVICE)
        pick = lambda x: x.reshape(-1, self.hkv, self.d)[slots].double()
        return at, pick(self.k), pick(self.v)


def attend(batch, q, s, new=None, causal=True, scale=None):
    """q [tokens, heads, D] of sequence s, the last `new` tokens of it (decode: all keys). Output [tokens, heads, D], weights [tokens, heads, keys],
    the keys' places, and the largest scale * sum |q||k| - what the rounding of a score goes by."""
    at, k, v = batch.keys(s)
    group = batch.hq // batch.hkv
    scale = batch.d ** -0.5 if scale is None else scale
    n = int(batch.lens_host[s])
    q = q.double()
    out = torch.zeros_like(q)
    p = torch.zeros((q.shape[0], batch.hq, len(at)), dtype=torch.float64, device=DEVICE)
    size = 0.0
    if len(at):
        for h in range(batch.hq):
            scores = scale * q[:, h] @ k[:, h // group].T
            size = max(size, float((scale * q[:, h].abs() @ k[:, h // group].abs().T).max()))
            if new is not None and causal:
                hidden = torch.from_numpy(at).to(DEVICE)[None, :] > torch.arange(n - new, n, device=DEVICE)[:, None]
                scores = scores.masked_fill(hidden, -torch.inf)
            some = torch.isfinite(scores).any(-1, keepdim=True)
            p[:, h] = torch.where(some, torch.softmax(torch.where(some, scores, 0.0), -1), 0.0)
            out[:, h] = p[:, h] @ v[:, h // group]
    return out, p, at, size


def weights_bound(d, keys, rows, size):
    """How far a sum of weights may be off, relative to the sum. A score is a sum of d products that are exact in 32 bits, each addition off by
    2^-23 of what is summed at most (the tensor core may cut instead of rounding): d * 2^-23 * size, where size is the sum of the products'
    sizes; scaling and the change to powers of two, 3 * 2^-24 of it more. An exponential takes that as a factor, once for the token and once for the
    sum of the row, and adds 2^-22 of its own each time; the sum of the row has `keys` additions, the sum over the rows `rows`."""
    score = (d + 2) * 2.0 ** -23 * size
    return 2 * score + 2 * 2.0 ** -22 + (keys + rows + 8) * 2.0 ** -24


def check_weights(got, before, added, bound, tag=""):
    """got = before + added: `bound` of what was added, and two roundings to 32 bits."""
    want = before.double() + added
    limit = bound * added.abs() + 2 * 2.0 ** -24 * want.abs() + 1e-37
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), tag
    worst = float((off / limit).max())
    assert worst <= 1, (worst, tag)
    return worst


def check_output(got, want, p, v, bound, p_step, tag=""):
    """got [heads, D] against want = p @ v [heads, D]: half a step of its type, and on the sum of p * |v| what a weight may be off (`bound`, see
    weights_bound) and the rounding of p to `p_step`, its product included; what is rounded at the end is off by that much, so a step of both."""
    group = want.shape[0] // v.shape[1]
    half = torch.finfo(got.dtype).eps / 2
    spread = torch.stack([p[h] @ v[:, h // group].abs() for h in range(want.shape[0])])
    limit = half * want.abs() + (1 + half) * (bound + p_step) * spread
    worst = float(((got.double() - want).abs() / limit).max())
    assert torch.isfinite(got).all() and worst <= 1, (worst, tag)


def evict(k, v, weights, table, lens, *, keep, recent=0, first=0):
    """New pools, weights and lengths, by the definition; all on the host as numpy arrays. k, v [blocks, bs, heads, row]."""
    k2, v2, w2 = k.copy(), v.copy(), weights.copy()
    bs, heads = k.shape[1], k.shape[2]
    new = lens.copy()
    for s, n in enumerate(lens):
        n = min(max(int(n), 0), table.shape[1] * bs)
        f = max(int(first[s]) if np.ndim(first) else int(first), 0)
        m = max(keep, f + recent)
        new[s] = min(n, m)
        if n <= m:
            continue
        for h in range(heads):
            w = weights[s, h]
            between = list(range(f, n - recent))
            weight = lambda j: (np.isnan(w[j]), 0.0 if np.isnan(w[j]) else w[j] + 0.0)
            kept = set(sorted(between, key=lambda j: (weight(j), -j), reverse=True)[:m - f - recent])
            free = [j for j in range(f, m - recent) if j not in kept]
            late = sorted(j for j in kept if j >= m - recent)
            moves = list(zip(late, free)) + [(n - recent + i, m - recent + i) for i in range(recent)]
            for src, dst in moves:
                a, b = table[s, src // bs], table[s, dst // bs]
                if 0 <= a < k.shape[0] and 0 <= b < k.shape[0]:
                    k2[b, dst % bs, h], v2[b, dst % bs, h] = k[a, src % bs, h], v[a, src % bs, h]
                w2[s, h, dst] = w[src]
            w2[s, h, m:n] = 0
    return k2, v2, w2, new
