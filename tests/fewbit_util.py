"""Shared by the tests of the few-bit entry points: types, 64-bit restatements, paged pools."""
import numpy as np
import torch

DT = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16)}


def half_step(name):
    """Largest relative error of one rounding to the type."""
    return torch.finfo(DT[name][1]).eps / 2


def ptr(t):
    return None if t is None else t.data_ptr()


def int8_rows(x):
    """The kernels' recipe in numpy, fp32 rows -> (int8, scale): scale = max|x| * (1/127), 1 where that is
    below 2^-126, q = clamp(rne(x * (1 / scale))); the maximum skips NaN, and a NaN product counts as
    INT_MIN."""
    x = np.ascontiguousarray(x, np.float32)
    with np.errstate(all="ignore"):
        sc = np.fmax.reduce(np.fmax(np.abs(x), 0), -1) * (np.float32(1) / np.float32(127))
        sc = np.where(sc < np.float32(2.0 ** -126), np.float32(1), sc)
        inv = (np.float32(1) / sc).astype(np.float32)
        p = x * inv[..., None]
        return np.where(np.isnan(p), -127, np.clip(np.rint(p), -127, 127)).astype(np.int8), sc


class Pool:
    """A paged cache on the GPU and the tables of its sequences.  `keys[b]` positions of sequence b
    lie on shuffled pages; every byte that belongs to no position is garbage (NaN scales)."""

    def __init__(self, sdq, rng, new, keys, heads, page, dim, spare=2, front=0, behind=0):
        self.sdq, self.heads, self.page, self.dim, self.new, self.keys = sdq, heads, page, dim, new, keys
        self.counts = [-(-k // page) for k in keys]
        self.pages = sum(self.counts) + spare
        self.wide = max(self.counts + [1])
        order = rng.permutation(self.pages)
        table = np.full((len(keys), self.wide), -7, np.int32)
        at = 0
        for b, n in enumerate(self.counts):
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table
        self.starts = np.concatenate([[front], front + np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + behind
        shape = (self.pages, heads, page)
        self.k = torch.from_numpy(rng.integers(-128, 128, shape + (dim,), dtype=np.int8)).cuda()
        self.v = torch.from_numpy(rng.integers(-128, 128, shape + (dim,), dtype=np.int8)).cuda()
        self.ks = torch.full(shape, float("nan"), device="cuda")
        self.vs = torch.full(shape, float("nan"), device="cuda")
        self.refresh()

    def refresh(self):
        self.d_start = torch.from_numpy(self.starts).cuda()
        self.d_len = torch.from_numpy(np.asarray(self.keys, np.int32)).cuda()
        self.d_table = torch.from_numpy(self.table).cuda()
        self.cache = self.sdq.kv_cache(ptr(self.k), ptr(self.v), ptr(self.ks), ptr(self.vs), self.pages, self.heads, self.page, self.dim)
        self.seqs = self.sdq.kv_seqs(ptr(self.d_start), ptr(self.d_len), ptr(self.d_table), len(self.keys), self.wide)

    def places(self, b):
        p = np.arange(self.keys[b])
        return self.table[b, p // self.page], p % self.page

    def fill(self, rng, spread=1.0):
        """Random codes and scales at every position of every sequence."""
        for b in range(len(self.keys)):
            pg, off = [torch.from_numpy(x.astype(np.int64)).cuda() for x in self.places(b)]
            for s in (self.ks, self.vs):
                sc = (0.005 + 0.02 * rng.random((self.keys[b], self.heads)) ** spread).astype(np.float32)
                s[pg, :, off] = torch.from_numpy(sc).cuda()

    def dense(self, b, which):
        """float64 [keys, heads, dim] of sequence b."""
        pg, off = self.places(b)
        q = (self.k if which == "k" else self.v).cpu().numpy()[pg, :, off].astype(np.float64)
        s = (self.ks if which == "k" else self.vs).cpu().numpy()[pg, :, off].astype(np.float64)
        return q * s[..., None]


def attention64(pool, q, heads, scale, causal, b):
    """Of the rows of sequence b: the output, sum p |v|, the largest sum |q k| of a score (each [rows, heads, ..]) and
    the sum of exp(score - largest score); q float64 [rows, heads, dim]."""
    group = heads // pool.heads
    k, v = pool.dense(b, "k"), pool.dense(b, "v")
    first, n, L = int(pool.starts[b]), pool.new[b], pool.keys[b]
    out = np.zeros((n, heads, pool.dim))
    mag = np.zeros_like(out)
    smag, total = np.zeros((n, heads)), np.ones((n, heads))
    if L == 0 or n == 0:
        return out, mag, smag, total
    qb = q[first:first + n]
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        s = scale * (qb[:, h] @ kk.T)
        a = scale * (np.abs(qb[:, h]) @ np.abs(kk).T)
        if causal:
            pos = L - n + np.arange(n)
            seen = np.arange(L)[None] <= pos[:, None]
        else:
            seen = np.ones((n, L), bool)
        s = np.where(seen, s, -np.inf)
        m = np.max(s, 1, keepdims=True)
        p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0.0)
        l = p.sum(1, keepdims=True)
        p = np.where(l > 0, p / np.where(l > 0, l, 1), 0.0)
        total[:, h] = np.maximum(l[:, 0], 1)
        out[:, h], mag[:, h], smag[:, h] = p @ vv, p @ np.abs(vv), np.max(np.where(seen, a, 0), 1)
    return out, mag, smag, total


def attention_tolerance(name, pool, b, heads, out, mag, smag, total):
    """What the kernel's roundings add up to at most, element by element.

    A score is off by its two factors' roundings (q in 11 bits of a power of two, or 22 with fp32; the
    codes are exact) and by an fp32 accumulation over at most 128 products: (2^-22 + 16 * 2^-23) sum|q k|.
    The maximum it is taken from and the multiplications by scales add 4 half steps of 2^-24 of it.
    exp turns that into a relative error of the weight, on the weight and on the sum: twice.  The
    weight is rounded once more to 11 bits (16-bit types) or 22 (fp32), and the exponential is good to
    2^-21.  Sums over the keys are fp32: 2^-23 for each addition of 16 keys, both in the weights'
    sum and in the output.  Then the output's own rounding: half a step relative to the value, and for
    fp16, whose numbers below 2^-14 lie on a grid of 2^-24, at least half of that grid (2^-25).

    Weights are fp16 numbers, and fp16's grid ends at 2^-24: a weight is off by 2^-25 units, however small it
    is.  With up to 32 rows to a sequence the units put the largest v_scale of the sequence into [2^14, 2^15):
    2^-39 of that scale, times codes of at most 2^7, for every key: keys * 2^-32 * max v_scale, over the sum
    of the p, which is 1 or more.  Tiles of 128 rows leave room above the running offset: their units are
    2^ev / 2^6 with 2^ev <= 2 max v_scale, so a weight is off by 2^-25 * 2^-5 = 2^-30 of that scale, and the
    keys by keys * 2^-23 * max v_scale over the sum of the p."""
    keys = pool.keys[b]
    pg, off = pool.places(b)
    vmax = float(pool.vs.cpu().numpy()[pg, :, off].max()) if keys else 0.0
    score = smag * (2.0 ** -22 + 16 * 2.0 ** -23 + 8 * 2.0 ** -24)
    few = pool.rows * (heads // pool.heads) <= 32 * len(pool.keys)
    grid = 2.0 ** -32 if few else 2.0 ** -23
    weight = 2.0 ** -11 if name != "f32" else 2.0 ** -21
    rel = 2 * score + weight + 2.0 ** -20 + 2 * (keys / 16 + 8) * 2.0 ** -23
    return rel[..., None] * mag + half_step(name) * np.abs(out) + (2.0 ** -25 if name == "f16" else 1e-30) + keys * grid * vmax / total[..., None]
