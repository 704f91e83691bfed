"""GPU: the paged int8 cache -- append and read back bit for bit, attention against 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from fewbit_util import DT, Pool, attention64, attention_tolerance, int8_rows, ptr

pytestmark = pytest.mark.gpu


def dense_rows(rng, rows, heads, dim, name):
    x = rng.standard_normal((rows, heads, dim)) * np.exp(rng.normal(0, 1, (rows, heads, 1)))
    x = torch.from_numpy(x.astype(np.float32)).to(DT[name][1])
    if rows > 3:
        x[1] = 0
        x[2, 0, dim // 2] = 300.0
    return x


def snapshot(pool):
    return [t.clone() for t in (pool.k, pool.v, pool.ks, pool.vs)]


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,keys,heads,page,dim,front,behind", [
    ([1], [1], 1, 16, 128, 0, 0), ([1, 1, 1], [5, 17, 64], 8, 16, 128, 0, 2), ([7], [7], 2, 4, 64, 0, 0),
    ([3, 0, 20, 1], [10, 4, 20, 33], 3, 7, 80, 2, 3), ([100, 31], [130, 31], 5, 64, 32, 0, 1), ([9, 9], [9, 900], 24, 48, 64, 0, 0),
    ([2] * 40, list(range(2, 42)), 1, 1, 16, 0, 0), ([300], [1000], 4, 128, 112, 5, 0), ([33], [64], 2, 32, 96, 0, 0),
])
def test_append_and_read_back(sdq, name, new, keys, heads, page, dim, front, behind):
    rng = np.random.default_rng(sum(keys) * 17 + dim)
    pool = Pool(sdq, rng, new, keys, heads, page, dim, front=front, behind=behind)
    k, v = [dense_rows(rng, pool.rows, heads, dim, name) for _ in range(2)]
    dk, dv = k.cuda(), v.cuda()
    before = snapshot(pool)
    sdq.kv_append(pool.cache, pool.seqs, ptr(dk), ptr(dv), DT[name][0], pool.rows)
    torch.cuda.synchronize()
    want = [t.cpu().numpy().copy() for t in before]
    back = [np.full((pool.rows, heads, dim), 9.0, np.float32) for _ in range(2)]
    for b in range(len(keys)):
        first, n = int(pool.starts[b]), new[b]
        pg, off = [x[keys[b] - n:] for x in pool.places(b)]
        for i, x in enumerate((k, v)):
            q, sc = int8_rows(x[first:first + n].float().numpy())
            want[i][pg, :, off], want[2 + i][pg, :, off] = q, sc
            back[i][first:first + n] = q.astype(np.float32) * sc[..., None]
    for got, w in zip((pool.k, pool.v, pool.ks, pool.vs), want):      # rows written, everything else left as it was
        assert np.array_equal(got.cpu().numpy().view(np.uint8), w.view(np.uint8))
    rk, rv = [torch.full((pool.rows, heads, dim), 9.0, device="cuda").to(DT[name][1]) for _ in range(2)]
    sdq.kv_read(pool.cache, pool.seqs, ptr(rk), ptr(rv), DT[name][0], pool.rows, flags=0x10)
    for got, w in zip((rk, rv), back):
        assert torch.equal(got.cpu(), torch.from_numpy(w).to(DT[name][1]))


def test_whole_sequences_read_in_one_call(sdq):
    rng = np.random.default_rng(3)
    keys = [100, 1, 57]
    pool = Pool(sdq, rng, keys, keys, 2, 16, 64)
    pool.fill(rng)
    k, v = [torch.empty(sum(keys), 2, 64, device="cuda") for _ in range(2)]
    sdq.kv_read(pool.cache, pool.seqs, ptr(k), ptr(v), 0, sum(keys), flags=0x10)
    for x, n in ((k, "k"), (v, "v")):
        want = np.concatenate([pool.dense(b, n) for b in range(3)]).astype(np.float32)
        assert np.array_equal(x.cpu().numpy(), want)


def test_strided_and_unaligned_rows(sdq):
    """k and v as slices of one fused projection, at an odd offset."""
    rng = np.random.default_rng(4)
    new, keys, heads, dim = [13, 6], [20, 6], 3, 48
    for name, ld, shift in (("bf16", 3 * heads * dim, 0), ("f32", 2 * heads * dim + 5, 1), ("f16", heads * dim + 8, 3)):
        pool = Pool(sdq, rng, new, keys, heads, 8, dim)
        flat = [torch.from_numpy(rng.standard_normal(pool.rows * ld + 8).astype(np.float32)).to(DT[name][1]).cuda() for _ in range(2)]
        k, v = [torch.as_strided(f, (pool.rows, heads, dim), (ld, dim, 1), shift) for f in flat]
        sdq.kv_append(pool.cache, pool.seqs, ptr(k), ptr(v), DT[name][0], pool.rows, ld=ld)
        out = [torch.full_like(f, 2.0) for f in flat]
        rk, rv = [torch.as_strided(f, (pool.rows, heads, dim), (ld, dim, 1), shift) for f in out]
        sdq.kv_read(pool.cache, pool.seqs, ptr(rk), ptr(rv), DT[name][0], pool.rows, ld=ld, flags=0x10)
        for x, r, f in ((k, rk, out[0]), (v, rv, out[1])):
            q, sc = int8_rows(x.float().cpu().numpy())
            want = torch.from_numpy(q.astype(np.float32) * sc[..., None]).to(DT[name][1])
            assert torch.equal(r.cpu(), want)
            mask = torch.ones_like(f, dtype=torch.bool)
            torch.as_strided(mask, (pool.rows, heads, dim), (ld, dim, 1), shift)[:] = False
            assert (f[mask] == 2.0).all()


def bad_pool(sdq, rng):
    """Sequences whose tables go wrong: a page outside the pool, a length beyond the table, more rows
    than positions, no positions at all."""
    pool = Pool(sdq, rng, [2, 4, 5, 3, 1], [40, 30, 2, 0, 16], 2, 8, 64, spare=4)
    pool.fill(rng)
    pool.table[0, 1] = pool.pages              # positions 8..15 of sequence 0
    pool.table[1, 3] = -1                      # 24..29 of sequence 1: all its new rows
    pool.keys[4] = 10 ** 6                     # far beyond the table
    pool.refresh()
    return pool


def test_bad_tables_stay_inside_the_pool(sdq):
    rng = np.random.default_rng(6)
    pool = bad_pool(sdq, rng)
    k, v = [dense_rows(rng, pool.rows, 2, 64, "f32") for _ in range(2)]
    dk, dv = k.cuda(), v.cuda()
    want = [t.cpu().numpy().copy() for t in snapshot(pool)]
    sdq.kv_append(pool.cache, pool.seqs, ptr(dk), ptr(dv), 0, pool.rows, flags=0x10)
    rk, rv = [torch.full((pool.rows, 2, 64), 9.0, device="cuda") for _ in range(2)]
    sdq.kv_read(pool.cache, pool.seqs, ptr(rk), ptr(rv), 0, pool.rows, flags=0x10)
    back = [np.zeros((pool.rows, 2, 64), np.float32) for _ in range(2)]
    # what has a place: both rows of sequence 0 (positions 38, 39), the last two rows of sequence 2
    for row, b, p in ((0, 0, 38), (1, 0, 39), (9, 2, 0), (10, 2, 1)):
        for i, x in enumerate((k, v)):
            q, sc = int8_rows(x[row].numpy())
            want[i][pool.table[b, p // 8], :, p % 8], want[2 + i][pool.table[b, p // 8], :, p % 8] = q, sc
            back[i][row] = q.astype(np.float32) * sc[:, None]
    for got, w in zip((pool.k, pool.v, pool.ks, pool.vs), want):
        assert np.array_equal(got.cpu().numpy().view(np.uint8), w.view(np.uint8))
    for got, w in zip((rk, rv), back):
        assert np.array_equal(got.cpu().numpy(), w)


# ---------------------------------------------------------------- attention
def attend(sdq, pool, q, heads, name, scale=None, causal=False, ldq=0, ldo=0, stream=None):
    out = torch.full((pool.rows, heads, pool.dim), 11.0, device="cuda").to(DT[name][1])
    sdq.kv_attention(pool.cache, pool.seqs, ptr(q), DT[name][0], pool.rows, heads, ptr(out), scale=scale, causal=causal,
                     ldq=ldq, ldo=ldo, stream=stream)
    torch.cuda.synchronize()
    return out


def compare(pool, out, q, heads, name, scale, causal):
    got, q64 = out.double().cpu().numpy(), q.double().cpu().numpy()
    covered = np.zeros(pool.rows, bool)
    for b in range(len(pool.keys)):
        want, *sizes = attention64(pool, q64, heads, scale, causal, b)
        rows = slice(int(pool.starts[b]), int(pool.starts[b]) + pool.new[b])
        covered[rows] = True
        tol = attention_tolerance(name, pool, b, heads, want, *sizes)
        err = np.abs(got[rows] - want)
        assert (err <= tol).all(), (b, np.nanmax(err / tol), np.isnan(err).sum())
    assert (got[~covered] == 11.0).all()      # rows of no sequence are left alone


SHAPES = [
    # new, keys, cache heads, query heads per cache head, page, dim
    ([1], [1], 1, 1, 16, 128), ([1], [2], 2, 1, 1, 64), ([1, 1], [16, 33], 2, 4, 16, 128), ([1], [1000], 1, 8, 64, 128),
    ([1, 1, 1, 1], [7, 300, 129, 64], 8, 4, 16, 64), ([1], [5000], 2, 1, 128, 80), ([1, 1], [777, 2049], 3, 5, 48, 112),
    ([1], [4097], 1, 16, 32, 128), ([1, 1], [90, 91], 2, 24, 16, 32), ([2, 1, 3], [50, 7, 200], 2, 4, 7, 16),
    ([5], [5], 4, 1, 16, 128), ([17, 1, 0, 40], [17, 600, 9, 90], 2, 2, 16, 64), ([64], [64], 2, 4, 64, 128),
    ([130], [700], 3, 1, 16, 128), ([65, 63], [1100, 65], 1, 8, 100, 96), ([200, 3], [200, 450], 2, 3, 32, 48),
    ([33], [3000], 24, 1, 64, 128), ([300], [301], 1, 2, 5, 128), ([257, 1], [513, 4000], 2, 4, 128, 128),
    # enough heads for the tiles of 128 rows, a tile to a block
    ([70, 5], [333, 640], 24, 4, 16, 128), ([9, 9, 9], [600, 9, 100], 40, 8, 7, 16), ([65], [65], 25, 5, 5, 112),
    ([2] * 70, list(range(2, 212, 3)), 4, 24, 16, 32), ([1000], [1000], 7, 1, 64, 64), ([33, 0, 40], [900, 5, 41], 30, 2, 100, 48),
    # few enough tiles for 2, 4 and 8 blocks to share one's keys; blocks that have none
    ([40, 1, 30], [500, 300, 30], 24, 4, 16, 64), ([130], [2100], 8, 4, 48, 128), ([3, 60], [100, 2500], 16, 2, 64, 80),
    ([28], [4097], 8, 4, 32, 128), ([257], [1030], 8, 3, 128, 96), ([34, 34], [2049, 34], 7, 3, 33, 16), ([128], [129], 8, 1, 2048, 128),
]


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, (len(s[0]), max(s[0]), max(s[1])) + s[2:])))
def test_attention(sdq, name, causal, shape):
    new, keys, kv, group, page, dim = shape
    rng = np.random.default_rng(sum(keys) * 7 + dim + group)
    pool = Pool(sdq, rng, new, keys, kv, page, dim, front=1, behind=2)
    pool.fill(rng)
    heads = kv * group
    q = torch.from_numpy((1.3 * rng.standard_normal((pool.rows, heads, dim))).astype(np.float32)).to(DT[name][1]).cuda()
    out = attend(sdq, pool, q, heads, name, causal=causal)
    compare(pool, out, q, heads, name, dim ** -0.5, causal)
    assert torch.equal(out, attend(sdq, pool, q, heads, name, causal=causal))      # same bits again


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,kv", [([1, 1], 2), ([70, 5], 2), ([70, 5], 24), ([70, 5], 12)])
def test_peaked_scores_and_uneven_scales(sdq, name, new, kv):
    """Large logits, and value scales five orders of magnitude apart."""
    rng = np.random.default_rng(31)
    pool = Pool(sdq, rng, new, [333, 640], kv, 16, 128)
    pool.fill(rng)
    for s, lo, hi in ((pool.ks, 0, 1.5), (pool.vs, -5, 0)):
        s *= torch.from_numpy(10.0 ** rng.uniform(lo, hi, tuple(s.shape)).astype(np.float32)).cuda()
    q = torch.from_numpy((2 * rng.standard_normal((pool.rows, 4 * kv, 128))).astype(np.float32)).to(DT[name][1]).cuda()
    out = attend(sdq, pool, q, 4 * kv, name, causal=True)
    compare(pool, out, q, 4 * kv, name, 128 ** -0.5, True)


@pytest.mark.parametrize("new,kv", [([1], 1), ([40], 1), ([40], 40)])
@pytest.mark.parametrize("factor", [1e-12, 1e8])
def test_magnitude_of_q_does_not_matter(sdq, new, kv, factor):
    """q far outside fp16's range, the scale its inverse."""
    rng = np.random.default_rng(32)
    pool = Pool(sdq, rng, new, [150], kv, 16, 64)
    pool.fill(rng)
    for name in ("f32", "bf16"):
        q = torch.from_numpy((factor * rng.standard_normal((pool.rows, 4 * kv, 64))).astype(np.float32)).to(DT[name][1]).cuda()
        out = attend(sdq, pool, q, 4 * kv, name, scale=0.125 / factor)
        compare(pool, out, q, 4 * kv, name, 0.125 / factor, False)


def test_extreme_cache_scales(sdq):
    """Scales near fp32's ends: a cache of tiny values, and one whose values are zero."""
    rng = np.random.default_rng(33)
    for new, keys, kv in (([1, 1], [100, 60], 2), ([20, 30], [100, 60], 2), ([20, 30], [100, 60], 52), ([40, 40], [600, 60], 18)):
        for ksc, vsc in ((1e-30, 1e-36), (1e-38, 1e30), (0.0, 0.0), (1.0, 0.0)):
            pool = Pool(sdq, rng, new, keys, kv, 16, 64)
            pool.fill(rng)
            pool.ks.fill_(ksc)
            pool.vs.fill_(vsc)
            q = torch.from_numpy(rng.standard_normal((pool.rows, 2 * kv, 64)).astype(np.float32)).cuda()
            out = attend(sdq, pool, q, 2 * kv, "f32", causal=True)
            compare(pool, out, q, 2 * kv, "f32", 0.125, True)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_rows_that_see_nothing_are_zero(sdq, name):
    rng = np.random.default_rng(34)
    pool = Pool(sdq, rng, [3, 6, 1, 40], [3, 2, 0, 10], 2, 8, 64)
    pool.fill(rng)
    q = torch.from_numpy(rng.standard_normal((pool.rows, 4, 64)).astype(np.float32)).to(DT[name][1]).cuda()
    out = attend(sdq, pool, q, 4, name, causal=True)
    assert (out[3:7] == 0).all() and (out[9] == 0).all() and (out[10:40] == 0).all()   # positions below zero, an empty sequence
    assert torch.isfinite(out.float()).all()
    compare(pool, out, q, 4, name, 0.125, True)
    out = attend(sdq, pool, q, 4, name, causal=False)
    assert (out[9] == 0).all()
    compare(pool, out, q, 4, name, 0.125, False)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("last,heads,dim", [(10, 14, 64), (560, 8, 64), (1100, 8, 128)])
def test_rows_that_see_nothing_in_tiles_of_many_rows(sdq, name, last, heads, dim):
    """The same with a tile to a block, and with 2 and 4 blocks that share its keys."""
    rng = np.random.default_rng(36)
    pool = Pool(sdq, rng, [3, 6, 1, 100], [3, 2, 0, last], heads, 8, dim)
    pool.fill(rng)
    q = torch.from_numpy(rng.standard_normal((pool.rows, heads * 4, dim)).astype(np.float32)).to(DT[name][1]).cuda()
    for causal in (True, False):
        out = attend(sdq, pool, q, heads * 4, name, causal=causal)
        assert (out[9] == 0).all() and torch.isfinite(out.float()).all()
        if causal:
            assert (out[3:7] == 0).all()
        compare(pool, out, q, heads * 4, name, dim ** -0.5, causal)


def test_nan_in_a_query_stays_in_its_row(sdq):
    rng = np.random.default_rng(35)
    for new, keys, kv in (([1] * 6, 100, 2), ([50], 100, 2), ([50], 100, 32), ([50], 700, 20)):
        pool = Pool(sdq, rng, new, [keys] * len(new), kv, 16, 128)
        pool.fill(rng)
        for name in ("f32", "bf16", "f16"):
            q = torch.from_numpy(rng.standard_normal((pool.rows, 4 * kv, 128)).astype(np.float32)).to(DT[name][1]).cuda()
            clean = attend(sdq, pool, q, 4 * kv, name)
            for value in (float("nan"), float("inf")):
                q2 = q.clone()
                q2[4, 3, 17] = value
                out = attend(sdq, pool, q2, 4 * kv, name)
                assert torch.isnan(out[4, 3]).all()
                out[4, 3] = clean[4, 3]
                assert torch.equal(out, clean)


@pytest.mark.parametrize("name", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,keys,kv,group", [([5], [100], 2, 2), ([40], [130], 1, 1), ([60], [400], 50, 4), ([60], [1000], 20, 4)])
def test_scales_that_are_not_finite_stay_with_the_rows_that_see_them(sdq, name, new, keys, kv, group):
    """A key that a causal row does not see may hold anything; the rows that see it have no finite answer."""
    rng = np.random.default_rng(37)
    pool = Pool(sdq, rng, new, keys, kv, 16, 64)
    pool.fill(rng)
    heads = kv * group
    q = torch.from_numpy(rng.standard_normal((pool.rows, heads, 64)).astype(np.float32)).to(DT[name][1]).cuda()
    want, *sizes = attention64(pool, q.double().cpu().numpy(), heads, 0.125, True, 0)
    before = new[0] - 3                  # the third-last position is not seen by the rows before it
    tol = attention_tolerance(name, pool, 0, heads, want, *sizes)[:before]
    pg, off = pool.places(0)
    place = int(pg[keys[0] - 3]), slice(None), int(off[keys[0] - 3])
    first = int(pool.starts[0])
    for which in (pool.ks, pool.vs):
        keep = which[place].clone()
        for value in (float("nan"), float("inf")):
            which[place] = value
            out = attend(sdq, pool, q, heads, name, causal=True)
            assert (np.abs(out[first:first + before].double().cpu().numpy() - want[:before]) <= tol).all()
            if which is pool.vs:
                assert not torch.isfinite(out[first + before:first + new[0]]).any()
        which[place] = keep


def test_bad_tables_are_not_seen(sdq):
    """Positions without a page take no part; the others are attended to as if they were all."""
    rng = np.random.default_rng(6)
    for many, heads in ((1, 4), (9, 4), (9, 300)):
        pool = bad_pool(sdq, rng)
        if many > 1:
            pool.new = [n * many for n in pool.new]
            pool.starts = np.concatenate([[0], np.cumsum(pool.new)]).astype(np.int32)
            pool.rows = int(pool.starts[-1])
            pool.refresh()
        q = torch.from_numpy(rng.standard_normal((pool.rows, heads, 64)).astype(np.float32)).cuda()
        out = attend(sdq, pool, q, heads, "f32").double().cpu().numpy()
        there = {0: [p for p in range(40) if not 8 <= p < 16], 1: list(range(24)), 2: [0, 1], 3: [], 4: list(range(16))}
        for b, pos in there.items():
            rows = slice(int(pool.starts[b]), int(pool.starts[b + 1]))
            if not pos:
                assert (out[rows] == 0).all()
                continue
            pg, off = pool.table[b, np.array(pos) // 8], np.array(pos) % 8
            k, v = [c.cpu().numpy()[pg, :, off].astype(np.float64) * s.cpu().numpy()[pg, :, off][..., None].astype(np.float64)
                    for c, s in ((pool.k, pool.ks), (pool.v, pool.vs))]
            for h in range(heads):
                s = 0.125 * (q[rows, h].double().cpu().numpy() @ k[:, h * 2 // heads].T)
                p = np.exp(s - s.max(1, keepdims=True))
                want = (p / p.sum(1, keepdims=True)) @ v[:, h * 2 // heads]
                assert np.max(np.abs(out[rows, h] - want)) <= 1e-5 * np.max(np.abs(v))   # fp32: far above 2^-20
            

@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("new,keys,kv", [([1, 1, 1], [60, 77, 9], 2), ([30, 50, 1], [60, 77, 9], 2), ([30, 50, 1], [60, 77, 9], 24),
                                         ([30, 50, 1], [1060, 77, 9], 11)])
def test_strided_and_unaligned_queries(sdq, name, new, keys, kv):
    rng = np.random.default_rng(41)
    pool = Pool(sdq, rng, new, keys, kv, 16, 64)
    pool.fill(rng)
    heads = 3 * kv
    for ldq, ldo, shift in ((heads * 64 * 2, heads * 64 + 8, 0), (heads * 64 + 3, heads * 64 + 1, 1)):
        flat = torch.from_numpy(rng.standard_normal(pool.rows * ldq + 8).astype(np.float32)).to(DT[name][1]).cuda()
        out = torch.full((pool.rows * ldo + 8,), 11.0, device="cuda").to(DT[name][1])
        q = torch.as_strided(flat, (pool.rows, heads, 64), (ldq, 64, 1), shift)
        o = torch.as_strided(out, (pool.rows, heads, 64), (ldo, 64, 1), shift)
        sdq.kv_attention(pool.cache, pool.seqs, ptr(q), DT[name][0], pool.rows, heads, ptr(o), causal=True, ldq=ldq, ldo=ldo, flags=0x10)
        compare(pool, o, q, heads, name, 0.125, True)
        mask = torch.ones_like(out, dtype=torch.bool)
        torch.as_strided(mask, (pool.rows, heads, 64), (ldo, 64, 1), shift)[:] = False
        assert (out[mask] == 11.0).all()


def test_one_token_at_a_time_equals_a_chunk(sdq):
    """The causal chunk's rows are what single-token calls give, to the rounding of the sums."""
    rng = np.random.default_rng(42)
    pool = Pool(sdq, rng, [24], [224], 2, 16, 128)
    pool.fill(rng)
    q = torch.from_numpy(rng.standard_normal((24, 8, 128)).astype(np.float32)).cuda()
    chunk = attend(sdq, pool, q, 8, "f32", causal=True)
    for i in (0, 11, 23):
        one = Pool.__new__(Pool)
        one.__dict__.update(pool.__dict__)
        one.new, one.keys, one.starts, one.rows = [1], [201 + i], np.array([0, 1], np.int32), 1
        one.refresh()
        got = attend(sdq, one, q[i:i + 1].contiguous(), 8, "f32", causal=True)
        compare(one, got, q[i:i + 1], 8, "f32", 128 ** -0.5, True)
        assert (got[0] - chunk[i]).abs().max() <= 2.0 ** -18 * pool.vs.nan_to_num().max() * 127


def test_a_pool_beyond_32_bit_offsets(sdq):
    """Pages whose byte offset passes 2^32: 40 million pool rows of 128 bytes."""
    rng = np.random.default_rng(43)
    pages, heads, page, dim = 40000, 8, 128, 128
    k, v = [torch.zeros(pages, heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    ks, vs = [torch.full((pages, heads, page), float("nan"), device="cuda") for _ in range(2)]
    use = np.array([39999, 17, 33333, 39998], np.int32)
    n = 4 * page - 30
    x = [torch.from_numpy(rng.standard_normal((n, heads, dim)).astype(np.float32)).cuda() for _ in range(2)]
    start, length, table = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, n], [n], use.tolist())]
    cache = sdq.kv_cache(ptr(k), ptr(v), ptr(ks), ptr(vs), pages, heads, page, dim)
    seqs = sdq.kv_seqs(ptr(start), ptr(length), ptr(table), 1, 4)
    sdq.kv_append(cache, seqs, ptr(x[0]), ptr(x[1]), 0, n)
    back = [torch.empty_like(t) for t in x]
    sdq.kv_read(cache, seqs, ptr(back[0]), ptr(back[1]), 0, n, flags=0x10)
    for t, r in zip(x, back):
        q, sc = int8_rows(t.cpu().numpy())
        assert np.array_equal(r.cpu().numpy(), q.astype(np.float32) * sc[..., None])
    for rows in (1, 60):
        qq = torch.from_numpy(rng.standard_normal((rows, heads, dim)).astype(np.float32)).cuda()
        s2 = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        out = torch.empty_like(qq)
        sdq.kv_attention(cache, sdq.kv_seqs(ptr(s2), ptr(length), ptr(table), 1, 4), ptr(qq), 0, rows, heads, ptr(out), flags=0x10)
        p = torch.softmax(torch.einsum("rhd,khd->rhk", qq.double(), back[0].double()) * dim ** -0.5, -1)
        want = torch.einsum("rhk,khd->rhd", p, back[1].double())
        assert (out.double() - want).abs().max() <= 1e-5 * back[1].abs().max()


def test_shared_pages_and_a_graph_with_new_lengths(sdq):
    """Two sequences read one prefix; a captured step sees tables that change between replays, and
    two graphs replayed side by side on different streams do not disturb each other."""
    rng = np.random.default_rng(44)
    pool = Pool(sdq, rng, [1, 1], [200, 180], 2, 16, 128, spare=8)
    pool.fill(rng)
    pool.table[1, :4] = pool.table[0, :4]
    pool.refresh()
    q = torch.from_numpy(rng.standard_normal((2, 8, 128)).astype(np.float32)).cuda()
    compare(pool, attend(sdq, pool, q, 8, "f32"), q, 8, "f32", 128 ** -0.5, False)
    outs, graphs, cap = [torch.zeros(2, 8, 128, device="cuda") for _ in range(2)], [], torch.cuda.Stream()
    qs = [q, q.flip(0).contiguous()]
    for x, o in zip(qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=cap):
            sdq.kv_attention(pool.cache, pool.seqs, ptr(x), 0, 2, 8, ptr(o), stream=C.c_void_p(cap.cuda_stream))
        graphs.append(g)
    for keys in ([200, 180], [33, 150], [1, 2]):
        pool.keys = keys
        pool.d_len.copy_(torch.tensor(keys, dtype=torch.int32))
        torch.cuda.synchronize()
        sts = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(10):
            for g, s in zip(graphs, sts):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for x, o in zip(qs, outs):
            got = attend(sdq, pool, x, 8, "f32")
            compare(pool, got, x, 8, "f32", 128 ** -0.5, False)
            assert torch.equal(o, got)


def test_nothing_to_do(sdq):
    pool = Pool(sdq, np.random.default_rng(1), [1], [3], 1, 16, 64)
    empty = sdq.kv_seqs(None, None, None, 0, 0)
    t = torch.full((64,), 4.0, device="cuda")
    sdq.kv_append(pool.cache, pool.seqs, None, None, 0, 0)
    sdq.kv_read(pool.cache, empty, ptr(t), ptr(t), 0, 1)
    sdq.kv_attention(pool.cache, empty, ptr(t), 0, 1, 1, ptr(t), flags=0x10)
    assert (t == 4.0).all()
