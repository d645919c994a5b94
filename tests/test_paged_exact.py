"""That attention over pages keeps all bits of an f32: three bf16 parts of a query, a weight, and an f32 key or value, and every
product of them down to 2^-22.  Each row sees two keys that weigh anything (or one), and a key has one entry that counts, so that few roundings
add up and a lost part shows.  The tolerances count them, in units of u = 2^-24, half a step of an f32 being u of its value:

A score is one product, cut into 1 (f32 instruction), 3 (bf16 pages) or 6 (f32 pages, many rows) exact ones, added at a step (2 u)
each; of f32 by f32 the products of parts (1, 2), (2, 1) and (2, 2) are left out: a query's parts are rounded (at most 2^-8 of the
part before), a key's cut off (2^-7), so 2^-22 + 2^-23 + 2^-30 < 6.1 u.  The scale, log2 e and their product are rounded (3 u), and
the difference to the row's base (1 u).  So a score is off by e = S u times its size, with S = 6 + 4 for bf16 pages and 12 + 6.1 + 4
for f32 ones, and S = 4 where a query and a key have so few bits that the product is exact.  A weight p of two is then
off by at most p (1 - p) (exp(2 e) - 1).

An output sums two values' products of 3 or 6 parts at a step each (12 u, 24 u and 6.1 u left out); exp2 is off by a step for
either (4 u); the weights' sum, a base that moves and the merges of waves and of splits round numerator and
denominator twice each (2 + 4 + 4 + 4 u), the quotient two times (2 u); S: 32 u for bf16 pages, 50.1 u for f32 ones."""
import numpy as np
import pytest

import ctorch_amd as ct
import oracle
from common import say

U = 2.0 ** -24
SCORE = {"bf16": 10.0, "f32": 22.1}
VALUE = {"bf16": 32.0, "f32": 50.1}
KINDS = ["queries", "weights", "values"]


def rounded(x):
    return oracle.bf16_decode(oracle.bf16_encode(np.ascontiguousarray(x, np.float32)))


def cut_off(x):
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)


def parts(x, cut):
    """Three bf16 parts of f32 values, exact."""
    x = np.asarray(x, np.float32)
    first = cut(x)
    second = cut(x - first)
    third = cut(x - first - second)
    assert np.array_equal(first.astype(np.float64) + second + third, x)
    return [p.astype(np.float64) for p in (first, second, third)]


class Rows:
    """A step whose rows see two keys (one, for "values") that weigh anything, in plain arrays."""

    def __init__(self, kind, lengths, counts, heads, kv, dim, pages, queries, scale=1.0, seed=0, shared=0):
        rng = np.random.default_rng(seed)
        self.kind, self.pages, self.queries, self.shared = kind, pages, queries, shared
        self.lengths, self.counts, self.heads, self.kv, self.dim = lengths, counts, heads, kv, dim
        of = rounded if pages == "bf16" else lambda x: np.asarray(x, np.float32)
        root, power = np.sqrt(dim), 2.0 ** np.floor(np.log2(np.sqrt(dim)))
        group, tokens = heads // kv, sum(counts)
        self.key, self.value = [], []
        self.q = np.zeros((tokens, heads, dim), np.float32)
        # of each row: its scores' factors [tokens, heads, 2] and its values [tokens, heads, 2, dim]
        self.factors, self.values = np.zeros((2, tokens, heads, 2)), np.zeros((tokens, heads, 2, dim))
        t = 0
        front = of(rng.standard_normal((2, kv, shared, dim)))
        for b, (n, c) in enumerate(zip(lengths, counts)):
            k, v = np.zeros((kv, n + c, dim), np.float32), of(rng.standard_normal((kv, n + c, dim)) * scale)
            first = rng.integers(0, shared or n) if b == 0 or not shared else place[0]
            place = first, rng.choice([i for i in rng.integers(shared, n, 9) if i != first])
            spots = rng.permutation(dim)[:2] if b == 0 or not shared else spots  # the entries of a key and a query that count
            if kind == "weights":
                k[:, :, spots] = -1024 * power
                k[:, place] = 0
                v[:, place[0]] = 0
            if kind == "queries":
                big = of(4 * root * rng.uniform(1, 2, (kv, 2)))
            else:
                big = np.full((kv, 2), power, np.float32)
            if shared:  # what the sequences have in common is the first one's
                if b == 0:
                    front = big.copy(), v[:, :shared].copy()
                big[:, 0], v[:, :shared] = front[0][:, 0], front[1]
            live = 1 if kind == "values" else 2
            for i in range(live):
                k[:, place[i], spots[i]] = big[:, i]
            for h in range(heads):
                a = big[h // group].astype(np.float64)
                if kind == "queries":
                    x = np.float32(128 * root / a[0] * rng.uniform(0.8, 1.2, c))
                    y = np.float32((x * a[0] + root * rng.uniform(-2, 2, c)) / a[1])
                elif kind == "weights":
                    x, y = rng.integers(128, 257, (2, c)) / np.float32(256)
                else:
                    x, y = np.float32(256.0) * np.ones(c, np.float32), np.zeros(c, np.float32)
                if queries == "bf16":
                    x, y = rounded(x), rounded(y)
                self.q[t:t + c, h, spots[0]], self.q[t:t + c, h, spots[1]] = x, y
                self.factors[0, t:t + c, h] = np.stack([x, y], -1)
                self.factors[1, t:t + c, h] = a
                self.values[t:t + c, h] = v[h // group, list(place)]
            self.key.append(k)
            self.value.append(v)
            t += c

    def exact(self, score=None, product=None):
        """(outputs in 64 bits, how far off they may be); score and product stand in for a mistake."""
        q, k = self.factors
        s = (q * k if score is None else score(q, k)) / np.sqrt(self.dim)
        if self.kind == "values":
            s[..., 1] = -np.inf
        w = np.exp(s - s.max(-1, keepdims=True))
        p = w / w.sum(-1, keepdims=True)
        v = self.values
        if product is None:
            out = (p[..., None] * v).sum(-2)
        else:
            out = product(np.float32(w)[..., None] * np.ones_like(v, np.float32), np.float32(v)).sum(-2) / w.sum(-1)[..., None]
        e = (4.0 if self.kind != "queries" else SCORE[self.pages]) * U * np.max(np.abs(q * k), -1) / np.sqrt(self.dim)
        moved = (p[..., 0] * p[..., 1] * np.expm1(2 * e))[..., None] * np.abs(v[..., 0, :] - v[..., 1, :])
        return out, moved + VALUE[self.pages] * U * (p[..., None] * np.abs(v)).sum(-2)


# lengths, counts, heads, kv, shared: 16 rows, 32, many, many and few, splits, and a shared prefix
STEPS = [([40, 77, 130, 50, 350, 51], [1] * 6, 12, 2, 0), ([300, 37], [1, 5], 8, 2, 0), ([700], [130], 8, 2, 0), ([50, 900], [60, 1], 6, 2, 0),
         ([6000, 5000], [1, 3], 8, 2, 0), ([3000, 40], [2, 90], 4, 4, 0), ([700, 720, 660], [1, 2, 40], 16, 4, 640)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(STEPS)))
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("pages", ["f32", "bf16"])
@pytest.mark.parametrize("queries", ["f32", "bf16"])
def test_products_keep_all_bits(case, dim, pages, queries):
    from test_gpu_paged import TYPES, fill, give

    lengths, counts, heads, kv, shared = STEPS[case]
    for kind in KINDS:
        say(f"case: exact {kind} {STEPS[case]} heads of {dim}, pages {pages}, queries {queries}")
        # (the largest values that a sum of n keys' weights holds, and small ones)
        rows = Rows(kind, lengths, counts, heads, kv, dim, pages, queries, [1.0, 2.0 ** -90, 1e36 / (8 * max(lengths))][case % 3], case, shared)
        page = [16, 32, 128][case % 3]
        order = np.random.default_rng(case).permutation(sum(-(-(n + c) // page) for n, c in zip(lengths, counts)) + 1)
        pools = [np.full((len(order), kv, page, dim), np.nan, np.float32) for _ in range(2)]
        tables, at = np.full((len(lengths), -(-max(n + c for n, c in zip(lengths, counts)) // page)), -1), 0
        for b, (n, c) in enumerate(zip(lengths, counts)):
            for i in range(-(-(n + c) // page)):
                if b and (i + 1) * page <= shared:
                    tables[b, i] = tables[0, i]
                    continue
                tables[b, i], at = order[at], at + 1
                for pool, held in zip(pools, (rows.key[b], rows.value[b])):
                    live = held[:, i * page:(i + 1) * page]
                    pool[tables[b, i], :, :live.shape[1]] = live
        cache = ct.PagedCache(1, len(order), page, kv, dim, TYPES[pages])
        fill(cache.key(0), pools[0])
        fill(cache.value(0), pools[1])
        batch = ct.PagedBatch(cache, heads, lengths, counts, tables, shared)
        got = ct.paged_attention(cache, 0, batch, give(rows.q, queries)[0]).numpy()
        want, bound = rows.exact()
        off = np.abs(got - want)
        assert np.all(off <= bound), (kind, float(np.nanmax(off / bound)), np.argwhere(~(off <= bound))[:3])


@pytest.mark.gpu
@pytest.mark.parametrize("pages", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1], [5], [200]])
@pytest.mark.parametrize("length", [40, 3000])
def test_the_largest_values(pages, counts, length):
    """Values of 1e36 over the number of keys, of one sign: their sum by weights of up to 2^8 still is an f32.  Keys of score 0,
    then one 5 above them, which leaves the row's base where it is, 2^7 below."""
    from test_gpu_paged import TYPES, fill, give

    say(f"case: largest values, {length} and {counts} pages {pages}")
    heads, kv, dim, page, keys = 8, 2, 64, 16, length + counts[0]
    cache = ct.PagedCache(1, -(-keys // page), page, kv, dim, TYPES[pages])
    value = np.float32(2.0 ** np.floor(np.log2(1e36 / keys)))
    key = np.zeros((-(-keys // page), kv, page, dim))
    key[length // 2 // page, :, length // 2 % page, 0] = 40
    fill(cache.key(0), key)
    fill(cache.value(0), np.full(key.shape, value))
    batch = ct.PagedBatch(cache, heads, [length], counts, [np.arange(len(key))])
    got = ct.paged_attention(cache, 0, batch, give(np.ones((counts[0], heads, dim)))[0]).numpy()
    # the mean of equal values: keys are added on both sides, a step each
    assert np.all(np.abs(got / value - 1) <= (4 * keys + 32) * U)


def products(a, b, left_out, cut_a=rounded, cut_b=cut_off):
    """a b from three by three parts without those that are left out."""
    return sum(x * y for i, x in enumerate(parts(a, cut_a)) for j, y in enumerate(parts(b, cut_b)) if (i, j) not in left_out)


SMALL = {(1, 2), (2, 1), (2, 2)}
MISTAKES = {
    "two parts of a query": ("queries", "bf16", dict(score=lambda q, k: products(q, k, {(2, 0)}, cut_b=rounded))),
    "two parts of a query, f32 pages": ("queries", "f32", dict(score=lambda q, k: products(q, k, SMALL | {(2, 0)}))),
    "two parts of a key": ("queries", "f32", dict(score=lambda q, k: products(q, k, SMALL | {(0, 2)}))),
    "no second by second of scores": ("queries", "f32", dict(score=lambda q, k: products(q, k, SMALL | {(1, 1)}))),
    "two parts of a weight": ("weights", "bf16", dict(product=lambda w, v: products(w, v, {(2, 0)}))),
    "two parts of a weight, f32 pages": ("weights", "f32", dict(product=lambda w, v: products(w, v, SMALL | {(2, 0)}))),
    "no second by second of outputs": ("weights", "f32", dict(product=lambda w, v: products(w, v, SMALL | {(1, 1)}))),
    "two parts of a value": ("values", "f32", dict(product=lambda w, v: products(w, v, SMALL | {(0, 2)}))),
}


@pytest.mark.parametrize("case", range(len(STEPS)))
@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("name", MISTAKES)
def test_a_lost_part_is_seen(name, case, dim):
    kind, pages, mistake = MISTAKES[name]
    lengths, counts, heads, kv, shared = STEPS[case]
    rows = Rows(kind, lengths, counts, heads, kv, dim, pages, "f32", 1.0, case, shared)
    want, bound = rows.exact()
    # the rule itself, with the products that are left out, stays within the bound
    kept = dict(score=lambda q, k: products(q, k, SMALL)) if "score" in mistake else dict(product=lambda w, v: products(w, v, SMALL))
    assert np.all(np.abs(rows.exact(**kept)[0] - want) <= bound)
    assert np.any(np.abs(rows.exact(**mistake)[0] - want) > bound)
