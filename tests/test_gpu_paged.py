"""The paged cache's operators on the GPU against numpy in 64 bits: rows at given positions, the append, attention over
the pages with and without a shared prefix, and a serving loop of them together.

Tolerances, from the arithmetic.  Rotation: two products and a sum in f32, each rounded by at most 2^-24, of values up to
|a| + |b| times the tables' entries.  Attention: queries, f32 keys and probabilities may be sums of no fewer than two bf16
parts, each off by half a step, so x = hi + lo within 2^-9 * 2^-9 = 2^-18 of x; of a product of two such values the parts'
errors and the dropped lo * lo add up to less than 2^-16 of it, and sums of n products add n * 2^-24.  A score off by e changes its
weight by a factor of at most exp(2 e), so an output is off by at most (2 e + 2^-16 + n * 2^-24) of sum_j p_j |v_j|."""
import random

import numpy as np
import pytest

import ctorch_amd as ct
import oracle
from common import say

pytestmark = pytest.mark.gpu
GPU = ct.device("gpu")
TYPES = {"f32": ct.F32, "bf16": ct.BF16}


def give(values, dtype="f32"):
    """The tensor on the GPU, and the values that it holds."""
    if dtype == "bf16":
        bits = oracle.bf16_encode(np.ascontiguousarray(values, np.float32))
        return ct.Tensor.from_numpy(bits, ct.BF16, GPU), oracle.bf16_decode(bits)
    if np.asarray(values).dtype == np.int64:
        return ct.Tensor.from_numpy(values, ct.I64, GPU), values
    return ct.Tensor.from_numpy(np.asarray(values, np.float32), ct.F32, GPU), np.asarray(values, np.float32)


def values_of(tensor):
    array = tensor.numpy()
    return oracle.bf16_decode(array) if tensor.dtype == ct.BF16 else array


def spans(tokens, heads, dim, dtype, rng, gap):
    """Rows [tokens, heads, dim], as they are or as a view of a wider projection output (gap)."""
    wide, whole = give(rng.standard_normal((tokens, heads + 2 * gap, dim)), dtype)
    return ct.narrow(wide, 1, gap, heads), whole[:, gap:gap + heads]


# ------------------------------------------------------------------------------------------------ rotation
def rotated(x, c, s, half):
    """In 64 bits: x [T, H, D], c and s [T, R/2]; and the sum of the magnitudes that each entry is made of."""
    x, c, s = x.astype(np.float64), c.astype(np.float64)[:, None], s.astype(np.float64)[:, None]
    n = c.shape[-1]
    first, second = (np.arange(n), np.arange(n) + n) if half else (2 * np.arange(n), 2 * np.arange(n) + 1)
    y, size = x.copy(), np.abs(x)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    size[..., first], size[..., second] = abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)
    return y, size


@pytest.mark.parametrize("T,H,D,part", [(1, 32, 64, 64), (7, 3, 128, 32), (1, 1, 2, 2), (5, 2, 30, 10), (300, 8, 80, 24),
                                        (2, 5, 64, 62), (33, 1, 7, 6), (1000, 4, 16, 16), (3, 12, 128, 128)])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_are_rotated_by_their_positions(T, H, D, part, half, dtype):
    say(f"case: rotary T={T} H={H} D={D} part={part} half={half} {dtype}")
    rng = np.random.default_rng(T + D)
    angles = rng.uniform(0, 6.3, (500, part // 2))
    c, s = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    gc, gs = give(c)[0], give(s)[0]
    at = rng.integers(0, 500, T)
    at[0], at[-1] = 499, 0
    for gap in (0, 1):
        x, values = spans(T, H, D, dtype, rng, gap)
        got = ct.rotary_positions(x, give(at)[0], gc, gs, int(half))
        want, size = rotated(values, c[at], s[at], half)
        assert got.shape == (T, H, D) and got.dtype == ct.F32
        assert np.all(np.abs(got.numpy() - want) <= 3 * 2.0 ** -24 * size)
        assert np.array_equal(got.numpy()[..., part:], values[..., part:])  # copied


def test_positions_beyond_the_tables_come_out_nan():
    x, values = give(np.ones((4, 2, 8)))
    angles = np.ones((6, 2))
    got = ct.rotary_positions(x, give(np.array([5, 6, -1, 2 ** 60]))[0], give(np.cos(angles))[0], give(np.sin(angles))[0]).numpy()
    assert np.all(np.isfinite(got[0])) and np.all(np.isnan(got[1:, :, :4])) and np.all(got[:, :, 4:] == 1)


def test_rows_of_columns_with_gaps_and_of_one_row_for_all():
    rng = np.random.default_rng(3)
    x, values = give(rng.standard_normal((6, 2, 16)))
    angles = rng.uniform(0, 6, (9, 4))
    c, s = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    part = ct.narrow(x, 2, 3, 9)  # rows of 9 entries, 4 bytes off any alignment
    at = np.arange(6)[::-1].copy()
    got = ct.rotary_positions(part, give(at)[0], give(c)[0], give(s)[0], ct.ROTARY_HALF).numpy()
    want, size = rotated(values[..., 3:12], c[at], s[at], True)
    assert np.all(np.abs(got - want) <= 3 * 2.0 ** -24 * size)


# ------------------------------------------------------------------------------------------------ a paged step
class Step:
    """A cache whose pages hold NaN where no position lies, a step over it, and the same in plain arrays."""

    def __init__(self, lengths, counts, heads, kv, dim, page, dtype, shared=0, seed=0, layers=1):
        rng, order = np.random.default_rng(seed), random.Random(seed)
        self.lengths, self.counts, self.page, self.dtype, self.shared = lengths, counts, page, dtype, shared
        self.heads, self.kv, self.dim = heads, kv, dim
        need = [max(0, -(-(n + c) // page) - shared // page) for n, c in zip(lengths, counts)]
        self.pages = shared // page + sum(need) + 2
        free = list(range(self.pages))
        order.shuffle(free)
        front = [free.pop() for _ in range(shared // page)]
        tables = [front + [free.pop() for _ in range(n)] for n in need]
        width = max(1, max(map(len, tables)))
        self.tables = np.array([t + [-1] * (width - len(t)) for t in tables], np.int64)
        self.cache = ct.PagedCache(layers, self.pages, page, kv, dim, TYPES[dtype])
        self.key, self.value = [], []
        for layer in range(layers):
            k, v = (np.full((self.pages, kv, page, dim), np.nan, np.float32) for _ in range(2))
            for n, c, table in zip(lengths, counts, tables):
                for i, p in enumerate(table):
                    live = min(page, n + c - i * page)
                    for pool in (k, v):
                        pool[p, :, :live] = rng.standard_normal((kv, live, dim))
            if dtype == "bf16":
                k, v = (oracle.bf16_decode(oracle.bf16_encode(a)) for a in (k, v))
            for pool, view in ((k, self.cache.key(layer)), (v, self.cache.value(layer))):
                fill(view, pool)
            self.key.append(k)
            self.value.append(v)
        self.batch = self.again()
        self.tokens = sum(counts)
        self.rng = rng

    def again(self):
        return ct.PagedBatch(self.cache, self.heads, self.lengths, self.counts, self.tables, self.shared)

    def held(self, pool, b, n):
        """The first n positions of sequence b, [kv, n, dim]."""
        pages = self.tables[b, :-(-n // self.page)]
        return pool[pages].transpose(1, 0, 2, 3).reshape(self.kv, -1, self.dim)[:, :n].astype(np.float64)

    def attend(self, q, layer=0):
        """(outputs, how far off they may be) for q [tokens, heads, dim]."""
        out, bound, t = np.empty(q.shape), np.empty(q.shape), 0
        group = self.heads // self.kv
        for b, (n, c) in enumerate(zip(self.lengths, self.counts)):
            k, v = (self.held(pool[layer], b, n + c) for pool in (self.key, self.value))
            hidden = np.arange(n + c)[None] > n + np.arange(c)[:, None]
            for h in range(self.heads if c else 0):
                x, kk, vv = q[t:t + c, h].astype(np.float64), k[h // group], v[h // group]
                z = np.where(hidden, -np.inf, x @ kk.T / np.sqrt(self.dim))
                with np.errstate(invalid="ignore"):
                    p = np.exp(z - z.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                size = np.max(np.where(hidden, 0, np.abs(x) @ np.abs(kk).T / np.sqrt(self.dim)), -1, keepdims=True)
                out[t:t + c, h] = p @ vv
                bound[t:t + c, h] = (2 * (2.0 ** -16 + self.dim * 2.0 ** -24) * size + 2.0 ** -16 + (n + c) * 2.0 ** -24) * (p @ np.abs(vv))
            t += c
        return out, bound


def fill(view, values):
    """Writes the whole of a pool's live storage, whatever the values."""
    bits = oracle.bf16_encode(values) if view.dtype == ct.BF16 else np.ascontiguousarray(values, np.float32)
    assert view.shape == bits.shape and ct.lib().dl_tensor_nbytes(view.handle) == bits.nbytes
    ct.synchronize()
    copy = ct.lib().hipMemcpy  # of the runtime that the library is linked with
    copy.argtypes, copy.restype = [ct.C.c_void_p, ct.C.c_void_p, ct.C.c_size_t, ct.C.c_int], ct.C.c_int
    assert copy(ct.lib().dl_tensor_data(view.handle), bits.ctypes.data_as(ct.C.c_void_p), bits.nbytes, 1) == 0


# lengths, counts, heads, kv, dim, page, shared
STEPS = [
    ([0], [1], 8, 2, 64, 16, 0), ([15], [1], 32, 8, 64, 16, 0), ([16], [1], 4, 4, 16, 16, 0), ([129], [1], 32, 8, 128, 32, 0),
    ([300, 5, 0, 77], [1, 1, 1, 1], 32, 8, 64, 16, 0), ([4000, 3], [1, 1], 8, 2, 128, 64, 0), ([511], [1], 40, 2, 32, 16, 0),
    ([31, 700, 64], [5, 2, 0], 32, 8, 64, 16, 0), ([0, 100], [70, 33], 12, 4, 64, 32, 0), ([0], [257], 6, 6, 32, 128, 0),
    ([90], [130], 16, 2, 128, 16, 0), ([2500], [9], 32, 4, 64, 16, 0), ([0, 0, 1000], [1, 40, 300], 8, 8, 16, 16, 0),
    ([70, 64, 400], [1, 1, 1], 32, 8, 64, 16, 64), ([1024 + 5, 1024], [1, 3], 8, 2, 128, 32, 1024),
    ([16] * 20, [1] * 20, 32, 8, 32, 16, 16), ([640 + 100 * i for i in range(4)], [5, 0, 1, 40], 12, 4, 64, 64, 640),
    ([3000, 2900 + 77], [17, 60], 16, 16, 64, 16, 2880), ([4096 + 3 * i for i in range(40)], [1] * 40, 16, 4, 128, 128, 4096),
    ([0, 900], [500, 1], 32, 8, 128, 16, 0), ([200, 12, 33], [129, 300, 16], 16, 4, 16, 16, 0),
]


@pytest.mark.parametrize("case", range(len(STEPS)))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("query", ["f32", "bf16"])
def test_attention_over_pages(case, dtype, query):
    lengths, counts, heads, kv, dim, page, shared = STEPS[case]
    say(f"case: paged attention {STEPS[case]} pages {dtype} queries {query}")
    step = Step(lengths, counts, heads, kv, dim, page, dtype, shared, case)
    for gap in (0, 1):
        q, values = spans(step.tokens, heads, dim, query, step.rng, gap)
        got = ct.paged_attention(step.cache, 0, step.batch, q)
        want, bound = step.attend(values)
        assert got.shape == (step.tokens, heads, dim) and got.dtype == ct.F32
        off = np.abs(got.numpy() - want)
        assert np.all(off <= bound), (float(np.nanmax(off / bound)), np.argwhere(~(off <= bound))[:3])
        # the same call, and a batch made anew, give the same bits
        assert np.array_equal(ct.paged_attention(step.cache, 0, step.batch, q).numpy(), got.numpy())
        assert np.array_equal(ct.paged_attention(step.cache, 0, step.again(), q).numpy(), got.numpy())


@pytest.mark.parametrize("seed", range(10))
def test_random_batches(seed):
    """Runs of few rows, of many and what is left of them side by side, with and without a prefix."""
    order = random.Random(seed)
    kv, dim, page = order.choice([1, 2, 4]), order.choice([16, 32, 64, 128]), order.choice([16, 32, 128])
    heads, shared = kv * order.choice([1, 3, 4, 7, 8]), order.choice([0, 0, page, 9 * page])
    batch = order.randint(1, 9)
    counts = [order.choice([0, 1, 1, 2, 5, 17, order.randint(20, 180)]) for _ in range(batch)]
    counts[0] = max(counts[0], 1)
    lengths = [shared + order.choice([0, 1, 31, order.randint(0, 300), order.randint(0, 1800)]) for _ in range(batch)]
    for dtype, query in (("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")):
        say(f"case: paged attention {lengths} {counts} heads {heads} of {kv}, {dim}, page {page}, shared {shared}, {dtype} {query}")
        step = Step(lengths, counts, heads, kv, dim, page, dtype, shared, 100 + seed)
        q, values = spans(step.tokens, heads, dim, query, step.rng, 0)
        want, bound = step.attend(values)
        assert np.all(np.abs(ct.paged_attention(step.cache, 0, step.batch, q).numpy() - want) <= bound)


def test_a_prefix_shared_or_not_is_the_same_attention():
    step = Step([2048 + 40, 2048, 2048 + 700], [1, 2, 20], 32, 8, 64, 32, "bf16", 2048, 4)
    q, values = spans(step.tokens, 32, 64, "f32", step.rng, 0)
    want, bound = step.attend(values)
    alone = ct.PagedBatch(step.cache, 32, step.lengths, step.counts, step.tables)
    for batch in (step.batch, alone):
        assert np.all(np.abs(ct.paged_attention(step.cache, 0, batch, q).numpy() - want) <= bound)


def test_queries_at_odd_places_are_read_through_a_copy():
    step = Step([50, 20], [1, 3], 8, 2, 32, 16, "f32", 0, 5)
    wide, whole = give(step.rng.standard_normal((step.tokens, 8, 37)))
    for start in (0, 3, 4):
        got = ct.paged_attention(step.cache, 0, step.batch, ct.narrow(wide, 2, start, 32))
        want, bound = step.attend(whole[..., start:start + 32])
        assert np.all(np.abs(got.numpy() - want) <= bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 1], [40, 3]])
def test_extreme_values(dtype, counts):
    """Scores far apart, and keys that are not finite."""
    step = Step([100, 200], counts, 8, 2, 64, 16, dtype, 0, 6)
    q, values = give(step.rng.standard_normal((step.tokens, 8, 64)) * 30)
    want, bound = step.attend(values)
    got = ct.paged_attention(step.cache, 0, step.batch, q).numpy()
    assert np.all(np.abs(got - want) <= bound)
    # a key of sequence 0 that is not finite (its rows are nobody's): sequence 1 does not notice
    k = step.key[0].copy()
    for p in range(40):
        k[step.tables[0, p // 16], :, p % 16] = -np.inf
    fill(step.cache.key(0), k)
    got = ct.paged_attention(step.cache, 0, step.batch, q).numpy()
    assert np.all(np.abs(got[counts[0]:] - want[counts[0]:]) <= bound[counts[0]:])


AHEAD = [([100], [4], 8, 2, 64), ([40], [8], 8, 2, 128), ([90], [150], 8, 2, 64), ([1000], [70], 16, 4, 128), ([33], [3], 4, 1, 16),
         ([0], [2], 40, 2, 32), ([3000], [6], 8, 2, 32), ([5], [400], 4, 4, 16)]


@pytest.mark.parametrize("case", range(len(AHEAD)))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_lies_ahead_of_a_row_does_not_reach_it(case, dtype):
    """Values and then keys that are not finite at a new position: the rows before it do not see them, and of the others only
    those entries change."""
    lengths, counts, heads, kv, dim = AHEAD[case]
    say(f"case: paged attention {AHEAD[case]} pages {dtype}, not finite ahead")
    step = Step(lengths, counts, heads, kv, dim, 16, dtype, 0, 50 + case)
    q, values = give(step.rng.standard_normal((step.tokens, heads, dim)))
    row, at, group = counts[0] // 2, lengths[0] + counts[0] // 2, heads // kv
    place = step.tables[0, at // 16], 0, at % 16  # KV head 0
    marks = {3: np.nan, 5: np.inf, dim - 1: -np.inf}
    for d in marks:
        step.value[0][place][d] = 0
    want, bound = step.attend(values)
    spoiled = step.value[0].copy()
    for d, x in marks.items():
        spoiled[place][d] = x
    fill(step.cache.value(0), spoiled)
    got = ct.paged_attention(step.cache, 0, step.batch, q).numpy()
    sees = np.zeros(got.shape, bool)
    for d in marks:
        sees[row:, :group, d] = True
    assert not np.isfinite(got[sees]).any()
    assert np.all(np.abs(got - want)[~sees] <= bound[~sees])
    fill(step.cache.value(0), step.value[0])
    key = step.key[0].copy()
    key[place] = np.nan
    fill(step.cache.key(0), key)
    got = ct.paged_attention(step.cache, 0, step.batch, q).numpy()
    sees[row:, :group] = True
    assert np.isnan(got[sees]).all() and np.all(np.abs(got - want)[~sees] <= bound[~sees])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1, 0], [1, 200], [9, 1]])
def test_scores_far_below_zero(dtype, counts):
    """A row's one key, and equal ones, still weigh what they weigh."""
    step = Step([0, 0], counts, 8, 2, 64, 16, dtype, 0, 8)
    fill(step.cache.key(0), np.full_like(step.key[0], -2.0 ** 12))
    q = give(np.full((step.tokens, 8, 64), 1.375 * 2.0 ** 13))[0]  # 64 * 1.375 * 2^25 / 8 = 1.375 * 2^28
    got, t = ct.paged_attention(step.cache, 0, step.batch, q).numpy(), 0
    for b, c in enumerate(counts):
        v = step.held(step.value[0], b, c)
        for i in range(c):  # the mean of i + 1 values: equal weights that round, their sum in f32, and the quotient
            want, size = v[:, :i + 1].mean(1), np.abs(v[:, :i + 1]).mean(1)
            assert np.all(np.abs(got[t + i].reshape(2, 4, 64) - want[:, None]) <= (2 * i + 16) * 2.0 ** -23 * size[:, None])
        t += c


def test_a_nan_stays_in_the_rows_that_see_it():
    step = Step([30, 30], [3, 3], 8, 2, 32, 16, "bf16", 0, 7)
    k = step.key[0].copy()
    k[step.tables[0, 31 // 16], 0, 31 % 16] = np.nan  # sequence 0, position 31, KV head 0: seen by its rows 1 and 2
    fill(step.cache.key(0), k)
    q, values = give(step.rng.standard_normal((6, 8, 32)))
    got = ct.paged_attention(step.cache, 0, step.batch, q).numpy()
    lost = np.isnan(got)
    assert lost[1:3, :4].all()
    lost[1:3, :4] = False
    assert not lost.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("source", ["f32", "bf16"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kv,dim,part", [(32, 8, 64, 64), (12, 4, 128, 32), (3, 1, 16, 6), (8, 2, 32, 16)])
def test_append_writes_its_places_and_nothing_else(heads, kv, dim, part, half, source, dtype):
    say(f"case: append heads={heads} kv={kv} dim={dim} part={part} half={half} {source} -> {dtype}")
    step = Step([5, 0, 47, 16, 200], [1, 33, 0, 16, 3], heads, kv, dim, 16, dtype, 0, dim + part, layers=2)
    at = np.concatenate([n + np.arange(c) for n, c in zip(step.lengths, step.counts)])
    angles = step.rng.uniform(0, 6.3, (210, part // 2))
    c, s = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    gc, gs = give(c)[0], give(s)[0]
    wide, whole = give(step.rng.standard_normal((step.tokens, heads + 2 * kv, dim)), source)
    q, k, v = (ct.narrow(wide, 1, a, n) for a, n in ((0, heads), (heads, kv), (heads + kv, kv)))
    before = [values_of(step.cache.key(0)), values_of(step.cache.value(0))]
    got = step.cache.append(1, step.batch, q, k, v, gc, gs, int(half))
    want, size = rotated(whole[:, :heads], c[at], s[at], half)
    assert np.all(np.abs(got.numpy() - want) <= 3 * 2.0 ** -24 * size)
    for a, b in zip(before, (step.cache.key(0), step.cache.value(0))):
        assert np.array_equal(a, values_of(b), equal_nan=True)  # the other layer
    seq = np.repeat(np.arange(5), step.counts)
    pages, rows = step.tables[seq, at // 16], at % 16
    want, size = rotated(whole[:, heads:heads + kv], c[at], s[at], half)
    key, value = values_of(step.cache.key(1)), values_of(step.cache.value(1))
    rounding = 2.0 ** -8 if dtype == "bf16" else 0.0
    assert np.all(np.abs(key[pages, :, rows] - want) <= 3 * 2.0 ** -24 * size + rounding * (np.abs(want) + 2.0 ** -20 * size))
    exact = whole[:, heads + kv:]
    assert np.array_equal(value[pages, :, rows], oracle.bf16_decode(oracle.bf16_encode(exact)) if dtype == "bf16" else exact)
    key[pages, :, rows], value[pages, :, rows] = step.key[1][pages, :, rows], step.value[1][pages, :, rows]
    assert np.array_equal(key, step.key[1], equal_nan=True) and np.array_equal(value, step.value[1], equal_nan=True)


def test_append_without_queries():
    step = Step([5], [2], 8, 2, 32, 16, "f32", 0, 1)
    k, v = (give(step.rng.standard_normal((2, 2, 32))) for _ in range(2))
    c, s = give(np.ones((7, 16)))[0], give(np.zeros((7, 16)))[0]
    assert step.cache.append(0, step.batch, None, k[0], v[0], c, s) is None
    pages, rows = step.tables[0, np.array([5, 6]) // 16], np.array([5, 6]) % 16
    assert np.array_equal(values_of(step.cache.key(0))[pages, :, rows], k[1])
    assert np.array_equal(values_of(step.cache.value(0))[pages, :, rows], v[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("by", [1, 16, -7])
def test_rows_of_the_pages_that_are_written(dtype, by):
    """Keys and values that lie in the layer's own pages, a few rows from their new places: what was there before the call."""
    page, dim, count = 1024, 32, 900
    cache = ct.PagedCache(2, 1, page, 1, dim, TYPES[dtype])
    rng = np.random.default_rng(by + 8)
    held = []
    for layer in range(2):
        for view in (cache.key(layer), cache.value(layer)):
            bits = rng.standard_normal(view.shape).astype(np.float32)
            held.append(oracle.bf16_decode(oracle.bf16_encode(bits)) if dtype == "bf16" else bits)
            fill(view, held[-1])
    start = 40  # the new positions; their rows come from `by` further
    batch = ct.PagedBatch(cache, 1, [start], [count], [[0]])
    c, s = give(np.ones((page, dim // 2)))[0], give(np.zeros((page, dim // 2)))[0]

    def rows(view):
        flat = ct.Tensor(ct._new(ct.lib().dl_reshape, view.handle, ct._shape((page, 1, dim))))
        return ct.narrow(flat, 0, start + by, count)

    query = cache.append(0, batch, rows(cache.value(0)), rows(cache.key(0)), rows(cache.value(0)), c, s).numpy()
    key, value = (h.reshape(page, dim) for h in held[:2])
    moved = slice(start + by, start + by + count)
    assert np.array_equal(query[:, 0], value[moved])
    for view, old in ((cache.key(0), key), (cache.value(0), value)):
        want = old.copy()
        want[start:start + count] = old[moved]
        assert np.array_equal(values_of(view).reshape(page, dim), want)


def test_tables_in_the_pages_that_are_written():
    page, dim, count = 1024, 32, 1000
    cache = ct.PagedCache(1, 1, page, 1, dim)
    fill(cache.key(0), np.ones((1, 1, page, dim)))
    fill(cache.value(0), np.zeros((1, 1, page, dim)))
    c, s = (ct.Tensor(ct._new(ct.lib().dl_reshape, view.handle, ct._shape((2 * page, dim // 2))))
            for view in (cache.key(0), cache.value(0)))
    k, v = (give(np.random.default_rng(i).standard_normal((count, 1, dim))) for i in range(2))
    batch = ct.PagedBatch(cache, 1, [0], [count], [[0]])
    assert np.array_equal(cache.append(0, batch, k[0], k[0], v[0], c, s).numpy(), k[1])
    for view, want, rest in ((cache.key(0), k[1], 1), (cache.value(0), v[1], 0)):
        got = values_of(view).reshape(page, 1, dim)
        assert np.array_equal(got[:count], want) and np.all(got[count:] == rest)


def test_a_pool_beyond_4_gib():
    """Pages whose offset passes 32 bits, in bytes and in elements."""
    kv, dim, page = 8, 128, 1024
    pages = 2 ** 32 // (kv * dim * page) + 2  # more elements than 32 bits count, in bf16
    cache = ct.PagedCache(1, pages, page, kv, dim, ct.BF16)
    tables = np.array([[pages - 1, 0], [pages // 2, pages - 2]])
    lengths, counts = [0, 0], [1030, 7]
    batch = ct.PagedBatch(cache, 16, lengths, counts, tables)
    rng = np.random.default_rng(8)
    tokens = sum(counts)
    k, v, q = (give(rng.standard_normal((tokens, n, dim)), "bf16") for n in (kv, kv, 16))
    c, s = give(np.ones((1030, 64)))[0], give(np.zeros((1030, 64)))[0]
    turned = cache.append(0, batch, q[0], k[0], v[0], c, s)
    assert np.array_equal(turned.numpy(), q[1])
    got = ct.paged_attention(cache, 0, batch, turned).numpy()
    for first, count in ((0, 1030), (1030, 7)):
        for row in (0, count // 2, count - 1):
            for h in (0, 15):
                kk, vv = (a[1][first:first + row + 1, h // 2].astype(np.float64) for a in (k, v))
                x = q[1][first + row, h].astype(np.float64)
                z = kk @ x / np.sqrt(dim)
                p = np.exp(z - z.max())
                p /= p.sum()
                size = np.max(np.abs(kk) @ np.abs(x)) / np.sqrt(dim)
                bound = (2 * (2.0 ** -16 + dim * 2.0 ** -24) * size + 2.0 ** -16 + row * 2.0 ** -24) * (p @ np.abs(vv))
                assert np.all(np.abs(got[first + row, h] - p @ vv) <= bound)


def test_a_serving_loop():
    """Requests that come and go over several steps: prompts in chunks, single tokens, drafted tokens of which some are taken
    back (their positions are written again), against attention over plain arrays that hold the same history."""
    rng, heads, kv, dim, page = np.random.default_rng(12), 8, 2, 64, 16
    cache = ct.PagedCache(2, 64, page, kv, dim, ct.F32)
    cosine, sine = ct.rotary_tables(dim, 400)
    c, s = cosine.numpy(), sine.numpy()
    free = list(range(64))
    random.Random(2).shuffle(free)
    tables, lengths = [[] for _ in range(3)], [0, 0, 0]
    history = [[(np.zeros((0, kv, dim)), np.zeros((0, kv, dim))) for _ in range(3)] for _ in range(2)]
    steps = [([40, 0, 0], None), ([30, 17, 0], None), ([1, 1, 100], None), ([5, 5, 1], [2, 5, 1]), ([1, 5, 1], [1, 3, 1]),
             ([0, 1, 1], None), ([5, 0, 33], [4, 0, 33])]
    for counts, kept in steps:
        for b in range(3):
            while len(tables[b]) * page < lengths[b] + counts[b]:
                tables[b].append(free.pop())
        width = max(map(len, tables))
        batch = ct.PagedBatch(cache, heads, lengths, counts, [t + [-1] * (width - len(t)) for t in tables])
        at = np.concatenate([n + np.arange(m) for n, m in zip(lengths, counts)])
        first = np.cumsum([0] + counts)
        for layer in range(2):
            wide, whole = give(rng.standard_normal((sum(counts), heads + 2 * kv, dim)))
            parts = [ct.narrow(wide, 1, a, n) for a, n in ((0, heads), (heads, kv), (heads + kv, kv))]
            q = cache.append(layer, batch, *parts, cosine, sine)
            got = ct.paged_attention(cache, layer, batch, q).numpy()
            rq, rk = (rotated(x, c[at], s[at], False)[0] for x in (whole[:, :heads], whole[:, heads:heads + kv]))
            for b in range(3):
                rows = slice(first[b], first[b + 1])
                k, v = (np.concatenate([old[:lengths[b]], new[rows]])
                        for old, new in zip(history[layer][b], (rk, whole[:, heads + kv:].astype(np.float64))))
                history[layer][b] = (k, v)
                for i in range(counts[b]):
                    n = lengths[b] + i + 1
                    for h in range(heads):
                        z = k[:n, h // 4] @ rq[first[b] + i, h] / np.sqrt(dim)
                        p = np.exp(z - z.max())
                        p /= p.sum()
                        size = np.max(np.abs(k[:n, h // 4]) @ np.abs(rq[first[b] + i, h])) / np.sqrt(dim)
                        bound = (2 * (2.0 ** -15 + dim * 2.0 ** -24) * size + 2.0 ** -16 + n * 2.0 ** -24) * (p @ np.abs(v[:n, h // 4]))
                        assert np.all(np.abs(got[first[b] + i, h] - p @ v[:n, h // 4]) <= bound)
        lengths = [n + m for n, m in zip(lengths, kept or counts)]


def test_two_batches_of_one_cache_in_turn():
    """Calls queued one behind another share no state: each gives what it gives alone."""
    step = Step([2000, 900], [1, 4], 32, 8, 64, 16, "bf16", 0, 9)
    other = ct.PagedBatch(step.cache, 32, [900], [1], step.tables[1:])
    q, q2 = (spans(n, 32, 64, "f32", step.rng, 0)[0] for n in (step.tokens, 1))
    alone = ct.paged_attention(step.cache, 0, step.batch, q).numpy(), ct.paged_attention(step.cache, 0, other, q2).numpy()
    outs = [ct.paged_attention(step.cache, 0, b, x) for _ in range(5) for b, x in ((step.batch, q), (other, q2))]
    for i, out in enumerate(outs):
        assert np.array_equal(out.numpy(), alone[i % 2])


def test_a_batch_outlives_its_cache_and_a_view_its_storage():
    step = Step([20], [1], 8, 2, 32, 16, "f32", 0, 3)
    same = Step([20], [1], 8, 2, 32, 16, "f32", 0, 3)
    q = give(step.rng.standard_normal((1, 8, 32)))[0]
    want = ct.paged_attention(step.cache, 0, step.batch, q).numpy()
    key = step.cache.key(0)
    held = values_of(key)
    batch = step.batch
    del step
    assert np.array_equal(ct.paged_attention(same.cache, 0, batch, q).numpy(), want)
    assert np.array_equal(values_of(key), held, equal_nan=True)


def test_refusals_come_back_as_errors():
    step = Step([20], [2], 8, 2, 32, 16, "f32", 0, 3)
    q, k = give(np.zeros((2, 8, 32)))[0], give(np.zeros((2, 2, 32)))[0]
    c = give(np.ones((30, 16)))[0]
    for call, said in [
            (lambda: ct.PagedCache(1, 4, 12, 2, 32), "power of two"),
            (lambda: ct.PagedCache(1, 4, 16, 2, 32, ct.F32, ct.device("cpu")), "GPU only"),
            (lambda: ct.PagedBatch(step.cache, 8, [20], [1], [[99, 0]]), "not in the cache"),
            (lambda: ct.PagedBatch(step.cache, 8, [5, 3], [1, 1], [[1], [1]]), "two places"),
            (lambda: step.cache.key(1), "layer out of range"),
            (lambda: ct.paged_attention(step.cache, 0, step.batch, k), "query must be"),
            (lambda: step.cache.append(0, step.batch, q, k, q, c, c), "value must be"),
            (lambda: step.cache.append(0, step.batch, q, k, k, ct.narrow(c, 0, 0, 21), ct.narrow(c, 0, 0, 21)), "position 21"),
            (lambda: ct.rotary_positions(q, give(np.zeros(3, np.int64))[0], c, c), "positions must be")]:
        with pytest.raises(ct.DLError, match=said.replace("[", r"\[")):
            call()
    lib = ct.lib()
    out = ct.C.c_void_p()
    assert lib.dl_paged_attention(None, 0, step.batch.handle, q.handle, ct.C.byref(out)) == 1 and "NULL" in ct.last_error()
    assert lib.dl_paged_attention(step.cache.handle, 0, None, q.handle, ct.C.byref(out)) == 1 and "NULL" in ct.last_error()
    assert lib.dl_paged_attention(step.cache.handle, 0, step.batch.handle, q.handle, None) == 1
    assert lib.dl_paged_cache_append(step.cache.handle, 0, step.batch.handle, q.handle, k.handle, k.handle, c.handle,
                                     c.handle, 0, None) == 1 and "together" in ct.last_error()
