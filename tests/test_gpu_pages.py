"""Copies, forks and compaction of a paged cache's pages on the GPU, bit for bit: what is copied, and that nothing else
changes.  (Which pages, who holds them and what is refused: test_serving_rules.py, without a GPU.)"""
import numpy as np
import pytest

import ctorch_amd as ct
from common import say, write

pytestmark = pytest.mark.gpu
GPU = ct.device("gpu")
TYPES = {"f32": ct.F32, "bf16": ct.BF16}


def fill(tensor, seed):
    """Random bits into a live view (through the HIP runtime: the library only reads such views)."""
    rng = np.random.default_rng(seed)
    values = rng.integers(0, 1 << 16, tensor.shape).astype(np.uint16) if tensor.dtype == ct.BF16 else \
        rng.integers(0, 1 << 31, tensor.shape).astype(np.int32)
    write(tensor, values)


def bits(tensor):
    values = tensor.numpy()
    return values.view(np.int32) if values.dtype == np.float32 else values


class Pools:
    def __init__(self, layers, pages, page, kv, dim, dtype, seed=0):
        self.cache = ct.PagedCache(layers, pages, page, kv, dim, TYPES[dtype])
        for layer in range(layers):
            fill(self.cache.key(layer), seed + 2 * layer)
            fill(self.cache.value(layer), seed + 2 * layer + 1)
        self.layers, self.before = layers, None
        self.before = self.all()

    def all(self):
        return [bits(f(layer)) for layer in range(self.layers) for f in (self.cache.key, self.cache.value)]

    def check(self, moves, page):
        """moves: (source, target, rows)."""
        for was, now in zip(self.before, self.all()):
            want = was.copy()
            for source, target, rows in moves:
                want[target, :, :rows] = was[source, :, :rows]
            assert np.array_equal(now, want)


@pytest.mark.parametrize("layers,pages,page,kv,dim,dtype", [(1, 6, 16, 1, 16, "bf16"), (3, 9, 16, 2, 64, "f32"), (2, 7, 128, 8, 128, "bf16"),
                                                            (33, 6, 16, 3, 32, "bf16"), (1, 6, 1024, 5, 128, "f32")])
def test_pages_are_copied_in_every_layer(layers, pages, page, kv, dim, dtype):
    say(f"case: copy {layers} x {pages} pages of {page}, {kv} x {dim} {dtype}")
    for sources, targets, rows in (([1], [4], None), ([0, 1, 2], [1, 2, 0], [page, 3, 1]), ([0, 0, 3], [1, 2, 5], [5, 0, page - 1]),
                                   ([4, 4], [4, 5], [page, 7])):
        pools = Pools(layers, pages, page, kv, dim, dtype)
        pools.cache.copy_pages(sources, targets, rows)
        pools.check([(s, t, page if rows is None else rows[i]) for i, (s, t) in enumerate(zip(sources, targets))], page)


def test_more_pairs_than_a_launch_takes():
    rng = np.random.default_rng(1)
    pools = Pools(2, 600, 16, 1, 16, "bf16")
    sources, targets, rows = rng.integers(0, 600, 500), rng.permutation(600)[:500], rng.integers(0, 17, 500)
    pools.cache.copy_pages(sources, targets, rows)
    pools.check(list(zip(sources, targets, rows)), 16)


@pytest.mark.parametrize("dtype,page,lengths", [("bf16", 16, [40, 16, 0, 15]), ("f32", 64, [200, 1, 63])])
def test_forked_requests_have_what_their_parents_hold(dtype, page, lengths):
    pools = Pools(2, 40, page, 2, 32, dtype)
    pool, rng = ct.PagePool(40), np.random.default_rng(2)
    order, width = list(rng.permutation(40)), 5
    tables = [[int(order.pop()) for _ in range(-(-n // page))] for n in lengths]
    tables = np.array([t + [-1] * (width - len(t)) for t in tables], np.int64)
    pool.claim(tables)
    parents = [0, 0, 1, 2, len(lengths) - 1]
    children = pools.cache.fork(pool, tables, lengths, parents)
    moves = []
    for b, child in zip(parents, children):
        whole, rest = divmod(lengths[b], page)
        assert child[:whole].tolist() == tables[b, :whole].tolist() and np.all(child[whole + (rest > 0):] == -1)
        if rest:
            assert pool.references(child[whole]) == 1
            moves.append((tables[b, whole], child[whole], rest))
    pools.check(moves, page)
    pool.release(children)
    assert pool.available == 40 - np.sum(tables >= 0)


def test_a_compacted_pool_holds_the_same_requests():
    pools = Pools(3, 50, 16, 2, 64, "bf16")
    rng, pool = np.random.default_rng(3), ct.PagePool(50)
    tables = np.append(rng.permutation(50)[:22], [-1, -1]).reshape(4, 6)
    pool.claim(tables)
    moved = pools.cache.compact(pool, tables)
    live = moved[moved >= 0]
    assert sorted(live) == list(range(22)) and pool.available == 28 and np.array_equal(moved < 0, tables < 0)
    pools.check([(s, t, 16) for s, t in zip(tables.ravel(), moved.ravel()) if s != t], 16)
    assert np.array_equal(pools.cache.compact(pool, moved), moved)  # nothing left to do


def test_states_are_copied_in_every_layer():
    states = ct.DeltaStates(3, 7, 2, 32, 96)
    for layer in range(3):
        assert not states.state(layer).numpy().any()  # zero at first
        fill(states.state(layer), layer)
    before = [bits(states.state(layer)) for layer in range(3)]
    states.copy([0, 1, 5], [1, 0, 6])
    for was, layer in zip(before, range(3)):
        assert np.array_equal(bits(states.state(layer)), was[[1, 0, 2, 3, 4, 5, 5]])
