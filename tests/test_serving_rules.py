"""What the host side of page pools, forks, compaction, delta batches and experts decides and refuses, without a GPU:
tests/clients/serving_checks.cpp calls the library's own functions, with the copy of pages done on the host."""
import os
import random
import subprocess

import numpy as np
import pytest

import ctorch_amd as ct

PROGRAM = os.path.join(os.path.dirname(os.path.abspath(__file__)), "clients", "_build", "serving_checks")


def checks(*arguments):
    if not os.path.exists(PROGRAM):
        import __graft_entry__
        __graft_entry__.build()
    return subprocess.run([PROGRAM, *map(str, arguments)], capture_output=True, text=True, timeout=60)


def text(values):
    return ",".join(map(str, values)) or "-"


# ------------------------------------------------------------------------------------------------ the pool
def test_a_pool_hands_out_its_lowest_free_pages():
    pool = ct.PagePool(9)
    pool.claim([2, 4, -1])
    assert pool.available == 7 and pool.take(4).tolist() == [0, 1, 3, 5] and pool.available == 3
    pool.share([4, 0, -1])
    assert [pool.references(i) for i in range(9)] == [2, 1, 1, 1, 2, 1, 0, 0, 0]
    pool.release([0, 1, 4, -7])
    assert [pool.references(i) for i in range(9)] == [1, 0, 1, 1, 1, 1, 0, 0, 0] and pool.available == 4
    assert pool.take(0).tolist() == [] and pool.take(4).tolist() == [1, 6, 7, 8] and pool.available == 0
    pool.release(np.array([[8, 0], [-1, 3]]))  # a table
    assert pool.take(2).tolist() == [0, 3]


@pytest.mark.parametrize("seed", range(5))
def test_a_pool_counts_as_a_plain_list_does(seed):
    rng, pool, held = random.Random(seed), ct.PagePool(40), [0] * 40
    for _ in range(300):
        kind, ids = rng.choice(["take", "claim", "share", "release"]), rng.choices(range(-1, 40), k=rng.randint(0, 6))
        if kind == "take":
            free = [i for i in range(40) if held[i] == 0]
            if len(ids) > len(free):
                with pytest.raises(ct.DLError, match="pages wanted"):
                    pool.take(len(ids))
                continue
            assert pool.take(len(ids)).tolist() == free[:len(ids)]
            for i in free[:len(ids)]:
                held[i] = 1
            continue
        after = list(held)
        for i in ids:
            if i >= 0:
                after[i] += -1 if kind == "release" else 1
        bad = any(n < 0 for n in after) or (kind == "share" and any(i >= 0 and held[i] == 0 for i in ids))
        if bad:
            with pytest.raises(ct.DLError, match="not held"):
                getattr(pool, kind)(ids)
        else:
            getattr(pool, kind)(ids)
            held = after
        assert [pool.references(i) for i in range(40)] == held and pool.available == held.count(0)


def test_a_pool_refuses():
    pool = ct.PagePool(4)
    for call, said in ((lambda: pool.claim([1, 4]), "not in the pool"), (lambda: pool.release([4]), "not in the pool"),
                       (lambda: pool.references(-1), "not in the pool"), (lambda: pool.take(-1), "below zero"),
                       (lambda: pool.take(5), "5 pages wanted, 4 are free"), (lambda: pool.take(2 ** 40), "pages wanted"),
                       (lambda: pool.share([0]), "not held"), (lambda: ct.PagePool(-3), "positive")):
        with pytest.raises(ct.DLError, match=said):
            call()
    assert pool.available == 4
    lib = ct.lib()
    assert lib.dl_page_pool_take(pool.handle, 1, None) == 1 and "NULL" in ct.last_error() and pool.available == 4
    assert lib.dl_page_pool_claim(pool.handle, 1, None) == 1 and "NULL" in ct.last_error()
    assert lib.dl_page_pool_claim(pool.handle, -1, None) == 1 and lib.dl_page_pool_claim(pool.handle, 0, None) == 0
    assert lib.dl_page_pool_take(None, 0, None) == 1 and lib.dl_page_pool_available(pool.handle, None) == 1


# ------------------------------------------------------------------------------------------------ copies
@pytest.mark.parametrize("sources,targets,rows", [
    ([1], [4], None), ([1, 1, 1], [2, 3, 4], None), ([0, 1], [1, 0], None), ([0, 1, 2], [1, 2, 0], [16, 3, 1]),
    ([0, 1, 2, 3], [1, 2, 3, 4], None), ([3, 3, 5], [5, 3, 1], [2, 16, 7]), ([2, 2, 2], [0, 1, 2], [1, 5, 9]), ([], [], None),
    ([0, 0, 1], [1, 2, 3], [4, 0, 16])])
@pytest.mark.parametrize("heads,page,size,pools", [(1, 16, 16, 1), (3, 32, 48, 2), (2, 16, 256, 70)])
def test_copies_take_their_sources_as_they_were(sources, targets, rows, heads, page, size, pools):
    run = checks("copy", 6, heads, page, size, pools, text(sources), text(targets), text(rows or []))
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("seed", range(6))
def test_copies_of_many_pages(seed):
    rng = random.Random(seed)
    pages = rng.choice([300, 700])
    count = rng.randint(241, pages)
    targets, page = rng.sample(range(pages), count), 16
    run = checks("copy", pages, 1, page, 16, 3, text(rng.choices(range(pages), k=count)), text(targets),
                 text([rng.randint(0, page) for _ in range(count)]) if seed % 2 else "-")
    assert run.returncode == 0, run.stderr


def plain_fork(pages, page, width, tables, lengths, parents):
    held = [0] * pages
    for i in sum(tables, []):
        if i >= 0:
            held[i] += 1
    free, children = [i for i in range(pages) if held[i] == 0], []
    for b in parents:
        whole, rest = divmod(lengths[b], page)
        table = tables[b][:whole]
        for i in table:
            held[i] += 1
        if rest:
            table = table + [free.pop(0)]
            held[table[-1]] += 1
        children.append(table + [-1] * (width - len(table)))
    return children, held


@pytest.mark.parametrize("seed", range(12))
def test_a_fork_shares_whole_pages_and_copies_the_last(seed):
    rng = random.Random(seed)
    page, width, batch = rng.choice([16, 32]), rng.randint(1, 7), rng.randint(1, 5)
    lengths = [rng.choice([0, page, width * page, rng.randint(0, width * page)]) for _ in range(batch)]
    parents = rng.choices(range(batch), k=rng.randint(0, 8))
    order = rng.sample(range(80), 80)
    tables = [[order.pop() for _ in range(-(-n // page))] for n in lengths]
    tables = [t + [order.pop() if rng.random() < 0.3 else -1 for _ in range(width - len(t))] for t in tables]  # (some reserved)
    children, held = plain_fork(80, page, width, tables, lengths, parents)
    run = checks("fork", 80, page, width, text(sum(tables, [])), text(lengths), text(parents))
    assert run.returncode == 0, run.stderr
    first, second = run.stdout.splitlines()
    assert list(map(int, first.split())) == sum(children, []) and list(map(int, second.split())) == held


@pytest.mark.parametrize("seed", range(12))
def test_compaction_moves_what_lies_behind_to_the_front(seed):
    rng = random.Random(seed)
    pages = rng.randint(1, 60)
    live = rng.sample(range(pages), rng.randint(0, pages))
    tables = live + rng.choices(live, k=5 if live else 0) + [-1] * rng.randint(0, 3)  # (some shared)
    rng.shuffle(tables)
    run = checks("compact", pages, 16, text(tables))
    assert run.returncode == 0, run.stderr
    far, near = sorted(i for i in live if i >= len(live)), [i for i in range(len(live)) if i not in live]
    moved = dict(zip(far, near))
    lines = run.stdout.splitlines()
    assert list(map(int, lines[0].split())) == [moved.get(i, i) for i in tables] and int(lines[1]) == len(far)


# ------------------------------------------------------------------------------------------------ hidden entries of experts
@pytest.mark.parametrize("unit", [4, 8])  # entries of a 16-byte piece: f32, bf16
@pytest.mark.parametrize("laid", [0, 1])
@pytest.mark.parametrize("hidden", [1, 3, 4, 5, 7, 8, 9, 12, 15, 16, 17, 33, 63, 64, 1025])
def test_hidden_entries_and_zeros_share_a_pairs_room(hidden, unit, laid):
    """Each place of a pair's room is written once, and nothing beside it: side by side the entries fill it, in pieces the last
    piece holds the last `unit` ones, those of them that stand in a piece before it as zeros."""
    if laid and hidden < unit:
        return  # (no piece: such products go entry by entry)
    run = checks("hidden", hidden, unit, laid)
    assert run.returncode == 0, run.stderr
    (room,), places, zeros = (list(map(int, line.split())) for line in run.stdout.splitlines())
    whole = hidden // unit * unit
    assert room == (-(-hidden // unit) * unit if laid else hidden)
    want = list(range(hidden))
    if laid and hidden > whole:
        want = list(range(whole)) + [i - (hidden - unit) + whole for i in range(whole, hidden)]
    assert places == want
    assert sorted(places + [z for z in zeros if z >= 0]) == list(range(room))


# ------------------------------------------------------------------------------------------------ refusals
REFUSED = {
    "pool empty": "positive", "pool large": "2^31", "copy unequal": "target", "copy rows unequal": "rows", "copy source": "not one of",
    "copy target": "not one of", "copy twice": "written twice", "copy rows": "from 0 to 16", "copy rows below": "from 0 to 16",
    "copy large": "2 GiB", "fork other pool": "other pages", "fork tables": "[sequences, width]", "fork parent": "not one of",
    "fork parent below": "not one of", "fork length": "outside its table", "fork length below": "outside its table",
    "fork missing page": "not held", "fork page beyond": "not held", "fork free page": "not held", "fork too many": "6 pages wanted",
    "fork failing": "HIP", "compact other pool": "other pages", "compact beyond": "not in the cache", "compact missing": "is held 1 times",
    "compact twice": "stands 2 times", "states layers": "positive", "states key_dim": "32, 64 or 128", "states value_dim": "multiple of 32",
    "states wide": "multiple of 32", "states slots": "too many", "states host": "delta states", "batch key_heads": "multiple of key_heads",
    "batch no key_heads": "multiple of key_heads", "batch empty": "each of its requests", "batch unequal": "each of its requests",
    "batch count": "below zero", "batch target": "slot 6", "batch no target": "slot -1", "batch source": "slot 6",
    "batch source below": "slot -2", "batch written twice": "two requests", "batch read and written": "read by another",
    "batch read and written before": "read by another", "batch many": "too many", "batch many heads": "too many", "batch many requests": "too many requests", "states heads": "too many",
    "experts large": "too many experts",
    "delta other states": "another layout", "delta fewer slots": "another layout", "delta layer": "layer out of range",
    "delta layer below": "layer out of range", "delta query": "query must be", "delta key heads": "key must be",
    "delta value": "value must be", "delta type": "f32 or bf16", "delta host": "another device", "delta decay": "decay must be",
    "delta rate type": "f32 or bf16", "delta host decay": "another device", "delta scale": "finite", "delta scale beyond f32": "finite in f32", "delta undefined": "undefined tensor",
    "delta undefined rate": "undefined tensor", "states copy twice": "written twice", "states copy beyond": "not one of",
    "experts router": "router [E, d]", "experts router rank": "router [E, d]", "experts gate": "gate and up", "experts up": "gate and up",
    "experts down": "down [E, d, F]", "experts top": "top must be", "experts no top": "top must be", "experts top beyond": "top must be",
    "experts many": "too many experts", "experts types": "one type", "experts weight type": "bf16 or f32",
    "experts input type": "f32 or bf16", "experts host": "expert_mixture", "experts host weights": "another device",
    "experts strides": "contiguous", "experts no width": "positive", "experts undefined": "undefined tensor", "experts module": "top from 1",
}


@pytest.mark.parametrize("name", REFUSED)
def test_an_operator_refuses(name):
    run = checks("call", name)
    assert run.returncode == 1 and REFUSED[name] in run.stderr, (run.returncode, run.stdout, run.stderr)


@pytest.mark.parametrize("name", ["copy nothing", "copy itself", "compact nothing", "delta nothing", "experts nothing"])
def test_nothing_to_do_launches_nothing(name):
    run = checks("call", name)
    assert run.returncode == 0 and run.stdout.strip() == "0", (run.stdout, run.stderr)


def test_rows_that_lie_in_the_states_that_are_written_are_copied_first():
    first, other = (checks("call", f"delta rows of {where}") for where in ("the states", "another layer"))
    assert first.returncode == other.returncode == 0, (first.stderr, other.stderr)
    assert int(first.stdout) == int(other.stdout) + 1


def test_the_python_wrappers_check_shapes():
    pool, holder = ct.PagePool(4), ct.PagedCache.__new__(ct.PagedCache)  # (a cache needs a GPU; the shapes are looked at first)
    holder.handle = None
    for call in (lambda: holder.copy_pages([1, 2], [3]), lambda: holder.copy_pages([1], [3], [1, 2]),
                 lambda: holder.fork(pool, [0, 1], [5], [0]), lambda: holder.fork(pool, [[0, 1]], [5, 6], [0]),
                 lambda: ct.DeltaBatch(holder, 1, [0], [0, 1], [1])):
        with pytest.raises(ValueError):
            call()
