"""What the paged cache's host side decides and refuses, without a GPU: tests/clients/paged_checks.cpp calls the library's
own functions and walks the plan of a step as the kernels do."""
import os
import random
import subprocess

import numpy as np
import pytest

import ctorch_amd as ct

U = 2.0 ** -24
PROGRAM = os.path.join(os.path.dirname(os.path.abspath(__file__)), "clients", "_build", "paged_checks")


def checks(*arguments):
    if not os.path.exists(PROGRAM):
        import __graft_entry__
        __graft_entry__.build()
    return subprocess.run([PROGRAM, *map(str, arguments)], capture_output=True, text=True, timeout=60)


def plan(lengths, counts, tables, page=16, pages=64, kv=2, heads=8, head_dim=64, bf16=0, shared=0):
    text = [",".join(map(str, a)) for a in (lengths, counts, sum(tables, []))]
    return checks("plan", pages, page, kv, heads, head_dim, bf16, shared, len(tables[0]), *text)


def layout(rng, lengths, counts, page, shared=0):
    """Page tables whose pages lie anywhere, the shared ones in front."""
    need = [-(-(n + c) // page) - shared // page for n, c in zip(lengths, counts)]
    order = list(range(shared // page + sum(max(0, n) for n in need) + 2))
    rng.shuffle(order)
    front = [order.pop() for _ in range(shared // page)]
    tables = [front + [order.pop() for _ in range(max(0, n))] for n in need]
    width = max(map(len, tables))
    return [t + [-1] * (width - len(t)) for t in tables], width, len(order) + sum(map(len, tables))


@pytest.mark.parametrize("heads,kv,head_dim", [(8, 2, 32), (32, 8, 64), (12, 4, 128), (16, 16, 64), (40, 2, 16), (6, 6, 64)])
@pytest.mark.parametrize("seed", range(6))
def test_a_plan_gives_every_row_each_of_its_keys_once(heads, kv, head_dim, seed):
    rng = random.Random(seed + heads)
    for _ in range(6):
        batch, page = rng.choice([1, 2, 5, 9]), rng.choice([16, 32, 64])
        shared = rng.choice([0, 0, page, 5 * page, 40 * page])
        counts = [rng.choice([0, 1, 1, 2, 5, rng.randint(1, 90)]) for _ in range(batch)]
        lengths = [shared + rng.choice([0, 1, 15, 16, 17, rng.randint(0, 900), rng.randint(0, 5000)]) for _ in range(batch)]
        tables, width, pages = layout(rng, lengths, counts, page, shared)
        if width == 0:
            continue
        run = plan(lengths, counts, tables, page, max(1, pages), kv, heads, head_dim, seed % 2, shared)
        assert run.returncode == 0, (lengths, counts, page, shared, run.stderr)
        assert int(run.stdout.split()[0]) == sum(counts)


def test_a_long_sequence_among_short_ones_is_split():
    lengths = [20000, 10, 10, 10]
    tables, width, pages = layout(random.Random(1), lengths, [1] * 4, 16)
    run = plan(lengths, [1] * 4, tables, 16, pages)
    assert run.returncode == 0, run.stderr
    tokens, items, shared, merges = map(int, run.stdout.split())
    assert tokens == 4 and items > 20 and shared == 0 and merges == 1


BAD = {
    "no sequences agree": ([5, 5], [1], [[0], [1]], {}, "length and a count"),
    "heads": ([5], [1], [[0]], dict(heads=9), "multiple"),
    "length below zero": ([-1], [1], [[0]], {}, "outside its table"),
    "count below zero": ([5], [-1], [[0]], {}, "outside its table"),
    "one page too few": ([16], [1], [[0]], {}, "outside its table"),
    "far beyond": ([2 ** 62], [2 ** 62], [[0]], {}, "outside its table"),
    "page below zero": ([17], [1], [[0, -1]], {}, "not in the cache"),
    "page beyond the cache": ([17], [1], [[64, 1]], {}, "not in the cache"),
    "one page for two sequences": ([5, 3], [1, 1], [[7], [7]], {}, "two places"),
    "one page twice in a sequence": ([10], [20], [[3, 3]], {}, "two places"),
    "written under another's history": ([20, 5], [1, 1], [[3, 4], [3, 9]], {}, "another place"),
    "written under its own history": ([20], [1], [[4, 4]], {}, "another place"),
    "shared prefix of half a page": ([20], [1], [[4, 5]], dict(shared=8), "whole pages"),
    "shared prefix below zero": ([20], [1], [[4, 5]], dict(shared=-16), "whole pages"),
    "shared prefix not held": ([15], [2], [[4, 5]], dict(shared=16), "does not hold"),
    "shared prefix in other pages": ([16, 16], [1, 1], [[4, 5], [6, 7]], dict(shared=16), "begin with"),
}


@pytest.mark.parametrize("name", BAD)
def test_a_batch_that_cannot_be_is_refused(name):
    lengths, counts, tables, more, said = BAD[name]
    run = plan(lengths, counts, tables, **more)
    assert run.returncode == 1 and said in run.stderr, (run.returncode, run.stdout, run.stderr)


def test_sequences_without_new_positions_are_not_looked_at():
    # their table may be empty and their pages anyone's
    run = plan([5, 40, 3], [1, 0, 2], [[7, -1, -1], [7, 7, 99], [8, -1, -1]])
    assert run.returncode == 0 and run.stdout.split()[0] == "3", run.stderr
    assert plan([5], [0], [[-1]]).stdout.split() == ["0"] * 4


REFUSED = {
    "cache layers": "positive", "cache pages": "positive", "cache page size 8": "power of two",
    "cache page size 24": "power of two", "cache page size 2048": "power of two", "cache head 48": "head size",
    "cache heads": "positive", "cache f64": "f32 or bf16", "cache on the host": "GPU only",
    "append layer": "layer out of range", "append layer below": "layer out of range", "append rows": "key must be [3, 2, 32]",
    "append heads": "value must be [3, 2, 32]", "append query heads": "query must be [3, 4, 32]", "append type": "f32 or bf16",
    "append host rows": "another device", "append short tables": "position 22", "append wide tables": "rotate 34 of 32",
    "append unequal tables": "alike", "append empty tables": "rotate 0", "append layout": "layout",
    "attend other cache": "another layout", "attend other type": "another layout", "attend fewer pages": "another layout",
    "attend layer": "layer out of range", "attend rows": "query must be [3, 4, 32]", "attend flat": "query must be",
    "attend type": "f32 or bf16", "attend host rows": "another device", "rotary rank": "[T, H, D]",
    "rotary positions": "positions must be", "rotary positions type": "positions must be",
    "rotary host positions": "another device", "rotary host rows": "GPU only", "rotary type": "f32 or bf16",
    "rotary wide tables": "rotate 32 of 30", "rotary layout": "layout", "rotary heads": "too many heads", "verify drafts": "2^20 drafts", "tables odd": "even", "tables empty": "capacity",
    "tables base": "base", "tables kind": "unknown scaling", "tables factor": "factor", "tables trained": "trained",
    "tables turns": "slow_turns", "tables one pair": "two pairs", "tables magnitude": "finite", "verify ids": "drafted must be",
    "verify target": "[B, K + 1, V]", "verify draft": "[B, K, V]", "verify uniforms": "uniforms must be",
    "verify uniforms type": "uniforms must be", "verify vocabulary": "empty vocabulary", "verify temperature": "finite",
    "verify temperature nan": "finite", "verify logits type": "f32 or bf16", "verify host ids": "different devices",
    "verify host draft": "different devices",
}


@pytest.mark.parametrize("name", REFUSED)
def test_an_operator_refuses(name):
    run = checks("call", name)
    assert run.returncode == 1 and REFUSED[name] in run.stderr, (run.returncode, run.stdout, run.stderr)


@pytest.mark.parametrize("name", ["append undefined tables", "append undefined sines", "append undefined rows"])
def test_undefined_tensors_are_refused(name):
    run = checks("call", name)
    assert run.returncode == 1 and "undefined tensor" in run.stderr, (run.returncode, run.stdout, run.stderr)


@pytest.mark.parametrize("name", ["cache elements", "cache bytes"])
def test_a_cache_whose_size_wraps_is_refused(name):
    run = checks("call", name)  # 2^67 elements, 2^64 bytes: both nothing in 64 bits
    assert run.returncode == 1 and "too many elements" in run.stderr, (run.returncode, run.stdout, run.stderr)


@pytest.mark.parametrize("name,said", [("batch heads", "too many heads"), ("batch of too many items", "too many new positions"),
                                       ("batch of too many merges", "too many new positions"), ("verify rows", "too many rows")])
def test_a_launch_has_fewer_than_2_to_the_32_threads(name, said):
    run = checks("call", name)
    assert run.returncode == 1 and said in run.stderr, (run.returncode, run.stdout, run.stderr)


def test_sizes_that_wrap_are_refused():
    cpu = ct.device("cpu")
    for call in (lambda: ct.rotary_tables(32, 2 ** 60, dev=cpu), lambda: ct.rotary_tables(32, 2 ** 58, dev=cpu),
                 lambda: ct.zeros((2 ** 32, 2 ** 32), ct.F32, cpu), lambda: ct.zeros((2 ** 32, 0, 2 ** 32), ct.F32, cpu),
                 lambda: ct.zeros((2 ** 61,), ct.F64, cpu)):
        with pytest.raises(ct.DLError, match="too many elements"):
            call()
    assert ct.zeros((2 ** 30, 0, 2 ** 28), ct.F32, cpu).shape == (2 ** 30, 0, 2 ** 28)  # (strides within 2^59)


@pytest.mark.parametrize("name", ["append nothing", "attend nothing", "rotary nothing", "verify nothing"])
def test_nothing_to_do_launches_nothing(name):
    run = checks("call", name)
    assert run.returncode == 0 and run.stdout.strip() == "0", (run.stdout, run.stderr)


@pytest.mark.parametrize("name,launches", [("append rows of the pages", 3), ("append rows of another layer", 1)])
def test_what_lies_in_the_pages_that_are_written_is_copied_first(name, launches):
    run = checks("call", name)
    assert run.returncode == 0 and run.stdout.strip() == str(launches), (run.stdout, run.stderr)


# ------------------------------------------------------------------------------------------------ tables
def frequencies(dims, base, kind, factor, trained, slow, fast):
    i = np.arange(dims // 2, dtype=np.float64)
    if kind == ct.ROTARY_BASE:
        base = base * factor ** (dims / (dims - 2))
    f = base ** (-2 * i / dims)
    if kind == ct.ROTARY_LINEAR:
        f = f / factor
    if kind == ct.ROTARY_PARTS:
        keep = np.clip((trained * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


@pytest.mark.parametrize("dims,base", [(64, 10000.0), (128, 500000.0), (6, 100.0), (2, 10.0)])
@pytest.mark.parametrize("kind", [ct.ROTARY_UNSCALED, ct.ROTARY_LINEAR, ct.ROTARY_BASE, ct.ROTARY_PARTS])
def test_rotary_tables_are_the_angles_rounded_once(dims, base, kind):
    if kind == ct.ROTARY_BASE and dims == 2:
        return
    rule = ct.RotaryScaling(kind, 8.0, 4096, 1.0, 32.0, 1.25)
    cosine, sine = ct.rotary_tables(dims, 5000, base, rule, ct.device("cpu"))
    angles = np.arange(5000)[:, None] * frequencies(dims, base, kind, 8.0, 4096, 1.0, 32.0)
    # an angle of at most 5000 is off by a few steps of 64 bits, the entry by half a step of 32 bits
    for table, exact in ((cosine, np.cos(angles)), (sine, np.sin(angles))):
        assert table.shape == (5000, dims // 2) and table.dtype == ct.F32
        assert np.max(np.abs(table.numpy() - 1.25 * exact)) <= 1.25 * 2.0 ** -24 + 5000 * 2.0 ** -49


def test_the_scalings_keep_what_they_say():
    at = lambda rule: frequencies(64, 10000.0, *rule)  # noqa: E731
    plain = at((ct.ROTARY_UNSCALED, 8.0, 8192, 1.0, 32.0))
    base = at((ct.ROTARY_BASE, 8.0, 8192, 1.0, 32.0))
    assert np.isclose(base[0], plain[0]) and np.isclose(base[-1], plain[-1] / 8)
    parts = at((ct.ROTARY_PARTS, 8.0, 8192, 1.0, 32.0))
    assert parts[0] == plain[0] and parts[-1] == plain[-1] / 8


@pytest.mark.parametrize("dims,base", [(64, 10000.0), (128, 500000.0)])
def test_the_tables_scale_as_they_say(dims, base):
    """The angles of the first position: which pairs a rule leaves alone, which it slows down by the factor, and by how much
    the others lie in between.  (sin f of f32, off by 2^-24 of it and less than twice that as an angle below 1.)"""
    cpu = ct.device("cpu")

    def angles(kind, slow=1.0, fast=32.0, magnitude=1.0):
        rule = ct.RotaryScaling(kind, 8.0, 8192, slow, fast, magnitude)
        cosine, sine = ct.rotary_tables(dims, 2, base, rule, cpu)
        return np.arctan2(sine.numpy()[1].astype(np.float64), cosine.numpy()[1].astype(np.float64))

    i = np.arange(dims // 2)
    plain = angles(ct.ROTARY_UNSCALED)
    assert np.allclose(plain, base ** (-2 * i / dims), rtol=4 * U, atol=0)
    assert np.allclose(angles(ct.ROTARY_LINEAR), plain / 8, rtol=8 * U, atol=0)
    raised = angles(ct.ROTARY_BASE)
    assert np.allclose(raised, plain * 8.0 ** (-2 * i / (dims - 2)), rtol=8 * U, atol=0)
    assert np.isclose(raised[0], plain[0], rtol=8 * U) and np.isclose(raised[-1], plain[-1] / 8, rtol=8 * U)
    parts, turns = angles(ct.ROTARY_PARTS), 8192 * plain / (2 * np.pi)
    assert np.allclose(parts[turns >= 32], plain[turns >= 32], rtol=8 * U, atol=0)
    assert np.allclose(parts[turns <= 1], plain[turns <= 1] / 8, rtol=8 * U, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and np.all(parts[between] < plain[between]) and np.all(parts[between] > plain[between] / 8)
    assert np.all(np.diff(parts) < 0)
    # other borders move the pairs that are kept
    assert np.sum(angles(ct.ROTARY_PARTS, 0.25, 4.0) == plain) > np.sum(parts == plain)
    # a magnitude leaves the angle
    assert np.allclose(angles(ct.ROTARY_PARTS, magnitude=1.25), parts, rtol=8 * U, atol=0)
