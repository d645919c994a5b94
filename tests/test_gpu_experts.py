"""A layer of experts on the GPU against numpy in 64 bits.

Tolerances, from the arithmetic (u = 2^-24): products keep all bits of an f32 and sums of n of them are of f32, so that a dot
product is off by at most (n + 4) u of the sum of its products' magnitudes, in any order (matrix instructions add four and more
products at once, within the same bound).  silu(g) has a slope of at most 1.1 and comes out within 8 u; the chosen experts' weights
are of 64 bits, rounded once, and the sum over them adds (top + 2) u."""
import numpy as np
import pytest

import ctorch_amd as ct
import oracle
from common import say, write

pytestmark = pytest.mark.gpu
GPU = ct.device("gpu")
TYPES = {"f32": ct.F32, "bf16": ct.BF16}
U = 2.0 ** -24


def give(values, dtype="f32"):
    """The tensor on the GPU, and the values that it holds."""
    if dtype == "bf16":
        bits = oracle.bf16_encode(np.ascontiguousarray(values, np.float32))
        return ct.Tensor.from_numpy(bits, ct.BF16, GPU), oracle.bf16_decode(bits).astype(np.float64)
    values = np.asarray(values, np.float32)
    return ct.Tensor.from_numpy(values, ct.F32, GPU), values.astype(np.float64)


def route(x, router, top, normalise):
    z = x @ router.T
    chosen = np.argsort(-z, axis=-1, kind="stable")[:, :top]
    p = np.exp(z - z.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    weights = np.take_along_axis(p, chosen, -1)
    return chosen, weights / weights.sum(-1, keepdims=True) if normalise else weights


def mixed(x, gate, up, down, chosen, weights):
    """Outputs and their tolerances."""
    T, d = x.shape
    F, top = gate.shape[1], chosen.shape[1]
    y, off = np.zeros((T, d)), np.zeros((T, d))
    size = np.zeros((T, d))
    for e in np.unique(chosen):
        t, j = np.nonzero(chosen == e)
        rows, w = x[t], weights[t, j][:, None]
        g, h = rows @ gate[e].T, rows @ up[e].T
        eg, eh = ((d + 4) * U * (np.abs(rows) @ np.abs(m[e]).T) for m in (gate, up))
        s = g / (1 + np.exp(-g))
        act = s * h
        ea = 1.1 * eg * (np.abs(h) + eh) + (np.abs(s) + 1.1 * eg) * eh + 8 * U * np.abs(act)
        part, ep = act @ down[e].T, ea @ np.abs(down[e]).T + (F + 4) * U * (np.abs(act) @ np.abs(down[e]).T)
        np.add.at(y, t, w * part)
        np.add.at(off, t, w * ep)
        np.add.at(size, t, w * np.abs(part))
    return y, off + (top + 2) * U * size


def check(T, d, F, E, top, weight="bf16", inputs="f32", normalise=True, seed=0, shape=None, change=None):
    say(f"case: experts T={T} d={d} F={F} E={E} top={top} {weight} {inputs} normalise={normalise}")
    rng = np.random.default_rng(seed + T + d)
    arrays = [rng.standard_normal((T, d))] + [rng.standard_normal(s) * s[-1] ** -0.5 for s in ((E, d), (E, F, d), (E, F, d), (E, d, F))]
    if change:
        change(arrays)
    tensors, values = zip(*[give(a if i or shape is None else a.reshape(shape), inputs if i == 0 else weight) for i, a in enumerate(arrays)])
    y, chosen, weights = ct.expert_mixture(*tensors, top, normalise)
    lead = (T,) if shape is None else tuple(shape[:-1])
    assert y.shape == lead + (d,) and chosen.shape == weights.shape == lead + (top,)
    assert y.dtype == weights.dtype == ct.F32 and chosen.dtype == ct.I64
    want_chosen, want_weights = route(values[0].reshape(T, d), values[1], top, normalise)
    assert np.array_equal(chosen.numpy().reshape(T, top), want_chosen)
    off = np.abs(weights.numpy().reshape(T, top) - want_weights)
    assert np.all(off <= U * want_weights + 2.0 ** -149 + 1e-13)
    want, tolerance = mixed(values[0].reshape(T, d), *values[2:], want_chosen, want_weights)
    off = np.abs(y.numpy().reshape(T, d) - want)
    assert np.all(off <= tolerance), (np.unravel_index(np.argmax(off / tolerance), off.shape), np.max(off / tolerance))
    say(f"  at most {np.max(off / tolerance):.3f} of the tolerance")
    return y.numpy()


SIZES = [(1, 64, 32, 4, 2), (2, 256, 688, 8, 2), (3, 128, 8, 3, 3), (5, 1000, 72, 16, 4), (16, 512, 256, 64, 8), (17, 96, 40, 5, 1),
         (33, 256, 136, 8, 8), (64, 264, 64, 6, 2), (130, 128, 192, 4, 3), (300, 192, 104, 7, 2), (1, 2048, 704, 2, 2), (7, 72, 1032, 2, 1)]


@pytest.mark.parametrize("T,d,F,E,top", SIZES)
@pytest.mark.parametrize("weight", ["f32", "bf16"])
@pytest.mark.parametrize("inputs", ["f32", "bf16"])
def test_rows_through_their_experts(T, d, F, E, top, weight, inputs):
    check(T, d, F, E, top, weight, inputs, normalise=T % 2 == 0)


@pytest.mark.parametrize("T,d,F,E,top", [(1, 1, 1, 1, 1), (4, 7, 5, 3, 2), (2, 65, 33, 9, 4), (20, 63, 64, 4, 2), (3, 64, 63, 4, 2),
                                         (9, 68, 36, 4, 2), (5, 100, 20, 130, 3), (40, 12, 4, 6, 2)])
@pytest.mark.parametrize("weight", ["f32", "bf16"])
def test_odd_sizes(T, d, F, E, top, weight):
    check(T, d, F, E, top, weight, "f32", normalise=T % 2 == 1)


@pytest.mark.parametrize("E,top", [(1024, 64), (64, 64), (65, 1), (1000, 3)])
def test_many_experts(E, top):
    check(6, 64, 16, E, top, "bf16")


@pytest.mark.parametrize("T,E,top,narrow,long", [(4, 64, 4, 32, 1032), (8, 64, 4, 40, 1064), (8, 128, 8, 24, 1040), (16, 64, 4, 32, 1040),
                                                 (64, 16, 2, 72, 520), (34, 64, 1, 32, 520), (40, 64, 1, 32, 1040), (60, 64, 1, 24, 1104),
                                                 (4, 64, 4, 39, 1031), (8, 64, 4, 41, 1063), (16, 64, 4, 33, 1039)])
@pytest.mark.parametrize("weight", ["f32", "bf16"])
@pytest.mark.parametrize("inputs", ["f32", "bf16"])
def test_long_matrices_of_few_and_of_many_experts(T, E, top, narrow, long, weight, inputs):
    """Each product with 512 to 4200 tiles of 16 rows, by itself: as many go to a wave as leave waves enough."""
    check(T, narrow, long, E, top, weight, inputs)
    check(T, long, narrow, E, top, weight, inputs, seed=1)


@pytest.mark.parametrize("weight", ["f32", "bf16"])
def test_many_pairs_of_few_rows(weight):
    check(16, 1024, 72, 64, 64, weight)
    check(32, 256, 24, 32, 32, weight)


@pytest.mark.parametrize("T,d,F,E,top", [(40, 65, 40, 32, 1), (64, 127, 33, 64, 2), (65, 127, 33, 64, 2), (33, 63, 64, 8, 8), (32, 2047, 24, 8, 3)])
@pytest.mark.parametrize("weight", ["f32", "bf16"])
@pytest.mark.parametrize("inputs", ["f32", "bf16"])
def test_odd_rows_one_by_one_and_together(T, d, F, E, top, weight, inputs):
    check(T, d, F, E, top, weight, inputs)


@pytest.mark.parametrize("T,E,long", [(20, 64, 16400), (40, 64, 32776), (60, 64, 65544)])
def test_more_rows_than_a_tile_through_one_of_many_experts(T, E, long):
    def change(a):
        a[0][:] = np.abs(a[0])
        a[1][:] = 0
        a[1][5] = 1
    check(T, 32, long // T, E, 1, change=change)


def test_all_rows_to_one_expert():
    def change(a):
        a[0][:] = np.abs(a[0])
        a[1][:] = 0
        a[1][5] = 1
    check(200, 64, 48, 8, 1, change=change)
    check(70, 64, 48, 8, 1, "f32", change=change)


def test_the_lowest_index_is_first_among_equals():
    def change(a):
        a[1][:] = a[1][:1]
        a[1][7:] += 1.0 / 64
        a[0][:] = np.abs(a[0])
    check(9, 64, 32, 20, 5, "bf16", change=change)
    check(9, 64, 32, 20, 20, "f32", change=lambda a: a[1].fill(0.0))


def test_near_ties_are_settled_in_64_bits():
    """Logits of about 30 that differ by one step of f32 of an entry, 2^-23: sums of f32 would round it away."""
    def change(a):
        a[0][:] = 1.0
        a[1][:] = 0.5
        a[1][3, 11] += 2.0 ** -24
        a[1][6, 12] += 2.0 ** -23
        a[1][9, 13] -= 2.0 ** -24
    check(3, 64, 32, 12, 3, "f32", change=change)


@pytest.mark.parametrize("weight", ["f32", "bf16"])
def test_large_and_small_values(weight):
    check(4, 128, 64, 4, 2, weight, change=lambda a: a[2].__imul__(60.0))  # silu far from zero, both sides
    check(4, 128, 64, 4, 2, weight, change=lambda a: a[0].__imul__(1e-4))


@pytest.mark.parametrize("T", [3, 40])
def test_rows_that_are_not_finite_stay_alone(T):
    rng = np.random.default_rng(T)
    arrays = [rng.standard_normal(s) * 0.2 for s in ((T, 64), (8, 64), (8, 32, 64), (8, 32, 64), (8, 64, 32))]
    tensors = [give(a, "bf16" if i else "f32")[0] for i, a in enumerate(arrays)]
    want = [t.numpy() for t in ct.expert_mixture(*tensors, 2)]
    arrays[0][1, 5], arrays[0][2, 3] = np.nan, np.inf
    tensors = (give(arrays[0])[0], *tensors[1:])
    y, chosen, weights = (t.numpy() for t in ct.expert_mixture(*tensors, 2))
    others = [t for t in range(T) if t not in (1, 2)]
    for got, right in zip((y, chosen, weights), want):
        assert np.array_equal(got[others], right[others])
    assert np.array_equal(chosen[1], [0, 1]) and np.isnan(weights[1]).all() and np.isnan(y[1]).all()
    assert np.all((chosen[2] >= 0) & (chosen[2] < 8)) and chosen[2, 0] != chosen[2, 1]


def test_leading_axes_and_strided_rows():
    check(12, 64, 32, 4, 2, shape=(3, 4, 64))
    check(1, 64, 32, 4, 2, shape=(64,))
    rng = np.random.default_rng(1)
    wide, values = give(rng.standard_normal((6, 3, 40)))
    weights = [give(rng.standard_normal(s) * 0.2, "bf16")[0] for s in ((4, 40), (4, 16, 40), (4, 16, 40), (4, 40, 16))]
    got = ct.expert_mixture(ct.narrow(wide, 1, 1, 2), *weights, 2)
    want = ct.expert_mixture(give(values[:, 1:3])[0], *weights, 2)
    assert all(np.array_equal(a.numpy(), b.numpy()) for a, b in zip(got, want))


def test_weights_off_their_alignment():
    """Matrices that begin 2 or 4 bytes behind a boundary of 16."""
    rng = np.random.default_rng(2)
    for dtype in ("bf16", "f32"):
        shapes = ((4, 64), (4, 32, 64), (4, 32, 64), (4, 64, 32))
        arrays = [rng.standard_normal(s) * 0.2 for s in shapes]
        x, _ = give(rng.standard_normal((5, 64)))
        plain = [give(a, dtype) for a in arrays]
        moved = []
        for a, s in zip(arrays, shapes):
            flat, _ = give(np.concatenate([[0.0], a.ravel()]), dtype)
            part = ct.narrow(flat, 0, 1, a.size)
            moved.append(ct.Tensor(ct._new(ct.lib().dl_reshape, part.handle, ct._shape(s))))
        y, chosen, weights = ct.expert_mixture(x, *moved, 2)
        want_chosen, want_weights = route(x.numpy().astype(np.float64), plain[0][1], 2, True)
        want, tolerance = mixed(x.numpy().astype(np.float64), *[v for _, v in plain[1:]], want_chosen, want_weights)
        assert np.array_equal(chosen.numpy(), want_chosen) and np.all(np.abs(y.numpy() - want) <= tolerance)


def test_the_module_is_the_operator():
    module = ct.expert_mixture_module(64, 32, 6, 2, False, ct.BF16)
    state = module.state()
    assert {n: t.shape for n, t in state.items()} == {"router": (6, 64), "gate": (6, 32, 64), "up": (6, 32, 64), "down": (6, 64, 32)}
    for name, inputs in (("gate", 64), ("down", 32)):  # drawn as a Linear's
        values = oracle.bf16_decode(state[name].numpy())
        assert np.abs(values).max() <= inputs ** -0.5 * (1 + 2.0 ** -8) and values.std() > 0.5 * inputs ** -0.5
    x, _ = give(np.random.default_rng(3).standard_normal((2, 5, 64)))
    want = ct.expert_mixture(x, state["router"], state["gate"], state["up"], state["down"], 2, False)[0]
    assert np.array_equal(module.forward(x).numpy(), want.numpy())
    rng = np.random.default_rng(4)
    module.load_state({n: (rng.standard_normal(t.shape) * 0.1).astype(np.float32) for n, t in state.items()})
    state = module.state()
    want = ct.expert_mixture(x, state["router"], state["gate"], state["up"], state["down"], 2, False)[0]
    assert np.array_equal(module.forward(x).numpy(), want.numpy())


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(6)
    arrays = [rng.standard_normal(s) * 0.2 for s in ((50, 256), (16, 256), (16, 128, 256), (16, 128, 256), (16, 256, 128))]
    tensors = [give(a, "bf16" if i else "f32")[0] for i, a in enumerate(arrays)]
    first = [t.numpy() for t in ct.expert_mixture(*tensors, 4)]
    for _ in range(3):
        assert all(np.array_equal(a, t.numpy()) for a, t in zip(first, ct.expert_mixture(*tensors, 4)))


@pytest.mark.parametrize("T,d,F", [(1, 65, 64), (40, 63, 24), (3, 64, 63), (150, 129, 40), (20, 96, 41), (9, 130, 66)])
@pytest.mark.parametrize("weight,inputs", [("bf16", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
def test_one_of_the_products_in_pieces(T, d, F, weight, inputs):
    check(T, d, F, 6, 3, weight, inputs)


@pytest.mark.parametrize("T,top", [(1001, 8), (8100, 1), (130, 64)])
def test_more_rows_than_a_launch_takes(T, top):
    check(T, 64, 32, max(10, top), top, "bf16", "f32")


@pytest.mark.parametrize("T", [1, 12, 90])
@pytest.mark.parametrize("weight,inputs", [("bf16", "f32"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("d,F", [(256, 128), (511, 128), (256, 129)])
def test_all_bits_of_an_f32_count(T, weight, inputs, d, F):
    """Roundings of different sums are independent, so that their number adds up by its root: sums of d and of F products are
    off by sqrt(d + F) u of their size in the mean over many.  A row or hidden entry whose third part of 8 bits is lost is off
    by 2^-17 in the mean, always to the same side: five times and more of that."""
    rng = np.random.default_rng(T)
    arrays = [rng.standard_normal((T, d))] + [rng.standard_normal(s) * s[-1] ** -0.5 for s in ((4, d), (4, F, d), (4, F, d), (4, d, F))]
    tensors, values = zip(*[give(a, inputs if i == 0 else weight) for i, a in enumerate(arrays)])
    chosen, weights = route(values[0], values[1], 2, True)
    want, _ = mixed(values[0], *values[2:], chosen, weights)
    error = ct.expert_mixture(*tensors, 2)[0].numpy() - want
    assert np.linalg.norm(error) <= (d + F) ** 0.5 * U * np.linalg.norm(want)


@pytest.mark.parametrize("weight,F", [("bf16", (1 << 24) + 1), ("bf16", (1 << 24) + 15), ("f32", (1 << 23) + 1), ("f32", (1 << 23) + 3)])
@pytest.mark.parametrize("T", [1, 3, 12])
def test_matrices_beyond_2_gib(weight, F, T):
    """Zero but for the hidden entries at both ends: what a row's last ones write must not reach its own or the next row's first.
    (A zero adds nothing to a sum, whose tolerance counts the others.)"""
    d, ends = 64, [8, 17]
    say(f"case: experts T={T} d={d} F={F} {weight}")
    rng = np.random.default_rng(T)
    n = sum(ends)
    x, rows = give(rng.standard_normal((T, d)))
    router, _ = give(np.ones((1, d)), weight)
    coded = lambda a: oracle.bf16_encode(np.ascontiguousarray(a, np.float32)) if weight == "bf16" else np.ascontiguousarray(a, np.float32)  # noqa: E731
    gate, up, down = (rng.standard_normal(s) * s[-1] ** -0.5 for s in ((n, d), (n, d), (d, n)))
    values = [give(a, weight)[1][None] for a in (gate, up, down)]

    def flat(shape):
        whole = ct.zeros(shape, TYPES[weight])
        return whole, ct.Tensor(ct._new(ct.lib().dl_reshape, whole.handle, ct._shape((F * d,))))

    matrices = []
    for a in (gate, up):
        whole, line = flat((1, F, d))
        write(ct.narrow(line, 0, 0, ends[0] * d), coded(a[:ends[0]]).ravel())
        write(ct.narrow(line, 0, (F - ends[1]) * d, ends[1] * d), coded(a[ends[0]:]).ravel())
        matrices.append(whole)
    whole, line = flat((1, d, F))
    for i in range(d):
        write(ct.narrow(line, 0, i * F, ends[0]), coded(down[i, :ends[0]]))
        write(ct.narrow(line, 0, (i + 1) * F - ends[1], ends[1]), coded(down[i, ends[0]:]))
    matrices.append(whole)
    y, chosen, weights = (t.numpy() for t in ct.expert_mixture(x, router, *matrices, 1))
    assert not chosen.any() and np.all(weights == 1.0)
    want, tolerance = mixed(rows, *values, chosen, weights.astype(np.float64))
    assert np.all(np.abs(y - want) <= tolerance), np.max(np.abs(y - want) / tolerance)


@pytest.mark.parametrize("T,d,F,E,top", [(1, 64, 32, 8, 2), (3, 65, 33, 8, 2), (12, 1, 40, 6, 2), (40, 63, 24, 8, 2), (100, 128, 72, 8, 2), (100, 65, 33, 8, 2),
                                         (64, 65, 65, 4, 2), (8, 40, 1064, 64, 4), (16, 39, 1031, 64, 4), (60, 65, 1104, 64, 1)])
@pytest.mark.parametrize("weight", ["f32", "bf16"])
@pytest.mark.parametrize("inputs", ["f32", "bf16"])
def test_numbers_that_are_not_finite_reach_what_they_take_part_in(T, d, F, E, top, weight, inputs):
    """In a row's and a matrix's first and last entries (which odd widths read twice).  All else is the same to the bit; but where a row
    goes to other experts the sums of the rows that it leaves or joins may begin elsewhere (by the first row of an expert), and
    are held to the tolerance."""
    rng = np.random.default_rng(T + d)
    arrays = [rng.standard_normal((T, d))] + [rng.standard_normal(s) * s[-1] ** -0.5 for s in ((E, d), (E, F, d), (E, F, d), (E, d, F))]
    kinds = [inputs] + [weight] * 4
    clean, values = zip(*[give(a, kind) for a, kind in zip(arrays, kinds)])
    want = [t.numpy() for t in ct.expert_mixture(*clean, top)]
    assert all(np.isfinite(a).all() for a in want)
    chosen = want[1]
    exact, tolerance = mixed(values[0], *values[2:], *route(values[0], values[1], top, True))
    counts = np.bincount(chosen.ravel(), minlength=E)
    busy, idle = int(np.argmax(counts)), int(np.argmin(counts))
    users = np.any(chosen == busy, -1)

    def with_bad(which, index, value):
        say(f"case: experts T={T} d={d} F={F} E={E} top={top} {weight} {inputs}: {value} at {index} of {which}")
        changed = arrays[which].copy()
        changed[index] = value
        tensors = [give(changed, kinds[which])[0] if i == which else t for i, t in enumerate(clean)]
        return [t.numpy() for t in ct.expert_mixture(*tensors, top)]

    for value in (np.nan, np.inf, -np.inf):
        for last in (0, -1):
            for which in (2, 3):  # a hidden entry, and by it all outputs of the rows that chose the expert
                y, now, weights = with_bad(which, (busy, last, last), value)
                assert not np.isfinite(y[users]).any() and np.array_equal(y[~users], want[0][~users])
                assert np.array_equal(now, chosen) and np.array_equal(weights, want[2])
            y, now, _ = with_bad(4, (busy, last, last), value)
            reached = np.zeros(y.shape, bool)
            reached[users, last] = True
            assert not np.isfinite(y[reached]).any() and np.array_equal(y[~reached], want[0][~reached]) and np.array_equal(now, chosen)
            y, now, weights = with_bad(0, (T // 2, last), value)
            others = np.arange(T) != T // 2
            assert not np.isfinite(y[T // 2]).any() and len(set(now[T // 2])) == top and np.all((now >= 0) & (now < E))
            assert np.array_equal(now[others], chosen[others]) and np.array_equal(weights[others], want[2][others])
            assert np.all(np.abs(y - exact)[others] <= tolerance[others])
        if counts[idle] == 0:  # an expert that no row chose
            for which in (2, 3, 4):
                assert all(np.array_equal(a, b) for a, b in zip(with_bad(which, (idle, -1, -1), value), want))
    y, now, weights = with_bad(1, (busy, -1), np.nan)  # the router's
    assert np.all(now[:, 0] == busy) and not np.isfinite(y).any() and np.isnan(weights).all()


def test_a_logit_of_minus_infinity_takes_part_with_nothing():
    for T in (1, 40):
        rng = np.random.default_rng(T)
        arrays = [np.abs(rng.standard_normal((T, 64)))] + [rng.standard_normal(s) * 0.2 for s in ((8, 64), (8, 32, 64), (8, 32, 64), (8, 64, 32))]
        arrays[1][5] = -1e3  # never chosen, and e^-1000 and less is nothing beside 1
        tensors = [give(a)[0] for a in arrays]
        arrays[1][5, 3] = -np.inf
        for normalise in (True, False):
            want = ct.expert_mixture(*tensors, 3, normalise)
            got = ct.expert_mixture(tensors[0], give(arrays[1])[0], *tensors[2:], 3, normalise)
            assert all(np.array_equal(a.numpy(), b.numpy()) for a, b in zip(got, want))
