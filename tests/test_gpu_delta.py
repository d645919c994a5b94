"""The gated delta rule on the GPU against numpy in 64 bits, token after token.

Tolerances, from the arithmetic (u = 2^-24).  Columns of a state are independent, so everything below is for one of them, with
2-norms over the rows.  With keys of length 1 (to u) and rates in [0, 2], the step S -> a (1 - rate k k^T) S does not lengthen an
error, so that errors add up: e_t <= a_t e_(t-1) + d_t.  What a step adds: token by token, sums of dk products and a few
roundings of parts no larger than a S and v: (dk + 10) u (|a S| + |v|).  In chunks of C <= 64 tokens, the same for the entries
of the triangular system (dk + 4 roundings each, of values up to |k_i . k_j| <= 1 times a fade) and for its solution by
substitution (up to C more): perturbations of w_t by (dk + 70) u sum_i fade_ti |w_i|, w_i the chunk's earlier writes.  With
R_t = a_t R_(t-1) + |w_t| >= that sum, d_t = (dk + 80) u (|a S| + |v| + R_t) covers both, and the output adds scale |q| (e_t +
(dk + 80) u (|S| + R_t)).  bf16 inputs are exact; a key rounded to bf16 is 2^-8 longer at most, which makes a (1 - rate k
k^T) of up to |1 - rate (1 + 2^-7)|: no more than 1 for the rates up to 1.9 that are drawn."""
import numpy as np
import pytest

import ctorch_amd as ct
import oracle
from common import agree, say, write

pytestmark = pytest.mark.gpu
GPU = ct.device("gpu")
U = 2.0 ** -24


def give(values, dtype="f32"):
    """The tensor on the GPU, and the values that it holds."""
    if dtype == "bf16":
        bits = oracle.bf16_encode(np.ascontiguousarray(values, np.float32))
        return ct.Tensor.from_numpy(bits, ct.BF16, GPU), oracle.bf16_decode(bits).astype(np.float64)
    values = np.asarray(values, np.float32)
    return ct.Tensor.from_numpy(values, ct.F32, GPU), values.astype(np.float64)


def put(states, layer, values):
    write(states.state(layer), np.ascontiguousarray(values, np.float32))


def rule(state, q, k, v, decay, rate, scale):
    """One request: state [H, dk, dv], q, k [T, H, dk], v [T, H, dv], decay, rate [T, H].  Outputs and state with their
    tolerances."""
    T, H, dk = k.shape
    norm = lambda x: np.sqrt(np.sum(x * x, -2))  # over the rows  # noqa: E731
    S, e, R = state.copy(), np.zeros((H, v.shape[2])), np.zeros((H, v.shape[2]))
    c = (dk + 80) * U
    out, tolerance = np.empty(v.shape), np.empty(v.shape)
    for t in range(T):
        a = np.exp(decay[t])[:, None]
        S = a[..., None] * S
        size = norm(S)
        w = rate[t][:, None] * (v[t] - np.einsum("hk,hkv->hv", k[t], S))
        S = S + k[t][..., None] * w[:, None]
        R = a * R + np.abs(w)
        e = a * e + c * (size + np.abs(v[t]) + R)
        out[t] = scale * np.einsum("hk,hkv->hv", q[t], S)
        tolerance[t] = abs(scale) * np.linalg.norm(q[t], axis=-1)[:, None] * (e + c * (norm(S) + R))
    return out, tolerance, S, e


def draw(rng, tokens, hk, h, dk, dv, alike=0.0):
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    q, k = unit(rng.standard_normal((tokens, hk, dk))), unit(rng.standard_normal((tokens, hk, dk)) + alike * rng.standard_normal((1, hk, dk)))
    return [q, k, rng.standard_normal((tokens, h, dv)), -np.exp(rng.uniform(-7, 1, (1, h))) * rng.uniform(0, 2, (tokens, h)),
            rng.uniform(0, 1.9, (tokens, h))]


def check(counts, sources, targets, hk, h, dk, dv, dtype="f32", seed=0, change=None, scale=None, alike=0.0, slots=None):
    """A step over states of random numbers; `change` may alter the drawn inputs."""
    say(f"case: delta counts={counts} heads={hk}/{h} {dk}x{dv} {dtype} seed={seed}")
    rng = np.random.default_rng(seed + sum(counts))
    slots = slots or max(targets + sources) + 2
    states = ct.DeltaStates(2, slots, h, dk, dv)
    held = [rng.standard_normal((slots, h, dk, dv)).astype(np.float32) for _ in range(2)]
    for layer in range(2):
        put(states, layer, held[layer])
    inputs = draw(rng, sum(counts), hk, h, dk, dv, alike)
    if change:
        change(inputs)
    tensors, values = zip(*[give(x, dtype if i < 3 else "f32") for i, x in enumerate(inputs)])
    batch = ct.DeltaBatch(states, hk, sources, targets, counts)
    got = ct.gated_delta(states, 1, batch, *tensors, scale)
    assert got.shape == (sum(counts), h, dv) and got.dtype == ct.F32
    got, after = got.numpy(), states.state(1).numpy()
    assert np.array_equal(states.state(0).numpy(), held[0])
    q, k, v, decay, rate = values
    q, k = (np.repeat(x, h // hk, 1) for x in (q, k))
    first, factor, kept = 0, dk ** -0.5 if scale is None else scale, held[1].astype(np.float64)
    worst = 0.0
    for b, n in enumerate(counts):
        if n == 0:
            continue
        at = slice(first, first + n)
        begin = kept[sources[b]] if sources[b] >= 0 else np.zeros((h, dk, dv))
        out, tolerance, S, e = rule(begin, q[at], k[at], v[at], decay[at], rate[at], factor)
        off = np.abs(got[at] - out)
        assert np.all(off <= tolerance), (b, np.unravel_index(np.argmax(off - tolerance), off.shape), np.max(off / tolerance))
        error = np.sqrt(np.sum((after[targets[b]] - S) ** 2, -2))
        assert np.all(error <= e), (b, float(np.max(error / e)))
        worst = max(worst, float(np.max(off / np.maximum(tolerance, 1e-300))), float(np.max(error / e)))
        first += n
    untouched = [s for s in range(slots) if s not in [t for t, n in zip(targets, counts) if n]]
    assert np.array_equal(after[untouched], held[1][untouched])
    say(f"  at most {worst:.3f} of the tolerance")


SHAPES = [(1, 1, 32, 32), (2, 2, 64, 64), (2, 4, 128, 128), (1, 3, 64, 96), (3, 3, 32, 256), (2, 8, 128, 64)]


@pytest.mark.parametrize("hk,h,dk,dv", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_single_and_drafted_tokens(hk, h, dk, dv, dtype):
    check([1], [0], [0], hk, h, dk, dv, dtype)  # in place
    check([1, 5, 0, 2], [3, -1, 77, 1], [0, 2, -9, 1], hk, h, dk, dv, dtype, 1, slots=5)
    check([9, 16], [-1, 0], [2, 0], hk, h, dk, dv, dtype, 2)


@pytest.mark.parametrize("hk,h,dk,dv", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompts(hk, h, dk, dv, dtype):
    check([200], [-1], [0], hk, h, dk, dv, dtype)
    check([63, 1, 129, 64, 65, 17], [0, -1, 3, 1, -1, -1], [0, 2, 4, 1, 5, 6], hk, h, dk, dv, dtype, 1)


@pytest.mark.parametrize("count", [2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 95, 96, 127, 128, 129, 191, 192, 193, 257])
def test_every_end_of_a_chunk(count):
    check([count, 3], [1, 0], [1, 0], 1, 2, 64, 64, "bf16", count)
    check([3, count], [-1, 0], [1, 2], 1, 2, 32, 32, "f32", count + 1)


def test_a_long_prompt():
    check([3001], [-1], [0], 1, 2, 128, 64, "bf16")


def test_many_requests():
    rng = np.random.default_rng(5)
    counts = rng.integers(0, 4, 70).tolist()
    check(counts, list(range(70)), list(range(70, 140)), 1, 2, 32, 32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_keys_that_are_alike(dtype):
    check([150], [0], [1], 2, 2, 64, 64, dtype, alike=8.0)


def test_keys_that_are_the_same_and_rates_of_one():
    def change(x):
        x[1][:] = x[1][:1]
        x[4][:] = 1.0
    check([130], [0], [0], 1, 2, 64, 64, change=change)


def test_decays_that_forget_everything_and_nothing():
    def change(x):
        x[3][5] = -np.inf
        x[3][70:75] = -np.inf
        x[3][80:90] = -1e30
        x[3][90:] = 0.0
        x[4][100:] = 0.0
    check([140], [0], [0], 1, 2, 64, 64, change=change)
    check([140, 3], [1, -1], [0, 2], 2, 2, 128, 32, change=lambda x: x[3].fill(-np.inf))
    check([140, 3], [1, -1], [0, 2], 2, 2, 128, 32, change=lambda x: x[3].fill(0.0))
    check([3, 140], [1, -1], [0, 2], 2, 2, 32, 32, change=lambda x: x[3].fill(-90.0))


def test_decays_whose_sums_are_long():
    # (differences within a chunk hold although the sums are large)
    check([64 * 3], [0], [0], 1, 1, 32, 32, change=lambda x: x[3].__setitem__(slice(0, 190), np.linspace(-60, -1e-3, 190)[:, None]))


@pytest.mark.parametrize("count", [9, 100])
def test_decays_above_zero(count):
    """(The tolerance grows with the state.)"""
    for change in (lambda x: x[3].fill(0.5), lambda x: x[3].__setitem__(slice(None), 1.0 * (np.arange(count) < 60)[:, None]),
                   lambda x: x[3].__setitem__(slice(None), np.where(np.arange(count) % 2, 20.0, -20.0)[:, None])):
        check([count], [0], [0], 1, 2, 64, 64, change=change)


@pytest.mark.parametrize("scale", [1.0, 0.0, -3.5])
def test_a_scale_of_ones_own(scale):
    check([7, 70], [0, -1], [0, 1], 1, 2, 64, 32, scale=scale)


def test_values_that_are_not_finite_stay_in_their_column_and_behind():
    rng = np.random.default_rng(9)
    counts, (hk, h, dk, dv) = [70, 90], (1, 2, 64, 64)
    for bad in (np.nan, np.inf):
        states = ct.DeltaStates(1, 4, h, dk, dv)
        inputs = draw(rng, 160, hk, h, dk, dv)
        inputs[2][100, 1, 7] = bad
        tensors = [give(x)[0] for x in inputs]
        got = ct.gated_delta(states, 0, ct.DeltaBatch(states, hk, [-1, -1], [0, 1], counts), *tensors).numpy()
        reached = ~np.isfinite(got)
        assert reached[101:, 1, 7].all()
        reached[64:, 1, 7] = False  # (from the first token of its chunk on at the latest)
        assert not reached[:100].any() and not reached.any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count", [2, 80])
def test_rows_are_views_of_a_projection(dtype, count):
    rng = np.random.default_rng(4)
    hk, h, d = 2, 4, 64
    q, k, v, decay, rate = draw(rng, count, hk, h, d, d)
    wide, values = give(np.concatenate([q, k, v, np.full((count, 1, d), np.nan)], 1), dtype)
    gates, gate_values = give(np.concatenate([decay, rate], 1))
    parts = [ct.narrow(wide, 1, 0, hk), ct.narrow(wide, 1, hk, hk), ct.narrow(wide, 1, 2 * hk, h)]
    states = ct.DeltaStates(1, 1, h, d, d)
    batch = ct.DeltaBatch(states, hk, [-1], [0], [count])
    got = ct.gated_delta(states, 0, batch, *parts, ct.narrow(gates, 1, 0, h), ct.narrow(gates, 1, h, h)).numpy()
    whole = [give(values[:, a:b], dtype)[0] for a, b in ((0, hk), (hk, 2 * hk), (2 * hk, 2 * hk + h))]
    want = ct.gated_delta(states, 0, batch, *whole, give(gate_values[:, :h])[0], give(gate_values[:, h:])[0]).numpy()
    assert np.isfinite(got).all() and np.array_equal(got, want)
    # entries that are not neighbours, and rows off their alignment: read from copies
    odd, odd_values = give(rng.standard_normal((count, hk, d + 3)), dtype)
    got = ct.gated_delta(states, 0, batch, ct.narrow(odd, 2, 1, d), *whole[1:], ct.narrow(gates, 1, 0, h), ct.narrow(gates, 1, h, h)).numpy()
    want = ct.gated_delta(states, 0, batch, give(odd_values[..., 1:d + 1], dtype)[0], *whole[1:], ct.narrow(gates, 1, 0, h),
                          ct.narrow(gates, 1, h, h)).numpy()
    assert np.array_equal(got, want)


@pytest.mark.parametrize("count", [3, 90])
@pytest.mark.parametrize("types", [("bf16", "f32", "f32"), ("f32", "bf16", "bf16"), ("bf16", "bf16", "f32"), ("f32", "f32", "bf16")])
def test_rows_of_different_types(types, count):
    rng = np.random.default_rng(13)
    hk, h, dk, dv = 1, 2, 64, 64
    inputs = draw(rng, count, hk, h, dk, dv)
    tensors, values = zip(*[give(x, types[i] if i < 3 else "f32") for i, x in enumerate(inputs)])
    states = ct.DeltaStates(1, 1, h, dk, dv)
    got = ct.gated_delta(states, 0, ct.DeltaBatch(states, hk, [-1], [0], [count]), *tensors).numpy()
    q, k = (np.repeat(x, h // hk, 1) for x in values[:2])
    want, tolerance, _, _ = rule(np.zeros((h, dk, dv)), q, k, *values[2:], dk ** -0.5)
    assert np.all(np.abs(got - want) <= tolerance)


def test_bf16_gates():
    rng = np.random.default_rng(8)
    inputs = draw(rng, 5, 1, 2, 32, 32)
    tensors = [give(x)[0] for x in inputs[:3]]
    (g, gv), (b, bv) = give(inputs[3], "bf16"), give(inputs[4], "bf16")
    states = ct.DeltaStates(1, 1, 2, 32, 32)
    batch = ct.DeltaBatch(states, 1, [-1], [0], [5])
    assert np.array_equal(ct.gated_delta(states, 0, batch, *tensors, g, b).numpy(),
                          ct.gated_delta(states, 0, batch, *tensors, give(gv)[0], give(bv)[0]).numpy())


def test_a_prompt_in_parts_is_the_prompt():
    """The parts' errors add up as a whole's do: both against the rule, the second with the states of the first's."""
    rng = np.random.default_rng(11)
    hk, h, dk, dv = 1, 2, 64, 64
    inputs = draw(rng, 300, hk, h, dk, dv)
    values = [give(x)[1] for x in inputs]
    q, k = (np.repeat(x, h // hk, 1) for x in values[:2])
    want, tolerance, S, e = rule(np.zeros((h, dk, dv)), q, k, *values[2:], dk ** -0.5)
    for cuts in ([300], [1, 299], [77, 3, 1, 219], [64, 64, 64, 64, 44]):
        states, first, slot = ct.DeltaStates(1, 2, h, dk, dv), 0, -1
        for n in cuts:
            part = [give(x[first:first + n])[0] for x in inputs]
            to = 0 if slot != 0 else 1
            got = ct.gated_delta(states, 0, ct.DeltaBatch(states, hk, [slot], [to], [n]), *part).numpy()
            assert np.all(np.abs(got - want[first:first + n]) <= tolerance[first:first + n])
            first, slot = first + n, to
        error = np.sqrt(np.sum((states.state(0).numpy()[slot] - S) ** 2, -2))
        assert np.all(error <= e)


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(12)
    inputs = draw(rng, 400, 2, 4, 128, 128)
    tensors = [give(x, "bf16" if i < 3 else "f32")[0] for i, x in enumerate(inputs)]
    states = ct.DeltaStates(1, 4, 4, 128, 128)
    batch = ct.DeltaBatch(states, 2, [-1, -1, -1], [0, 1, 2], [300, 97, 3])
    first = ct.gated_delta(states, 0, batch, *tensors).numpy(), states.state(0).numpy()
    for _ in range(3):
        again = ct.gated_delta(states, 0, batch, *tensors).numpy(), states.state(0).numpy()
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_chunks_in_several_rounds_of_launches():
    """(8192 chunks of a head in all: 128 of 64 heads.)  Long requests go on from round to round, many take turns."""
    check([8300, 700], [0, -1], [1, 2], 64, 64, 32, 32)
    check([65] * 130, [-1] * 130, list(range(130)), 64, 64, 32, 32, slots=130)


@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 128)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("count", [9, 100, 640])
def test_all_bits_of_an_f32_count(dk, dv, dtype, count):
    """Roundings of different sums are independent, so that their number adds up by its root: an output is made of sums of dk
    and of up to 64 products, one rounding each, and is off by about sqrt(dk + 64) u of its size, in the mean over many.  A factor
    whose third part of 8 bits is lost is off by 2^-17 in the mean, always to the same side: five times and more of that."""
    rng = np.random.default_rng(dk + count)
    hk, h = 1, 2
    inputs = draw(rng, count, hk, h, dk, dv)
    inputs[3][:] = -np.exp(rng.uniform(-5, -1, (1, h)))  # (states of a size that stays)
    tensors, values = zip(*[give(x, dtype if i < 3 else "f32") for i, x in enumerate(inputs)])
    states = ct.DeltaStates(1, 1, h, dk, dv)
    begin = rng.standard_normal((1, h, dk, dv)).astype(np.float32)
    put(states, 0, begin)
    got = ct.gated_delta(states, 0, ct.DeltaBatch(states, hk, [0], [0], [count]), *tensors).numpy()
    q, k = (np.repeat(x, h // hk, 1) for x in values[:2])
    want, _, state, _ = rule(begin[0].astype(np.float64), q, k, *values[2:], dk ** -0.5)
    bound = (dk + 64) ** 0.5 * U
    assert np.linalg.norm(got - want) <= bound * np.linalg.norm(want)
    agree(states.state(0).numpy()[0].reshape(-1, dv), state.reshape(-1, dv), bound)


def test_rows_of_one_head_for_all_tokens():
    """Rows that lie in one place (no step between tokens), and rows far apart."""
    rng = np.random.default_rng(14)
    inputs = draw(rng, 70, 1, 2, 32, 32)
    for i in range(3):
        inputs[i][:] = inputs[i][:1]
    tensors = [give(x)[0] for x in inputs]
    states = ct.DeltaStates(1, 1, 2, 32, 32)
    batch = ct.DeltaBatch(states, 1, [-1], [0], [70])
    want = ct.gated_delta(states, 0, batch, *tensors).numpy()
    far = give(np.concatenate([np.broadcast_to(x.reshape(70, 1, -1), (70, 1, x.shape[1] * 32)) for x in inputs[:3]], 2))[0]
    views, at = [], 0
    for x in inputs[:3]:
        part = ct.narrow(far, 2, at, x.shape[1] * 32)
        views.append(ct.Tensor(ct._new(ct.lib().dl_reshape, part.handle, ct._shape(x.shape))))
        at += x.shape[1] * 32
    assert np.array_equal(ct.gated_delta(states, 0, batch, *views, *tensors[3:]).numpy(), want)


def test_states_beyond_4_gib():
    """The same tokens through the last slots of a large pool and through a small one, bit for bit."""
    h, d, results = 32, 128, []
    rng = np.random.default_rng(3)
    steps = [(n, [give(x)[0] for x in draw(rng, n, 16, h, d, d)]) for n in (1, 100, 1, 100)]
    for slots in (3, 2200):
        say(f"case: delta {slots} slots of {h} x {d} x {d}")
        states, last = ct.DeltaStates(1, slots, h, d, d), slots - 1
        run = lambda i, source, target: ct.gated_delta(states, 0, ct.DeltaBatch(states, 16, [source], [target], [steps[i][0]]), *steps[i][1]).numpy()
        out = [run(0, -1, last), run(1, last, last - 1)]
        states.copy([last - 1], [last])
        out += [run(2, last, 0), run(3, last, last)]
        states.copy([last], [0])
        results.append(out + [run(0, 0, 1)])
    for small, large in zip(*results):
        assert np.array_equal(small, large)


WHERE = [(9, 0), (9, 4), (9, 8), (150, 0), (150, 13), (150, 16), (150, 63), (150, 64), (150, 100), (150, 127), (150, 149)]  # (new tokens, which)


def step_of(inputs, dtype, begin, counts, sources, key_heads):
    tensors = [give(x, dtype if i < 3 else "f32")[0] for i, x in enumerate(inputs)]
    h, dk, dv = begin.shape[1:]
    states = ct.DeltaStates(1, len(begin), h, dk, dv)
    put(states, 0, begin)
    batch = ct.DeltaBatch(states, key_heads, sources, list(range(len(counts))), counts)
    return ct.gated_delta(states, 0, batch, *tensors).numpy(), states.state(0).numpy()


@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 32), (128, 96)])
@pytest.mark.parametrize("of", ["value", "key", "decay", "rate", "query", "state"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_is_not_finite_reaches_what_follows_it_alone(of, bad, dtype, dk, dv):
    """Of the same request, and of its column (a value), its heads (a key or a gate) or its row (a query); all else is the same
    to the bit as without it.  A later decay of -inf does not take it back."""
    if of == "decay" and bad < 0:
        return  # (forgets: a number like others)
    hk, h = 2, 4
    rng = np.random.default_rng(21)
    for count, t in WHERE:
        say(f"case: delta {of} {bad} at {t} of {count} {dk}x{dv} {dtype}")
        counts = [70, count, 40]  # (the second request is looked at; the first and the last must not know)
        first, end = 70 + t, 70 + count
        inputs = draw(rng, sum(counts), hk, h, dk, dv)
        begin = rng.standard_normal((3, h, dk, dv)).astype(np.float32)
        if t + 1 < count:
            inputs[3][first + 1] = -np.inf
        whole, state = step_of(inputs, dtype, begin, counts, [0, 1, 2], hk)
        assert np.isfinite(whole).all() and np.isfinite(state).all()
        reached, left = np.zeros(whole.shape, bool), np.zeros(state.shape, bool)
        if of == "value":
            inputs[2][first, 1, 7] = bad
            reached[first:end, 1, 7], left[1, 1, :, 7] = True, True
        elif of in ("key", "query"):
            inputs[1 if of == "key" else 0][first, 1, 21] = bad
            if of == "key":
                reached[first:end, 2:], left[1, 2:] = True, True
            else:
                reached[first, 2:] = True
        elif of in ("decay", "rate"):
            inputs[3 if of == "decay" else 4][first, 1] = bad
            reached[first:end, 1], left[1, 1] = True, True
        else:
            begin[1, 1, 5, 7] = bad
            reached[70:end, 1, 7], left[1, 1, :, 7] = True, True
        got, after = step_of(inputs, dtype, begin, counts, [0, 1, 2], hk)
        assert not np.isfinite(got[reached]).any() and np.array_equal(got[~reached], whole[~reached])
        assert not np.isfinite(after[left]).any() and np.array_equal(after[~left], state[~left])


@pytest.mark.parametrize("count,t,other", [(9, 3, 7), (150, 0, 1), (150, 17, 18), (150, 50, 63), (150, 70, 140)])
def test_what_f32_does_not_hold_reaches_what_follows_it_alone(count, t, other):
    """Two long keys that are alike: their product is 1e50.  (The first one's own write is so too, but for a state of zero.)"""
    rng = np.random.default_rng(22)
    hk, h, dk, dv = 1, 2, 64, 32
    inputs = draw(rng, count, hk, h, dk, dv)
    inputs[3][:] = -1e-3
    begin = np.zeros((1, h, dk, dv), np.float32)
    whole, _ = step_of(inputs, "f32", begin, [count], [-1], hk)
    inputs[1][t] *= 1e25
    inputs[1][other] = inputs[1][t]
    got, after = step_of(inputs, "f32", begin, [count], [-1], hk)
    assert np.array_equal(got[:t], whole[:t]) and (t > 0 or np.isfinite(got[0]).all())
    assert not np.isfinite(got[other:]).any() and not np.isfinite(after).any()
