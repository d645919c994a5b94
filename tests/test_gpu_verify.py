"""dl_verify_drafted against the rule in 64-bit numpy: whole numbers, which have to be equal.  (The uniform numbers of a
case stand at least 1e-9 from any border of its decisions, so that no rounding of 64 bits decides one; the test says so.)"""
import numpy as np
import pytest

import ctorch_amd as ct
import oracle
from common import say

pytestmark = pytest.mark.gpu
GPU = ct.device("gpu")


def softmax(x, t):
    x = x.astype(np.float64) / t
    e = np.exp(x - x.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def verify(drafted, target, draft, t, u):
    """(tokens, accepted, the smallest distance of a decision from its border)."""
    B, K = drafted.shape
    tokens, accepted, near = np.full((B, K + 1), -1), np.zeros(B, np.int64), 1.0
    for b in range(B):
        n, refused = 0, False
        while n < K and drafted[b, n] >= 0:
            x = drafted[b, n]
            if t <= 0:
                keep = x == np.argmax(target[b, n])
            elif x >= target.shape[2]:
                keep = False
            else:
                p, q = softmax(target[b, n], t)[x], 1.0 if draft is None else softmax(draft[b, n], t)[x]
                keep = u[b, n] * q < p
                near = min(near, abs(float(u[b, n]) - p / q) if q > 0 else 1.0)
            if not keep:
                refused = True
                break
            tokens[b, n] = x
            n += 1
        accepted[b] = n
        if t <= 0:
            tokens[b, n] = np.argmax(target[b, n])
            continue
        w = softmax(target[b, n], t)
        if refused:
            q = np.zeros_like(w)
            if draft is not None:
                q = softmax(draft[b, n], t)
            elif drafted[b, n] < len(w):
                q[drafted[b, n]] = 1.0
            over = np.maximum(w - q, 0)
            w = over if over.sum() > 0 else w
        reach = np.cumsum(w) / w.sum()
        near = min(near, np.min(np.abs(reach[:-1] - u[b, K])) if len(reach) > 1 else 1.0)
        tokens[b, n] = min(int(np.searchsorted(reach, float(u[b, K]), side="right")), np.flatnonzero(w > 0)[-1])
    return tokens, accepted, near


def run(drafted, target, draft, t, u, dtype="f32"):
    def give(x):
        if dtype == "bf16":
            return ct.Tensor.from_numpy(oracle.bf16_encode(x), ct.BF16, GPU)
        return ct.Tensor.from_numpy(x, ct.F32, GPU)

    tokens, accepted = ct.verify_drafted(ct.Tensor.from_numpy(drafted.astype(np.int64), ct.I64, GPU), give(target),
                                         give(draft) if draft is not None else None, t,
                                         ct.Tensor.from_numpy(u.astype(np.float32), ct.F32, GPU))
    return tokens.numpy(), accepted.numpy()


@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 32000), (3, 0, 50), (7, 8, 257), (2, 3, 2), (33, 5, 1000), (4, 2, 65537),
                                   (1, 70, 100), (64, 1, 4096), (5, 4, 16), (2, 4, 63)])
@pytest.mark.parametrize("t", [0.0, 0.7, 1.0, 2.5])
@pytest.mark.parametrize("kind", ["draft", "certain", "bf16"])
def test_verification_is_the_rule(B, K, V, t, kind):
    say(f"case: verify B={B} K={K} V={V} T={t} {kind}")
    rng = np.random.default_rng(B * K + V)
    target = (rng.standard_normal((B, K + 1, V)) * 3).astype(np.float32)
    draft = (target[:, :K] + rng.standard_normal((B, K, V))).astype(np.float32)
    if kind == "bf16":
        target, draft = (oracle.bf16_decode(oracle.bf16_encode(x)) for x in (target, draft))
    drafted = np.zeros((B, K), np.int64)
    for b in range(B):
        for i in range(K):
            # as the draft model would, and the target's best now and then, so that some rows are accepted whole
            p = softmax(draft[b, i], max(t, 0.5))
            drafted[b, i] = rng.choice(V, p=p / p.sum()) if rng.random() < 0.7 else np.argmax(target[b, i])
        if b % 3 == 2 and K:
            drafted[b, rng.integers(0, K + 1):] = -1
    u = rng.random((B, K + 1)).astype(np.float32)
    given = None if kind == "certain" else draft
    tokens, accepted, near = verify(drafted, target, given, t, u)
    assert near > 1e-9  # (a property of the inputs, not of the kernel)
    got = run(drafted, target, given, t, u, "bf16" if kind == "bf16" else "f32")
    assert np.array_equal(got[1], accepted), (got[1], accepted)
    assert np.array_equal(got[0], tokens), np.argwhere(got[0] != tokens)[:5]


def test_borders():
    """Uniform numbers of 0 and just below 1, equal models, a certain draft of probability 1, ids beyond the vocabulary."""
    V = 300
    rng = np.random.default_rng(4)
    target = (rng.standard_normal((1, 2, V)) * 2).astype(np.float32)
    below = np.float32(1 - 2.0 ** -24)
    # the same logits: every draft is kept, whatever the number (u < 1)
    for x in (0, 17, V - 1):
        tokens, accepted = run(np.array([[x]]), target, target[:, :1], 1.0, np.array([[below, 0.5]]))
        assert accepted[0] == 1 and tokens[0, 0] == x
    # the draw: 0 gives the first index with any weight, just below 1 the last
    target[0, 1, :5] = target[0, 1, -3:] = -np.inf
    for u, x in ((0.0, 5), (below, V - 4)):
        got = run(np.array([[3]]), target, target[:, :1], 1.0, np.array([[0.0, u]]))[0]
        want = verify(np.array([[3]]), target, target[:, :1], 1.0, np.array([[0.0, u]], np.float32))[0]
        assert got[0, 1] == want[0, 1] and (u > 0 or got[0, 1] == x)
    # an id beyond the vocabulary, and a draft that the target gives no weight, are refused
    target[0, 0, 8] = -np.inf
    for x in (V, 2 ** 40, 8):
        tokens, accepted = run(np.array([[x]]), target, None, 1.0, np.array([[0.0, 0.3]]))
        assert accepted[0] == 0 and tokens[0, 1] == -1 and 0 <= tokens[0, 0] < V and tokens[0, 0] != 8
    # a certain draft that is refused is not drawn again
    sharp = np.full((1, 2, V), -20, np.float32)
    sharp[0, 0, 7], sharp[0, 0, 9] = 5.0, 4.9
    tokens, accepted = run(np.array([[7]]), sharp, None, 1.0, np.array([[0.9, 0.0001]]))
    assert accepted[0] == 0 and tokens[0, 0] == 9


def test_a_row_without_a_sum_takes_its_argmax():
    target = np.random.default_rng(1).standard_normal((3, 1, 40)).astype(np.float32)
    target[0, 0, 12] = np.nan
    target[1, 0, 30] = np.inf
    target[2, 0, :] = -np.inf
    tokens, accepted = run(np.zeros((3, 0)), target, None, 1.0, np.full((3, 1), 0.5))
    assert tokens[:, 0].tolist() == [12, 30, 0] and accepted.tolist() == [0, 0, 0]


def test_ties_of_a_greedy_verification_go_to_the_lower_index():
    target = np.zeros((1, 3, 1000), np.float32)
    target[0, 1, [400, 900]] = 1
    tokens, accepted = run(np.array([[0, 900]]), target, None, 0.0, np.zeros((1, 3)))
    assert accepted[0] == 1 and tokens[0].tolist() == [0, 400, -1]
    tokens, accepted = run(np.array([[0, 400]]), target, None, -1.0, np.zeros((1, 3)))
    assert accepted[0] == 2 and tokens[0].tolist() == [0, 400, 0]


def test_views_are_read_as_they_lie():
    rng = np.random.default_rng(6)
    wide = (rng.standard_normal((2, 4, 90)) * 3).astype(np.float32)
    t = ct.narrow(ct.Tensor.from_numpy(wide, ct.F32, GPU), 2, 7, 50)
    ids = rng.integers(0, 50, (2, 6))
    d = ct.narrow(ct.Tensor.from_numpy(ids, ct.I64, GPU), 1, 2, 3)
    u = rng.random((2, 9)).astype(np.float32)
    gu = ct.narrow(ct.Tensor.from_numpy(u, ct.F32, GPU), 1, 5, 4)
    tokens, accepted = ct.verify_drafted(d, t, None, 1.0, gu)
    want = verify(ids[:, 2:5], wide[:, :, 7:57], None, 1.0, u[:, 5:])
    assert np.array_equal(tokens.numpy(), want[0]) and np.array_equal(accepted.numpy(), want[1])


def test_long_rows_of_nothing_but_few_entries():
    """A vocabulary of many slices and parts whose weight lies in a few entries far apart, and many drafts of a sequence."""
    rng = np.random.default_rng(8)
    V = 200001
    target = np.full((2, 3, V), -np.inf, np.float32)
    draft = np.full((2, 2, V), -np.inf, np.float32)
    for b in range(2):
        for i in range(3):
            target[b, i, [70000, 130000 + i, V - 1]] = rng.standard_normal(3)
        draft[b, :, [70000, 150000]] = 0.5
    for u in (0.0, 0.3, 0.6, 0.95):
        numbers = np.full((2, 3), u, np.float32)
        for given in (draft, None):
            for ids in ([70000, 150000], [150000, 70000]):
                drafted = np.array([ids, ids])
                want = verify(drafted, target, given, 1.0, numbers)
                got = run(drafted, target, given, 1.0, numbers)
                assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (u, ids)
    K = 300  # more than one round of comparisons
    logits = rng.standard_normal((2, K + 1, 7)).astype(np.float32)
    drafted = rng.integers(0, 7, (2, K))
    for numbers in (np.zeros((2, K + 1)), np.where(np.arange(K + 1) == 270, 1 - 2.0 ** -24, 0.0) * np.ones((2, 1))):
        for given in (logits[:, :K] * np.float32(1.5), None):
            want = verify(drafted, logits, given, 0.9, numbers.astype(np.float32))
            got = run(drafted, logits, given, 0.9, numbers)
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_a_greedy_verification_takes_a_nan_for_the_largest():
    target = np.random.default_rng(2).standard_normal((1, 3, 5000)).astype(np.float32)
    target[0, 0, 4321] = np.nan
    target[0, 1, :] = -np.inf
    tokens, accepted = run(np.array([[4321, 0]]), target, None, 0.0, np.zeros((1, 3)))
    assert accepted[0] == 2 and tokens[0].tolist() == [4321, 0, int(target[0, 2].argmax())]


@pytest.mark.parametrize("V", [5, 300, 1024, 5000, 32000])
@pytest.mark.parametrize("t", [0.7, 1.0, 3.0])
def test_a_refusal_where_both_models_agree_draws_from_the_target(V, t):
    """Rows that are the same for both models leave nothing of p - q, not even a rounding: the token comes from p.  (The draft
    has no weight in either, so that 0 < 0 refuses it.)"""
    say(f"case: verify, equal rows, V={V} T={t}")
    rng = np.random.default_rng(V)
    target = (rng.standard_normal((8, 2, V)) * 3).astype(np.float32)
    drafted = rng.integers(0, V, (8, 1))
    for b in range(8):
        target[b, 0, drafted[b, 0]] = -np.inf if b % 2 else -2400.0  # exp(-800) at most: no number of 64 bits
    u = rng.random((8, 2)).astype(np.float32)
    u[0, 1], u[1, 1] = 0.0, 1 - 2.0 ** -24
    tokens, accepted, near = verify(drafted, target, target[:, :1], t, u)
    assert near > 1e-12 and not accepted.any()  # (a property of the inputs)
    got = run(drafted, target, target[:, :1], t, u)
    assert np.array_equal(got[1], accepted) and np.array_equal(got[0], tokens), (got[0][:, 0], tokens[:, 0])


@pytest.mark.parametrize("t", [1e-250, 1e-33, 1e-29, 1e29, 1e31, 1e38, 1e46, 1e300])
@pytest.mark.parametrize("V", [3, 50, 1500, 5001])
@pytest.mark.parametrize("kind", ["draft", "certain"])
def test_temperatures_beyond_32_bits(V, t, kind):
    """Any finite temperature: masked logits weigh nothing, and logits as far apart as the type holds what they weigh."""
    say(f"case: verify V={V} T={t} {kind}")
    rng = np.random.default_rng(V)
    unit = np.float32(1e38 if t >= 1e37 and V != 50 else np.clip(t, 1e-33, 1.0))  # (V = 50: ordinary logits)
    target = (np.clip(rng.standard_normal((6, 3, V)), -3, 3)).astype(np.float32) * unit
    draft = (np.clip(rng.standard_normal((6, 2, V)), -3, 3)).astype(np.float32) * unit
    target[1::2, :, 0] = draft[1::3, :, 0] = -np.inf
    target[2::4, :, V // 2] = np.finfo(np.float32).min
    drafted = rng.integers(0, V, (6, 2))
    drafted[1::2, 1] = 0
    drafted[2::4, 0] = V // 2
    u = rng.random((6, 3)).astype(np.float32)
    u[4, :2] = 0.0
    given = draft if kind == "draft" else None
    tokens, accepted, near = verify(drafted, target, given, t, u)
    # a property of the inputs (at 1e-250 weights are equal or nothing, and the decisions exact where they meet their border)
    assert near > 1e-9 or t < 1e-200
    got = run(drafted, target, given, t, u)
    assert np.array_equal(got[1], accepted), (got[1], accepted)
    assert np.array_equal(got[0], tokens), (got[0], tokens)
