"""Page pools, forks, compaction, the delta rule, experts, and the paged cache's operators together, as a serving loop uses
them: a decoder of two layers (attention over pages, the gated delta rule; experts behind both), requests that come, are forked,
have drafts refused, end and move; every output against numpy in 64 bits over the request's whole history.

Tolerance: every operator is off by at most a few hundred steps of 2^-24 of the magnitudes that it sums, which here are
within ten times its results; a dozen of them follow one another, so that outputs are off by less than 12 * 10 * 300 * 2^-24 < 2^-8 of
the largest of a row.  A wrong page, state or expert is off by as much as the row itself."""
import numpy as np
import pytest

import ctorch_amd as ct
from common import say

pytestmark = pytest.mark.gpu
GPU = ct.device("gpu")
D, H, KV, HD, HK, HV, DK, DV, E, F, TOP, PAGE = 64, 4, 2, 16, 2, 4, 32, 32, 6, 48, 2, 16


def give(values):
    return ct.Tensor.from_numpy(np.asarray(values, np.float32), ct.F32, GPU)


class Model:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        draw = lambda *s: (rng.standard_normal(s) * s[-1] ** -0.5).astype(np.float32)  # noqa: E731
        self.weights = dict(q=draw(H * HD, D), k=draw(KV * HD, D), v=draw(KV * HD, D), o=draw(D, H * HD),
                            dq=draw(HK * DK, D), dk=draw(HK * DK, D), dv=draw(HV * DV, D), gate=draw(2 * HV, D), do=draw(D, HV * DV),
                            **{f"{n}{layer}": draw(*s) for layer in (0, 1)
                               for n, s in (("router", (E, D)), ("up", (E, F, D)), ("act", (E, F, D)), ("down", (E, D, F)))})
        self.given = {n: give(w) for n, w in self.weights.items()}
        self.cosine, self.sine = ct.rotary_tables(HD, 256)
        self.tables = self.cosine.numpy().astype(np.float64), self.sine.numpy().astype(np.float64)

    # in 64 bits, a whole history x [T, D]
    def exact(self, x):
        w = {n: a.astype(np.float64) for n, a in self.weights.items()}
        norm = lambda z: z / np.sqrt(np.mean(z * z, -1, keepdims=True) + 1e-5)  # noqa: E731
        T = len(x)

        def turn(z):
            c, s = (t[:T, None] for t in self.tables)
            y = z.copy()
            y[..., 0::2], y[..., 1::2] = z[..., 0::2] * c - z[..., 1::2] * s, z[..., 0::2] * s + z[..., 1::2] * c
            return y

        def experts(z, layer):
            scores = z @ w[f"router{layer}"].T
            y = np.zeros_like(z)
            for t in range(T):
                best = np.argsort(-scores[t], kind="stable")[:TOP]
                p = np.exp(scores[t, best] - scores[t, best[0]])
                for e, share in zip(best, p / p.sum()):
                    g = w[f"act{layer}"][e] @ z[t]
                    y[t] += share * (w[f"down{layer}"][e] @ (g / (1 + np.exp(-g)) * (w[f"up{layer}"][e] @ z[t])))
            return y

        x = x.astype(np.float64)
        z = norm(x)
        q, k, v = turn((z @ w["q"].T).reshape(T, H, HD)), turn((z @ w["k"].T).reshape(T, KV, HD)), (z @ w["v"].T).reshape(T, KV, HD)
        k, v = (np.repeat(a, H // KV, 1) for a in (k, v))
        scores = np.einsum("thd,shd->hts", q, k) / np.sqrt(HD) + np.triu(np.full((T, T), -np.inf), 1)
        p = np.exp(scores - scores.max(-1, keepdims=True))
        x = x + np.einsum("hts,shd->thd", p / p.sum(-1, keepdims=True), v).reshape(T, H * HD) @ w["o"].T
        x = x + experts(norm(x), 0)
        z = norm(x)
        unit = lambda a: a / np.sqrt(np.sum(a * a, -1, keepdims=True) + DK * 1e-5)  # noqa: E731
        q, k = (np.repeat(unit((z @ w[n].T).reshape(T, HK, DK)), HV // HK, 1) for n in ("dq", "dk"))
        v, gate = (z @ w["dv"].T).reshape(T, HV, DV), z @ w["gate"].T
        state, out = np.zeros((HV, DK, DV)), np.empty((T, HV, DV))
        for t in range(T):
            state *= np.exp(-np.abs(gate[t, :HV]))[:, None, None]
            wrong = v[t] - np.einsum("hk,hkv->hv", k[t], state)
            state += k[t][..., None] * (1 / (1 + np.exp(-gate[t, HV:])))[:, None, None] * wrong[:, None]
            out[t] = np.einsum("hk,hkv->hv", q[t], state) * DK ** -0.5
        x = x + out.reshape(T, HV * DV) @ w["do"].T
        return x + experts(norm(x), 1)


class Server:
    """The loop: who holds which pages and which state, and a step over some of the requests."""

    def __init__(self, model, pages, slots):
        self.model, self.width = model, 8
        self.cache, self.pool = ct.PagedCache(1, pages, PAGE, KV, HD), ct.PagePool(pages)
        self.states, self.slots = ct.DeltaStates(1, slots, HV, DK, DV), list(range(slots))
        self.requests, self.names = {}, 0

    def begin(self):
        self.names += 1
        self.requests[self.names] = dict(table=np.full(self.width, -1), length=0, slot=-1, history=np.zeros((0, D), np.float32))
        return self.names

    def step(self, inputs, keep=None):
        """inputs: {name: rows}; keep: {name: how many of them stay} (drafts behind are refused)."""
        m, g = self.model, self.model.given
        names = list(inputs)
        counts = [len(inputs[n]) for n in names]
        x = np.concatenate([inputs[n] for n in names])
        T = len(x)
        for n in names:
            r = self.requests[n]
            need = -(-(r["length"] + len(inputs[n])) // PAGE)
            have = int(np.sum(r["table"] >= 0))
            if need > have:
                r["table"][have:need] = self.pool.take(need - have)
        targets = [self.slots.pop() for _ in names]
        batch = ct.PagedBatch(self.cache, H, [self.requests[n]["length"] for n in names], counts, np.stack([self.requests[n]["table"] for n in names]))
        delta = ct.DeltaBatch(self.states, HK, [self.requests[n]["slot"] for n in names], targets, counts)
        given = give(x)
        h = x.astype(np.float32)
        norm = lambda a: ct.rms_norm(give(a), (D,), None, 1e-5)  # noqa: E731
        view = lambda t, *s: ct.Tensor(ct._new(ct.lib().dl_reshape, t.handle, ct._shape(s)))  # noqa: E731
        z = ct.rms_norm(given, (D,), None, 1e-5)
        q = self.cache.append(0, batch, view(ct.linear(z, g["q"]), T, H, HD), view(ct.linear(z, g["k"]), T, KV, HD),
                              view(ct.linear(z, g["v"]), T, KV, HD), m.cosine, m.sine)
        h = h + ct.linear(view(ct.paged_attention(self.cache, 0, batch, q), T, H * HD), g["o"]).numpy()
        mix = lambda a, layer: ct.expert_mixture(norm(a), *(g[f"{n}{layer}"] for n in ("router", "act", "up", "down")), TOP)[0].numpy()  # noqa: E731
        h = h + mix(h, 0)
        z = norm(h)
        unit = lambda t: ct.rms_norm(view(t, T, HK, DK), (DK,), give(np.full(DK, DK ** -0.5)), 1e-5)  # (of length 1)  # noqa: E731
        gate = ct.linear(z, g["gate"]).numpy()
        out = ct.gated_delta(self.states, 0, delta, unit(ct.linear(z, g["dq"])), unit(ct.linear(z, g["dk"])), view(ct.linear(z, g["dv"]), T, HV, DV),
                             give(-np.abs(gate[:, :HV])), give(1 / (1 + np.exp(-gate[:, HV:]))))
        h = h + ct.linear(view(out, T, HV * DV), g["do"]).numpy()
        h = h + mix(h, 1)
        first, outputs = 0, {}
        for n, c, target in zip(names, counts, targets):
            r = self.requests[n]
            outputs[n] = h[first:first + c]
            want = m.exact(np.concatenate([r["history"], inputs[n]]))[r["length"]:]
            error = np.max(np.abs(outputs[n] - want), -1) / np.max(np.abs(want), -1)
            assert np.all(error < 2.0 ** -8), (n, r["length"], c, float(error.max()))
            kept = c if keep is None or n not in keep else keep[n]
            if kept == c:
                if r["slot"] >= 0:
                    self.slots.append(r["slot"])
                r["slot"], r["length"], r["history"] = target, r["length"] + c, np.concatenate([r["history"], inputs[n]])
            else:  # refused: the old state stays, and the step is taken again with what was accepted
                self.slots.append(target)
                if kept:
                    self.step({n: inputs[n][:kept]})
            first += c
        say(f"  step of {counts}: ok, {self.pool.available} pages free")

    def fork(self, name, children):
        """New requests that go on from `name`: pages shared but the last, the state copied."""
        r = self.requests[name]
        tables = self.cache.fork(self.pool, r["table"][None], [r["length"]], [0] * children)
        slots = [self.slots.pop() for _ in range(children)]
        self.states.copy([r["slot"]] * children, slots)
        out = []
        for table, slot in zip(tables, slots):
            child = self.begin()
            self.requests[child] |= dict(table=table, length=r["length"], slot=slot, history=r["history"].copy())
            out.append(child)
        return out

    def end(self, name):
        r = self.requests.pop(name)
        self.pool.release(r["table"])
        self.slots.append(r["slot"])

    def compact(self):
        names = list(self.requests)
        tables = self.cache.compact(self.pool, np.stack([self.requests[n]["table"] for n in names]))
        for n, table in zip(names, tables):
            self.requests[n]["table"] = table
        return int(tables.max())


@pytest.mark.parametrize("seed", [1, 2])
def test_a_serving_loop_of_a_decoder_with_experts(seed):
    rng = np.random.default_rng(seed)
    rows = lambda n: rng.standard_normal((n, D)).astype(np.float32)  # noqa: E731
    server = Server(Model(seed), 48, 24)
    a, b, c = server.begin(), server.begin(), server.begin()
    server.step({a: rows(37), b: rows(70), c: rows(1)})  # prompts, in chunks and token by token
    server.step({a: rows(1), b: rows(1), c: rows(5)}, keep={c: 2})  # three drafts refused
    d, e = server.fork(a, 2)  # two more answers
    f, = server.fork(b, 1)
    server.step({n: rows(1) for n in (a, b, c, d, e, f)})
    server.step({a: rows(20), d: rows(3), f: rows(1)})  # parents and children part
    server.end(b)
    server.end(a)
    live = 48 - server.pool.available
    assert server.compact() == live - 1
    server.step({c: rows(30), d: rows(1), e: rows(1), f: rows(4)}, keep={f: 0})
    g, = server.fork(e, 1)
    server.end(e)
    server.step({g: rows(9), f: rows(1)})
    assert server.compact() == 47 - server.pool.available
    server.step({n: rows(2) for n in (c, d, f, g)})
    for n in (c, d, f, g):
        server.end(n)
    assert server.pool.available == 48 and len(server.slots) == 24
