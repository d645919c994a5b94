"""The operators of a serving step beyond the paged attention's, as measurable cases: a layer of experts over few tokens,
the gated delta rule over states of fixed size (single tokens, drafted ones, prompts), and forking and compacting the
pages of a cache.

A case is a dict of plain values with a "kind":

  experts   rows [tokens, dim] through a router and the `top` best of `experts` SwiGLU experts of `hidden` entries each
  delta     the step's queries, keys and values [tokens, heads, d] through the states of their requests: `count` new
            tokens of each of `batch` requests, a share of which begins with this step
  fork      `children` copies of each of `batch` requests: whole pages are shared, the last, partly filled one is copied
            in every layer; then the copies' pages are given back
  compact   `live` of `pages` pages, which lie anywhere, moved to the front of the pool in every layer

With `own` false the operators run in their plain form, elementary torch operations; with `own` true through
ctorch_amd's entry points.
"""
import math
import random

import numpy as np
import torch

own = False


def listed():
    return [
        # one token of one request through a small layer of experts: the smallest call
        dict(name="experts_token", kind="experts", tokens=1, dim=1024, hidden=704, experts=16, top=2, normalise=True,
             weight="bf16", input="f32"),
        # f32 weights at the tiny decoder's widths, a few drafted tokens
        dict(name="experts_f32", kind="experts", tokens=5, dim=256, hidden=688, experts=8, top=2, normalise=False,
             weight="f32", input="f32"),
        # a decode step of a serving batch at the 1B decoder's width: nearly all experts are read
        dict(name="experts_step", kind="experts", tokens=16, dim=2048, hidden=1024, experts=64, top=8, normalise=True,
             weight="bf16", input="f32"),
        # a chunk of prompts beside it
        dict(name="experts_chunk", kind="experts", tokens=200, dim=2048, hidden=768, experts=32, top=4, normalise=True,
             weight="bf16", input="bf16"),
        # one token of one request through its states
        dict(name="delta_token", kind="delta", batch=1, count=1, key_heads=8, heads=8, key_dim=64, value_dim=64, input="f32"),
        # a decode step of 64 requests, two value heads to a key head
        dict(name="delta_step", kind="delta", batch=64, count=1, key_heads=16, heads=32, key_dim=128, value_dim=128,
             input="bf16"),
        # drafted tokens of a batch, from the states of before them
        dict(name="delta_drafts", kind="delta", batch=12, count=5, key_heads=16, heads=16, key_dim=128, value_dim=64,
             input="f32"),
        # one long prompt: the longest chain
        dict(name="delta_prompt", kind="delta", batch=1, count=8191, key_heads=16, heads=32, key_dim=128, value_dim=128,
             input="bf16"),
        # prompts of several requests, of odd lengths
        dict(name="delta_prompts", kind="delta", batch=6, count=1500, key_heads=8, heads=16, key_dim=64, value_dim=128,
             input="f32"),
        # three more answers to one prompt: a few rows of one page in 16 layers
        dict(name="fork_one", kind="fork", batch=1, children=3, held=1000, layers=16, kv=8, head_dim=64, page=16, dtype="bf16"),
        # a beam of four for each of 16 requests, f32 pages
        dict(name="fork_many", kind="fork", batch=16, children=4, held=900, layers=16, kv=8, head_dim=64, page=64, dtype="f32"),
        # what is left of a pool after many requests have ended, moved to its front
        dict(name="compact", kind="compact", pages=480, live=230, layers=16, kv=8, head_dim=64, page=64, dtype="bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["experts", "experts", "delta", "delta", "prompt", "fork", "compact"])
    if kind == "experts":
        experts = rng.choice([4, 8, 16, 32, 64, 128])
        dim = 8 * _log(rng, 16, 256)
        # (the weights within those of 64 experts of 2048 x 1024)
        hidden = 8 * _log(rng, 8, min(256, 64 * 2048 * 1024 // (8 * dim * experts)))
        return dict(kind=kind, tokens=_log(rng, 1, 200), dim=dim - rng.choice([0, 0, 0, 1]), hidden=hidden, experts=experts,
                    top=rng.randint(1, min(8, experts)), normalise=rng.random() < 0.6, weight=rng.choice(["f32", "bf16", "bf16"]),
                    input=rng.choice(["f32", "bf16"]))
    if kind in ("delta", "prompt"):
        heads, key_heads = rng.choice([(8, 8), (16, 16), (16, 8), (32, 16), (12, 4), (6, 2)])
        key_dim, value_dim = rng.choice([(32, 32), (64, 64), (64, 128), (128, 64), (128, 128), (128, 128)])
        if kind == "delta":
            batch, count = _log(rng, 1, 64), rng.choice([1, 1, rng.randint(2, 9)])
        else:
            batch = _log(rng, 1, 8)
            count = _log(rng, 10, 6000 // batch)
        return dict(kind="delta", batch=batch, count=count, key_heads=key_heads, heads=heads, key_dim=key_dim,
                    value_dim=value_dim, input=rng.choice(["f32", "bf16"]))
    layers, kv = rng.choice([(4, 8), (16, 8), (24, 4), (30, 2)])
    common = dict(layers=layers, kv=kv, head_dim=rng.choice([32, 64, 128]), page=rng.choice([16, 32, 64, 128]),
                  dtype=rng.choice(["f32", "bf16", "bf16"]))
    row = 2 * layers * kv * common["head_dim"] * {"f32": 4, "bf16": 2}[common["dtype"]]  # bytes of a position
    if kind == "fork":
        batch = _log(rng, 1, 24)
        return dict(kind=kind, batch=batch, children=rng.randint(1, 6), held=_log(rng, 5, min(4000, (1 << 29) // (row * batch))),
                    **common)
    pages = _log(rng, 6, max(6, min(3000, (1 << 30) // (row * common["page"]))))
    return dict(kind=kind, pages=pages, live=rng.randint(pages // 4 + 1, pages // 2 + 1), **common)


# ------------------------------------------------------------------------------------------------ inputs
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _spread(case, name):
    """A number for each request, half of the case's to the whole of it: the case's own, so that its work is known."""
    rng = random.Random(1000 * case["batch"] + case[name])
    n = case[name]
    return [n if case["batch"] == 1 else rng.randint((n + 1) // 2, n) for _ in range(case["batch"])]


def _counts(case):
    return _spread(case, "count") if case["count"] > 9 else [case["count"]] * case["batch"]


def _fresh(case):
    """Which requests begin with this step: a third of those with prompts (not a lone one's, which is continued)."""
    return [case["count"] > 9 and b % 3 == 2 for b in range(case["batch"])]


def _places(case):
    """Page tables of the case's requests, whose pages lie anywhere in the pool, and the pool's size."""
    rng = random.Random(case.get("held", 0) + case["page"])
    if case["kind"] == "compact":
        live = rng.sample(range(case["pages"]), case["live"])
        width = max(1, min(9, case["live"]))
        rows = [live[i:i + width] for i in range(0, len(live), width)]
        return np.array([r + [-1] * (width - len(r)) for r in rows], np.int64), case["pages"]
    held = _spread(case, "held")
    need = [-(-n // case["page"]) for n in held]
    pages = sum(need) + case["batch"] * case["children"] + 2
    order = rng.sample(range(pages), pages)
    width = max(need) + 1
    tables = [[order.pop() for _ in range(n)] for n in need]
    return np.array([t + [-1] * (width - len(t)) for t in tables], np.int64), pages


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    kind = case["kind"]
    state = dict(case=case, kind=kind)
    if kind == "experts":
        t, d, h, e = case["tokens"], case["dim"], case["hidden"], case["experts"]
        weight = TYPES[case["weight"]]

        def matrices(*shape):  # one expert after another: the f32 draw is never held for all
            out = torch.empty(*shape, dtype=weight, device="cuda")
            for part in out:
                part.copy_(normal(*shape[1:]) * 0.02)
            return out

        # rows behind a norm, and weights of the decoders' scale
        state |= dict(x=normal(t, d).to(TYPES[case["input"]]), router=(normal(e, d) * 0.02).to(weight),
                      gate=matrices(e, h, d), up=matrices(e, h, d), down=matrices(e, d, h), top=case["top"],
                      normalise=case["normalise"])
        return state
    if kind == "delta":
        batch, hk, h, dk, dv = (case[n] for n in ("batch", "key_heads", "heads", "key_dim", "value_dim"))
        counts, kind_of = _counts(case), TYPES[case["input"]]
        tokens = sum(counts)
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        mean = normal(1, hk, dk)  # the keys of a text have a direction in common
        # heads forget at rates from a thousandth to about one a token
        pace = torch.exp(torch.linspace(math.log(1e-3), math.log(1.0), h, device="cuda"))
        order = random.Random(batch + 7 * tokens).sample(range(2 * batch + 3), 2 * batch)
        state |= dict(q=unit(normal(tokens, hk, dk)).to(kind_of), k=unit(normal(tokens, hk, dk) + 0.3 * mean).to(kind_of),
                      v=normal(tokens, h, dv).to(kind_of), decay=-pace * torch.nn.functional.softplus(normal(tokens, h) + 0.5),
                      rate=torch.sigmoid(normal(tokens, h)), states=normal(2 * batch + 3, h, dk, dv) * 0.3,
                      # the states of before the step are kept (a draft may be refused): it writes others
                      sources=[-1 if new else s for new, s in zip(_fresh(case), order)], targets=order[batch:], counts=counts)
        seq = torch.repeat_interleave(torch.arange(batch), torch.tensor(counts))
        at = torch.arange(tokens) - (torch.tensor(counts).cumsum(0) - torch.tensor(counts))[seq]
        state |= dict(seq=seq.cuda(), at=at.cuda(), into=torch.tensor(state["targets"]).cuda(),
                      whence=torch.tensor(state["sources"]).clamp(min=0).cuda(),
                      kept=torch.tensor([float(s >= 0) for s in state["sources"]]).cuda())
        return state
    tables, pages = _places(case)
    shape = (case["layers"], pages, case["kv"], case["page"], case["head_dim"])
    state |= dict(tables=tables, pages=pages, page=case["page"])
    for name in ("key", "value"):
        pool = torch.empty(*shape, dtype=TYPES[case["dtype"]], device="cuda")
        for layer in pool:
            layer.copy_(normal(*shape[1:]))
        state[name] = list(pool)
    if kind == "fork":
        state |= dict(lengths=_spread(case, "held"), parents=[b for b in range(case["batch"]) for _ in range(case["children"])])
    return state


def _library(inputs):
    """The same inputs in the library's hands: its tensors, its cache or states and the step's batch, as a program keeps
    them."""
    import ctorch_amd as ct

    kind = inputs["kind"]
    state = dict(kind=kind, ct=ct)
    types = {torch.float32: ct.F32, torch.bfloat16: ct.BF16}

    def hand(x):
        t = ct.zeros(x.shape, types[x.dtype])
        ct.synchronize()
        _torch(ct, t).copy_(x)
        return t

    if kind == "experts":
        state |= {name: hand(inputs.pop(name)) for name in ("x", "router", "gate", "up", "down")}
        state |= dict(top=inputs["top"], normalise=inputs["normalise"])
    elif kind == "delta":
        state |= {name: hand(inputs[name]) for name in ("q", "k", "v", "decay", "rate")}
        slots, heads, key_dim, value_dim = inputs["states"].shape
        state["states"] = states = ct.DeltaStates(1, slots, heads, key_dim, value_dim)
        state["state"] = _torch(ct, states.state(0))
        ct.synchronize()
        state["state"].copy_(inputs["states"])
        state["batch"] = ct.DeltaBatch(states, inputs["k"].shape[1], inputs["sources"], inputs["targets"], inputs["counts"])
    else:
        layers = len(inputs["key"])
        pages, kv, page, d = inputs["key"][0].shape
        state["cache"] = cache = ct.PagedCache(layers, pages, page, kv, d, types[inputs["key"][0].dtype])
        for name, of in (("key", cache.key), ("value", cache.value)):
            state[name] = [_torch(ct, of(layer)) for layer in range(layers)]
            ct.synchronize()
            for held, given in zip(state[name], inputs[name]):
                held.copy_(given)
        state |= {name: inputs[name] for name in ("tables", "pages", "lengths", "parents") if name in inputs}
        if kind == "fork":
            state["pool"] = ct.PagePool(pages)
            state["pool"].claim(inputs["tables"])
    torch.cuda.synchronize()
    return state


def prepare(case, seed):
    inputs = _inputs(case, seed)
    if own:
        return _library(inputs)
    if case["kind"] == "fork":  # how many hold each page
        inputs["references"] = np.bincount(inputs["tables"][inputs["tables"] >= 0], minlength=inputs["pages"])
    return inputs


class _View:
    """A library tensor as a device array (the view holds the tensor)."""

    def __init__(self, ct, tensor):
        kind = {ct.F32: "<f4", ct.I64: "<i8", ct.BF16: "<i2"}[tensor.dtype]
        self.tensor = tensor
        self.__cuda_array_interface__ = dict(shape=tensor.shape, typestr=kind, version=3,
                                             data=(ct.lib().dl_tensor_data(tensor.handle), False))


def _torch(ct, tensor):
    view = torch.as_tensor(_View(ct, tensor), device="cuda")
    return view.view(torch.bfloat16) if tensor.dtype == ct.BF16 else view


# ------------------------------------------------------------------------------------------------ one pass
def _route(x, router, top, normalise):
    """The chosen experts and their weights in 64 bits (a choice is a comparison), the lowest index first among equals."""
    p = torch.softmax(x.double() @ router.double().T, -1)
    weights, chosen = torch.sort(p, descending=True, stable=True)
    weights, chosen = weights[:, :top], chosen[:, :top]
    return chosen.contiguous(), weights / weights.sum(-1, keepdim=True) if normalise else weights


def _experts(s):
    x, (tokens, dim) = s["x"].float(), s["x"].shape
    chosen, weights = _route(s["x"], s["router"], s["top"], s["normalise"])
    weights = weights.float()
    experts = len(s["gate"])
    silu = lambda z: z / (1 + torch.exp(-z))  # noqa: E731
    if chosen.numel() <= experts:  # each pair's own matrices
        flat, rows = chosen.flatten(), x.repeat_interleave(s["top"], 0)[..., None]
        hidden = silu(s["gate"][flat].float() @ rows) * (s["up"][flat].float() @ rows)
        y = (s["down"][flat].float() @ hidden).view(tokens, s["top"], dim)
        y = (y * weights[..., None]).sum(1)
    else:  # every expert over all rows, with weight zero where it was not chosen
        dense = torch.zeros(tokens, experts, device=x.device).scatter_(1, chosen, weights)
        hidden = silu(x @ s["gate"].float().transpose(1, 2)) * (x @ s["up"].float().transpose(1, 2))
        y = ((hidden @ s["down"].float().transpose(1, 2)) * dense.T[..., None]).sum(0)
    return {"y": y, "chosen": chosen, "weights": weights}


def _delta(s):
    """Chunks of up to 64 tokens, the requests side by side and padded to the longest: within a chunk the rule is a
    triangular system, between chunks the states go on."""
    batch, most = len(s["counts"]), max(s["counts"])
    chunk = min(64, most)
    padded = -(-most // chunk) * chunk
    heads, dv = s["v"].shape[1:]
    dk, group = s["k"].shape[2], heads // s["k"].shape[1]

    def lay(x, dtype=torch.float32):  # [batch, heads, chunks, chunk, ...]
        out = torch.zeros(batch, padded, *x.shape[1:], dtype=dtype, device=x.device)
        out[s["seq"], s["at"]] = x.to(dtype)
        if x.ndim == 3 and x.shape[1] != heads:
            out = out.repeat_interleave(group, 2)
        return out.transpose(1, 2).unflatten(2, (-1, chunk))

    q, k, v, rate = (lay(s[n]) for n in ("q", "k", "v", "rate"))
    reach = lay(s["decay"], torch.float64).cumsum(-1)  # the sums are long, and their differences short
    fade = torch.exp((reach[..., :, None] - reach[..., None, :]).float()).tril()
    since, left = torch.exp(reach.float()), torch.exp((reach[..., -1:] - reach).float())
    kt = k.transpose(-1, -2).contiguous()
    a = ((k @ kt) * fade * rate[..., None]).tril(-1)
    solve = torch.eye(chunk, device=q.device).expand_as(a).contiguous()  # the inverse of 1 + a, row by row
    for i in range(1, chunk):
        solve[..., i, :i] = -(a[..., i:i + 1, :i] @ solve[..., :i, :i])[..., 0, :]
    own_part = solve @ (v * rate[..., None])
    held_part = solve @ (k * (rate * since)[..., None])
    within, queries = (q @ kt) * fade, q * since[..., None]
    keys = (k * left[..., None]).transpose(-1, -2).contiguous()
    state = s["states"][s["whence"]] * s["kept"][:, None, None, None]
    outs = []
    for c in range(padded // chunk):
        u = own_part[:, :, c] - held_part[:, :, c] @ state
        outs.append(queries[:, :, c] @ state + within[:, :, c] @ u)
        state = state * since[:, :, c, -1, None, None] + keys[:, :, c] @ u
    out = torch.cat(outs, 2).transpose(1, 2)[s["seq"], s["at"]] / math.sqrt(dk)
    s["states"][s["into"]] = state
    return {"out": out, "states": s["states"]}


def _fork(s):
    page, children = s["page"], []
    free = np.flatnonzero(s["references"] == 0)
    moves, taken = [], 0
    for parent in s["parents"]:
        whole, rest = divmod(s["lengths"][parent], page)
        table = s["tables"][parent].copy()
        table[whole + (rest > 0):] = -1
        s["references"][table[:whole]] += 1
        if rest:
            moves.append((table[whole], free[taken], rest))
            table[whole] = free[taken]
            s["references"][free[taken]] = 1
            taken += 1
        children.append(table)
    if moves:  # row by row of the pages, all at once in each layer
        source, target, row = (torch.from_numpy(np.concatenate(x)).cuda() for x in zip(
            *[(np.full(rows, s_), np.full(rows, t_), np.arange(rows)) for s_, t_, rows in moves]))
        for pool in s["key"] + s["value"]:
            pool[target, :, row] = pool[source, :, row]
    children = np.stack(children)
    np.subtract.at(s["references"], children[children >= 0], 1)
    return {"tables": children, "key": s["key"], "value": s["value"]}


def _compact(s):
    tables = s["tables"].copy()
    live = np.unique(tables[tables >= 0])
    source = live[live >= len(live)]
    target = np.setdiff1d(np.arange(len(live)), live)
    rename = np.arange(s["pages"])
    rename[source] = target
    tables[tables >= 0] = rename[tables[tables >= 0]]
    source, target = torch.from_numpy(source).cuda(), torch.from_numpy(target).cuda()
    for pool in s["key"] + s["value"]:
        pool[target] = pool[source]
    return {"tables": tables, "key": s["key"], "value": s["value"]}


def run(state):
    kind = state["kind"]
    if not own:
        return {"experts": _experts, "delta": _delta, "fork": _fork, "compact": _compact}[kind](state)
    ct = state["ct"]
    if kind == "experts":
        y, chosen, weights = ct.expert_mixture(state["x"], state["router"], state["gate"], state["up"], state["down"],
                                               state["top"], state["normalise"])
        return {"y": _torch(ct, y), "chosen": _torch(ct, chosen), "weights": _torch(ct, weights)}
    if kind == "delta":
        out = ct.gated_delta(state["states"], 0, state["batch"], state["q"], state["k"], state["v"], state["decay"],
                             state["rate"])
        return {"out": _torch(ct, out), "states": state["state"]}
    if kind == "fork":
        tables = state["cache"].fork(state["pool"], state["tables"], state["lengths"], state["parents"])
        state["pool"].release(tables)
    else:
        pool = ct.PagePool(state["pages"])
        pool.claim(state["tables"])
        tables = state["cache"].compact(pool, state["tables"])
    return {"tables": tables, "key": state["key"], "value": state["value"]}


# ------------------------------------------------------------------------------------------------ accounts
def work(case):
    """Bytes: each input once and each output once (of experts those that are likely to be chosen, of pages what is
    copied).  Operations: the chosen experts' products; three products with the state for each token and head."""
    size = {"f32": 4, "bf16": 2}
    kind = case["kind"]
    if kind == "experts":
        t, d, h, e, k = (case[n] for n in ("tokens", "dim", "hidden", "experts", "top"))
        active = e * (1 - (1 - k / e) ** t)
        return {"bytes": round((3 * active * h + e) * d * size[case["weight"]] + t * d * (size[case["input"]] + 4) + 12 * t * k),
                "flops": 6 * t * k * d * h + 2 * t * d * e}
    if kind == "delta":
        hk, h, dk, dv, e = *(case[n] for n in ("key_heads", "heads", "key_dim", "value_dim")), size[case["input"]]
        tokens, read = sum(_counts(case)), _fresh(case).count(False)
        return {"bytes": tokens * (2 * hk * dk * e + h * dv * e + 8 * h + 4 * h * dv) + 4 * h * dk * dv * (read + case["batch"]),
                "flops": 6 * tokens * h * dk * dv}
    row = 2 * case["layers"] * case["kv"] * case["head_dim"] * size[case["dtype"]]
    tables, _ = _places(case)
    if kind == "fork":
        rows = case["children"] * sum(n % case["page"] for n in _spread(case, "held"))
    else:
        rows = case["page"] * int((tables >= case["live"]).sum())
    return {"bytes": max(1, 2 * rows * row), "flops": 0}


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "compact"):  # copies
        return None
    s = _inputs(case, seed)
    if kind == "experts":
        x = s["x"].double()
        z = (x[:, None] * s["router"].double()).sum(-1)
        p = torch.exp(z - z.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        left, chosen, weights = p.clone(), [], []
        for _ in range(case["top"]):
            best = left.argmax(-1, keepdim=True)
            chosen.append(best)
            weights.append(p.gather(1, best))
            left.scatter_(1, best, -1.0)
        chosen, weights = torch.cat(chosen, 1), torch.cat(weights, 1)
        if case["normalise"]:
            weights = weights / weights.sum(-1, keepdim=True)
        y = torch.zeros_like(x)
        for e in range(case["experts"]):
            at, slot = torch.nonzero(chosen == e, as_tuple=True)
            if len(at):
                gate = x[at] @ s["gate"][e].double().T
                hidden = gate * torch.sigmoid(gate) * (x[at] @ s["up"][e].double().T)
                y.index_add_(0, at, weights[at, slot, None] * (hidden @ s["down"][e].double().T))
        return {"y": y, "chosen": None, "weights": weights}
    # the rule, one token after another
    batch, most = case["batch"], max(s["counts"])
    heads, dv = s["v"].shape[1:]
    group = heads // s["k"].shape[1]

    def lay(x):  # [most, batch, heads, ...], nothing where a request has no such token
        out = torch.zeros(most, batch, *x.shape[1:], dtype=torch.float64, device=x.device)
        out[s["at"], s["seq"]] = x.double()
        return out.repeat_interleave(group, 2) if x.shape[1] != heads else out

    q, k, v, decay, rate = (lay(s[n]) for n in ("q", "k", "v", "decay", "rate"))
    state = s["states"].double()
    now = state[s["whence"]] * s["kept"].double()[:, None, None, None]
    out = torch.empty(most, batch, heads, dv, dtype=torch.float64, device=q.device)
    for t in range(most):
        now = now * torch.exp(decay[t])[..., None, None]
        wrong = v[t] - (k[t][..., None] * now).sum(-2)
        now = now + k[t][..., None] * (rate[t][..., None] * wrong)[..., None, :]
        out[t] = (q[t][..., None] * now).sum(-2)
    state[s["into"]] = now
    return {"out": out[s["at"], s["seq"]] * case["key_dim"] ** -0.5, "states": state}
