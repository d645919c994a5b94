"""The operators of a serving step over a paged key/value cache, as measurable cases: rotary positions, the append that
rotates on the way, attention over the pages (of single tokens, drafted tokens and prompts), the same for a batch that
shares a long prefix, and the verification of drafted tokens.

A case is a dict of plain values with a "kind":

  rotary   rows [tokens, heads, head_dim] at given positions, rotated by cosine and sine tables: interleaved or half
           layout, the first `part` of the head, tables scaled for a longer context or not
  append   the queries, keys and values of a step's new tokens: queries and keys rotated, keys and values written to
           their places in the pages
  attend   the step's queries over the pages, each row over the positions up to its own
  shared   the same where every sequence begins with the same `shared` positions, which lie in the same pages
  verify   drafted tokens against the target model's logits, from given uniform numbers

With `own` false the operators run in their plain form, elementary torch operations; with `own` true through
ctorch_amd's entry points.
"""
import math
import random

import torch

own = False

BASE = 10000.0


def listed():
    return [
        # one token of one request at the 1B decoder's heads: the smallest call
        dict(name="rotary_token", kind="rotary", tokens=1, heads=32, head_dim=64, part=64, layout="interleaved", far=2048,
             scaled=False, dtype="f32"),
        # a long prompt's queries at 8B heads, half of each head rotated, positions far beyond the trained context
        dict(name="rotary_prompt", kind="rotary", tokens=4093, heads=32, head_dim=128, part=64, layout="half", far=131072,
             scaled=True, dtype="bf16"),
        # a decode step of a serving batch: one token of each of 32 sequences
        dict(name="append_step", kind="append", batch=32, held=2048, count=1, heads=32, kv=8, head_dim=64, part=64,
             layout="interleaved", page=16, dtype="bf16", input="f32"),
        # the prompts of four requests of odd lengths, two of them continued
        dict(name="append_prompts", kind="append", batch=4, held=1000, count=1500, heads=32, kv=8, head_dim=128, part=128,
             layout="half", page=64, dtype="f32", input="f32"),
        # a chat's next token over a short history
        dict(name="attend_one", kind="attend", batch=1, held=128, count=1, heads=32, kv=8, head_dim=64, page=16,
             dtype="f32"),
        # a serving batch in flight, sequences of very different lengths
        dict(name="attend_batch", kind="attend", batch=32, held=4096, count=1, heads=32, kv=8, head_dim=64, page=16,
             dtype="bf16"),
        # long contexts at 8B heads: the largest
        dict(name="attend_long", kind="attend", batch=8, held=32767, count=1, heads=32, kv=8, head_dim=128, page=64,
             dtype="bf16"),
        # prompts in chunks: up to 1024 new tokens of four sequences after up to 1024 held ones, f32 pages
        dict(name="attend_prompts", kind="attend", batch=4, held=1024, count=1024, heads=32, kv=8, head_dim=64, page=16,
             dtype="f32"),
        # 64 chats behind one long system prompt
        dict(name="shared_chats", kind="shared", batch=64, shared=4096, held=400, count=1, heads=32, kv=8, head_dim=128,
             page=16, dtype="bf16"),
        # eight answers to one long document, four drafted tokens each to be checked with the next
        dict(name="shared_drafts", kind="shared", batch=8, shared=8192, held=1000, count=5, heads=32, kv=8, head_dim=64,
             page=64, dtype="f32"),
        # one request's four drafted tokens
        dict(name="verify_one", kind="verify", batch=1, drafts=4, vocab=32000, temperature=0.8, draft_logits=True),
        # a batch of 32 requests with up to seven drafted tokens
        dict(name="verify_batch", kind="verify", batch=32, drafts=7, vocab=32000, temperature=1.0, draft_logits=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend", "attend", "prompt", "shared", "shared", "verify"])
    heads, kv = rng.choice([(8, 2), (32, 8), (32, 8), (16, 16), (32, 4), (12, 4)])
    head_dim = rng.choice([32, 64, 64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    layout = rng.choice(["interleaved", "half"])
    if kind == "rotary":
        return dict(kind=kind, tokens=_log(rng, 1, 4000), heads=heads, head_dim=head_dim,
                    part=rng.choice([head_dim, head_dim // 2, head_dim // 4]), layout=layout, far=_log(rng, 4096, 131072),
                    scaled=rng.random() < 0.5, dtype=rng.choice(["f32", "bf16"]))
    if kind == "append":
        batch = _log(rng, 1, 64)
        return dict(kind=kind, batch=batch, held=_log(rng, 1, 4096), count=rng.choice([1, _log(rng, 1, 4000 // batch)]),
                    heads=heads, kv=kv, head_dim=head_dim, part=rng.choice([head_dim, head_dim // 2]), layout=layout,
                    page=page, dtype=dtype, input=rng.choice(["f32", "bf16"]))
    if kind == "attend":
        batch = _log(rng, 1, 64)
        return dict(kind=kind, batch=batch, held=_log(rng, 16, 200000 // batch if batch > 6 else 32000),
                    count=rng.choice([1, 1, rng.randint(2, 9)]), heads=heads, kv=kv, head_dim=head_dim, page=page,
                    dtype=dtype)
    if kind == "prompt":
        batch = _log(rng, 1, 8)
        return dict(kind="attend", batch=batch, held=_log(rng, 1, 1024), count=_log(rng, 16, 3000 // batch), heads=heads,
                    kv=kv, head_dim=head_dim, page=page, dtype=dtype)
    if kind == "shared":
        return dict(kind=kind, batch=_log(rng, 2, 128), shared=page * _log(rng, 512 // page, 16384 // page),
                    held=_log(rng, 1, 600), count=rng.choice([1, 1, rng.randint(2, 6)]), heads=heads, kv=kv,
                    head_dim=head_dim, page=page, dtype=dtype)
    return dict(kind=kind, batch=_log(rng, 1, 48), drafts=rng.randint(1, 8), vocab=_log(rng, 200, 60000),
                temperature=rng.choice([0.0, 0.7, 1.0, 1.3]), draft_logits=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Positions held by each sequence (behind the shared ones, if any) and its new ones.  They are the case's own, so
    that its work is known: spread over a quarter to the whole of `held`, and for prompts (count above 16) of `count`."""
    rng = random.Random(1000 * case["batch"] + case["held"])
    spread = lambda n: n if case["batch"] == 1 else rng.randint((n + 3) // 4, n)  # noqa: E731
    held = [spread(case["held"]) for _ in range(case["batch"])]
    counts = [spread(case["count"]) if case["count"] > 16 else case["count"] for _ in range(case["batch"])]
    return held, counts


def _frequencies(case):
    """Turns per position in 64 bits.  A scaled table is stretched by 8 where a pair turns fewer than 1 time over the
    trained 8192 positions, left alone where it turns more than 32 times, and blended between the two."""
    part = case["part"]
    f = BASE ** (-torch.arange(0, part, 2, dtype=torch.float64, device="cuda") / part)
    if not case.get("scaled"):
        return f
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return f * keep + f / 8.0 * (1 - keep)


def _angles(case, positions):
    return positions.double()[:, None] * _frequencies(case)


def _magnitude(case):
    """What a scaled table multiplies its entries by (0.1 ln 8 + 1)."""
    return 0.1 * math.log(8.0) + 1.0 if case.get("scaled") else 1.0


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}
    kind = case["kind"]
    state = dict(case=case, kind=kind)
    if kind == "verify":
        b, n, v, t = case["batch"], case["drafts"], case["vocab"], case["temperature"]
        target = normal(b, n + 1, v) * 3.0  # a draft model's logits are near the target's
        draft = target[:, :n] + normal(b, n, v) if case["draft_logits"] else None
        guess = (draft if draft is not None else target[:, :n]) / (t if t > 0 else 1.0)
        noise = -torch.log(-torch.log(torch.rand(b, n, v, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
        drafted = (guess + noise * (1.0 if t > 0 else 0.3)).argmax(-1)
        # some sequences have fewer drafts: the rest of their row is -1
        have = torch.randint((n + 1) // 2, n + 1, (b, 1), generator=g, device="cuda")
        drafted = torch.where(torch.arange(n, device="cuda") < have, drafted, -1)
        state |= dict(target=target, draft=draft, drafted=drafted, temperature=t,
                      uniforms=torch.rand(b, n + 1, generator=g, device="cuda"))
        return state
    if kind == "rotary":
        positions = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda")
        angles = _angles(case, torch.arange(case["far"], device="cuda"))
        scale = _magnitude(case)
        state |= dict(x=normal(case["tokens"], case["heads"], case["head_dim"]).to(dtype[case["dtype"]]),
                      positions=positions, cosine=(angles.cos() * scale).float(), sine=(angles.sin() * scale).float(),
                      layout=case["layout"])
        return state
    # a paged cache: each sequence's pages lie anywhere in the pool, which has some more than the step needs
    held, counts = _lengths(case)
    shared, page, kv, d = case.get("shared", 0), case["page"], case["kv"], case["head_dim"]
    need = [-(-(h + c) // page) for h, c in zip(held, counts)]
    width = shared // page + max(need)
    pages = shared // page + sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    front = [order.pop() for _ in range(shared // page)]
    tables = [front + [order.pop() for _ in range(n)] for n in need]
    tables = torch.tensor([t + [-1] * (width - len(t)) for t in tables])
    state |= dict(held=[shared + h for h in held], counts=counts, tables=tables, shared=shared, page=page, heads=case["heads"],
                  key=normal(pages, kv, page, d).to(dtype[case["dtype"]]),
                  value=normal(pages, kv, page, d).to(dtype[case["dtype"]]))
    tokens = sum(counts)
    if kind == "append":
        # the projections' output, queries, keys and values side by side
        qkv = normal(tokens, case["heads"] + 2 * kv, d).to(dtype[case["input"]])
        angles = _angles(case, torch.arange(case["held"] + case["count"], device="cuda"))
        state |= dict(qkv=qkv, cosine=angles.cos().float(), sine=angles.sin().float(), layout=case["layout"])
    else:
        state |= dict(q=normal(tokens, case["heads"], d) * 1.5)
    # where each new token stands: its sequence, its position, and the page and row of that position (the plain form's plan)
    seq = torch.repeat_interleave(torch.arange(case["batch"]), torch.tensor(counts))
    at = torch.arange(tokens) - (torch.tensor(counts).cumsum(0) - torch.tensor(counts))[seq]
    position = torch.tensor(state["held"])[seq] + at
    state |= {name: x.cuda() for name, x in dict(seq=seq, at=at, position=position, pages=tables.clamp(min=0),
                                                 page_of=tables[seq, position // page], row_of=position % page).items()}
    return state


def _library(inputs):
    """The same inputs in the library's hands: its tensors, its cache and the step's batch, as a program keeps them."""
    import ctorch_amd as ct

    kind = inputs["kind"]
    state = dict(kind=kind, ct=ct)
    types = {torch.float32: ct.F32, torch.bfloat16: ct.BF16, torch.int64: ct.I64}

    def hand(x):
        if x is None:
            return None
        t = ct.zeros(x.shape, types[x.dtype])
        ct.synchronize()
        _torch(ct, t).copy_(x)
        return t

    for name in ("x", "positions", "cosine", "sine", "q", "target", "draft", "drafted", "uniforms"):
        if name in inputs:
            state[name] = hand(inputs[name])
    if kind == "verify":
        state["temperature"] = inputs["temperature"]
    if "layout" in inputs:
        state["layout"] = {"interleaved": ct.ROTARY_INTERLEAVED, "half": ct.ROTARY_HALF}[inputs["layout"]]
    if "key" in inputs:
        pages, kv, page, d = inputs["key"].shape
        state["cache"] = cache = ct.PagedCache(1, pages, page, kv, d, types[inputs["key"].dtype])
        state["key"], state["value"] = _torch(ct, cache.key(0)), _torch(ct, cache.value(0))
        ct.synchronize()
        state["key"].copy_(inputs["key"])
        state["value"].copy_(inputs["value"])
        state["batch"] = ct.PagedBatch(cache, inputs["heads"], inputs["held"], inputs["counts"], inputs["tables"].numpy(),
                                       inputs["shared"])
    if "qkv" in inputs:
        h, kv = inputs["heads"], inputs["key"].shape[1]
        qkv = hand(inputs["qkv"])
        state["parts"] = [ct.narrow(qkv, 1, *piece) for piece in ((0, h), (h, kv), (h + kv, kv))]
    torch.cuda.synchronize()
    return state


def prepare(case, seed):
    inputs = _inputs(case, seed)
    return _library(inputs) if own else inputs


class _View:
    """A library tensor as a device array (the view holds the tensor)."""

    def __init__(self, ct, tensor):
        kind, size = {ct.F32: ("<f4", 4), ct.I64: ("<i8", 8), ct.BF16: ("<i2", 2)}[tensor.dtype]
        self.tensor = tensor
        self.__cuda_array_interface__ = dict(shape=tensor.shape, typestr=kind, version=3,
                                             data=(ct.lib().dl_tensor_data(tensor.handle), False))


def _torch(ct, tensor):
    view = torch.as_tensor(_View(ct, tensor), device="cuda")
    return view.view(torch.bfloat16) if tensor.dtype == ct.BF16 else view


# ------------------------------------------------------------------------------------------------ one pass
def _rotate(x, cosine, sine, layout):
    """x [tokens, heads, d] with the first 2 * cosine.size(1) of d rotated by the rows' cosine and sine, in f32."""
    x, c, s = x.float(), cosine[:, None], sine[:, None]
    half = cosine.shape[1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if layout == "interleaved":
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, rest], -1)


def _attend(s, shared):
    """Softmax attention of the step's queries in f32: the shared positions once for all rows, the others gathered by each
    sequence's table and padded to the longest."""
    q, page, kv = s["q"], s["page"], s["key"].shape[1]
    tokens, heads, d = q.shape
    group, batch = heads // kv, len(s["counts"])
    front = shared // page
    gather = lambda pool: pool[s["pages"][:, front:]].transpose(1, 2).flatten(2, 3).float()  # noqa: E731
    keys, values = gather(s["key"]), gather(s["value"])  # [batch, kv, positions, d]
    most = max(s["counts"])
    rows = torch.zeros(batch, most, heads, d, device=q.device)
    rows[s["seq"], s["at"]] = q / math.sqrt(d)
    limit = torch.full((batch, most), -1, device=q.device)
    limit[s["seq"], s["at"]] = s["position"] - shared
    rows = rows.view(batch, most, kv, group, d).transpose(1, 2)  # [batch, kv, most, group, d]
    scores = (rows.flatten(2, 3) @ keys.transpose(2, 3)).view(batch, kv, most, group, -1)
    hidden = torch.arange(keys.shape[2], device=q.device) > limit[:, None, :, None, None]
    scores = scores.masked_fill(hidden, -1e30)
    top = scores.amax(-1, keepdim=True)
    if shared:
        k, v = (s[n][s["pages"][0, :front]].transpose(0, 1).flatten(1, 2).float() for n in ("key", "value"))  # [kv, shared, d]
        flat = rows.transpose(0, 1).reshape(kv, -1, d)
        first = (flat @ k.transpose(1, 2)).view(kv, batch, most, group, shared).transpose(0, 1)
        top = torch.maximum(top, first.amax(-1, keepdim=True))
        first = torch.exp(first - top)
    weights = torch.exp(scores - top).masked_fill(hidden, 0.0)
    out = (weights.flatten(2, 3) @ values).view(batch, kv, most, group, d)
    total = weights.sum(-1, keepdim=True)
    if shared:
        out = out + (first.transpose(0, 1).reshape(kv, -1, shared) @ v).view(kv, batch, most, group, d).transpose(0, 1)
        total = total + first.sum(-1, keepdim=True)
    return (out / total).transpose(1, 2).reshape(batch, most, heads, d)[s["seq"], s["at"]]


def _verify(s):
    """Speculative verification in 64 bits (a decision is a comparison, and a draw a place in a long sum)."""
    drafted, uniforms, t = s["drafted"], s["uniforms"].double(), s["temperature"]
    batch, n = drafted.shape
    live = drafted >= 0
    have = live.long().cumprod(1).sum(1)  # drafts before the first -1
    token = drafted.clamp(min=0)
    if t > 0:
        p = torch.softmax(s["target"].double() / t, -1)
        if s["draft"] is not None:
            q = torch.softmax(s["draft"].double() / t, -1)
        else:
            q = torch.zeros_like(p[:, :n]).scatter_(2, token[..., None], 1.0)
        pick = lambda x: x[:, :n].gather(2, token[..., None])[..., 0]  # noqa: E731
        keep = uniforms[:, :n] * pick(q) < pick(p)
    else:
        best = s["target"].argmax(-1)
        keep = token == best[:, :n]
    accepted = (keep & live).long().cumprod(1).sum(1)
    row = torch.arange(batch, device=drafted.device)
    if t > 0:
        weight = p[row, accepted]
        refused = (accepted < have)[:, None]  # a draft was refused there: what the target has over the draft
        over = (weight - q[row, accepted.clamp(max=n - 1)]).clamp(min=0)
        over = torch.where(over.sum(1, keepdim=True) > 0, over, weight)
        weight = torch.where(refused, over, weight)
        reach = weight.cumsum(1)
        last = (reach <= uniforms[:, n:] * reach[:, -1:]).sum(1)
        last = torch.minimum(last, reach.shape[1] - 1 - (weight > 0).flip(1).long().argmax(1))
    else:
        last = best[row, accepted]
    slots = torch.arange(n + 1, device=drafted.device)
    tokens = torch.where(slots < accepted[:, None], torch.nn.functional.pad(drafted, (0, 1)), -1)
    return {"tokens": torch.where(slots == accepted[:, None], last[:, None], tokens), "accepted": accepted}


def run(state):
    kind = state["kind"]
    if own:
        ct = state["ct"]
        if kind == "rotary":
            return _torch(ct, ct.rotary_positions(state["x"], state["positions"], state["cosine"], state["sine"],
                                                  state["layout"]))
        if kind == "append":
            q = state["cache"].append(0, state["batch"], *state["parts"], state["cosine"], state["sine"], state["layout"])
            return {"query": _torch(ct, q), "key": state["key"], "value": state["value"]}
        if kind == "verify":
            tokens, accepted = ct.verify_drafted(state["drafted"], state["target"], state["draft"], state["temperature"],
                                                 state["uniforms"])
            return {"tokens": _torch(ct, tokens), "accepted": _torch(ct, accepted)}
        return _torch(ct, ct.paged_attention(state["cache"], 0, state["batch"], state["q"]))
    if kind == "rotary":
        at = state["positions"]
        return _rotate(state["x"], state["cosine"][at], state["sine"][at], state["layout"])
    if kind == "append":
        h, kv = state["heads"], state["key"].shape[1]
        q, k, v = state["qkv"].split([h, kv, kv], 1)
        c, s = state["cosine"][state["position"]], state["sine"][state["position"]]
        page, row = state["page_of"], state["row_of"]
        state["key"][page, :, row] = _rotate(k, c, s, state["layout"]).to(state["key"].dtype)
        state["value"][page, :, row] = v.to(state["value"].dtype)
        return {"query": _rotate(q, c, s, state["layout"]), "key": state["key"], "value": state["value"]}
    if kind == "verify":
        return _verify(state)
    return _attend(state, state["shared"])


# ------------------------------------------------------------------------------------------------ accounts
def work(case):
    """Bytes: each input once and each output once (of an append's pages what it writes; of a shared prefix one reading).
    Operations: products of the rows with the positions that they see."""
    size = {"f32": 4, "bf16": 2}
    kind = case["kind"]
    if kind == "verify":
        b, n, v = case["batch"], case["drafts"], case["vocab"]
        rows = n + 1 + (n if case["draft_logits"] and case["temperature"] > 0 else 0)
        return {"bytes": b * (4 * rows * v + 8 * n + 4 * (n + 1) + 8 * (n + 2)), "flops": 10 * b * rows * v}
    if kind == "rotary":
        t, row = case["tokens"], case["heads"] * case["head_dim"]
        return {"bytes": t * (row * (size[case["dtype"]] + 4) + 4 * case["part"] + 8),
                "flops": 3 * t * case["heads"] * case["part"]}
    held, counts = _lengths(case)
    h, kv, d, e = case["heads"], case["kv"], case["head_dim"], size[case["dtype"]]
    tokens = sum(counts)
    if kind == "append":
        return {"bytes": tokens * d * ((h + 2 * kv) * size[case["input"]] + 4 * h + 2 * kv * e) + tokens * 4 * case["part"],
                "flops": 3 * tokens * (h + kv) * case["part"]}
    shared = case.get("shared", 0)
    seen = sum(c * (shared + n) + c * (c + 1) // 2 for n, c in zip(held, counts))
    return {"bytes": 2 * kv * d * e * (shared + sum(held) + tokens) + 8 * tokens * h * d, "flops": 4 * h * d * seen}


# ------------------------------------------------------------------------------------------------ 64-bit results
def _turn(x, angles, layout, scale):
    """x [tokens, heads, d] in 64 bits, each rotated pair as a complex number times scale * e^(i angle)."""
    half = angles.shape[1]
    y = x.double().clone()
    pairs = torch.arange(half, device=x.device)
    first, second = (2 * pairs, 2 * pairs + 1) if layout == "interleaved" else (pairs, pairs + half)
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angles, scale), angles)[:, None]
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "verify":  # whole numbers
        return None
    if kind == "rotary":
        return _turn(s["x"], _angles(case, s["positions"]), case["layout"], _magnitude(case))
    page = s["page"]
    if kind == "append":
        h, kv = case["heads"], case["kv"]
        angles = _angles(case, s["position"])
        key, value = s["key"].double(), s["value"].double()
        q, k = (_turn(x, angles, case["layout"], 1.0) for x in (s["qkv"][:, :h], s["qkv"][:, h:h + kv]))
        key[s["page_of"], :, s["row_of"]], value[s["page_of"], :, s["row_of"]] = k, s["qkv"][:, h + kv:].double()
        return {"query": q, "key": key, "value": value}
    out, first = torch.empty(*s["q"].shape, dtype=torch.float64, device="cuda"), 0
    group = case["heads"] // case["kv"]
    for held, count, table in zip(s["held"], s["counts"], s["tables"].tolist()):
        seen = held + count
        pages = table[:-(-seen // page)]
        k, v = (s[n][pages].permute(1, 0, 2, 3).flatten(1, 2)[:, :seen].double() for n in ("key", "value"))
        late = torch.arange(seen, device="cuda")[None] > held + torch.arange(count, device="cuda")[:, None]
        for i in range(case["heads"]):
            z = s["q"][first:first + count, i].double() @ k[i // group].T / math.sqrt(case["head_dim"])
            out[first:first + count, i] = torch.softmax(z.masked_fill(late, -math.inf), -1) @ v[i // group]
        first += count
    return out
