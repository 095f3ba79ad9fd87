"""Many continuations of one prompt: attention over a shared prefix, and draws from given random numbers.

Two kinds of cases, each a call that a serving program makes in every step:

    prefix   attention of a batch whose requests share their first positions in groups, over the paged cache:
             single tokens, or the short portions that follow a common system prompt
    draw     tokens from rows of logits by temperature, top-k, top-p and min-p, with the caller's uniform numbers; one
             draw a row, or the first tokens of many continuations from one row; and the probability of each

Head layouts, vocabularies and page size are the benchmark's Qwen2.5 shapes'.
"""

from __future__ import annotations

import math
import random

import torch

own = False

SHAPES = {
    "0.5b": dict(heads=14, kv_heads=2, dim=64, vocab=151936),
    "7b": dict(heads=28, kv_heads=4, dim=128, vocab=152064),
    "14b": dict(heads=40, kv_heads=8, dim=128, vocab=152064),
}
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
SMALLEST = 2.0 ** -44        # a weight below it (the largest is 1) counts as none


def listed():
    return [
        # two continuations of a short prompt on the smallest model: latency
        dict(name="prefix-0.5b-2-of-176", kind="prefix", shape="0.5b", dtype="bfloat16", page=16,
             groups=1, members=2, prefix=176, own=9, tokens=1),
        # eight samples of the benchmark's prompt, some way into their answers
        dict(name="prefix-7b-8-of-2048", kind="prefix", shape="7b", dtype="bfloat16", page=16,
             groups=1, members=8, prefix=2048, own=257, tokens=1),
        # a loaded server with one long system prompt
        dict(name="prefix-7b-64-of-8192", kind="prefix", shape="7b", dtype="bfloat16", page=16,
             groups=1, members=64, prefix=8192, own=511, tokens=1),
        # four applications on one server, each with a system prompt of its own
        dict(name="prefix-14b-4x16-of-4000", kind="prefix", shape="14b", dtype="bfloat16", page=16,
             groups=4, members=16, prefix=4000, own=1001, tokens=1),
        # questions about one document: their prompts' few tokens behind a long prefix
        dict(name="prefix-7b-portions-24-of-20000", kind="prefix", shape="7b", dtype="bfloat16", page=16,
             groups=1, members=24, prefix=20000, own=0, tokens=47),
        # the command line's default type
        dict(name="prefix-0.5b-float32-8-of-1504", kind="prefix", shape="0.5b", dtype="float32", page=16,
             groups=1, members=8, prefix=1504, own=100, tokens=1),
        # a chat with one user: latency
        dict(name="draw-1-filtered", kind="draw", vocab=151936, dtype="float32", rows=1, draws=1, filters="all"),
        # a batch without filters: every token can be drawn
        dict(name="draw-8-plain", kind="draw", vocab=152064, dtype="float32", rows=8, draws=1, filters="none"),
        # the first tokens of 64 continuations of one prompt
        dict(name="draw-1x64-filtered", kind="draw", vocab=152064, dtype="float32", rows=1, draws=64, filters="all"),
        # a loaded server, every request with settings of its own
        dict(name="draw-64-mixed", kind="draw", vocab=152064, dtype="float32", rows=64, draws=1, filters="mixed"),
        # logits in 16 bits (many equal values) and a mass to be found among all tokens
        dict(name="draw-256-bf16-top-p", kind="draw", vocab=152064, dtype="bfloat16", rows=256, draws=1, filters="mass"),
    ]


def draw(rng):
    most = {k: max(_cost(c) for c in listed() if c["kind"] == k) for k in ("prefix", "draw")}
    while True:
        case = _draw(rng)
        if _cost(case) <= most[case["kind"]]:
            return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.6e15)


def _draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if rng.random() < 0.5:
        page = rng.choice([16, 16, 32])
        return dict(kind="prefix", shape=rng.choice(list(SHAPES)), dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]),
                    page=page, groups=rng.choice([1, 1, 2, 3, 5]), members=size(2, 80),
                    prefix=page * max(1, size(128, 24000) // page), own=size(1, 1500), tokens=rng.choice([1, 1, 1, size(2, 60)]))
    return dict(kind="draw", vocab=rng.choice([151936, 152064, size(1000, 152064)]), dtype=rng.choice(["float32", "float32", "bfloat16"]),
                rows=size(1, 256), draws=rng.choice([1, 1, 1, size(2, 64)]), filters=rng.choice(["all", "none", "mixed", "mass"]))


def _lengths(case):
    """Cached positions behind the prefix, and new tokens, of every request: they follow from the case alone."""
    r = random.Random("%(groups)d %(members)d %(prefix)d %(own)d %(tokens)d" % case)
    n = case["groups"] * case["members"]
    return [r.randint(0, case["own"]) for _ in range(n)], [r.randint(1, case["tokens"]) for _ in range(n)]


def _generator(seed, stream):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + stream) % (1 << 62))


def prepare(case, seed):
    return (_prepare_prefix if case["kind"] == "prefix" else _prepare_draw)(case, seed)


def run(state):
    if own:
        return _own_prefix(state) if state["kind"] == "prefix" else _own_draw(state)
    return _plain_prefix(state) if state["kind"] == "prefix" else _plain_draw(state)


# ------------------------------------------------------------------------------------------- a shared prefix
def _prepare_prefix(case, seed):
    s, dtype, page = SHAPES[case["shape"]], DTYPES[case["dtype"]], case["page"]
    behind, new = _lengths(case)
    n, P = len(new), case["prefix"]
    blocks = [-(-(P + b + t) // page) for b, t in zip(behind, new)]
    shared = P // page
    pages = case["groups"] * shared + sum(b - shared for b in blocks)
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table = torch.full((n, max(blocks)), -1, dtype=torch.int32)
    firsts = [ids[g * shared:(g + 1) * shared] for g in range(case["groups"])]
    at = case["groups"] * shared
    for r, b in enumerate(blocks):
        table[r, :shared] = torch.tensor(firsts[r // case["members"]], dtype=torch.int32)
        table[r, shared:b] = torch.tensor(ids[at:at + b - shared], dtype=torch.int32)
        at += b - shared

    def normal(stream, *shape):
        return torch.randn(shape, generator=_generator(seed, stream), device="cuda").to(dtype)

    # keys as a trained model has them: one direction that all share, and queries that find some of them
    d, rows = s["dim"], sum(new)
    store = normal(1, 2, pages, s["kv_heads"], page, d)
    store[0] += normal(2, 1, s["kv_heads"], 1, d)
    q = normal(3, rows, s["heads"] * d) * 1.5

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    return dict(kind="prefix", case=case, q=q, keys=store[0], values=store[1], table=table.cuda(), cu_q=ints(cu),
                ctx_len=ints([P + b for b in behind]), prefix_len=ints([P] * case["groups"]),
                group_off=ints([g * case["members"] for g in range(case["groups"] + 1)]), single=case["tokens"] == 1,
                heads=s["heads"], kv_heads=s["kv_heads"], dim=d, scale=d ** -0.5, out=torch.empty_like(q))


def _own_prefix(t):
    from somi_inference_b200.ops import cuda_ops
    cuda_ops().shared_prefix_attention(t["q"], t["keys"], t["values"], t["table"], t["ctx_len"], t["prefix_len"], t["group_off"],
                                       t["heads"], t["kv_heads"], t["dim"], t["scale"], t["out"],
                                       cu_q=None if t["single"] else t["cu_q"])
    return t["out"]


def _plain_prefix(t):
    """The prefix as one product a group over all of its rows, the requests' own positions padded to the longest."""
    c, nk, d = t["case"], t["kv_heads"], t["dim"]
    G, B, P, page = c["groups"], c["members"], c["prefix"], c["page"]
    R, per = G * B, t["heads"] // t["kv_heads"]
    new = t["cu_q"][1:] - t["cu_q"][:-1]
    N = c["tokens"]
    # rows [R, N] of the padded batch, and where each token lies in it
    col = torch.arange(N, device=new.device)
    live = col[None] < new[:, None]
    row = (t["cu_q"][:-1, None] + col[None]).clamp(max=t["q"].shape[0] - 1)
    q = t["q"][row.reshape(-1).long()].float().view(R, N, nk, per, d).permute(0, 2, 1, 3, 4)        # [R, nk, N, per, d]
    q = q.reshape(R, nk, N * per, d) * t["scale"]

    def gathered(store, pages):
        x = store[pages.long().clamp(min=0)]                    # [.., blocks, nk, page, d]
        x = x.transpose(-3, -4) if x.dim() == 4 else x.transpose(1, 2)
        return x.reshape(x.shape[0], nk, -1, d).float()

    first = t["table"][::B, :P // page]
    kp, vp = gathered(t["keys"], first), gathered(t["values"], first)                               # [G, nk, P, d]
    mine = t["table"][:, P // page:]
    ko, vo = gathered(t["keys"], mine), gathered(t["values"], mine)                                 # [R, nk, L, d]
    sp = q.view(G, B, nk, N * per, d).transpose(1, 2).reshape(G, nk, B * N * per, d) @ kp.transpose(-1, -2)
    so = q @ ko.transpose(-1, -2)
    last = (t["ctx_len"][:, None] + col[None]).repeat_interleave(per, 1)                            # [R, N * per]
    at = P + torch.arange(ko.shape[2], device=new.device)
    so = so.masked_fill((at[None, None] > last[..., None])[:, None], float("-inf"))
    sp_r = sp.view(G, nk, B, N * per, P).transpose(1, 2).reshape(R, nk, N * per, P)
    m = torch.maximum(sp_r.amax(-1), so.amax(-1))[..., None]
    ep, eo = (sp_r - m).exp(), (so - m).exp()
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    op = ep.view(G, B, nk, N * per, P).transpose(1, 2).reshape(G, nk, B * N * per, P) @ vp
    o = op.view(G, nk, B, N * per, d).transpose(1, 2).reshape(R, nk, N * per, d) + eo @ vo
    o = (o / total).view(R, nk, N, per, d).transpose(1, 2).reshape(R, N, nk * per * d)
    return o[live].to(t["q"].dtype)


def _exact_prefix(case, seed):
    """Every request by itself: softmax over all of its positions, in 64 bits."""
    t = prepare(case, seed)
    d, per = t["dim"], t["heads"] // t["kv_heads"]
    behind, new = _lengths(case)
    out, row = [], 0
    for r, (b, n) in enumerate(zip(behind, new)):
        length = case["prefix"] + b + n
        pages = t["table"][r, :-(-length // case["page"])].long()
        k = t["keys"][pages].double().permute(1, 0, 2, 3).reshape(t["kv_heads"], -1, d)[:, :length]
        v = t["values"][pages].double().permute(1, 0, 2, 3).reshape(t["kv_heads"], -1, d)[:, :length]
        q = t["q"][row:row + n].double().view(n, t["kv_heads"], per, d)
        s = torch.einsum("nkpd,kld->nkpl", q, k) * t["scale"]
        seen = torch.arange(length, device="cuda")[None] <= (length - n + torch.arange(n, device="cuda"))[:, None]
        s = s.masked_fill(~seen[:, None, None], float("-inf"))
        out.append(torch.einsum("nkpl,kld->nkpd", torch.softmax(s, -1), v).reshape(n, -1))
        row += n
    return torch.cat(out)


# ------------------------------------------------------------------------------------------------------ draws
def _prepare_draw(case, seed):
    R, V = case["rows"], case["vocab"]
    g = _generator(seed, 7)
    x = torch.randn((R, V), generator=g, device="cuda") * 2.2
    # a few dozen likely tokens above the rest, as a language model's rows have them
    n = min(V, 40)
    at = torch.randint(0, V, (R, n), generator=g, device="cuda")
    x.scatter_add_(1, at, 4 + 8 * torch.rand((R, n), generator=g, device="cuda"))
    pick = random.Random(int(seed) * 7 + 1)
    kind = case["filters"]
    if kind == "all":
        rows = [(0.7, 20, 0.8, 0.05)] * R
    elif kind == "none":
        rows = [(1.0, -1, 1.0, 0.0)] * R
    elif kind == "mass":
        rows = [(1.0, -1, 0.95, 0.0)] * R
    else:
        rows = [(pick.choice([0.0, 0.6, 0.8, 1.0, 1.3]), pick.choice([-1, 1, 20, 50, 1000]), pick.choice([1.0, 0.95, 0.9, 0.5]),
                 pick.choice([0.0, 0.0, 0.02, 0.1])) for _ in range(R)]
    temperature, top_k, top_p, min_p = zip(*rows)

    def floats(v):
        return torch.tensor(v, dtype=torch.float32, device="cuda")

    u = torch.rand((R, case["draws"]), generator=g, device="cuda")
    return dict(kind="draw", logits=x.to(DTYPES[case["dtype"]]), uniform=u, temperature=floats(temperature),
                top_k=torch.tensor(top_k, dtype=torch.int32, device="cuda"), top_p=floats(top_p), min_p=floats(min_p),
                out=torch.empty((R, case["draws"]), dtype=torch.int32, device="cuda"), prob=torch.empty_like(u))


def _own_draw(t):
    from somi_inference_b200.ops import cuda_ops
    cuda_ops().draw_tokens(t["logits"], t["uniform"], t["temperature"], t["top_k"], t["top_p"], t["min_p"], t["out"],
                           prob=t["prob"])
    return t["out"], t["prob"]


def _plain_draw(t):
    """Sorted rows, cumulated masses; 64 bits, since a number may lie next to a border of two tokens."""
    x = t["logits"].double()
    V = x.shape[1]
    s, order = torch.sort(x, dim=1, descending=True, stable=True)       # equal values: the lowest index first
    greedy = (t["temperature"] <= 0)[:, None]
    heat = torch.where(greedy, torch.ones_like(s[:, :1]), t["temperature"][:, None].double())
    w = ((s - s[:, :1]) / heat).exp()
    w = torch.where(w < SMALLEST, torch.zeros_like(w), w)
    k = torch.where(t["top_k"] > 0, t["top_k"], torch.full_like(t["top_k"], V))[:, None]
    w = torch.where(torch.arange(V, device=x.device)[None] < k, w, torch.zeros_like(w))
    before = w.cumsum(1) - w
    p = t["top_p"].double()[:, None]
    kept = (before <= p * w.sum(1, keepdim=True)) | (p >= 1)
    w = torch.where(kept & (w >= t["min_p"].double()[:, None]), w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)
    cdf = w.cumsum(1)
    token = torch.searchsorted(cdf, t["uniform"].double() * cdf[:, -1:], right=True)
    last = V - 1 - (w.flip(1) > 0).int().argmax(1, keepdim=True)
    token = torch.minimum(token, last)
    prob = torch.where(greedy, torch.ones_like(t["uniform"]), (w.gather(1, token) / cdf[:, -1:]).float())
    return torch.where(greedy, order[:, :1].expand_as(token), token).int(), prob


def _exact_draw(case, seed):
    """Row by row from the definition: cut-offs by value, ties by index, a walk over the kept tokens."""
    t = prepare(case, seed)
    out, prob = torch.empty(t["uniform"].shape, dtype=torch.int32), torch.ones(t["uniform"].shape, dtype=torch.float64)
    for r in range(case["rows"]):
        x = t["logits"][r].double()
        top = x.max()
        heat, k, p, least = (float(t[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if heat <= 0:
            out[r] = int(torch.nonzero(x == top)[0])
            continue
        ids = torch.arange(len(x), device=x.device)
        if 0 < k < len(x):
            edge = x.topk(int(k)).values[-1]
            above, ties = ids[x > edge], ids[x == edge]
            ids = torch.cat([above, ties[:int(k) - len(above)]]).sort().values
        w = torch.exp((x[ids] - top) / heat)
        w[w < SMALLEST] = 0
        if p < 1:
            rank = torch.argsort(x[ids], descending=True, stable=True)
            mass = torch.cumsum(w[rank], 0)
            keep = rank[:int((mass[:-1] <= p * mass[-1]).sum()) + 1].sort().values
            ids, w = ids[keep], w[keep]
        ids, w = ids[w >= least], w[w >= least]
        cdf = torch.cumsum(w, 0)
        place = torch.searchsorted(cdf, t["uniform"][r].double() * cdf[-1], right=True)
        place = place.clamp(max=int(torch.nonzero(w)[-1]))
        out[r], prob[r] = ids[place].int().cpu(), (w[place] / cdf[-1]).cpu()
    return out, prob


# ------------------------------------------------------------------------------------------------------- both
def exact(case, seed):
    return (_exact_prefix if case["kind"] == "prefix" else _exact_draw)(case, seed)


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] == "draw":
        # the logits once; a row's settings; a number, a token and its probability a draw; an exponential and a sum an element
        return {"bytes": case["rows"] * (case["vocab"] * size + 16 + 12 * case["draws"]), "flops": 2 * case["rows"] * case["vocab"]}
    s = SHAPES[case["shape"]]
    behind, new = _lengths(case)
    keys = case["groups"] * case["prefix"] + sum(b + n for b, n in zip(behind, new))
    pairs = sum(n * (case["prefix"] + b) + n * (n + 1) // 2 for b, n in zip(behind, new))
    return {"bytes": size * s["dim"] * (2 * keys * s["kv_heads"] + 2 * sum(new) * s["heads"]) + 4 * keys // case["page"],
            "flops": 4 * s["heads"] * s["dim"] * pairs}
