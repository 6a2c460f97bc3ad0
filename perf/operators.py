"""The context operators' cases: attention of one new token over a paged key/value cache, eviction from that cache by
accumulated attention weight, and linear attention with a decay per head (prompts and single tokens).

`run` computes a case in plain torch operations (float32, rounded once) where `own` is false, and through
strata_mlx_b200.context where it is true. Sizes: 16 query / 2 key-value heads of 256 at 8K and 128K contexts and
batches of 8 are the synthetic decoder's (decoder.py, bench.py); the rest are generic.
"""

import math
import random

import numpy as np
import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
MAX_LINEAR_TOKENS = 32768 * 16  # tokens x heads of the longest prompt
MAX_CACHE_VALUES = 8 * 131072 * 2 * 256  # keys of the largest cache
CHUNK = 128  # tokens a chunk of the plain linear attention


def listed():
    return [
        # one user's decode step at the decoder's 8K context: a latency case
        {"name": "attend_one_8k", "op": "attend", "batch": 1, "tokens": 8192, "ragged": False, "q_heads": 16,
         "kv_heads": 2, "dim": 256, "page": PAGE, "type": "bf16", "tracked": False},
        # eight users at the decoder's 128K context: the cache's bytes
        {"name": "attend_8x128k", "op": "attend", "batch": 8, "tokens": 131072, "ragged": False, "q_heads": 16,
         "kv_heads": 2, "dim": 256, "page": PAGE, "type": "bf16", "tracked": False},
        # a serving batch of conversations of every length, an empty one among them, their weights accumulated
        {"name": "attend_ragged_tracked", "op": "attend", "batch": 32, "tokens": 9001, "ragged": True, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": PAGE, "type": "f16", "tracked": True},
        # the first tokens of a few short conversations, three query heads a key/value head
        {"name": "attend_short_tracked", "op": "attend", "batch": 4, "tokens": 300, "ragged": True, "q_heads": 12,
         "kv_heads": 4, "dim": 64, "page": PAGE, "type": "bf16", "tracked": True},
        # one conversation a little past its budget: latency
        {"name": "evict_one_2k", "op": "evict", "batch": 1, "tokens": 2304, "ragged": False, "keep": 2048, "sinks": 4,
         "recent": 256, "kv_heads": 2, "dim": 256, "page": PAGE, "type": "bf16"},
        # a serving batch: some sequences within the budget, some far past it
        {"name": "evict_ragged", "op": "evict", "batch": 16, "tokens": 8191, "ragged": True, "keep": 3001, "sinks": 4,
         "recent": 500, "kv_heads": 8, "dim": 128, "page": PAGE, "type": "f16"},
        # long prompts cut to a quarter
        {"name": "evict_8x128k", "op": "evict", "batch": 8, "tokens": 131072, "ragged": False, "keep": 32768,
         "sinks": 4, "recent": 1024, "kv_heads": 2, "dim": 256, "page": PAGE, "type": "bf16"},
        # short prompts, no state yet, small heads
        {"name": "linear_prompt_short", "op": "linear", "batch": 2, "tokens": 77, "ragged": False, "k_heads": 2,
         "v_heads": 4, "k_dim": 64, "v_dim": 64, "stated": False, "type": "bf16"},
        # a batch of prompts of every length behind an earlier state, two value heads a key head
        {"name": "linear_prompt_ragged", "op": "linear", "batch": 6, "tokens": 1535, "ragged": True, "k_heads": 8,
         "v_heads": 16, "k_dim": 128, "v_dim": 128, "stated": True, "type": "bf16"},
        # one long prompt: few heads, a long axis
        {"name": "linear_prompt_long", "op": "linear", "batch": 1, "tokens": 32768, "ragged": False, "k_heads": 16,
         "v_heads": 16, "k_dim": 128, "v_dim": 128, "stated": True, "type": "bf16"},
        # one user's decode step
        {"name": "linear_step_one", "op": "step", "batch": 1, "k_heads": 16, "v_heads": 16, "k_dim": 128, "v_dim": 128,
         "type": "bf16"},
        # a serving batch's decode step: the states' bytes
        {"name": "linear_step_batch", "op": "step", "batch": 64, "k_heads": 8, "v_heads": 32, "k_dim": 128,
         "v_dim": 128, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "evict", "linear", "linear", "step"])
    if op in ("attend", "evict"):
        heads, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 80, 96, 128, 160, 256])
        tokens = _log(rng, 1, 131072)
        most = max(1, MAX_CACHE_VALUES // (2 * tokens * heads * dim))
        c = {"op": op, "batch": _log(rng, 1, min(64, most)), "tokens": tokens, "ragged": rng.random() < 0.7}
        if op == "attend":
            c |= {"q_heads": heads * rng.choice([1, 2, 3, 4, 5, 8, 16]), "kv_heads": heads, "dim": dim,
                  "page": rng.choice([8, 16, 16, 32, 64]), "type": rng.choice(["bf16", "f16"]),
                  "tracked": rng.random() < 0.5}
        else:
            keep = max(1, round(tokens * rng.uniform(0.1, 0.95)))
            sinks = min(keep, rng.choice([0, 1, 4]))
            c |= {"keep": keep, "sinks": sinks, "recent": int((keep - sinks) * rng.uniform(0, 0.5)), "kv_heads": heads,
                  "dim": dim, "page": rng.choice([8, 16, 16, 32, 64]), "type": rng.choice(["bf16", "f16"])}
        return c
    heads, rep = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 3])
    c = {"op": op, "k_heads": heads, "v_heads": heads * rep, "k_dim": rng.choice([32, 64, 72, 96, 128, 128]),
         "v_dim": rng.choice([32, 64, 80, 128, 128])}
    if op == "step":
        return c | {"batch": _log(rng, 1, 2048 // (heads * rep)), "type": rng.choice(["bf16", "f16"])}
    c["tokens"] = _log(rng, 1, 32768)
    most = max(1, MAX_LINEAR_TOKENS // (c["tokens"] * heads * rep))
    return c | {"batch": _log(rng, 1, min(16, most)), "ragged": rng.random() < 0.5, "stated": rng.random() < 0.5,
                "type": "bf16"}


def _lengths(case):
    """The sequences' lengths: a case's own, so that its work is known; ragged ones hold 0, 1 and the longest."""
    n, most = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [most] * n
    r = random.Random(n * 1000003 + most)
    got = [most, 0, 1][:n] + [r.randint(max(1, most // 16), most) for _ in range(n - 3)]
    r.shuffle(got)
    return got


def _gen(seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def _cache(case, seed, dev):
    """A pool of pages, each sequence's pages scattered over it, every slot holding something."""
    g, n, page = _gen(seed, dev), case["batch"], case["page"]
    per = -(-case["tokens"] // page)
    shape = (n * per, page, case["kv_heads"], case["dim"])
    dtype = TYPES[case["type"]]
    s = {"k": torch.randn(shape, generator=g, device=dev, dtype=dtype),
         "v": torch.randn(shape, generator=g, device=dev, dtype=dtype),
         "table": torch.randperm(n * per, generator=g, device=dev).to(torch.int32).reshape(n, per),
         "lengths": torch.tensor(_lengths(case), dtype=torch.int32, device=dev)}
    return s, g, per * page


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    if case["op"] == "attend":
        s, g, slots = _cache(case, seed, dev)
        s["q"] = torch.randn((case["batch"], case["q_heads"], case["dim"]), generator=g, device=dev,
                             dtype=TYPES[case["type"]])
        s["weight"] = None
        if case["tracked"]:  # what the tokens gathered in earlier steps
            s["weight"] = torch.rand((case["batch"], slots), generator=g, device=dev)
        if own:
            from strata_mlx_b200 import context

            s["cache"] = context.KVPages(s["k"], s["v"], s["table"], s["lengths"], weight=s["weight"])
    elif case["op"] == "evict":
        s, g, slots = _cache(case, seed, dev)
        n = case["batch"]
        # a few tokens hold most of the weight; values on a grid, so that some are equal
        w = torch.rand((n, slots), generator=g, device=dev)
        s["weight"] = torch.round(w.pow(-0.5) * 4096) / 4096
        # slots in about the order of their tokens (an eviction fills a hole with a later token)
        at = torch.arange(slots, device=dev) + 64 * torch.rand((n, slots), generator=g, device=dev)
        at = torch.where(torch.arange(slots, device=dev) < s["lengths"][:, None], at, float("inf"))
        s["position"] = at.argsort(-1).argsort(-1).to(torch.int32)
        s["seen"] = s["lengths"].clone()
        s["out"] = (torch.zeros((n, case["keep"]), device=dev), torch.zeros((n, case["keep"]), device=dev,
                                                                          dtype=torch.int32),
                    torch.zeros_like(s["lengths"]))
        if own:
            from strata_mlx_b200 import context

            s["cache"] = context.KVPages(s["k"], s["v"], s["table"], s["lengths"], weight=s["weight"],
                                         position=s["position"])
    else:
        g, dtype = _gen(seed, dev), TYPES[case["type"]]
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        lead = (case["batch"],) if case["op"] == "step" else (case["batch"], case["tokens"])
        s = {"q": torch.randn((*lead, hk, dk), generator=g, device=dev, dtype=dtype),
             "k": (torch.randn((*lead, hk, dk), generator=g, device=dev) * dk ** -0.5).to(dtype),
             "v": torch.randn((*lead, hv, dv), generator=g, device=dev, dtype=dtype)}
        # heads that forget within tokens next to heads that hold thousands, each token with its own step
        rate = -torch.logspace(-3, -0.3, hv, device=dev)
        x = torch.randn((*lead, hv), generator=g, device=dev)
        s["decay"] = rate * torch.log1p(torch.exp(x))
        s["state"] = None
        if case["op"] == "step" or case["stated"]:
            s["state"] = torch.randn((case["batch"], hv, dk, dv), generator=g, device=dev)
        if case["op"] == "linear":
            s["lengths"] = None
            if case["ragged"]:
                s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    s["case"] = case
    return s


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from strata_mlx_b200 import context

    case = s["case"]
    if case["op"] == "attend":
        out = s["cache"].attend(s["q"])
        return {"out": out, "weight": s["weight"]} if case["tracked"] else {"out": out}
    if case["op"] == "evict":
        s["cache"].evict(s["seen"], case["keep"], sinks=case["sinks"], recent=case["recent"], out=s["out"])
        return {"k": s["k"], "v": s["v"], "weight": s["out"][0], "position": s["out"][1], "lengths": s["out"][2]}
    if case["op"] == "step":
        return {"out": context.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"]),
                "state": s["state"]}
    out, state = context.linear_attention(s["q"], s["k"], s["v"], s["decay"], state=s["state"], lengths=s["lengths"])
    return {"out": out, "state": state}


# ---- plain forms


def _rows(s, slots):
    """The pool's row of every slot, (batch, slots)."""
    page = s["k"].shape[1]
    at = torch.arange(slots, device=s["k"].device)
    return s["table"].long()[:, at // page] * page + at % page


def _run_plain(s):
    case = s["case"]
    return {"attend": _attend, "evict": _evict, "linear": _linear, "step": _step}[case["op"]](s)


def _attend(s):
    q, k, v = s["q"], s["k"], s["v"]
    n, hq, d = q.shape
    hk = k.shape[2]
    slots = s["table"].shape[1] * k.shape[1]
    rows = _rows(s, slots)
    valid = torch.arange(slots, device=q.device) < s["lengths"][:, None]
    kf = k.reshape(-1, hk, d)[rows].permute(0, 2, 3, 1).float()  # (n, hk, d, slots)
    qf = q.float().reshape(n, hk, hq // hk, d) * d ** -0.5
    scores = (qf @ kf).masked_fill(~valid[:, None, None], float("-inf"))
    del kf
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    vf = v.reshape(-1, hk, d)[rows].permute(0, 2, 1, 3).float()
    vf.masked_fill_(~valid[:, None, :, None], 0.0)
    out = (p @ vf).reshape(n, hq, d).to(q.dtype)
    if s["weight"] is None:
        return {"out": out}
    s["weight"] += p.sum((1, 2))
    return {"out": out, "weight": s["weight"]}


def _evict(s):
    case, keep = s["case"], s["case"]["keep"]
    w, pos, n = s["weight"], s["position"], s["lengths"][:, None]
    slots = w.shape[1]
    at = torch.arange(slots, device=w.device)
    valid = at < n
    kept_by_place = (pos < case["sinks"]) | (pos >= s["seen"][:, None] - case["recent"])
    rank = torch.where(valid, 1 + (valid & kept_by_place).int(), 0)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    by = torch.sort(rank.gather(1, order), dim=-1, descending=True, stable=True).indices
    order = order.gather(1, by)
    left = torch.minimum(n, torch.full_like(n, keep))
    stays = torch.zeros_like(valid).scatter(1, order, at.expand_as(order) < left)
    src = (stays & (at >= left)).nonzero(as_tuple=True)
    dst = (~stays & (at < left)).nonzero(as_tuple=True)
    rows = _rows(s, slots)
    for pool in (s["k"], s["v"]):
        flat = pool.view(-1, *pool.shape[2:])
        flat[rows[dst]] = flat[rows[src]]
    outs = []
    for a, out in ((w, s["out"][0]), (pos, s["out"][1])):
        moved = a.clone()
        moved[dst] = a[src]
        m = min(keep, slots)
        out[:, :m] = torch.where((at < left)[:, :m], moved[:, :m], out[:, :m])
        outs.append(out)
    s["out"][2].copy_(left[:, 0])
    return {"k": s["k"], "v": s["v"], "weight": outs[0], "position": outs[1], "lengths": s["out"][2]}


def _linear(s):
    q, k, v = s["q"], s["k"], s["v"]
    n, t, hk, dk = q.shape
    hv, dv = v.shape[2:]
    rep, c = hv // hk, min(CHUNK, t)
    m = -(-t // c)

    def chunks(x, per_head=1):  # (n, t, h, ...) -> (n, h * per_head, m, c, ...) float32, zeros past the end
        x = x.float().repeat_interleave(per_head, 2) if per_head > 1 else x.float()
        if s["lengths"] is not None:
            live = torch.arange(t, device=x.device) < s["lengths"][:, None]
            x = x.masked_fill(~live.reshape(n, t, *[1] * (x.dim() - 2)), 0.0)
        pad = torch.zeros((n, m * c - t, *x.shape[2:]), device=x.device)
        return torch.cat([x, pad], 1).unflatten(1, (m, c)).movedim(3, 1)

    qc, kc, vc, g = chunks(q, rep) * dk ** -0.5, chunks(k, rep), chunks(v), chunks(s["decay"])
    since = g.cumsum(-1)  # (n, h, m, c): the decay from a chunk's start
    causal = torch.ones((c, c), dtype=torch.bool, device=q.device).tril()
    gap = (since[..., :, None] - since[..., None, :]).masked_fill(~causal, float("-inf"))
    out = (qc @ kc.transpose(-1, -2) * torch.exp(gap)) @ vc
    added = (kc * torch.exp(since[..., -1:] - since)[..., None]).transpose(-1, -2) @ vc  # (n, h, m, dk, dv)
    first = torch.zeros((n, hv, dk, dv), device=q.device) if s["state"] is None else s["state"]
    parts = torch.cat([first[:, :, None], added], 2).flatten(3)
    # the state before chunk j (and at the end): every earlier chunk's part, decayed over the chunks between
    total = torch.cat([torch.zeros_like(since[..., :1, -1]), since[..., -1].cumsum(-1)], -1)
    before = torch.ones((m + 1, m + 1), dtype=torch.bool, device=q.device).tril()
    states = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~before, float("-inf"))) @ parts
    states = states.unflatten(-1, (dk, dv))
    out = out + torch.exp(since)[..., None] * (qc @ states[:, :, :-1])
    out = out.movedim(1, 3).flatten(1, 2)[:, :t]
    if s["lengths"] is not None:
        live = torch.arange(t, device=q.device) < s["lengths"][:, None]
        out = out.masked_fill(~live[..., None, None], 0.0)
    return {"out": out.to(q.dtype), "state": states[:, :, -1].contiguous()}


def _step(s):
    q, k, v, state = s["q"].float(), s["k"].float(), s["v"].float(), s["state"]
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1) * q.shape[-1] ** -0.5, k.repeat_interleave(rep, 1)
    state *= torch.exp(s["decay"])[..., None, None]
    state += k[..., :, None] * v[..., None, :]
    return {"out": (q[..., None, :] @ state)[..., 0, :].to(s["q"].dtype), "state": state}


# ---- what a pass cannot do without


def work(case):
    if case["op"] in ("linear", "step"):
        hk, hv, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
        n = case["batch"]
        tokens = n if case["op"] == "step" else sum(_lengths(case))
        rows = n if case["op"] == "step" else n * case["tokens"]  # the output's rows, empty ones among them
        states = n * hv * dk * dv * 4
        stated = case["op"] == "step" or case["stated"]
        return {"bytes": tokens * (2 * hk * dk * 2 + hv * dv * 2 + hv * 4) + rows * hv * dv * 2
                + states * (2 if stated else 1), "flops": 4 * tokens * hv * dk * dv}
    tokens, n, page = sum(_lengths(case)), case["batch"], case["page"]
    row = 2 * case["kv_heads"] * case["dim"] * 2  # a token's keys and values
    table = sum(-(-t // page) for t in _lengths(case)) * 4
    if case["op"] == "attend":
        return {"bytes": tokens * row + table + 2 * n * case["q_heads"] * case["dim"] * 2
                + (8 * tokens if case["tracked"] else 0), "flops": 4 * tokens * case["q_heads"] * case["dim"]}
    # every weight and position once; the kept ones written; the kept tokens past the budget moved into holes
    # (how many those are goes by the weights: here, as many as even odds for every token give)
    keep = case["keep"]
    moved = sum((t - keep) * keep / t for t in _lengths(case) if t > keep)
    left = sum(min(t, keep) for t in _lengths(case))
    return {"bytes": 8 * tokens + 8 * left + table + 2 * moved * row, "flops": tokens}


# ---- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "evict": _exact_evict, "linear": _exact_linear, "step": _exact_linear}[
        case["op"]](s)


def _exact_attend(s):
    q, k, v = s["q"].double(), s["k"], s["v"]
    n, hq, d = q.shape
    page, hk = k.shape[1:3]
    out = torch.zeros_like(q)
    weight = None if s["weight"] is None else s["weight"].double()
    for b, length in enumerate(s["lengths"].tolist()):
        if length == 0:
            continue
        pages = s["table"][b, : -(-length // page)].long()
        for h in range(hk):
            keys, values = (x[pages, :, h].reshape(-1, d)[:length].double() for x in (k, v))
            mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
            p = torch.softmax(torch.einsum("qd,td->qt", q[b, mine], keys) / math.sqrt(d), -1)
            out[b, mine] = torch.einsum("qt,td->qd", p, values)
            if weight is not None:
                weight[b, :length] += p.sum(0)
    return {"out": out, "weight": weight} if weight is not None else {"out": out}


def _exact_evict(s):
    case, keep = s["case"], s["case"]["keep"]
    w, pos = s["weight"].cpu().numpy().astype(np.float64), s["position"].cpu().numpy()
    ow, op = np.zeros((len(w), keep)), np.zeros((len(w), keep), dtype=np.int32)
    lengths = s["lengths"].cpu().numpy().copy()
    for b, n in enumerate(lengths.tolist()):
        m = min(n, keep)
        a, p = w[b, :n], pos[b, :n]
        safe = (p < case["sinks"]) | (p >= n - case["recent"])
        stays = np.zeros(n, dtype=bool)
        stays[np.lexsort((np.arange(n), -a, ~safe))[:m]] = True
        take = np.arange(m)
        take[~stays[:m]] = m + np.flatnonzero(stays[m:])
        ow[b, :m], op[b, :m], lengths[b] = a[take], p[take], m
    return {"k": None, "v": None, "weight": ow, "position": op, "lengths": lengths}


def _exact_linear(s):
    """S = exp(g) S + k v^T, o = q S, token by token."""
    q, k, v, g = (s[x].double() for x in ("q", "k", "v", "decay"))
    if s["case"]["op"] == "step":
        q, k, v, g = (x[:, None] for x in (q, k, v, g))
    n, t, hk, dk = q.shape
    hv, dv = v.shape[2:]
    head = torch.arange(hv, device=q.device) // (hv // hk)
    S = torch.zeros((n, hv, dk, dv), device=q.device, dtype=torch.float64) if s["state"] is None else s["state"].double()
    out = torch.zeros((n, t, hv, dv), device=q.device, dtype=torch.float64)
    live = None
    if s.get("lengths") is not None:
        live = torch.arange(t, device=q.device) < s["lengths"][:, None]
    a = torch.exp(g)
    for i in range(t):
        new = torch.addcmul(S * a[:, i, :, None, None], k[:, i, head, :, None], v[:, i, :, None, :])
        o = torch.einsum("nhk,nhkv->nhv", q[:, i, head], new) / math.sqrt(dk)
        if live is None:
            S, out[:, i] = new, o
        else:
            alive = live[:, i, None, None]
            S, out[:, i] = torch.where(alive[..., None], new, S), torch.where(alive, o, 0.0)
    return {"out": out[:, 0] if s["case"]["op"] == "step" else out, "state": S}
