"""The serving operators of a ragged batch, case by case: the page tables of its requests, the rotary positions written
with K and V into the paged cache, and the attention of a batch that shares a long prefix.

Where `own` is false `run` computes them in elementary torch operations in 32 bits; where it is true it calls
edgeexpert_b200.paged, as a serving loop does."""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases ----
def _pages(name, requests, page, old, grow, finish, idle, spare=64):
    return {"name": name, "op": "pages", "requests": requests, "page": page, "old_min": old[0], "old_max": old[1],
            "grow_min": grow[0], "grow_max": grow[1], "finish": finish, "idle": idle, "spare": spare}


def _rope(name, tokens, heads, kv_heads, dim, rot, layout, scaling, norm, dtype, fused, page, longest, padding):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "layout": layout, "scaling": scaling, "norm": norm, "dtype": dtype, "fused": fused, "page": page,
            "longest": longest, "padding": padding}


def _attention(name, requests, prefix, history, query, heads, kv_heads, dim, dtype, page, window):
    return {"name": name, "op": "attention", "requests": requests, "prefix": prefix, "history_min": history[0],
            "history_max": history[1], "query_min": query[0], "query_max": query[1], "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "window": window}


def listed():
    return [
        # a decode step of the batch-32 decoder: every request one token longer, now and then a page
        _pages("pages-decode-32", 32, 16, (1, 2048), (1, 1), 0, 0),
        # a busy server's step: most requests one token (some drafts of up to 4) longer, some finish, some wait
        _pages("pages-step-1000", 1000, 32, (0, 4000), (1, 4), 60, 41),
        # admission: hundreds of prompts of up to 4096 tokens at once, the finished ones' pages handed back
        _pages("pages-admit-512", 512, 16, (0, 100), (1, 4000), 37, 5),
        # the decoder's own layer at batch 1: 16 query and 8 KV heads of 256 with their norms
        _rope("rope-token-1", 1, 16, 8, 256, 256, "half", "none", True, "fp16", False, 16, 4096, 0),
        # the same at the batch-256 decode step, a few rows of it padding
        _rope("rope-decode-256", 256, 16, 8, 256, 256, "half", "none", True, "fp16", False, 16, 4096, 3),
        # a long-context prompt: half of each head rotated, interleaved, frequencies ramped, out of one fused projection
        _rope("rope-prompt-8191", 8191, 16, 8, 256, 128, "interleaved", "ramp", False, "bf16", True, 32, 131072, 0),
        # two users behind a short system prompt: latency
        _attention("attention-2", 2, 317, (0, 40), (1, 1), 16, 8, 256, "fp16", 16, 0),
        # the batch-32 decode step, half of its 4096 positions shared
        _attention("attention-decode-32", 32, 2048, (1, 2047), (1, 1), 16, 8, 256, "fp16", 16, 0),
        # another head layout, an odd batch
        _attention("attention-decode-101", 101, 1500, (0, 900), (1, 1), 16, 4, 128, "bf16", 32, 0),
        # the batch-256 decode step behind a full-length shared prompt
        _attention("attention-decode-256", 256, 4096, (1, 1000), (1, 1), 16, 8, 256, "fp16", 64, 0),
        # drafts of 1 to 5 tokens checked at once; eight query heads to a KV head, sliding window over both parts
        _attention("attention-drafts-61", 61, 3001, (3, 700), (1, 5), 16, 2, 64, "bf16", 16, 1024),
        # the users' own prompts, prefilled together behind the shared one
        _attention("attention-prompts-24", 24, 2050, (0, 100), (1, 300), 16, 8, 256, "fp16", 32, 0),
    ]


def draw(rng):
    def spread(lo, hi):  # evenly over the logarithm
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["pages", "rope", "attention", "attention"])
    if op == "pages":
        requests = spread(1, 1000)
        grow = min(spread(1, 4000), 1000000 // requests)
        c = _pages("", requests, rng.choice([4, 8, 16, 17, 32, 64, 128]),
                   (rng.randint(0, 5), min(spread(10, 4000), 500000 // requests)), (1, grow), requests // rng.randint(3, 40), requests // rng.randint(3, 40))
    elif op == "rope":
        tokens = spread(1, 8191)
        heads, kv_heads, dim = rng.choice([(16, 8, 256), (16, 4, 128), (16, 2, 64), (8, 1, 128), (12, 4, 256), (4, 4, 80)])
        rot = rng.choice([dim, dim // 2, dim // 4 * 2 - 4 if dim == 80 else dim // 4])
        c = _rope("", tokens, heads, kv_heads, dim, rot, rng.choice(["half", "interleaved"]),
                  rng.choice(["none", "linear", "base", "ramp", "bands"]), rng.random() < 0.5,
                  rng.choice(["fp16", "bf16"]), rng.random() < 0.5, rng.choice([1, 16, 24, 64]), spread(64, 131072),
                  rng.randint(0, tokens // 8))
    else:
        heads, kv_heads, dim = rng.choice([(16, 8, 256), (16, 4, 128), (16, 2, 64), (8, 1, 128), (12, 4, 256), (4, 4, 80)])
        if rng.random() < 0.25:  # prompts
            requests, query, history = spread(1, 24), (1, spread(6, 300)), (0, spread(1, 100))
        else:
            requests, query = spread(2, 256), (1, rng.choice([1, 1, 1, 5]))
            history = (rng.randint(0, 3), spread(4, 1000))
        prefix = spread(16, 2050 if query[1] > 5 else 4096) - rng.choice([0, 0, 1, 7])
        c = _attention("", requests, prefix, history, query, heads, kv_heads, dim,
                       rng.choice(["fp16", "bf16"]), rng.choice([8, 16, 24, 32, 64, 128]), rng.choice([0, 0, 0, 512, 1024]))
    del c["name"]
    return c


def _spaced(lo, hi, n):
    """n whole numbers from lo to hi, evenly: the same ones for every seed, which only deals them out."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _ceil(a, b):
    return -(-a // b)


def work(c):
    if c["op"] == "pages":
        live = c["requests"] - c["finish"] - c["idle"]
        old, grow = (c["old_min"] + c["old_max"]) / 2, (c["grow_min"] + c["grow_max"]) / 2
        tokens = c["requests"] * grow + c["spare"]
        moved = (live * grow + c["finish"] * old) / c["page"]  # pages handed out or back: read once, written once
        return {"bytes": c["requests"] * 16 + 12 * tokens + 8 * moved + 32, "flops": 0}
    if c["op"] == "rope":
        row = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        flops = c["tokens"] * ((c["heads"] + c["kv_heads"]) * c["rot"] * 3 + (row * 4 if c["norm"] else 0))
        return {"bytes": c["tokens"] * (row * 4 + 8) + c["rot"] * 4, "flops": flops}
    B, P, W = c["requests"], c["prefix"], c["window"] or 1 << 40
    hist, query = _spaced(c["history_min"], c["history_max"], B), _spaced(c["query_min"], c["query_max"], B)
    n = sum(query) / B
    own_kv = sum(min(h + n, n + W - 1) for h in hist)
    shared = max(0, min(P, W - 1 - min(hist)))
    seen = sum(n * min(W, P + h + (n + 1) / 2) for h in hist)
    tokens = sum(query)
    nbytes = (own_kv + shared) * c["kv_heads"] * c["dim"] * 4 + tokens * c["heads"] * (c["dim"] * 4 + 4)
    nbytes += (own_kv + shared) / c["page"] * 4 + 8 * B
    return {"bytes": nbytes, "flops": 4 * c["dim"] * c["heads"] * seen}


# --------------------------------------------------------------- inputs ----
def prepare(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    host = torch.Generator().manual_seed(seed * 104729 + 5)
    return {"pages": _prepare_pages, "rope": _prepare_rope, "attention": _prepare_attention}[c["op"]](c, gen, host)


def _dealt(lo, hi, n, host):
    return torch.tensor(_spaced(lo, hi, n))[torch.randperm(n, generator=host)]


def _i32(t):
    return t.to(device="cuda", dtype=torch.int32)


def _prepare_pages(c, gen, host):
    B, ps = c["requests"], c["page"]
    old = _dealt(c["old_min"], c["old_max"], B, host)
    target = old + _dealt(c["grow_min"], c["grow_max"], B, host)
    order = torch.randperm(B, generator=host)
    target[order[:c["finish"]]] = 0
    target[order[c["finish"]:c["finish"] + c["idle"]]] = -1
    max_pages = _ceil(c["old_max"] + c["grow_max"], ps)
    held = (old + ps - 1) // ps
    used = int(held.sum())
    grow = _spaced(c["grow_min"], c["grow_max"], B)
    N = sum(_ceil(n, ps) for n in _spaced(c["old_min"], c["old_max"], B)) + sum(n // ps + 1 for n in grow) + 16
    ids = torch.randperm(N, generator=host).to(torch.int32)
    table = torch.full((B, max_pages), -1, dtype=torch.int32)
    inside = torch.arange(max_pages)[None, :] < held[:, None]
    table[inside] = ids[:used]
    head = int(torch.randint(0, N, (1,), generator=host))
    ring = torch.full((N,), -1, dtype=torch.int32)
    ring[(head + torch.arange(N - used)) % N] = ids[used:]
    tokens = sum(grow) + c["spare"]
    s = dict(op="pages", page=ps, tokens=tokens, base=c["page"] * 7 + 3, lens=_i32(old), targets=_i32(target),
             table=table.cuda(), ring=ring.cuda(), state=_i32(torch.tensor([head, N - used, 0, 0])),
             new_lens=_i32(torch.zeros(B)), new_state=_i32(torch.zeros(4)), starts=_i32(torch.zeros(B + 1)),
             slots=_i32(torch.zeros(tokens)), positions=_i32(torch.zeros(tokens)), requests=_i32(torch.zeros(tokens)))
    if own:
        from edgeexpert_b200.paged import KVPages
        s["handle"] = KVPages()
        s["workspace"] = torch.empty(s["handle"].workspace_bytes(B), dtype=torch.uint8, device="cuda")
    return s


SCALINGS = {
    "none": {},
    "linear": {"scaling": "linear", "factor": 4.0},
    "base": {"scaling": "base", "factor": 8.0},
    "ramp": {"scaling": "ramp", "factor": 16.0, "original_context": 8192, "beta_fast": 32.0, "beta_slow": 1.0},
    "bands": {"scaling": "bands", "factor": 8.0, "original_context": 8192, "low_factor": 1.0, "high_factor": 4.0},
}
THETA = 10000.0


def _frequencies(rot, scaling):
    """Radians per position of each pair, in 64 bits, and what cos and sin are multiplied by."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    p = SCALINGS[scaling]
    if scaling == "base":
        return (THETA * p["factor"] ** (rot / (rot - 2))) ** (-i / rot), 1.0
    f = THETA ** (-i / rot)
    if scaling == "linear":
        return f / p["factor"], 1.0
    if scaling == "ramp":  # pairs with fewer turns over the original context than beta_slow are slowed, over beta_fast kept
        def pair(turns):
            return rot * math.log(p["original_context"] / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(math.floor(pair(p["beta_fast"])), 0), min(math.ceil(pair(p["beta_slow"])), rot - 1)
        slow = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f / p["factor"] * slow + f * (1 - slow), 0.1 * math.log(p["factor"]) + 1.0
    if scaling == "bands":  # by wavelength against the original context
        turns = p["original_context"] * f / (2 * math.pi)
        keep = ((turns - p["low_factor"]) / (p["high_factor"] - p["low_factor"])).clamp(0, 1)
        return f / p["factor"] * (1 - keep) + f * keep, 1.0
    return f, 1.0


def _prepare_rope(c, gen, host):
    T, nq, nkv, hd, ps, dt = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"], DTYPES[c["dtype"]]

    def normal(*shape):
        return (torch.randn(*shape, generator=gen, device="cuda") * 2).to(dt)

    if c["fused"]:  # one projection's rows: q, k and v side by side
        qkv = normal(T, (nq + 2 * nkv) * hd)
        q, k, v = (x.view(T, -1, hd) for x in qkv.split([nq * hd, nkv * hd, nkv * hd], 1))
    else:
        q, k, v = normal(T, nq, hd), normal(T, nkv, hd), normal(T, nkv, hd)
    pages = _ceil(T, ps) + 8
    slots = torch.randperm(pages * ps, generator=host)[:T]
    positions = torch.randint(0, c["longest"], (T,), generator=host)
    if c["padding"]:
        slots[T - c["padding"]:] = -1
        positions[T - c["padding"]:] = -1
    freq, factor = _frequencies(c["rot"], c["scaling"])
    s = dict(op="rope", rot=c["rot"], layout=c["layout"], factor=factor, q=q, k=k, v=v, slots=_i32(slots),
             positions=_i32(positions), freq=freq.cuda(), q_out=torch.zeros(T, nq, hd, dtype=dt, device="cuda"),
             k_cache=torch.zeros(pages, ps, nkv, hd, dtype=dt, device="cuda"),
             v_cache=torch.zeros(pages, ps, nkv, hd, dtype=dt, device="cuda"), q_weight=None, k_weight=None)
    if c["norm"]:
        s["q_weight"], s["k_weight"] = ((1 + 0.1 * torch.randn(hd, generator=gen, device="cuda")).to(torch.bfloat16)
                                        for _ in range(2))
    if own:
        from edgeexpert_b200.paged import PagedKV, RotaryKVWrite
        s["handle"], s["kv"] = RotaryKVWrite(), PagedKV(s["k_cache"], s["v_cache"])
    return s


def _prepare_attention(c, gen, host):
    B, P, ps, dt = c["requests"], c["prefix"], c["page"], DTYPES[c["dtype"]]
    nq, nkv, hd = c["heads"], c["kv_heads"], c["dim"]
    query = _dealt(c["query_min"], c["query_max"], B, host)
    lens = _dealt(c["history_min"], c["history_max"], B, host) + query
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), query.cumsum(0)])
    longest = c["history_max"] + c["query_max"]
    max_pages, shared, held = _ceil(longest, ps), _ceil(P, ps), (lens + ps - 1) // ps
    total = shared + int(held.sum())
    ids = torch.randperm(total + 8, generator=host).to(torch.int32)  # pages lie anywhere
    table = torch.full((B, max_pages), -1, dtype=torch.int32)
    table[torch.arange(max_pages)[None, :] < held[:, None]] = ids[shared:total]
    T = int(starts[-1])

    def normal(std, *shape):
        x = torch.empty(*shape, dtype=dt, device="cuda")
        return x.normal_(0, std, generator=gen)

    s = dict(op="attention", prefix=P, window=c["window"], max_query=c["query_max"], longest=longest,
             scale=hd ** -0.5, q=normal(1.5, T, nq, hd), k=normal(1.0, total + 8, ps, nkv, hd),
             v=normal(1.0, total + 8, ps, nkv, hd), table=table.cuda(), prefix_pages=ids[:shared].cuda(),
             lens=_i32(lens), starts=_i32(starts), out=torch.zeros(T, nq, hd, dtype=dt, device="cuda"),
             lse=torch.zeros(T, nq, device="cuda"))
    if own:
        from edgeexpert_b200.paged import PagedKV, SharedPrefixAttention
        s["handle"], s["kv"] = SharedPrefixAttention(), PagedKV(s["k"], s["v"])
        s["workspace"] = torch.empty(s["handle"].workspace_bytes(s["kv"], nq, T, B, P, c["query_max"]), dtype=torch.uint8,
                                     device="cuda")
    return s


# ------------------------------------------------------------------ run ----
def run(s):
    if own:
        return {"pages": _own_pages, "rope": _own_rope, "attention": _own_attention}[s["op"]](s)
    return {"pages": _plain_pages, "rope": _plain_rope, "attention": _plain_attention}[s["op"]](s)


def _answer_pages(s):
    return {k: s[k] for k in ("new_lens", "table", "ring", "new_state", "starts", "slots", "positions", "requests")}


def _own_pages(s):
    s["handle"].encode_resize(s["lens"], s["targets"], s["table"], s["ring"], s["state"], s["new_lens"], s["new_state"],
                              s["starts"], s["slots"], s["positions"], s["requests"], s["page"], s["workspace"],
                              position_base=s["base"])
    return _answer_pages(s)


def _plain_pages(s):
    ps, table, ring, B, cap = s["page"], s["table"], s["ring"], s["lens"].numel(), s["tokens"]
    N, width = ring.numel(), table.shape[1]
    old, target = s["lens"].long(), s["targets"].long()
    head, free = s["state"][0].long(), s["state"][1].long()
    valid = (target >= 0) & (target <= width * ps)
    grow, shrink = valid & (target > old), valid & (target < old)
    have, want = (old + ps - 1) // ps, (target + ps - 1) // ps
    need = torch.where(grow, want - have, 0)
    taken = need.cumsum(0)
    paged = grow & ((need == 0) | (taken <= free))
    added = torch.where(paged, target - old, 0).cumsum(0)
    granted = paged & (added <= cap)
    grown = torch.where(granted, target - old, 0).cumsum(0)
    starts = torch.cat([torch.zeros_like(grown[:1]), grown])
    given = torch.where(granted, need, 0).sum()
    back = torch.where(shrink, have - want, 0)
    page = torch.arange(width, device=table.device)[None, :]
    gets = granted[:, None] & (page >= have[:, None]) & (page < want[:, None])
    leaves = shrink[:, None] & (page >= want[:, None]) & (page < have[:, None])
    to = (head + free + (back.cumsum(0) - back)[:, None] + page - want[:, None]) % N
    padded = torch.cat([ring, ring[:1]])  # one more place, for what is not handed back
    padded[torch.where(leaves, to, N)] = table
    source = (head + (taken - need)[:, None] + page - have[:, None]) % N
    table.copy_(torch.where(gets, ring[source], table))
    ring.copy_(padded[:N])
    s["new_lens"].copy_(torch.where(granted | shrink, target, old))
    s["new_state"].copy_(torch.stack([(head + given) % N, free - given + back.sum(),
                                      ((target > old) & ~granted).sum(), grown[-1]]))
    s["starts"].copy_(starts)
    token = torch.arange(cap, device=table.device)
    request = torch.searchsorted(grown, token, right=True).clamp(max=B - 1)
    at = old[request] + token - starts[request]
    live = token < grown[-1]
    s["slots"].copy_(torch.where(live, table[request, (at // ps).clamp(max=width - 1)] * ps + at % ps, -1))
    s["positions"].copy_(torch.where(live, at + s["base"], -1))
    s["requests"].copy_(torch.where(live, request, -1))
    return _answer_pages(s)


def _own_rope(s):
    s["handle"].encode(s["q"], s["k"], s["v"], s["q_out"], s["kv"], s["slots"], s["positions"], s["freq"],
                       rotary_dim=s["rot"], layout=s["layout"], attention_factor=s["factor"], q_weight=s["q_weight"],
                       k_weight=s["k_weight"], norm=s["q_weight"] is not None)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _normed(x, weight, eps=1e-6):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.float()


def _rotated(x, cos, sin, layout):
    half = cos.shape[-1]
    a, b = (x[..., :half], x[..., half:2 * half]) if layout == "half" else (x[..., 0:2 * half:2], x[..., 1:2 * half:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([u, w], -1) if layout == "half" else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _plain_rope(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["q_weight"] is not None:
        q, k, v = _normed(q, s["q_weight"]), _normed(k, s["k_weight"]), _normed(v, None)
    # 131072 positions of up to a radian each leave 32 bits no digits of a turn: the angles alone are formed in 64
    angle = (s["positions"].double()[:, None] * s["freq"]).remainder(2 * math.pi).float()[:, None, :]
    cos, sin = angle.cos() * s["factor"], angle.sin() * s["factor"]
    live = s["slots"] >= 0
    s["q_out"].copy_(torch.where(live[:, None, None], _rotated(q, cos, sin, s["layout"]), 0))
    for cache, x in ((s["k_cache"], _rotated(k, cos, sin, s["layout"])), (s["v_cache"], v)):
        cache.flatten(0, 1)[s["slots"][live].long()] = x[live].to(cache.dtype)
    return s["q_out"], s["k_cache"], s["v_cache"]


def _own_attention(s):
    s["handle"].encode(s["q"], s["kv"], s["table"], s["lens"], s["starts"], s["out"], s["workspace"],
                       prefix_pages=s["prefix_pages"], prefix_len=s["prefix"], max_query=s["max_query"], scale=s["scale"],
                       window=s["window"], lse=s["lse"])
    return s["out"], s["lse"]


def _plain_attention(s):
    q, P, (T, nq, hd) = s["q"].float(), s["prefix"], s["q"].shape
    nkv, B, n = s["k"].shape[2], s["lens"].numel(), s["max_query"]
    start, count = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    j = torch.arange(n, device=q.device)
    rows = q[(start[:, None] + j).clamp(max=T - 1)].view(B, n, nkv, nq // nkv, hd)
    at = (P + s["lens"].long() - count)[:, None] + j  # [B][n]: the position of each query token
    table = s["table"].clamp(min=0).long()

    def shared(x):
        return x[s["prefix_pages"].long()].flatten(0, 1)[:P].float()

    def mine(x):
        return x[table].flatten(1, 2)[:, :s["longest"]].float()

    scores = torch.cat([torch.einsum("bnkgd,pkd->bkgnp", rows, shared(s["k"])),
                        torch.einsum("bnkgd,bpkd->bkgnp", rows, mine(s["k"]))], -1) * s["scale"]
    key = torch.arange(P + s["longest"], device=q.device)
    seen = key <= at[:, :, None]
    if s["window"]:
        seen &= key > at[:, :, None] - s["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    # what the masks leave out has weight 0, and lies in pages that other requests have written
    out = torch.einsum("bkgnp,pkd->bnkgd", scores[..., :P], shared(s["v"]))
    out += torch.einsum("bkgnp,bpkd->bnkgd", scores[..., P:], mine(s["v"]))
    out = (out / total.permute(0, 3, 1, 2, 4)).reshape(B, n, nq, hd)
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(B, n, nq)
    token = torch.arange(T, device=q.device)
    request = torch.searchsorted(s["starts"][1:].long(), token, right=True)
    s["out"].copy_(out[request, token - start[request]])
    s["lse"].copy_(lse[request, token - start[request]])
    return s["out"], s["lse"]


# ---------------------------------------------------------------- exact ----
def exact(c, seed):
    """The answers from the definitions, in 64 bits, a request or a head at a time."""
    if c["op"] == "pages":
        return None  # whole numbers
    s = prepare(c, seed)
    return _exact_rope(s, c) if c["op"] == "rope" else _exact_attention(s)


def _exact_rope(s, c):
    half = s["rot"] // 2
    live = s["slots"] >= 0
    phase = torch.polar(torch.full_like(s["freq"], s["factor"]).expand(live.numel(), half).contiguous(),
                        s["positions"].double()[:, None] * s["freq"][None, :])

    def turn(x):
        x = x.clone()
        i = torch.arange(half, device=x.device)
        a, b = (i, i + half) if s["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(x[:, :, a], x[:, :, b]) * phase[:, None, :]
        x[:, :, a], x[:, :, b] = z.real, z.imag
        return x

    def norm(x, w):
        x = x.double()
        if not c["norm"]:
            return x
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt()
        return x if w is None else x * w.double()

    q = turn(norm(s["q"], s["q_weight"]))
    q[~live] = 0
    caches = []
    for cache, x in ((s["k_cache"], turn(norm(s["k"], s["k_weight"]))), (s["v_cache"], norm(s["v"], None))):
        flat = cache.double().flatten(0, 1)
        flat[s["slots"][live].long()] = x[live]
        caches.append(flat.view(cache.shape))
    return q, caches[0], caches[1]


def _exact_attention(s):
    T, nq, hd = s["q"].shape
    nkv, P = s["k"].shape[2], s["prefix"]
    out = torch.zeros(T, nq, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(T, nq, dtype=torch.float64, device="cuda")
    shared = [x[s["prefix_pages"].long()].reshape(-1, nkv, hd)[:P].double() for x in (s["k"], s["v"])]
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    ps = s["k"].shape[1]
    for b, length in enumerate(lens):
        t0, t1 = starts[b], starts[b + 1]
        pages = s["table"][b, :_ceil(length, ps)].long()
        k, v = (torch.cat([both, x[pages].reshape(-1, nkv, hd)[:length].double()])
                for both, x in zip(shared, (s["k"], s["v"])))
        at = torch.arange(P + length - (t1 - t0), P + length, device="cuda")
        key = torch.arange(P + length, device="cuda")
        hidden = key[None, :] > at[:, None]
        if s["window"]:
            hidden |= key[None, :] <= at[:, None] - s["window"]
        for h in range(nkv):
            g = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            z = torch.matmul(s["q"][t0:t1, g].double().transpose(0, 1), k[:, h].T) * s["scale"]
            z = z.masked_fill(hidden[None], -math.inf)
            lse[t0:t1, g] = torch.logsumexp(z, -1).T
            out[t0:t1, g] = torch.matmul(torch.softmax(z, -1), v[:, h]).transpose(0, 1)
    return out, lse
