"""The operators of a serving step of many sequences, for timing: low-rank adapters beside a shared projection, attention of the newest tokens over caches of keys and values, eviction from
such caches by accumulated attention weight, and sampling.  Each case is one call (or the calls that belong together) as a serving loop makes it; `own` picks this framework's kernels, else the
same operator in elementary torch operations."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the smallest call: one token of one sequence, the smallest model's heads, float32 as the framework's own cache
        {"name": "attn-token-f32", "op": "attn", "type": "f32", "seqs": 1, "heads": 14, "kv_heads": 2, "dim": 64, "slots": 4096, "shortest": 101, "longest": 101, "new": 1, "mask": "causal", "weights": False},
        # a decode step of 32 conversations of very different lengths whose cache will be evicted from: the 8B shape
        {"name": "attn-batch-bf16", "op": "attn", "type": "bf16", "seqs": 32, "heads": 32, "kv_heads": 8, "dim": 128, "slots": 8192, "shortest": 17, "longest": 8191, "new": 1, "mask": "causal", "weights": True},
        # a speculative step: four sequences verify a tree of up to 24 drafted tokens each
        {"name": "attn-tree-f16", "op": "attn", "type": "f16", "seqs": 4, "heads": 32, "kv_heads": 8, "dim": 128, "slots": 4096, "shortest": 1801, "longest": 4001, "new": 24, "mask": "tree", "weights": True},
        # a portion of a long prompt behind what is cached, with the weights that the eviction behind it goes by
        {"name": "attn-portion-bf16", "op": "attn", "type": "bf16", "seqs": 1, "heads": 32, "kv_heads": 8, "dim": 128, "slots": 4096, "shortest": 2047, "longest": 2047, "new": 2048, "mask": "causal", "weights": True},
        # every step: one token more than the cache is to hold, eight sequences
        {"name": "evict-step-f16", "op": "evict", "type": "f16", "seqs": 8, "kv_heads": 8, "dim": 128, "slots": 2064, "shortest": 2049, "longest": 2049, "keep": 2048, "recent": 512, "first": 4},
        # behind long prompts: down to the bound at once
        {"name": "evict-prompt-bf16", "op": "evict", "type": "bf16", "seqs": 16, "kv_heads": 8, "dim": 128, "slots": 16384, "shortest": 2100, "longest": 16384, "keep": 2048, "recent": 512, "first": 4},
        # one conversation, the sampler's usual settings
        {"name": "sample-one", "op": "sample", "type": "f32", "rows": 1, "n": 128256, "mix": "usual"},
        # a batch whose requests bring settings of their own, some without any filter
        {"name": "sample-batch", "op": "sample", "type": "f32", "rows": 256, "n": 128256, "mix": "any"},
        # logits as a 16-bit head leaves them (many equal ones), the largest vocabulary, no count limit
        {"name": "sample-bf16", "op": "sample", "type": "bf16", "rows": 33, "n": 151936, "mix": "nucleus"},
        # a decode step of few requests: latency
        {"name": "adapt-few", "op": "adapt", "type": "f32", "tokens": 4, "k": 2048, "n": 2048, "adapters": 3, "rank": 16, "runs": 1},
        # a decode step of many requests with adapters of many ranks, beside a feed-forward's projection
        {"name": "adapt-batch", "op": "adapt", "type": "bf16", "tokens": 253, "k": 4096, "n": 14336, "adapters": 64, "rank": 64, "runs": 1},
        # prompts of four requests
        {"name": "adapt-portion", "op": "adapt", "type": "bf16", "tokens": 2048, "k": 4096, "n": 4096, "adapters": 4, "rank": 16, "runs": 512},
    ]


def draw(rng):
    def spread(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["attn", "attn", "evict", "sample", "adapt"])
    if op == "sample":
        rows = spread(1, 256)
        return {"op": op, "type": rng.choice(["f32", "f32", "bf16", "f16"]), "rows": rows, "n": spread(50, 151936) if rows < 128 else spread(50, 128256), "mix": rng.choice(["usual", "any", "nucleus"])}
    if op == "adapt":
        tokens = spread(1, 2048)
        return {"op": op, "type": rng.choice(["f32", "bf16"]), "tokens": tokens, "k": spread(256, 4096), "n": spread(256, 4096 if tokens > 256 else 14336), "adapters": spread(1, 64),
                "rank": rng.choice([4, 8, 16, 32, 64]) if tokens <= 256 else rng.choice([4, 8, 16]), "runs": spread(1, 64) if tokens <= 256 else spread(16, 512)}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (32, 8, 64), (32, 8, 128)])
    if op == "evict":
        seqs, keep = spread(1, 16), spread(64, 4096)
        longest = keep + spread(1, 8192)
        return {"op": op, "type": rng.choice(["f32", "f16", "bf16"]), "seqs": seqs, "kv_heads": kv_heads, "dim": dim, "slots": longest + rng.randint(0, 64), "shortest": max(1, keep - rng.randint(0, keep)),
                "longest": longest, "keep": keep, "recent": keep // rng.randint(2, 5), "first": rng.randint(0, 8)}
    mask = rng.choice(["causal", "causal", "tree"])
    new = 1 if mask == "causal" and rng.random() < 0.5 else rng.randint(2, 40) if mask == "tree" else spread(2, 1024)
    kind = rng.choice(["f32", "f16", "bf16", "bf16"])
    seqs = spread(1, 24) if new <= 40 else 1
    longest = spread(9, 6000 if new <= 40 else 3000)
    return {"op": op, "type": kind, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "slots": longest + new + rng.randint(0, 100), "shortest": rng.randint(0, longest), "longest": longest, "new": new,
            "mask": mask, "weights": rng.random() < 0.6}


def _lengths(case):
    """Slots held by each sequence: from the shortest to the longest, evenly over the logarithm, neighbours in the batch not neighbours in length."""
    n, a, b = case["seqs"], case["shortest"] + 1, case["longest"] + 1
    got = [int(round(a * (b / a) ** (i / max(1, n - 1)))) - 1 for i in range(n)]
    got = got if n > 1 else [case["longest"]]
    return [got[(i * 5) % n] for i in range(n)] if n % 5 else got


def _counts(case):
    """New tokens of each sequence: a tree's size differs from sequence to sequence."""
    return [max(1, case["new"] - (3 * i) % case["new"] if case["mask"] == "tree" else case["new"]) for i in range(case["seqs"])]


def _ranks(case):
    return [max(1, case["rank"] >> (i % 3)) for i in range(case["adapters"])]


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------------------------- inputs
def _prepare_attn(c, g):
    t, S, G, D, T, N = TYPES[c["type"]], c["seqs"], c["kv_heads"], c["dim"], c["new"], c["slots"]
    s = {"c": c, "n_kv": _int32(_lengths(c)), "count": _int32(_counts(c)), "tree": None}
    s["q"], s["k_new"], s["v_new"] = 1.5 * _normal(g, (S, T, c["heads"], D)), _normal(g, (S, T, G, D), t), _normal(g, (S, T, G, D), t)
    s["q"] = s["q"].to(t)
    s["k"], s["v"] = (torch.stack([_normal(g, (N, G, D), t) for _ in range(S)]) for _ in range(2))
    s["out"] = torch.zeros((S, T, c["heads"], D), dtype=t, device="cuda")
    if c["mask"] == "tree":  # every token sees itself and its ancestors; the parent is a token before it
        parent = (torch.rand((S, T), generator=g, device="cuda") * torch.arange(T, device="cuda")).long()
        see = torch.eye(T, dtype=torch.bool, device="cuda").repeat(S, 1, 1)
        for i in range(1, T):
            see[:, i] |= see[torch.arange(S, device="cuda"), parent[:, i]]
        s["tree"] = see.to(torch.uint8).contiguous()
    s["weight"] = torch.rand((S, G, N), generator=g, device="cuda") * 4 if c["weights"] else None
    s["weight_out"] = torch.zeros((S, G, N), device="cuda") if c["weights"] else None
    return s


def _prepare_evict(c, g):
    t, S, G, D, N = TYPES[c["type"]], c["seqs"], c["kv_heads"], c["dim"], c["slots"]
    s = {"c": c, "n_kv": _int32(_lengths(c)), "n_kv_out": torch.zeros(S, dtype=torch.int32, device="cuda")}
    s["k"], s["v"] = (torch.stack([_normal(g, (N, G, D), t) for _ in range(S)]) for _ in range(2))
    # positions as they are behind earlier evictions: in no order; weights with few large ones and many zeros, as a soft-max leaves them
    s["pos"] = torch.argsort(torch.rand((S, G, N), generator=g, device="cuda"), -1).to(torch.int32)
    s["weight"] = torch.clamp(torch.exp(2.0 * _normal(g, (S, G, N))) - 0.3, min=0)
    s["weight_out"], s["pos_out"] = torch.zeros_like(s["weight"]), torch.zeros_like(s["pos"])
    return s


def _prepare_sample(c, g):
    R, n = c["rows"], c["n"]
    # logits of a trained head: a broad bulk and a tail of likely tokens
    logits = 2.0 * _normal(g, (R, n)) + 9.0 * torch.rand((R, n), generator=g, device="cuda") ** 24
    s = {"c": c, "logits": logits.to(TYPES[c["type"]]), "u": torch.rand(R, generator=g, device="cuda")}
    i = torch.arange(R, device="cuda")
    s["temperature"], s["top_p"], s["min_p"] = torch.full((R,), 0.8, device="cuda"), torch.full((R,), 0.95, device="cuda"), torch.zeros(R, device="cuda")
    s["top_k"] = torch.full((R,), 40, dtype=torch.int32, device="cuda")
    if c["mix"] == "nucleus":
        s["temperature"], s["top_k"], s["top_p"] = torch.ones(R, device="cuda"), torch.zeros_like(s["top_k"]), torch.full((R,), 0.9, device="cuda")
    if c["mix"] == "any":
        s["temperature"] = torch.tensor([0.8, 1.0, 0.0, 1.3, 0.6], device="cuda")[i % 5].contiguous()
        s["top_k"] = _int32([40, 0, 0, 1000, 20000, 5, 0])[i % 7].contiguous()
        s["top_p"] = torch.tensor([0.95, 1.0, 0.9, 0.5], device="cuda")[(i // 2) % 4].contiguous()
        s["min_p"] = torch.tensor([0.0, 0.05, 0.0], device="cuda")[(i // 3) % 3].contiguous()
    s["ids"], s["prob"] = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, device="cuda")
    return s


def _prepare_adapt(c, g):
    T, K, N, A, R = c["tokens"], c["k"], c["n"], c["adapters"], c["rank"]
    s = {"c": c, "x": _normal(g, (T, K), TYPES[c["type"]]), "base": _normal(g, (T, N)), "out": torch.zeros((T, N), device="cuda")}
    # the adapters present change every `runs` tokens; one token in nine has none
    run = torch.arange(T, device="cuda") // c["runs"]
    ids = torch.randint(0, A, (T,), generator=g, device="cuda")[run]
    s["ids"] = torch.where(run % 9 == 8, -1, ids).to(torch.int32)
    used = torch.arange(R, device="cuda") < _int32(_ranks(c))[:, None]
    s["down"] = (_normal(g, (A, R, K)) / math.sqrt(K) * used[:, :, None]).to(torch.bfloat16)
    s["up"] = (_normal(g, (A, N, R)) * used[:, None, :]).to(torch.bfloat16)
    s["scale"] = 0.5 + torch.rand(A, generator=g, device="cuda")
    return s


_CTX = []


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)
    s = {"attn": _prepare_attn, "evict": _prepare_evict, "sample": _prepare_sample, "adapt": _prepare_adapt}[case["op"]](case, g)
    if own:  # what a serving loop keeps: the context, descriptions of its buffers, workspaces, and adapters in the framework's layout
        from powerserve_amd import hip
        if not _CTX:
            _CTX.append(hip.Ctx(0))
        ctx = s["ctx"] = _CTX[0]
        kind = {"f32": hip.F32, "f16": hip.F16, "bf16": hip.BF16}[case["type"]]
        if case["op"] in ("attn", "evict"):
            s["cache"] = hip.kv_cache(kind, s["k"], s["v"], s["n_kv"], case["seqs"], case["slots"], case["kv_heads"], case["dim"], weight=s["weight"], pos=s.get("pos"))
        if case["op"] == "attn":
            s["call"] = hip.cache_attn_args(s["q"], s["out"], case["heads"], case["new"], 1.0 / math.sqrt(case["dim"]), k_new=s["k_new"], v_new=s["v_new"], count=s["count"], tree=s["tree"],
                                            weight_out=s["weight_out"])
            need = ctx.cache_attn_workspace(s["cache"], s["call"])
        elif case["op"] == "evict":
            s["call"] = hip.cache_evict_args(case["keep"], recent=case["recent"], first=case["first"], weight_out=s["weight_out"], pos_out=s["pos_out"], n_kv_out=s["n_kv_out"])
            need = ctx.cache_evict_workspace(s["cache"], s["call"])
        elif case["op"] == "sample":
            s["call"] = hip.sample_params(temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], u=s["u"])
            s["kind"] = kind
            need = ctx.sample_workspace(case["n"], case["rows"])
        else:
            s["set"] = hip.Adapters(ctx, case["n"], case["k"], case["adapters"], case["rank"])
            for i, r in enumerate(_ranks(case)):
                s["set"].load(i, s["down"][i, :r].contiguous().view(torch.int16).cpu().numpy(), s["up"][i, :, :r].contiguous().view(torch.int16).cpu().numpy(), float(s["scale"][i]))
            s["kind"] = kind
            need = s["set"].workspace(case["tokens"])
        s["need"], s["space"] = need, torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------------------- plain forms
def _new_rows(s):
    """The new tokens' rows in the cache, and which of them there are."""
    n, t = s["n_kv"].long()[:, None], torch.arange(s["c"]["new"], device="cuda")
    rows, there = (n + t).clamp(max=s["c"]["slots"] - 1), t < s["count"][:, None]
    seq = torch.arange(s["c"]["seqs"], device="cuda")[:, None]
    for old, new in ((s["k"], s["k_new"]), (s["v"], s["v_new"])):
        old[seq, rows] = torch.where(there[:, :, None, None], new, old[seq, rows])
    return there


def _visible(s):
    """[seqs, new, slots]"""
    n, T, N = s["n_kv"].long()[:, None, None], s["c"]["new"], s["c"]["slots"]
    j, t = torch.arange(N, device="cuda")[None, None, :], torch.arange(T, device="cuda")[None, :, None]
    i = j - n
    inside = (i >= 0) & (i < s["count"].long()[:, None, None])
    if s["tree"] is None:
        return (i < 0) | (inside & (i <= t))
    return (i < 0) | (inside & torch.gather(s["tree"].bool(), 2, i.clamp(0, T - 1).expand(-1, T, -1)))


def _plain_attn(s):
    c = s["c"]
    S, T, H, G, D, N = c["seqs"], c["new"], c["heads"], c["kv_heads"], c["dim"], c["slots"]
    there, R = _new_rows(s), H // G
    q = s["q"].float().view(S, T, G, R, D).permute(0, 2, 1, 3, 4).reshape(S * G, T * R, D)
    k = s["k"].float().permute(0, 2, 3, 1).reshape(S * G, D, N)
    z = torch.bmm(q, k).mul_(1.0 / math.sqrt(D)).view(S, G, T, R, N)
    z.masked_fill_(~_visible(s)[:, None, :, None, :], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    v = s["v"].float().permute(0, 2, 1, 3).reshape(S * G, N, D)
    o = torch.bmm(p.view(S * G, T * R, N), v).view(S, G, T, R, D).permute(0, 2, 1, 3, 4).reshape(S, T, H, D)
    s["out"].copy_(torch.where(there[:, :, None, None], o.to(s["out"].dtype), s["out"]))
    r = {"out": s["out"], "k": s["k"], "v": s["v"]}
    if c["weights"]:
        w = (p * there[:, None, :, None, None]).sum((2, 3))
        j, n = torch.arange(N, device="cuda"), s["n_kv"].long()[:, None, None]
        w = torch.where(j < n, s["weight"] + w, w)
        s["weight_out"].copy_(torch.where(j < n + s["count"].long()[:, None, None], w, s["weight_out"]))
        r["weight"] = s["weight_out"]
    return r


def _plain_evict(s):
    c = s["c"]
    N, keep = c["slots"], c["keep"]
    j, n = torch.arange(N, device="cuda"), s["n_kv"].long()[:, None, None]
    held, pos = j < n, s["pos"].long()
    newest = torch.where(held, pos, -1).amax(-1, keepdim=True)
    rank = torch.where(held, torch.where((pos < c["first"]) | (pos > newest - c["recent"]), 2, 1), 0)
    by_weight = torch.sort(torch.where(held, s["weight"], -1.0), dim=-1, descending=True, stable=True)[1]
    order = torch.gather(by_weight, -1, torch.sort(torch.gather(rank, -1, by_weight), dim=-1, descending=True, stable=True)[1])
    place = torch.empty_like(order).scatter_(-1, order, j.expand_as(order).contiguous())  # a slot's place in the order
    kept = held & (place < keep)
    hole, moved = ~kept & held & (j < keep), kept & (j >= keep)
    # the i-th hole takes the i-th kept slot at or behind the bound
    nth = torch.where(moved, torch.cumsum(moved, -1) - 1, N - 1)
    source = torch.zeros_like(order).scatter_(-1, nth, torch.where(moved, j, 0))
    take = torch.where(hole, torch.gather(source, -1, (torch.cumsum(hole, -1) - 1).clamp(min=0)), j)[..., :min(keep, N)]
    rows = take.permute(0, 2, 1)[..., None].expand(-1, -1, -1, c["dim"])
    for x in (s["k"], s["v"]):
        x[:, :take.shape[-1]] = torch.gather(x, 1, rows)
    left, stay = torch.minimum(n, torch.full_like(n, keep)), take.shape[-1]
    for x, y in ((s["weight"], s["weight_out"]), (s["pos"], s["pos_out"])):
        y[..., :stay] = torch.where(j[:stay] < left, torch.gather(x, -1, take), y[..., :stay])
    s["n_kv_out"].copy_(left.view(-1))
    return {"k": s["k"], "v": s["v"], "weight": s["weight_out"], "pos": s["pos_out"], "n_kv": s["n_kv_out"]}


def _plain_sample(s):
    n = s["c"]["n"]
    v, ids = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    z, t = v.double(), s["temperature"].double()[:, None]
    greedy = t <= 0
    w = torch.exp((z - z[:, :1]) / torch.where(greedy, 1.0, t))
    at, k = torch.arange(n, device="cuda"), s["top_k"].long()[:, None]
    w = torch.where((k > 0) & (at >= k) | greedy & (at > 0), 0.0, w)
    sums = torch.cumsum(w, -1)
    p = s["top_p"].double()[:, None]
    last = torch.where(p < 1, (sums < p * sums[:, -1:]).sum(-1, keepdim=True), n - 1)
    last = torch.minimum(last, ((w > 0) & (w >= s["min_p"].double()[:, None])).sum(-1, keepdim=True) - 1).clamp(0, n - 1)
    total = torch.gather(sums, -1, last)
    take = torch.minimum((sums <= s["u"].double()[:, None] * total).sum(-1, keepdim=True), last)
    s["ids"].copy_(torch.gather(ids, -1, take).view(-1))
    s["prob"].copy_((torch.gather(w, -1, take) / total).view(-1))
    return {"ids": s["ids"], "prob": s["prob"]}


def _plain_adapt(s):
    has, i = s["ids"] >= 0, s["ids"].long().clamp(min=0)
    h = torch.bmm(s["down"][i].float(), s["x"].float()[:, :, None])
    d = torch.bmm(s["up"][i].float(), h)[:, :, 0] * s["scale"][i][:, None]
    s["out"].copy_(torch.where(has[:, None], s["base"] + d, s["base"]))
    return s["out"]


def run(s):
    op = s["c"]["op"]
    if not own:
        return {"attn": _plain_attn, "evict": _plain_evict, "sample": _plain_sample, "adapt": _plain_adapt}[op](s)
    ctx, c = s["ctx"], s["c"]
    if op == "attn":
        ctx.cache_attn(s["cache"], s["call"], s["space"], s["need"])
        return {"out": s["out"], "k": s["k"], "v": s["v"]} | ({"weight": s["weight_out"]} if c["weights"] else {})
    if op == "evict":
        ctx.cache_evict(s["cache"], s["call"], s["space"], s["need"])
        return {"k": s["k"], "v": s["v"], "weight": s["weight_out"], "pos": s["pos_out"], "n_kv": s["n_kv_out"]}
    if op == "sample":
        ctx.sample(s["logits"], c["n"], c["rows"], s["call"], s["ids"], prob=s["prob"], dtype=s["kind"], space=s["space"], space_bytes=s["need"])
        return {"ids": s["ids"], "prob": s["prob"]}
    s["set"].apply(s["x"], c["tokens"], s["ids"], s["out"], base=s["base"], dtype=s["kind"], space=s["space"], space_bytes=s["need"])
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------------------- work, and the results in 64 bits
def work(case):
    c, size = case, {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if c["op"] == "attn":
        b = f = 0
        for n, t in zip(_lengths(c), _counts(c)):
            pairs = n * t + (t * (t + 1) // 2 if c["mask"] == "causal" else t)  # a tree's token sees itself at least
            f += 4 * c["heads"] * c["dim"] * pairs
            b += (2 * n * c["kv_heads"] + 2 * t * c["heads"] + 4 * t * c["kv_heads"]) * c["dim"] * size + (c["kv_heads"] * (8 * n + 4 * t) if c["weights"] else 0)
        return {"bytes": b, "flops": f}
    if c["op"] == "evict":  # weights and positions of all that is held, those of what stays written, and rows that move: at least half of what stays where most goes
        b = 0
        for n in _lengths(c):
            moved = 0 if n <= c["keep"] else min(c["keep"], n - c["keep"]) * max(0, n - c["keep"]) / n
            b += c["kv_heads"] * (8 * n + 8 * min(n, c["keep"]) + 4 * moved * c["dim"] * size)
        return {"bytes": b, "flops": 0}
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (c["n"] * size + 28), "flops": 0}
    have, ranks = min(c["adapters"], -(-c["tokens"] // c["runs"])), _ranks(c)
    rank = sum(ranks) / len(ranks)
    return {"bytes": c["tokens"] * (c["k"] * size + 8 * c["n"] + 4) + have * rank * (c["k"] + c["n"]) * 2, "flops": 2 * c["tokens"] * rank * (c["k"] + c["n"])}


def _exact_attn(s):
    c = s["c"]
    S, H, G, D = c["seqs"], c["heads"], c["kv_heads"], c["dim"]
    out, k, v = s["out"].double(), s["k"].clone(), s["v"].clone()
    weight = s["weight_out"].double() if c["weights"] else None
    for i, (n, t) in enumerate(zip(_lengths(c), _counts(c))):
        k[i, n:n + t], v[i, n:n + t] = s["k_new"][i, :t], s["v_new"][i, :t]
        see = torch.ones((t, n + t), dtype=torch.bool, device="cuda")
        see[:, n:] = torch.ones((t, t), dtype=torch.bool, device="cuda").tril() if s["tree"] is None else s["tree"][i, :t, :t] != 0
        for g in range(G):
            kg, vg, total = k[i, :n + t, g].double(), v[i, :n + t, g].double(), 0.0
            for h in range(g * (H // G), (g + 1) * (H // G)):
                z = (s["q"][i, :t, h].double() @ kg.t().contiguous()) / math.sqrt(D)
                p = torch.softmax(z.masked_fill(~see, -math.inf), -1)
                out[i, :t, h] = p @ vg
                total = total + p.sum(0)
            if c["weights"]:
                weight[i, g, :n + t] = total
                weight[i, g, :n] += s["weight"][i, g, :n].double()
    return {"out": out, "k": None, "v": None} | ({"weight": weight} if c["weights"] else {})


def _exact_sample(s):
    ids, prob = [], []
    for r in range(s["c"]["rows"]):
        z = s["logits"][r].double().cpu()
        t, k, p, m, u = (float(s[x][r]) for x in ("temperature", "top_k", "top_p", "min_p", "u"))
        order = torch.argsort(z, descending=True, stable=True)
        if t <= 0:
            order, t = order[:1], 1.0
        if k > 0:
            order = order[:int(k)]
        w = torch.exp((z[order] - z[order[0]]) / t)
        if p < 1:
            order = order[:int((torch.cumsum(w, 0) < p * w.sum()).sum()) + 1]
        order = order[:max(1, int((w[:len(order)] >= m).sum()))]
        w = w[:len(order)]
        i = min(int((torch.cumsum(w, 0) <= u * w.sum()).sum()), len(order) - 1)
        ids.append(int(order[i]))
        prob.append(float(w[i] / w.sum()))
    return {"ids": _int32(ids), "prob": torch.tensor(prob, dtype=torch.float64, device="cuda")}


def _exact_adapt(s):
    out, x = s["base"].double(), s["x"].double()
    for a in range(s["c"]["adapters"]):
        mine = torch.nonzero(s["ids"] == a)[:, 0]
        out[mine] += float(s["scale"][a]) * (x[mine] @ s["down"][a].double().t().contiguous()) @ s["up"][a].double().t().contiguous()
    return out


def exact(case, seed):
    if case["op"] == "evict":
        return None  # nothing is computed: numbers move
    s = {"attn": _prepare_attn, "sample": _prepare_sample, "adapt": _prepare_adapt}[case["op"]](case, torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13))
    return {"attn": _exact_attn, "sample": _exact_sample, "adapt": _exact_adapt}[case["op"]](s)
