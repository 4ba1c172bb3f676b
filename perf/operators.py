"""Operators of a serving step whose requests share a base model and a prompt, as cases to be measured: low-rank adapters beside a shared
projection, norms of queries and keys with their rotation, and attention over shared prefixes.  `own` says whether a case runs through this
framework or in its plain form."""
import math

import torch

own = False

HIDDEN, FFN, THETA, EPS = 4096, 14336, 500000.0, 1e-5


# ---- cases ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one request generating with its adapter: the smallest call, all latency; four projections of a step
        dict(name="lora_one", op="lora", rows="1", plain=0, slots=8, rank=16, mixed=False, k=HIDDEN, n=HIDDEN, layers=4),
        # a decode batch of many tenants at the fused q/k/v projection: a few rows for each adapter
        dict(name="lora_decode", op="lora", rows="4*64", plain=0, slots=64, rank=16, mixed=False, k=HIDDEN, n=6144, layers=2),
        # prompts of three tenants beside generating rows, some without an adapter, ranks that differ; gate and up
        dict(name="lora_mixed", op="lora", rows="700,683,129,2*29", plain=13, slots=33, rank=64, mixed=True, k=HIDDEN, n=2 * FFN, layers=1),
        # long prompts at the down projection
        dict(name="lora_prompts", op="lora", rows="2048,2048,1999,1500,597", plain=0, slots=5, rank=32, mixed=False, k=FFN, n=HIDDEN, layers=1),
        # one generated token, far into a long text
        dict(name="norm_rope_one", op="norm_rope", rows=1, hq=32, hkv=8, d=128, rot=128, interleaved=False, far=1000000),
        # a decode batch, small heads of which half rotates, in neighbouring pairs
        dict(name="norm_rope_decode", op="norm_rope", rows=257, hq=16, hkv=4, d=64, rot=32, interleaved=True, far=100000),
        # prompts of a step
        dict(name="norm_rope_prompt", op="norm_rope", rows=8192, hq=32, hkv=8, d=128, rot=128, interleaved=False, far=32768),
        # four answers to one short prompt
        dict(name="attn_few", op="attn", rows=4, system=500, docs=0, doc=0, most=40, hq=32, hkv=8, d=128, fp8=False, layers=4),
        # a chat service's batch under one system prompt
        dict(name="attn_batch", op="attn", rows=64, system=2048, docs=0, doc=0, most=512, hq=32, hkv=8, d=128, fp8=False, layers=2),
        # questions about three documents under a common instruction: a tree of prefixes
        dict(name="attn_tree", op="attn", rows=97, system=300, docs=3, doc=3001, most=200, hq=16, hkv=4, d=64, fp8=False, layers=2),
        # the same kind of batch on 8-bit pages
        dict(name="attn_fp8", op="attn", rows=128, system=4096, docs=0, doc=0, most=300, hq=32, hkv=8, d=128, fp8=True, layers=1),
        # a large batch over a long common text
        dict(name="attn_large", op="attn", rows=256, system=8192, docs=0, doc=0, most=512, hq=32, hkv=8, d=128, fp8=False, layers=1),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lora", "norm_rope", "attn"])
    most = max(work(c)["flops"] for c in listed() if c["op"] == op)
    while True:
        if op == "lora":
            prompts = [str(_log(rng, 17, 2048)) for _ in range(rng.randint(0, 4))]
            tenants = _log(rng, 1, 64)
            rows = prompts + ["%d*%d" % (_log(rng, 1, 8), tenants)]
            k, n = rng.choice([(HIDDEN, HIDDEN), (HIDDEN, 6144), (HIDDEN, 2 * FFN), (FFN, HIDDEN), (8 * rng.randint(8, 512), 8 * rng.randint(8, 1024))])
            case = dict(op=op, rows=",".join(rows), plain=rng.choice([0, 0, _log(rng, 1, 64)]), slots=len(prompts) + tenants + rng.randint(0, 3),
                        rank=rng.choice([8, 16, 32, 64, 128, rng.randint(1, 128)]), mixed=rng.random() < 0.5, k=k, n=n, layers=rng.randint(1, 2))
        elif op == "norm_rope":
            d = rng.choice([64, 128])
            hkv = rng.choice([1, 2, 4, 8])
            case = dict(op=op, rows=_log(rng, 1, 8192), hq=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv, d=d, rot=rng.choice([d, d, d // 2, d // 4]),
                        interleaved=rng.random() < 0.5, far=_log(rng, 100, 1000000))
        else:
            docs = rng.choice([0, 0, 2, 3, 5])
            hkv = rng.choice([2, 4, 8])
            fp8 = rng.random() < 0.3
            case = dict(op=op, rows=max(_log(rng, 1, 256), docs), system=_log(rng, 20, 8192), docs=docs, doc=_log(rng, 100, 4000) if docs else 0, most=_log(rng, 1, 600),
                        hq=hkv * rng.choice([1, 2, 4, 4, 8]), hkv=hkv, d=128 if fp8 else rng.choice([64, 128, 128]), fp8=fp8, layers=rng.randint(1, 2))
        if work(case)["flops"] <= most and case.get("hq", 0) <= 32:
            return case


# ---- what a case holds ----------------------------------------------------------------------------------------------------
def _counts(case):
    """Rows of each adapter, one after the other."""
    counts = []
    for part in case["rows"].split(","):
        each, _, times = part.partition("*")
        counts += [int(each)] * int(times or 1)
    return counts


def _ranks(case):
    return [max(1, case["rank"] >> (i % 4)) if case["mixed"] else case["rank"] for i in range(case["slots"])]


def _contexts(case):
    """Own tokens of each row: 1 to `most`, spread evenly, in an order that is no order."""
    return [1 + (i * 37 % case["rows"]) * (case["most"] - 1) // max(1, case["rows"] - 1) for i in range(case["rows"])]


def work(case):
    if case["op"] == "lora":
        counts, ranks = _counts(case), _ranks(case)
        rows, used = sum(counts) + case["plain"], ranks[:len(counts)]
        width = case["k"] + case["n"]
        return {"bytes": case["layers"] * 2 * (rows * (case["k"] + 2 * case["n"]) + sum(used) * width),
                "flops": case["layers"] * 2 * sum(c * r for c, r in zip(counts, used)) * width}
    if case["op"] == "norm_rope":
        elements = case["rows"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 4 * elements, "flops": 8 * elements}
    own_tokens = _contexts(case)
    shared = case["system"] + case["doc"]
    distinct = case["system"] + case["docs"] * case["doc"] + sum(own_tokens)
    total = case["rows"] * shared + sum(own_tokens)
    return {"bytes": case["layers"] * (2 * distinct * case["hkv"] * case["d"] * (1 if case["fp8"] else 2) + 4 * case["rows"] * case["hq"] * case["d"]),
            "flops": case["layers"] * 4 * total * case["hq"] * case["d"]}


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, scale=1.0: (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)  # noqa: E731
    if case["op"] == "lora":
        counts, ranks = _counts(case), _ranks(case)
        rows, slots, k, n, layers = sum(counts) + case["plain"], case["slots"], case["k"], case["n"], case["layers"]
        order = torch.randperm(slots, generator=g, device="cuda")[:len(counts)]
        pieces = list(zip(order.tolist(), counts)) + ([(-1, case["plain"])] if case["plain"] else [])
        row_adapter = torch.cat([torch.full((c,), a, dtype=torch.int32, device="cuda") for a, c in pieces])
        if max(counts) <= 16:  # generating rows come in the order in which requests arrived
            row_adapter = row_adapter[torch.randperm(rows, generator=g, device="cuda")].contiguous()
        rank_of = torch.zeros(slots, dtype=torch.int64, device="cuda")
        rank_of[order] = torch.tensor(ranks[:len(counts)], device="cuda")
        there = torch.arange(case["rank"], device="cuda")[None] < rank_of[:, None]
        a = [normal(slots, case["rank"], k, scale=k ** -0.5) * there[:, :, None] for _ in range(layers)]
        b = [normal(slots, n, case["rank"], scale=case["rank"] ** -0.5) * there[:, None, :] for _ in range(layers)]
        return dict(row_adapter=row_adapter, rank_of=rank_of, a=a, b=b, scale=0.5 + torch.rand(slots, generator=g, device="cuda"),
                    x=[normal(rows, k) for _ in range(layers)], y=[normal(rows, n) for _ in range(layers)])
    if case["op"] == "norm_rope":
        rows, hq, hkv, d = case["rows"], case["hq"], case["hkv"], case["d"]
        qkv = normal(rows, (hq + 2 * hkv) * d, scale=2.0)  # a fused projection's rows: q, k, v
        start = int(torch.randint(0, case["far"], (1,), generator=g, device="cuda").item())
        return dict(q=qkv[:, :hq * d].unflatten(1, (hq, d)), k=qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d)),
                    positions=(start + torch.arange(rows, device="cuda")).remainder(case["far"]).to(torch.int32),
                    q_weight=1 + normal(d, scale=0.2), k_weight=1 + normal(d, scale=0.2))
    rows, hkv, d, layers = case["rows"], case["hkv"], case["d"], case["layers"]
    own_tokens = _contexts(case)
    pages_of = lambda tokens: -(-tokens // 32)  # noqa: E731
    # pages of the prompt, of each document behind it and of each row behind that; a part that ends inside a page is copied by whoever goes on in it
    system_pages = list(range(case["system"] // 32))
    n_pages = len(system_pages)
    prefixes = []
    for _ in range(max(1, case["docs"])):
        more = (case["system"] + case["doc"]) // 32 - len(system_pages)
        prefixes.append(system_pages + list(range(n_pages, n_pages + more)))
        n_pages += more
    table = torch.zeros((rows, pages_of(case["system"] + case["doc"] + max(own_tokens))), dtype=torch.int64)
    contexts = []
    for r, tokens in enumerate(own_tokens):
        shared = prefixes[r % len(prefixes)]
        contexts.append(case["system"] + case["doc"] + tokens)
        more = pages_of(contexts[-1]) - len(shared)
        pages = shared + list(range(n_pages, n_pages + more))
        n_pages += more
        table[r, :len(pages)] = torch.tensor(pages)
    state = dict(table=table.cuda(), contexts=torch.tensor(contexts, dtype=torch.int32, device="cuda"), q=[normal(rows, case["hq"], d, scale=2.0) for _ in range(layers)])
    for name in "kv":
        rows_of = normal(layers, n_pages, hkv, 32, d)
        if case["fp8"]:
            scale = rows_of.float().abs().amax((3, 4)) / 448
            state[name] = (rows_of.float() / scale[..., None, None]).to(torch.float8_e4m3fn)
            state[name + "_scale"] = scale
        else:
            state[name] = rows_of
    return state


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        from dmlx_b200 import device
        if case["op"] == "lora":
            state["adapters"] = []
            for a, b in zip(state["a"], state["b"]):
                weights = device.LoraAdapters(case["slots"], case["n"], case["k"], case["rank"])
                for slot, rank in enumerate(state["rank_of"].tolist()):
                    if rank:
                        weights.set(slot, a[slot, :rank], b[slot, :, :rank], float(state["scale"][slot]))
                state["adapters"].append(weights)
            state["batch"] = device.LoraBatch(len(state["row_adapter"]), case["slots"], case["rank"])
        elif case["op"] == "attn":
            state["cache"] = _cache(device, state, case)
            state["attention"] = device.SharedPrefixAttention(state["cache"], case["rows"])
            state["row_seq"] = torch.arange(case["rows"], dtype=torch.int32, device="cuda")
    return state


def _cache(device, state, case):
    """The framework's cache with the state's pages: every shared page held once, by all the rows that go through it."""
    rows, n_pages = case["rows"], state["k"].shape[1]
    widest = state["table"].shape[1]
    cache = device.PagedKVCache(case["layers"], case["hkv"], case["d"], n_pages + 1, rows + 1, widest, case["hq"], max_rows=max(rows, 64),
                                kv_dtype=device.KV_FP8_E4M3 if case["fp8"] else device.KV_BF16)
    held = {}  # page of the state -> page of the cache, and a row that holds it
    table = state["table"].tolist()
    for r, context in enumerate(state["contexts"].tolist()):
        pages = table[r][:-(-context // 32)]
        known = 0
        while known < len(pages) and pages[known] in held:
            known += 1
        if known:
            cache.fork(held[pages[known - 1]][1], r, known * 32)
        mine = cache.alloc(r, len(pages) - known)
        held.update({p: (c, r) for p, c in zip(pages[known:], mine)})
        cache.set_len(r, context)
    raw = lambda t: t.view(torch.uint8 if case["fp8"] else torch.uint16).cpu().numpy()  # noqa: E731
    k, v = raw(state["k"]), raw(state["v"])
    scales = [state[n + "_scale"].cpu().numpy() if case["fp8"] else None for n in "kv"]
    for layer in range(case["layers"]):
        for page, (at, _) in held.items():
            cache.page_load(layer, at, k[layer, page], v[layer, page], *(None if s is None else s[layer, page] for s in scales))
    return cache


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        if case["op"] == "lora":
            state["batch"].plan(state["row_adapter"])
            return [w.apply(state["batch"], x, y) for w, x, y in zip(state["adapters"], state["x"], state["y"])]
        if case["op"] == "norm_rope":
            from dmlx_b200 import device
            return device.qk_norm_rope(state["q"], state["k"], state["positions"], state["q_weight"], state["k_weight"], eps=EPS, theta=THETA,
                                       rot_dim=case["rot"], interleaved=case["interleaved"])
        state["attention"].plan(state["row_seq"], state["contexts"])
        return [state["attention"].run(layer, q) for layer, q in enumerate(state["q"])]
    if case["op"] == "lora":
        return [_lora(state, *of_layer) for of_layer in zip(state["a"], state["b"], state["x"], state["y"])]
    if case["op"] == "norm_rope":
        turn = _rotation(state["positions"], case["rot"])
        return [_norm_rope(x, w, turn, case) for x, w in ((state["q"], state["q_weight"]), (state["k"], state["k_weight"]))]
    return [_attention(state, layer, q) for layer, q in enumerate(state["q"])]


def _lora(state, a, b, x, y):
    """All adapters' products, those of other adapters set to zero in between."""
    slots, rank, k = a.shape
    u = x.float() @ a.reshape(slots * rank, k).float().T
    mine = torch.arange(slots, device="cuda")[None] == state["row_adapter"][:, None]
    u = u.unflatten(1, (slots, rank)) * (mine * state["scale"])[:, :, None]
    return (y.float() + u.flatten(1) @ b.permute(0, 2, 1).reshape(slots * rank, -1).float()).to(torch.bfloat16)


def _rotation(positions, rot):
    angle = positions.double()[:, None] * THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _norm_rope(x, w, turn, case):
    x, (cos, sin), rot = x.float(), turn, case["rot"]
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    first, second = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    pair = first * cos - second * sin, first * sin + second * cos
    turned = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
    return torch.cat([turned, x[..., rot:]], -1).to(torch.bfloat16)


def _attention(state, layer, q):
    """Every row's pages gathered, then softmax(q k / sqrt(d)) v over the tokens it has."""
    case, table = state["case"], state["table"]
    k, v = (state[n][layer][table].float() for n in "kv")  # [row, page, head, token, d]
    if case["fp8"]:
        k, v = (x * state[n + "_scale"][layer][table][..., None, None] for n, x in (("k", k), ("v", v)))
    k, v = (x.permute(0, 2, 1, 3, 4).flatten(2, 3) for x in (k, v))
    rows, hkv, tokens, d = k.shape
    scores = q.float().reshape(rows, hkv, -1, d) @ k.transpose(2, 3) * d ** -0.5
    seen = torch.arange(tokens, device="cuda")[None] < state["contexts"][:, None]
    scores = torch.where(seen[:, None, None], scores, torch.full_like(scores, -math.inf))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return ((p @ v) / p.sum(-1, keepdim=True)).reshape(rows, -1, d).to(torch.bfloat16)


# ---- the definitions, in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "lora":
        outs = []
        for a, b, x, y in zip(s["a"], s["b"], s["x"], s["y"]):
            out = y.double()
            for slot in s["row_adapter"].unique().tolist():
                if slot >= 0:
                    at = (s["row_adapter"] == slot).nonzero()[:, 0]
                    u = torch.einsum("tk,rk->tr", x[at].double(), a[slot].double())
                    out[at] += s["scale"][slot].double() * torch.einsum("tr,nr->tn", u, b[slot].double())
            outs.append(out)
        return outs
    if case["op"] == "norm_rope":
        rot = case["rot"]
        both = []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["d"] + EPS) * w.double()
            out = x.clone()
            for i in range(rot // 2):
                p, q = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
                angle = s["positions"].double()[:, None] * THETA ** (-2.0 * i / rot)
                out[..., p] = x[..., p] * angle.cos() - x[..., q] * angle.sin()
                out[..., q] = x[..., q] * angle.cos() + x[..., p] * angle.sin()
            both.append(out)
        return both
    outs = []
    for layer, q in enumerate(s["q"]):
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        for r, context in enumerate(s["contexts"].tolist()):
            pages = s["table"][r, :-(-context // 32)]
            k, v = (s[n][layer, pages].double() for n in "kv")
            if case["fp8"]:
                k, v = k * s["k_scale"][layer, pages][:, :, None, None].double(), v * s["v_scale"][layer, pages][:, :, None, None].double()
            k, v = (x.permute(1, 0, 2, 3).reshape(case["hkv"], -1, case["d"])[:, :context] for x in (k, v))
            heads = q[r].double().view(case["hkv"], -1, case["d"])
            weights = torch.softmax(torch.einsum("hgd,htd->hgt", heads, k) / math.sqrt(case["d"]), -1)
            out[r] = torch.einsum("hgt,htd->hgd", weights, v).flatten(0, 1)
        outs.append(out)
    return outs
